// learn_policy.inl -- the clipped policy loss with its gradients, and the sampling of actions.
//
// Both are one pass over the logits: a row is in registers (or, beyond 8192 kinds, read twice) while its maximum, the sum s of e^(z - max) and
// u = sum of e^(z - max) (z - max) are taken; log s and u / s give the log-probabilities and the entropy, and the gradient is written from the same registers:
// reading the logits once and writing their gradient once is all the memory traffic there has to be (8209 rows of 6144 bf16, masked, with all gradients: 252 MB in 64 us,
// 3.9 TB/s, where a large copy reaches 4.76: two exps and a dozen other instructions per kind stand beside it).  Up to 8 kinds a row is one thread's, up to 2048
// a group of 1 to 64 lanes', beyond that a workgroup's.

static const int kUnits = 256;      // compute units of an MI355X
static const int kLossBlocks = 2560, kWeightBlocks = 256;
static const int64_t kLossWork = 8 * kLossBlocks + kWeightBlocks;
static const float kHalfLog2Pi = 0.91893853320467274f, kHalfLog2PiE = 1.4189385332046727f;

template <class T> __device__ __forceinline__ float log_std_at(const void *p, int per_row, int64_t row, int d) {
  return per_row ? to_f(((const T *)p)[2 * row + d]) : ((const float *)p)[d];
}

__global__ __launch_bounds__(256) void k_weight_sum(const float *__restrict__ w, int64_t rows, double *__restrict__ out) {
  __shared__ double part[4];
  double s = 0;
  int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  for (; i + 4 <= rows; i += (int64_t)gridDim.x * 1024) {
    Raw<float, 4> r; load_raw<float, 4>(r, w + i);
    s += ((double)r[0] + (double)r[1]) + ((double)r[2] + (double)r[3]);
  }
  for (; i < rows; ++i) s += (double)w[i];      // (one thread's: the others' i is beyond rows, or their four were whole)
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) out[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// VE neighbouring logits of a row, still as they were loaded; what is not allowed is made -inf in place, once, so that nothing after it needs to know
template <class T, int VE> struct Kinds {
  Raw<T, VE> raw; uint32_t ok[(VE + 3) / 4];
  __device__ __forceinline__ void load(const T *z, const uint8_t *allowed) {
    load_raw<T, VE>(raw, z);
    if (allowed) {
      struct __attribute__((packed)) Bytes { uint8_t b[VE]; };
      ok[(VE - 1) / 4] = 0;
      __builtin_memcpy(ok, (const Bytes *)allowed, VE);
    }
  }
  __device__ __forceinline__ void none() {
#pragma unroll
    for (auto &w : raw.w) w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, bf16_t>::value ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
    for (auto &w : ok) w = 0;
  }
  __device__ __forceinline__ void mask() {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < VE; ++k) raw.w[k] = ok[k / 4] >> (8 * (k % 4)) & 255u ? raw.w[k] : 0xff800000u;
    } else {      // two at a time: 0 / nonzero bytes to 0 / 0xffff halves
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      const uint32_t none = std::is_same<T, bf16_t>::value ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
      for (int k = 0; k < (VE + 1) / 2; ++k) {
        const uint32_t pair = __builtin_amdgcn_perm(0u, ok[k / 2], k & 1 ? 0x0c030c02u : 0x0c010c00u);
        u16x2 h = __builtin_bit_cast(u16x2, pair);
        h = (u16x2)(0) - __builtin_elementwise_min(h, (u16x2)(1));
        const uint32_t m = __builtin_bit_cast(uint32_t, h);
        raw.w[k] = (raw.w[k] & m) | (none & ~m);
      }
    }
  }
  __device__ __forceinline__ float operator[](int k) const { return raw[k]; }
};

// what a row's kinds come to, relative to the maximum m: s = sum of e^(z - m), u = sum of e^(z - m) (z - m)
struct RowSums { float m, s, u; };
// z - m, and nothing so low that the product with e^(z - m) = 0 would not be 0.  (The maximum that passes a NaN on: a NaN among the logits is to be seen in the
// loss.  And the difference before the factor log2 e: one multiply-add of both, 2 % faster, overflows where a mask is the type's lowest value.)
__device__ __forceinline__ float below(float z, float m) { return __builtin_elementwise_maximum(z - m, -200.f); }
// the reference point of a row: its maximum, or anything finite where nothing is allowed
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void sums_add(RowSums &r, float z) { const float d = below(z, r.m), e = __expf(d); r.s += e; r.u = fmaf(e, d, r.u); }
// r's sums relative to another maximum
__device__ __forceinline__ void sums_shift(RowSums &r, float m) {
  if (r.s > 0.f && m != r.m) { const float d = below(r.m, m), k = __expf(d); r.u = k * fmaf(r.s, d, r.u); r.s *= k; }
  r.m = m;
}

// what of a row is not per kind, loaded ahead of its logits
struct RowIn { float w, A, old, ref, za; int32_t kind; bool counts; };
template <class T> __device__ __forceinline__ RowIn row_in(const agarcl_policy_loss_args &a, int64_t row) {
  RowIn r;
  r.kind = a.kind[row]; r.w = a.weight ? a.weight[row] : 1.f; r.A = a.advantage[row]; r.old = a.old_log_prob[row]; r.ref = a.ref_log_prob ? a.ref_log_prob[row] : r.old;
  return r;
}
template <class T> __device__ __forceinline__ void row_kind(const agarcl_policy_loss_args &a, RowIn &r, const T *z, const uint8_t *ok) {      // (its kind's own logit)
  r.counts = r.w != 0.f && r.kind >= 0 && r.kind < a.kinds;
  const int32_t k = r.counts ? r.kind : 0;
  r.za = to_f(z[k]);
  r.counts = r.counts && r.za != -INFINITY && (!ok || ok[k]);
}

// dlogit[j] = e^d[j] (c1 d[j] + c0) + (j == kind ? sg : 0), d[j] = z[j] - m
struct LossRow { float sg, c0, c1; };
struct LossTotals { float inv; bool shared_std; };

// e^x - 1 and e^x - 1 - x: near 0, where both are the difference of near numbers, from the series (|x| < 0.35: of
// e^x - 1 - x 1e-7 is left out, of e^x - 1 2e-8)
__device__ __forceinline__ void exp_less(float x, float &less1, float &less1x) {
  const float p = fmaf(x, fmaf(x, fmaf(x, fmaf(x, fmaf(x, 1.f / 5040, 1.f / 720), 1.f / 120), 1.f / 24), 1.f / 6), 0.5f) * x * x, e = __expf(x) - 1.f;
  const bool near = fabsf(x) < 0.35f;
  less1x = near ? p : e - x; less1 = near ? p + x : e;
}

template <class T> __device__ __forceinline__ LossRow loss_row(const agarcl_policy_loss_args &a, const LossTotals &t, int64_t row, const RowIn &in, const RowSums &r, bool leader,
    float (&acc)[7]) {
  LossRow o;
  const float log_s = logf(r.s), rs = __builtin_amdgcn_rcpf(r.s), hcat = log_s - r.u * rs, A = in.A;
  float lp = in.za - r.m - log_s, ent = hcat;
  float dev[2] = {0.f, 0.f}, istd[2] = {0.f, 0.f};
  if (a.mean) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const float ls = log_std_at<T>(a.log_std, a.log_std_per_row, row, d);
      istd[d] = __expf(-ls);
      dev[d] = (a.move[2 * row + d] - to_f(((const T *)a.mean)[2 * row + d])) * istd[d];
      lp -= 0.5f * dev[d] * dev[d] + ls + kHalfLog2Pi;
      ent += ls + kHalfLog2PiE;
    }
  }
  const float ratio = __expf(lp - in.old), high = 1.f + a.clip_high, lowest = 1.f - a.clip_low;
  const bool clipped = A >= 0.f ? ratio > high : ratio < lowest;
  float eb, kl;
  exp_less(in.ref - lp, eb, kl);
  float g = clipped || A == 0.f ? 0.f : -A * ratio;
  if (a.kl_coef != 0.f) g -= a.kl_coef * eb;
  const float share = in.w * t.inv, ce = a.entropy_coef;
  o.sg = share * g; o.c1 = share * ce * rs; o.c0 = (ce != 0.f ? share * ce * (hcat - log_s) - o.sg : -o.sg) * rs;
  if (leader) {
    // (the minimum and maximum that pass a NaN on, as in `below`: the others would make a clipped ratio of it.  And an infinite ratio of no advantage is nothing)
    const float limited = __builtin_elementwise_minimum(__builtin_elementwise_maximum(ratio, lowest), high), w = in.w;
    const float low = A == 0.f && ratio == ratio ? 0.f : __builtin_elementwise_minimum(ratio * A, limited * A);
    acc[0] += w;
    if (in.counts) {
      acc[1] += w * low; acc[2] += w * kl; acc[3] += w * ent; acc[4] += clipped ? w : 0.f;
      if (t.shared_std) {
#pragma unroll
        for (int d = 0; d < 2; ++d) acc[5 + d] += w * (g * (dev[d] * dev[d] - 1.f) - ce);
      }
    }
    if (a.dmean) {
      float v[2];
#pragma unroll
      for (int d = 0; d < 2; ++d) v[d] = in.counts ? o.sg * dev[d] * istd[d] : 0.f;
      store_pack<T, 2>((T *)a.dmean + 2 * row, v);
    }
    if (a.dlog_std && a.log_std_per_row) {
      float v[2];
#pragma unroll
      for (int d = 0; d < 2; ++d) v[d] = in.counts ? o.sg * (dev[d] * dev[d] - 1.f) - share * ce : 0.f;
      store_pack<T, 2>((T *)a.dlog_std + 2 * row, v);
    }
  }
  return o;
}

// the gradient of kinds j0 ... of a row, into dz.  The probabilities are worked out once more: holding 8 of them for every 4 registers of logits would cost more
// (registers, and with them wavefronts) than a second exp
template <class T, int VE> __device__ __forceinline__ void loss_kinds(const RowIn &in, const LossRow &o, float m, int64_t j0, Kinds<T, VE> &z, T *dz) {
  z.raw.anew();
  float v[VE];
  if (in.counts) {
#pragma unroll
    for (int k = 0; k < VE; ++k) { const float d = below(z[k], m); v[k] = __expf(d) * fmaf(o.c1, d, o.c0); }
    const int64_t at = in.kind - j0;
    if (at >= 0 && at < VE) {
#pragma unroll
      for (int k = 0; k < VE; ++k) v[k] += k == (int)at ? o.sg : 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < VE; ++k) v[k] = 0.f;
  }
  store_pack<T, VE>(dz + j0, v);
}

// what comes before the rows; false: there is nothing to do
__device__ __forceinline__ bool loss_begin(const agarcl_policy_loss_args &a, LossTotals &t, double *lds) {
  const bool grads = a.dlogits || a.dmean || (a.dlog_std && a.log_std_per_row);
  t.shared_std = a.dlog_std && !a.log_std_per_row;
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.want_stats) {
    if (t.shared_std && blockIdx.x == 0 && threadIdx.x < 2) ((float *)a.dlog_std)[threadIdx.x] = a.dlog_std_one[threadIdx.x] * up;
    if (!grads || (a.skip_if_one && up == 1.f)) return false;
  }
  t.inv = up;
  if (a.mean_over_weight) {
    double total = (double)a.rows;
    if (a.weight && grads) {
      if (a.weight_sum) total = (double)*a.weight_sum;
      else {
        double w = 0;
        for (int i = threadIdx.x; i < kWeightBlocks; i += blockDim.x) w += a.work[8 * kLossBlocks + i];
        w = wave_sum(w);
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = w;
        __syncthreads();
        total = 0;
        for (int i = 0; i < (int)blockDim.x / 64; ++i) total += lds[i];
        __syncthreads();
      }
    }
    t.inv = total != 0 ? (float)((double)up / total) : 0.f;
  }
  return true;
}
// the workgroup's sums.  A thread adds up its own few rows in 32 bits, everything above that is added in 64
__device__ __forceinline__ void loss_end(const agarcl_policy_loss_args &a, const float (&acc)[7], double *lds) {
  if (!a.want_stats) return;
#pragma unroll
  for (int i = 0; i < 7; ++i) { const double s = wave_sum((double)acc[i]); if ((threadIdx.x & 63) == 0) lds[8 * (threadIdx.x >> 6) + i] = s; }
  __syncthreads();
  if (threadIdx.x < 7) {
    double s = 0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += lds[8 * i + threadIdx.x];
    a.work[threadIdx.x * kLossBlocks + blockIdx.x] = s;
  }
}

// V kinds, one thread per row
template <class T, int V>
__global__ __launch_bounds__(256) void k_loss_thread(const agarcl_policy_loss_args a) {
  __shared__ double lds[32];
  LossTotals t;
  if (!loss_begin(a, t, lds)) return;
  float acc[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    const T *zp = (const T *)a.logits + row * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    RowIn in = row_in<T>(a, row);
    Kinds<T, V> z; z.load(zp, ok);
    row_kind<T>(a, in, zp, ok);
    if (ok) z.mask();
    RowSums r = {-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < V; ++k) r.m = fmaxf(r.m, z[k]);
    r.m = finite_max(r.m);
#pragma unroll
    for (int k = 0; k < V; ++k) sums_add(r, z[k]);
    const LossRow o = loss_row<T>(a, t, row, in, r, true, acc);
    if (a.dlogits) loss_kinds<T, V>(in, o, r.m, 0, z, (T *)a.dlogits + row * a.kinds);
  }
  loss_end(a, acc, lds);
}

// a thread's chunks of 8 kinds of a row (of 8 kinds or more).  The row's last chunk begins 8 kinds before its end: the kinds that the chunk before it has, too,
// are left out of the sums (skip of them) and get the same gradient from both.
template <class T, int CHUNKS> struct Share {
  Kinds<T, 8> z[CHUNKS]; int32_t skip[CHUNKS]; uint32_t there;
  __device__ __forceinline__ static int64_t begin(int64_t j, int64_t kinds) { return j + 8 <= kinds ? j : kinds - 8; }
  __device__ __forceinline__ void load(const T *zp, const uint8_t *ok, int64_t j0, int64_t stride, int64_t kinds, bool on) {
    there = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int64_t j = j0 + c * stride, b = begin(j, kinds);
      skip[c] = (int32_t)(j - b);
      if (on && j < kinds) { there |= 1u << c; z[c].load(zp + b, ok ? ok + b : nullptr); }
      else z[c].none();
    }
  }
  __device__ __forceinline__ float top(bool flags) {
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (flags) z[c].mask();
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, z[c][k]);
      __builtin_amdgcn_sched_barrier(0);      // (chunk after chunk: all at once would take the registers of a second wavefront)
    }
    return m;
  }
  __device__ __forceinline__ void sum(RowSums &r) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      z[c].raw.anew();
      if (__any(skip[c] > 0 && (there >> c & 1))) {
#pragma unroll
        for (int k = 0; k < 8; ++k) sums_add(r, k < skip[c] ? -INFINITY : z[c][k]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) sums_add(r, z[c][k]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __device__ __forceinline__ void gradient(const RowIn &in, const LossRow &o, float m, int64_t j0, int64_t stride, T *dz) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (there >> c & 1) loss_kinds<T, 8>(in, o, m, j0 + c * stride - skip[c], z[c], dz);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// CHUNKS x 8 << g_log kinds, a group of 1 << g_log lanes per row; W wavefronts per SIMD
template <class T, int CHUNKS, int W>
__global__ __launch_bounds__(256, W) void k_loss_lanes(const agarcl_policy_loss_args a, const int g_log) {
  __shared__ double lds[32];
  LossTotals t;
  if (!loss_begin(a, t, lds)) return;
  float acc[7] = {0, 0, 0, 0, 0, 0, 0};
  const int g = 1 << g_log, lane = threadIdx.x & (g - 1), per = 256 >> g_log;
  for (int64_t first = (int64_t)blockIdx.x * per; first < a.rows; first += (int64_t)gridDim.x * per) {
    const int64_t row = first + (threadIdx.x >> g_log), safe = row < a.rows ? row : 0;
    const bool on = row < a.rows;
    const T *zp = (const T *)a.logits + safe * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + safe * a.allowed_stride : nullptr;
    RowIn in = row_in<T>(a, safe);
    Share<T, CHUNKS> z; z.load(zp, ok, lane * 8, g * 8, a.kinds, on);
    row_kind<T>(a, in, zp, ok);
    RowSums r = {z.top(ok), 0.f, 0.f};
    for (int d = 1; d < g; d <<= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, d));
    r.m = finite_max(r.m);
    z.sum(r);
    for (int d = 1; d < g; d <<= 1) { r.s += __shfl_xor(r.s, d); r.u += __shfl_xor(r.u, d); }
    if (!on) continue;      // (a whole group, behind the last of the shuffles of this turn)
    const LossRow o = loss_row<T>(a, t, row, in, r, lane == 0, acc);
    if (a.dlogits) z.gradient(in, o, r.m, lane * 8, g * 8, (T *)a.dlogits + row * a.kinds);
  }
  loss_end(a, acc, lds);
}

// a row's sums from those of its workgroup's wavefronts; one barrier, the two halves of lds in turn
template <int NT> __device__ __forceinline__ RowSums join_waves(const RowSums &mine, float (*lds)[NT / 64][4], int parity) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) { lds[parity][wave][0] = mine.m; lds[parity][wave][1] = mine.s; lds[parity][wave][2] = mine.u; }
  __syncthreads();
  RowSums all = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) all.m = fmaxf(all.m, lds[parity][i][0]);
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    RowSums w = {lds[parity][i][0], lds[parity][i][1], lds[parity][i][2]};
    sums_shift(w, all.m);
    all.s += w.s; all.u += w.u;
  }
  all.m = finite_max(all.m);
  return all;
}

// NT x 8 x CHUNKS kinds in registers, a workgroup per row; CHUNKS = 0: any number, read twice
template <class T, int NT, int CHUNKS, int W>
__global__ __launch_bounds__(NT, W) void k_loss_block(const agarcl_policy_loss_args a) {
  __shared__ double lds[NT / 64 * 8];
  __shared__ float wl[2][NT / 64][4];
  LossTotals t;
  if (!loss_begin(a, t, lds)) return;
  float acc[7] = {0, 0, 0, 0, 0, 0, 0};
  int parity = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
    const T *zp = (const T *)a.logits + row * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    T *dz = (T *)a.dlogits + row * a.kinds;
    RowIn in = row_in<T>(a, row);
    if constexpr (CHUNKS > 0) {
      Share<T, CHUNKS> z; z.load(zp, ok, threadIdx.x * 8, NT * 8, a.kinds, true);
      row_kind<T>(a, in, zp, ok);
      const float top = wave_max(z.top(ok));
      RowSums r = {finite_max(top), 0.f, 0.f};
      z.sum(r);
      r.s = wave_sum(r.s); r.u = wave_sum(r.u);
      r.m = top;
      const RowSums all = join_waves<NT>(r, wl, parity);
      const LossRow o = loss_row<T>(a, t, row, in, all, threadIdx.x == 0, acc);
      if (a.dlogits) z.gradient(in, o, all.m, threadIdx.x * 8, NT * 8, dz);
    } else {
      row_kind<T>(a, in, zp, ok);
      RowSums r = {-INFINITY, 0.f, 0.f};
      for (int64_t j0 = (int64_t)threadIdx.x * 8; j0 < a.kinds; j0 += NT * 8) {
        const int64_t b = Share<T, 1>::begin(j0, a.kinds);
        Kinds<T, 8> z; z.load(zp + b, ok ? ok + b : nullptr);
        if (ok) z.mask();
        float m = r.m;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, z[k]);
        sums_shift(r, m);
        RowSums c = {finite_max(m), 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; ++k) sums_add(c, k < (int)(j0 - b) ? -INFINITY : z[k]);
        r.s += c.s; r.u += c.u;
      }
      sums_shift(r, wave_max(r.m));
      r.s = wave_sum(r.s); r.u = wave_sum(r.u);
      const RowSums all = join_waves<NT>(r, wl, parity);
      const LossRow o = loss_row<T>(a, t, row, in, all, threadIdx.x == 0, acc);
      if (a.dlogits) {
        for (int64_t j0 = (int64_t)threadIdx.x * 8; j0 < a.kinds; j0 += NT * 8) {
          const int64_t b = Share<T, 1>::begin(j0, a.kinds);
          Kinds<T, 8> z; z.load(zp + b, ok ? ok + b : nullptr);
          if (ok) z.mask();
          loss_kinds<T, 8>(in, o, all.m, b, z, dz);
        }
      }
    }
  }
  loss_end(a, acc, lds);
}

// the workgroups' sums in a fixed order: the same inputs give the same bits.  One wavefront per sum, so that its loads are all under way at once (a wavefront that
// took all seven in turn needed 6.7 us for 2048 workgroups, this 4)
__global__ __launch_bounds__(512) void k_loss_stats(const agarcl_policy_loss_args a, int blocks) {
  __shared__ double sums[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave < 7) {
    double s = 0;
#pragma unroll 8
    for (int b = lane; b < blocks; b += 64) s += a.work[wave * kLossBlocks + b];
    s = wave_sum(s);
    if (lane == 0) sums[wave] = s;
  }
  __syncthreads();
  if (threadIdx.x) return;
  const double inv = sums[0] != 0 ? 1. / sums[0] : 0., by = a.mean_over_weight ? inv : 1.;
  const double kl = a.kl_coef != 0.f ? (double)a.kl_coef * sums[2] : 0., ent = a.entropy_coef != 0.f ? (double)a.entropy_coef * sums[3] : 0.;
  a.loss[0] = (float)((kl - sums[1] - ent) * by);
  for (int i = 1; i < 5; ++i) a.stats[i - 1] = (float)(sums[i] * inv);
  a.stats[4] = (float)sums[0]; a.stats[5] = a.stats[6] = a.stats[7] = 0.f;
  if (a.dlog_std && !a.log_std_per_row) {
    const double up = a.upstream ? (double)*a.upstream : 1.;
    for (int d = 0; d < 2; ++d) ((float *)a.dlog_std)[d] = (float)(sums[5 + d] * by * up);
  }
}

// How many kinds call for which kernel.  What a row needs besides its kinds (a logarithm, exponentials, the sums over its lanes) is a few hundred instructions of every
// wavefront that works on it, so lanes hold several chunks: 65536 rows of 500 bf16 kinds with 64 / 32 lanes of 1 / 2 chunks 112 / 56 us.  As many workgroups as are
// resident at once, for the most wavefronts per SIMD whose registers hold the chunks: those that wait for a place come late and alone.  40 to 50 million kinds, us:
//   lanes       2 chunks or, of 16-bit kinds, 3 where their lanes are filled better; bf16 with a mask / f32 of 350 kinds 3 chunks 56 / 45, 2 chunks more than 62 / 44;
//               of 1000 kinds 2 chunks 55 / 43, 4 chunks 56 / 44, with 4 workgroups per unit instead of as many as are resident 68 / 43; of 2048 4 chunks 55 / 43
//   workgroups  4000 kinds 128 x 4 chunks 66 / 52, 256 x 2 71 / 51; 6144 kinds 256 x 3 64 / 49, 128 x 6 68 / 54; 8000 kinds 256 x 4 66 / 53, 128 x 8 75 / 61.
//               Twice as many workgroups as are resident: 6144 kinds 68 instead of 64, f32 71 instead of 49
//   beyond      a workgroup of 256 reads a row twice: 9000 kinds 79 / 62; 1024 threads that hold a row of 16384 took 74 us where this took 58
static unsigned loss_grid(int64_t rows, int64_t per, int64_t most) { const int64_t n = (rows + per - 1) / per; return (unsigned)(n < 1 ? 1 : n < most ? n : most); }
template <class T, int CHUNKS, int W> static unsigned lanes_launch(const agarcl_policy_loss_args &a, hipStream_t st) {
  int g_log = 0;
  while ((CHUNKS * 8 << g_log) < a.kinds) ++g_log;
  const unsigned grid = loss_grid(a.rows, 256 >> g_log, kUnits * W);
  k_loss_lanes<T, CHUNKS, W><<<dim3(grid), 256, 0, st>>>(a, g_log);
  return grid;
}
template <class T, int NT, int CHUNKS, int W> static unsigned block_launch(const agarcl_policy_loss_args &a, hipStream_t st) {
  static_assert(kUnits * W * 256 / NT <= kLossBlocks, "work holds the sums of kLossBlocks workgroups");
  const unsigned grid = loss_grid(a.rows, 1, kUnits * W * 256 / NT);
  k_loss_block<T, NT, CHUNKS, W><<<dim3(grid), NT, 0, st>>>(a);
  return grid;
}
template <class T> static unsigned loss_launch(const agarcl_policy_loss_args &a, hipStream_t st) {
  const int64_t V = a.kinds;
  constexpr bool H = sizeof(T) == 2;
  const auto room = [&](int64_t chunks) { int64_t n = chunks * 8; while (n < V) n *= 2; return n; };      // the kinds that the lanes of a row hold
  if (V <= 8) {
    const unsigned grid = loss_grid(a.rows, 256, kUnits * 4);
    switch ((int)V) {
#define ONE(n) case n: k_loss_thread<T, n><<<dim3(grid), 256, 0, st>>>(a); break;
      ONE(1) ONE(2) ONE(3) ONE(4) ONE(5) ONE(6) ONE(7) ONE(8)
#undef ONE
    }
    return grid;
  }
  if (V <= 1536 && (V > 1024 || (H && room(3) < room(2)))) return lanes_launch<T, 3, H ? 6 : 5>(a, st);
  if (V <= 1024) return lanes_launch<T, 2, H ? 7 : 5>(a, st);
  if (V <= 2048) return lanes_launch<T, 4, H ? 5 : 4>(a, st);
  if (V <= 128 * 8 * 4) return block_launch<T, 128, 4, H ? 5 : 4>(a, st);
  if (V <= 256 * 8 * 3) return block_launch<T, 256, 3, H ? 6 : 5>(a, st);
  if (V <= 256 * 8 * 4) return block_launch<T, 256, 4, H ? 5 : 4>(a, st);
  return block_launch<T, 256, 0, 7>(a, st);
}

// Sampling: the same pass with the largest score beside the sums.  65536 rows of 24 bf16 kinds, masked, with gumbel 5.2 us (2.2 TB/s: latency); 4096 of 3 with a move 3.1,
// a launch.
// ---- sampling -----------------------------------------------------------------------------------------------------------------------------------
// a thread's share of a row: its sums, and the largest score with its (lowest) index; NONE: nothing allowed
static const int NONE = INT32_MAX;
struct Pick { RowSums r; float best; int at; };
__device__ __forceinline__ void pick_join(Pick &p, float best, int at) { if (at != NONE && (p.at == NONE || best > p.best || (best == p.best && at < p.at))) { p.best = best; p.at = at; } }

template <class T, int VE> __device__ __forceinline__ void pick_kinds(Pick &p, const T *z, const uint8_t *ok, const float *gum, int64_t j0, int skip) {
  Kinds<T, VE> k; k.load(z + j0, ok ? ok + j0 : nullptr);
  Raw<float, VE> gu;
  if (gum) load_raw<float, VE>(gu, gum + j0);
  if (ok) k.mask();
  float m = p.r.m;
#pragma unroll
  for (int i = 0; i < VE; ++i) m = fmaxf(m, k[i]);
  sums_shift(p.r, m);
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const float v = k[i];
    if (v == -INFINITY || i < skip) continue;
    p.r.s += __expf(below(v, m));
    const float score = gum ? v + gu[i] : v;
    if (p.at == NONE || score > p.best) { p.best = score; p.at = (int)(j0 + i); }      // (indices rise within a thread: the first of equals stays)
  }
}
template <class T> __device__ __forceinline__ void pick_write(const agarcl_sample_args &a, int64_t row, const Pick &p, const T *z) {
  float lp = p.at != NONE ? to_f(z[p.at]) - p.r.m - logf(p.r.s) : 0.f;
  a.kind[row] = p.at != NONE ? p.at : 0;
  if (a.mean) {
    float raw[2], move[2];
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const float ls = log_std_at<T>(a.log_std, a.log_std_per_row, row, d), n = a.normal ? a.normal[2 * row + d] : 0.f;
      raw[d] = fmaf(expf(ls), n, to_f(((const T *)a.mean)[2 * row + d]));
      move[d] = __builtin_elementwise_minimum(__builtin_elementwise_maximum(raw[d], -1.f), 1.f);      // (a NaN stays one, and shows in the log-probability, where a NaN mean would not)
      lp -= raw[d] == raw[d] ? 0.5f * n * n + ls + kHalfLog2Pi : raw[d];
    }
    store_pack<float, 2>(a.raw + 2 * row, raw); store_pack<float, 2>(a.move + 2 * row, move);
  }
  a.log_prob[row] = lp;
}

template <class T, int V>
__global__ __launch_bounds__(256) void k_sample_thread(const agarcl_sample_args a) {
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    const T *z = (const T *)a.logits + row * a.logits_stride;
    Pick p = {{-INFINITY, 0.f, 0.f}, -INFINITY, NONE};
    pick_kinds<T, V>(p, z, a.allowed ? a.allowed + row * a.allowed_stride : nullptr, a.gumbel ? a.gumbel + row * a.gumbel_stride : nullptr, 0, 0);
    pick_write<T>(a, row, p, z);
  }
}

// a group of 1 << g_log lanes per row; g_log = 8: the workgroup
template <class T>
__global__ __launch_bounds__(256) void k_sample_lanes(const agarcl_sample_args a, const int g_log) {
  __shared__ float wl[2][4][4];
  __shared__ Pick picks[2][4];
  const int g = 1 << g_log, lane = threadIdx.x & (g - 1), per = 256 >> g_log, in_wave = g < 64 ? g : 64;
  int parity = 0;
  for (int64_t first = (int64_t)blockIdx.x * per; first < a.rows; first += (int64_t)gridDim.x * per, parity ^= 1) {
    const int64_t row = first + (threadIdx.x >> g_log);
    const bool on = row < a.rows;
    const T *z = (const T *)a.logits + (on ? row : 0) * a.logits_stride;
    Pick p = {{-INFINITY, 0.f, 0.f}, -INFINITY, NONE};
    if (on) {
      const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
      const float *gum = a.gumbel ? a.gumbel + row * a.gumbel_stride : nullptr;
      for (int64_t j0 = (int64_t)lane * 8; j0 < a.kinds; j0 += (int64_t)g * 8) {
        const int64_t b = Share<T, 1>::begin(j0, a.kinds);
        pick_kinds<T, 8>(p, z, ok, gum, b, (int)(j0 - b));
      }
    }
    float m = p.r.m;
    for (int d = 1; d < in_wave; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    sums_shift(p.r, m);
    for (int d = 1; d < in_wave; d <<= 1) {
      p.r.s += __shfl_xor(p.r.s, d);
      const float best = __shfl_xor(p.best, d); const int at = __shfl_xor(p.at, d);
      pick_join(p, best, at);
    }
    if (g_log == 8) {
      p.r = join_waves<256>(p.r, wl, parity);
      if ((threadIdx.x & 63) == 0) picks[parity][threadIdx.x >> 6] = p;
      __syncthreads();
      for (int w = 0; w < 4; ++w) pick_join(p, picks[parity][w].best, picks[parity][w].at);
    }
    if (on && lane == 0) pick_write<T>(a, row, p, z);
  }
}

template <class T> static void sample_launch(const agarcl_sample_args &a, hipStream_t st) {
  const int64_t V = a.kinds;
  const auto grid = [&](int64_t per) { const int64_t n = (a.rows + per - 1) / per; return dim3((unsigned)(n < 65536 ? n : 65536)); };
  if (V <= 8) {
    switch ((int)V) {
#define ONE(n) case n: k_sample_thread<T, n><<<grid(256), 256, 0, st>>>(a); break;
      ONE(1) ONE(2) ONE(3) ONE(4) ONE(5) ONE(6) ONE(7) ONE(8)
#undef ONE
    }
    return;
  }
  int g_log = 1;
  while (g_log < 6 && (8 << g_log) < V) ++g_log;
  if (V > 1024) g_log = 8;
  k_sample_lanes<T><<<grid(256 >> g_log), 256, 0, st>>>(a, g_log);
}
