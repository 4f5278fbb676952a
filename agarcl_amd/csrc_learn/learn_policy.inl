// learn_policy.inl -- the clipped policy loss with its gradients, and the sampling of actions.
//
// Both are one pass over the logits: a row is in registers (or, beyond 32768 kinds, read twice) while its maximum, the sum s of e^(z - max) and
// u = sum of e^(z - max) (z - max) are taken; log s and u / s give the log-probabilities and the entropy, and the gradient is written from the same registers:
// reading the logits once and writing their gradient once is all the memory traffic there has to be.  Up to 8 kinds a row is one thread's, up to 1024
// a group of 2 to 64 lanes', beyond that a workgroup's.

static const int kLossBlocks = 2048, kWeightBlocks = 256;
static const int64_t kLossWork = 8 * kLossBlocks + kWeightBlocks;
static const float kHalfLog2Pi = 0.91893853320467274f, kHalfLog2PiE = 1.4189385332046727f;

template <class T> __device__ __forceinline__ float log_std_at(const void *p, int per_row, int64_t row, int d) {
  return per_row ? to_f(((const T *)p)[2 * row + d]) : ((const float *)p)[d];
}

__global__ __launch_bounds__(256) void k_weight_sum(const float *__restrict__ w, int64_t rows, double *__restrict__ out) {
  __shared__ double part[4];
  double s = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows; i += (int64_t)gridDim.x * 256) s += (double)w[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) out[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// bit k: kind k of these VE may be chosen
template <int VE> __device__ __forceinline__ uint32_t load_allowed(const uint8_t *p, int nv) {
  uint32_t bits = 0;
  if (VE == 8 && nv == 8) {
    struct __attribute__((packed)) Eight { uint32_t w[2]; };
    const Eight e = *(const Eight *)p;
#pragma unroll
    for (int k = 0; k < 8; ++k) bits |= (e.w[k / 4] >> (8 * (k % 4))) & 255u ? 1u << k : 0u;
  } else {
#pragma unroll
    for (int k = 0; k < VE; ++k) if (k < nv) bits |= p[k] ? 1u << k : 0u;
  }
  return bits;
}

// VE neighbouring logits of a row: what is not allowed, or not there, as -inf
template <class T, int VE> struct Kinds {
  Raw<T, VE> raw; uint32_t ok;
  __device__ __forceinline__ void load(const T *z, const uint8_t *allowed, int nv) {
    load_raw<T, VE>(raw, z, nv);
    ok = allowed ? load_allowed<VE>(allowed, nv) : (1u << nv) - 1u;
  }
  __device__ __forceinline__ float operator[](int k) const { return (ok >> k) & 1 ? raw[k] : -INFINITY; }
};

// what a row's kinds come to, relative to the maximum m
struct RowSums { float m, s, u; };
__device__ __forceinline__ float exp_below(float z, float m) { return z == -INFINITY ? 0.f : __expf(z - m); }
__device__ __forceinline__ void sums_add(RowSums &r, float z, float e) { r.s += e; if (e > 0.f) r.u += e * (z - r.m); }
// r's sums relative to another maximum
__device__ __forceinline__ void sums_shift(RowSums &r, float m) {
  if (r.s > 0.f && m != r.m) { const float d = r.m - m, k = __expf(d); r.u = k * (r.u + r.s * d); r.s *= k; }
  r.m = m;
}

// everything of a row that is not per kind
struct LossRow { bool counts; int32_t kind; float share, g, log_s, hcat, dev[2], istd[2]; };
struct LossTotals { float inv; bool shared_std; };

template <class T> __device__ __forceinline__ LossRow loss_row(const agarcl_policy_loss_args &a, const LossTotals &t, int64_t row, const RowSums &r, const T *z, const uint8_t *ok,
    bool leader, double (&acc)[7]) {
  LossRow o;
  const float w = a.weight ? a.weight[row] : 1.f, A = a.advantage[row], old = a.old_log_prob[row], ref = a.ref_log_prob ? a.ref_log_prob[row] : old;
  const int32_t kind = o.kind = a.kind[row];
  o.counts = w != 0.f && kind >= 0 && kind < a.kinds;
  float za = 0.f;
  if (o.counts) { za = to_f(z[kind]); o.counts = za != -INFINITY && (!ok || ok[kind]); }
  o.log_s = logf(r.s); o.hcat = o.log_s - r.u / r.s;
  float lp = za - r.m - o.log_s, ent = o.hcat;
#pragma unroll
  for (int d = 0; d < 2; ++d) o.dev[d] = o.istd[d] = 0.f;
  if (a.mean) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const float ls = log_std_at<T>(a.log_std, a.log_std_per_row, row, d);
      o.istd[d] = expf(-ls);
      o.dev[d] = (a.move[2 * row + d] - to_f(((const T *)a.mean)[2 * row + d])) * o.istd[d];
      lp -= 0.5f * o.dev[d] * o.dev[d] + ls + kHalfLog2Pi;
      ent += ls + kHalfLog2PiE;
    }
  }
  const float ratio = expf(lp - old);
  const float low = A == 0.f ? 0.f : fminf(ratio * A, fminf(fmaxf(ratio, 1.f - a.clip_low), 1.f + a.clip_high) * A);
  const bool clipped = A >= 0.f ? ratio > 1.f + a.clip_high : ratio < 1.f - a.clip_low;
  const float back = ref - lp, eb = expm1f(back), kl = eb - back;      // (expm1: near 0 the KL term is the difference of near numbers)
  o.g = clipped || A == 0.f ? 0.f : -A * ratio;
  if (a.kl_coef != 0.f) o.g -= a.kl_coef * eb;
  o.share = w * t.inv;
  if (leader) {
    acc[0] += (double)w;
    if (o.counts) {
      acc[1] += (double)w * low; acc[2] += (double)w * kl; acc[3] += (double)w * ent; acc[4] += clipped ? (double)w : 0.;
      if (t.shared_std) {
#pragma unroll
        for (int d = 0; d < 2; ++d) acc[5 + d] += (double)w * (o.g * (o.dev[d] * o.dev[d] - 1.f) - a.entropy_coef);
      }
    }
    if (a.dmean) {
      float v[2];
#pragma unroll
      for (int d = 0; d < 2; ++d) v[d] = o.counts ? o.share * o.g * o.dev[d] * o.istd[d] : 0.f;
      store_pack<T, 2>((T *)a.dmean + 2 * row, v, 2);
    }
    if (a.dlog_std && a.log_std_per_row) {
      float v[2];
#pragma unroll
      for (int d = 0; d < 2; ++d) v[d] = o.counts ? o.share * (o.g * (o.dev[d] * o.dev[d] - 1.f) - a.entropy_coef) : 0.f;
      store_pack<T, 2>((T *)a.dlog_std + 2 * row, v, 2);
    }
  }
  return o;
}

// the gradient of kinds j0 ... of a row.  The probabilities are worked out once more: holding 8 of them for every 4 registers of logits would cost more
// (registers, and with them wavefronts) than a second exp
template <class T, int VE> __device__ __forceinline__ void loss_kinds(const agarcl_policy_loss_args &a, const LossRow &o, const RowSums &r, int64_t row, int64_t j0, int nv, Kinds<T, VE> &z) {
  const float rs = 1.f / r.s;
  z.raw.anew();
  float v[VE];
#pragma unroll
  for (int k = 0; k < VE; ++k) {
    const float p = exp_below(z[k], r.m) * rs;
    float d = o.g * ((j0 + k == o.kind ? 1.f : 0.f) - p);
    if (a.entropy_coef != 0.f && p > 0.f) d += a.entropy_coef * p * (z[k] - r.m - o.log_s + o.hcat);
    v[k] = o.counts && (z.ok >> k) & 1 ? o.share * d : 0.f;
  }
  store_pack<T, VE>((T *)a.dlogits + row * a.kinds + j0, v, nv);
}

// what comes before the rows; false: there is nothing to do
__device__ __forceinline__ bool loss_begin(const agarcl_policy_loss_args &a, LossTotals &t, double *lds) {
  const bool grads = a.dlogits || a.dmean || (a.dlog_std && a.log_std_per_row);
  t.shared_std = a.mean && !a.log_std_per_row && a.dlog_std;
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
__device__ __forceinline__ void loss_end(const agarcl_policy_loss_args &a, double (&acc)[7], double *lds) {
  if (!a.want_stats) return;
#pragma unroll
  for (int i = 0; i < 7; ++i) { const double s = wave_sum(acc[i]); if ((threadIdx.x & 63) == 0) lds[8 * (threadIdx.x >> 6) + i] = s; }
  __syncthreads();
  if (threadIdx.x < 7) {
    double s = 0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += lds[8 * i + threadIdx.x];
    a.work[8 * blockIdx.x + threadIdx.x] = s;
  }
}

// V kinds, one thread per row
template <class T, int V>
__global__ __launch_bounds__(256) void k_loss_thread(const agarcl_policy_loss_args a) {
  __shared__ double lds[32];
  LossTotals t;
  if (!loss_begin(a, t, lds)) return;
  double acc[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    const T *zp = (const T *)a.logits + row * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    Kinds<T, V> z; z.load(zp, ok, V);
    RowSums r = {-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < V; ++k) r.m = fmaxf(r.m, z[k]);
#pragma unroll
    for (int k = 0; k < V; ++k) sums_add(r, z[k], exp_below(z[k], r.m));
    const LossRow o = loss_row<T>(a, t, row, r, zp, ok, true, acc);
    if (a.dlogits) loss_kinds<T, V>(a, o, r, row, 0, V, z);
  }
  loss_end(a, acc, lds);
}

// 8 << g_log (x CHUNKS) kinds, a group of 1 << g_log lanes per row
template <class T, int CHUNKS>
__global__ __launch_bounds__(256) void k_loss_lanes(const agarcl_policy_loss_args a, const int g_log) {
  __shared__ double lds[32];
  LossTotals t;
  if (!loss_begin(a, t, lds)) return;
  double acc[7] = {0, 0, 0, 0, 0, 0, 0};
  const int g = 1 << g_log, lane = threadIdx.x & (g - 1), per = 256 >> g_log;
  for (int64_t first = (int64_t)blockIdx.x * per; first < a.rows; first += (int64_t)gridDim.x * per) {
    const int64_t row = first + (threadIdx.x >> g_log);
    const bool on = row < a.rows;
    const T *zp = (const T *)a.logits + (on ? row : 0) * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + (on ? row : 0) * a.allowed_stride : nullptr;
    Kinds<T, 8> z[CHUNKS]; int nv[CHUNKS];
    RowSums r = {-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int64_t j0 = (int64_t)(c * g + lane) * 8, left = a.kinds - j0;
      nv[c] = on ? (left < 0 ? 0 : left < 8 ? (int)left : 8) : 0;
      z[c].load(zp + j0, ok ? ok + j0 : nullptr, nv[c]);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int k = 0; k < 8; ++k) r.m = fmaxf(r.m, z[c][k]);
    }
    for (int d = 1; d < g; d <<= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, d));
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      z[c].raw.anew();
#pragma unroll
      for (int k = 0; k < 8; ++k) sums_add(r, z[c][k], exp_below(z[c][k], r.m));
    }
    for (int d = 1; d < g; d <<= 1) { r.s += __shfl_xor(r.s, d); r.u += __shfl_xor(r.u, d); }
    if (!on) continue;      // (a whole group, behind the last of the shuffles of this turn)
    const LossRow o = loss_row<T>(a, t, row, r, zp, ok, lane == 0, acc);
    if (a.dlogits) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) loss_kinds<T, 8>(a, o, r, row, (int64_t)(c * g + lane) * 8, nv[c], z[c]);
    }
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
  return all;
}

// NT x 8 x CHUNKS kinds in registers, a workgroup per row; CHUNKS = 0: any number, read twice
template <class T, int NT, int CHUNKS>
__global__ __launch_bounds__(NT) void k_loss_block(const agarcl_policy_loss_args a) {
  __shared__ double lds[NT / 64 * 8];
  __shared__ float wl[2][NT / 64][4];
  LossTotals t;
  if (!loss_begin(a, t, lds)) return;
  double acc[7] = {0, 0, 0, 0, 0, 0, 0};
  int parity = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
    const T *zp = (const T *)a.logits + row * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    RowSums r = {-INFINITY, 0.f, 0.f};
    if constexpr (CHUNKS > 0) {
      Kinds<T, 8> z[CHUNKS]; int nv[CHUNKS];
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int64_t j0 = (int64_t)(c * NT + threadIdx.x) * 8, left = a.kinds - j0;
        nv[c] = left < 0 ? 0 : left < 8 ? (int)left : 8;
        z[c].load(zp + j0, ok ? ok + j0 : nullptr, nv[c]);
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
        for (int k = 0; k < 8; ++k) r.m = fmaxf(r.m, z[c][k]);
      }
      r.m = wave_max(r.m);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        z[c].raw.anew();
#pragma unroll
        for (int k = 0; k < 8; ++k) sums_add(r, z[c][k], exp_below(z[c][k], r.m));
      }
      r.s = wave_sum(r.s); r.u = wave_sum(r.u);
      const RowSums all = join_waves<NT>(r, wl, parity);
      const LossRow o = loss_row<T>(a, t, row, all, zp, ok, threadIdx.x == 0, acc);
      if (a.dlogits) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) loss_kinds<T, 8>(a, o, all, row, (int64_t)(c * NT + threadIdx.x) * 8, nv[c], z[c]);
      }
    } else {
      for (int64_t j0 = (int64_t)threadIdx.x * 8; j0 < a.kinds; j0 += NT * 8) {
        Kinds<T, 8> z; z.load(zp + j0, ok ? ok + j0 : nullptr, a.kinds - j0 < 8 ? (int)(a.kinds - j0) : 8);
        float m = r.m;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, z[k]);
        sums_shift(r, m);
#pragma unroll
        for (int k = 0; k < 8; ++k) sums_add(r, z[k], exp_below(z[k], m));
      }
      sums_shift(r, wave_max(r.m));
      r.s = wave_sum(r.s); r.u = wave_sum(r.u);
      const RowSums all = join_waves<NT>(r, wl, parity);
      const LossRow o = loss_row<T>(a, t, row, all, zp, ok, threadIdx.x == 0, acc);
      if (a.dlogits) {
        for (int64_t j0 = (int64_t)threadIdx.x * 8; j0 < a.kinds; j0 += NT * 8) {
          const int nv = a.kinds - j0 < 8 ? (int)(a.kinds - j0) : 8;
          Kinds<T, 8> z; z.load(zp + j0, ok ? ok + j0 : nullptr, nv);
          loss_kinds<T, 8>(a, o, all, row, j0, nv, z);
        }
      }
    }
  }
  loss_end(a, acc, lds);
}

// the workgroups' sums in a fixed order: the same inputs give the same bits
__global__ __launch_bounds__(1024) void k_loss_stats(const agarcl_policy_loss_args a, int blocks) {
  __shared__ double part[16][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double acc[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int b = threadIdx.x; b < blocks; b += 1024) for (int i = 0; i < 7; ++i) acc[i] += a.work[8 * b + i];
  for (int i = 0; i < 7; ++i) { acc[i] = wave_sum(acc[i]); if (lane == 0) part[wave][i] = acc[i]; }
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 0; i < 7; ++i) { acc[i] = 0; for (int w = 0; w < 16; ++w) acc[i] += part[w][i]; }
  const double inv = acc[0] != 0 ? 1. / acc[0] : 0., by = a.mean_over_weight ? inv : 1.;
  const double kl = a.kl_coef != 0.f ? (double)a.kl_coef * acc[2] : 0., ent = a.entropy_coef != 0.f ? (double)a.entropy_coef * acc[3] : 0.;
  a.loss[0] = (float)((kl - acc[1] - ent) * by);
  for (int i = 1; i < 5; ++i) a.stats[i - 1] = (float)(acc[i] * inv);
  a.stats[4] = (float)acc[0]; a.stats[5] = a.stats[6] = a.stats[7] = 0.f;
  if (a.dlog_std && !a.log_std_per_row) for (int d = 0; d < 2; ++d) ((float *)a.dlog_std)[d] = (float)(acc[5 + d] * by);
}

// how many kinds call for which kernel; the workgroups a launch needs
static unsigned loss_grid(int64_t rows, int64_t per) { const int64_t n = (rows + per - 1) / per; return (unsigned)(n < kLossBlocks ? n : kLossBlocks); }
template <class T> static unsigned loss_launch(const agarcl_policy_loss_args &a, hipStream_t st) {
  const int64_t V = a.kinds;
  unsigned grid;
  if (V <= 8) {
    grid = loss_grid(a.rows, 256);
    switch ((int)V) {
#define ONE(n) case n: k_loss_thread<T, n><<<dim3(grid), 256, 0, st>>>(a); break;
      ONE(1) ONE(2) ONE(3) ONE(4) ONE(5) ONE(6) ONE(7) ONE(8)
#undef ONE
    }
  } else if (V <= 1024) {
    int g_log = 1;
    while (g_log < 6 && (8 << g_log) < V) ++g_log;
    grid = loss_grid(a.rows, 256 >> g_log);
    if (V <= 512) k_loss_lanes<T, 1><<<dim3(grid), 256, 0, st>>>(a, g_log);
    else k_loss_lanes<T, 2><<<dim3(grid), 256, 0, st>>>(a, g_log);
  } else {
    grid = loss_grid(a.rows, 1);
    if (V <= 4096) k_loss_block<T, 256, 2><<<dim3(grid), 256, 0, st>>>(a);
    else if (V <= 8192) k_loss_block<T, 256, 4><<<dim3(grid), 256, 0, st>>>(a);
    else if (V <= 16384) k_loss_block<T, 1024, 2><<<dim3(grid), 1024, 0, st>>>(a);
    else if (V <= 32768) k_loss_block<T, 1024, 4><<<dim3(grid), 1024, 0, st>>>(a);
    else k_loss_block<T, 1024, 0><<<dim3(grid), 1024, 0, st>>>(a);
  }
  return grid;
}

// ---- sampling -----------------------------------------------------------------------------------------------------------------------------------
// a thread's share of a row: its sums, and the largest score with its (lowest) index; NONE: nothing allowed
static const int NONE = INT32_MAX;
struct Pick { RowSums r; float best; int at; };
__device__ __forceinline__ void pick_join(Pick &p, float best, int at) { if (at != NONE && (p.at == NONE || best > p.best || (best == p.best && at < p.at))) { p.best = best; p.at = at; } }

template <class T, int VE> __device__ __forceinline__ void pick_kinds(Pick &p, const T *z, const uint8_t *ok, const float *gum, int64_t j0, int nv) {
  Kinds<T, VE> k; k.load(z + j0, ok ? ok + j0 : nullptr, nv);
  Raw<float, VE> gu;
  if (gum) load_raw<float, VE>(gu, gum + j0, nv);
  float m = p.r.m;
#pragma unroll
  for (int i = 0; i < VE; ++i) m = fmaxf(m, k[i]);
  sums_shift(p.r, m);
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const float v = k[i];
    if (v == -INFINITY) continue;
    p.r.s += __expf(v - m);
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
      move[d] = fminf(fmaxf(raw[d], -1.f), 1.f);
      lp -= 0.5f * n * n + ls + kHalfLog2Pi;
    }
    store_pack<float, 2>(a.raw + 2 * row, raw, 2); store_pack<float, 2>(a.move + 2 * row, move, 2);
  }
  a.log_prob[row] = lp;
}

template <class T, int V>
__global__ __launch_bounds__(256) void k_sample_thread(const agarcl_sample_args a) {
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    const T *z = (const T *)a.logits + row * a.logits_stride;
    Pick p = {{-INFINITY, 0.f, 0.f}, -INFINITY, NONE};
    pick_kinds<T, V>(p, z, a.allowed ? a.allowed + row * a.allowed_stride : nullptr, a.gumbel ? a.gumbel + row * a.gumbel_stride : nullptr, 0, V);
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
      for (int64_t j0 = (int64_t)lane * 8; j0 < a.kinds; j0 += (int64_t)g * 8) pick_kinds<T, 8>(p, z, ok, gum, j0, a.kinds - j0 < 8 ? (int)(a.kinds - j0) : 8);
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
