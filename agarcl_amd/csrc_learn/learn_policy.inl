// learn_policy.inl -- the clipped policy loss with its gradients, and the sampling of actions: one wavefront per row, two passes over it

static const int kLossBlocks = 1024, kWeightBlocks = 64;
static const int64_t kLossWork = 8 * kLossBlocks + kWeightBlocks;
static __device__ const float kHalfLog2Pi = 0.91893853320467274f, kHalfLog2PiE = 1.4189385332046727f;

template <class T> __device__ inline float log_std_at(const void *p, int per_row, int64_t row, int d) {
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

// max, sum of exp, sum of exp x (z - max) over the allowed kinds of a row, in every lane
template <class T> __device__ inline void row_sums(const T *z, const uint8_t *ok, int64_t n, int lane, float &m, float &s, float &u) {
  m = -INFINITY;
  for (int64_t j = lane; j < n; j += 64) if (!ok || ok[j]) m = fmaxf(m, to_f(z[j]));
  m = wave_max(m);
  s = u = 0.f;
  if (m == -INFINITY) return;
  for (int64_t j = lane; j < n; j += 64) if (!ok || ok[j]) {
    const float d = to_f(z[j]) - m, e = __expf(d);
    s += e; u += e > 0.f ? e * d : 0.f;
  }
  s = wave_sum(s); u = wave_sum(u);
}

template <class T>
__global__ __launch_bounds__(256) void k_policy_loss(const agarcl_policy_loss_args a) {
  __shared__ double part[4][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool grads = a.dlogits || a.dmean || (a.dlog_std && a.log_std_per_row);
  const bool shared_std = a.mean && !a.log_std_per_row;
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.want_stats) {
    if (a.dlog_std && shared_std && blockIdx.x == 0 && threadIdx.x < 2) ((float *)a.dlog_std)[threadIdx.x] = a.dlog_std_one[threadIdx.x] * up;
    if (!grads || (a.skip_if_one && up == 1.f)) return;
  }
  float inv = up;
  if (a.mean_over_weight) {
    double total = (double)a.rows;
    if (a.weight && grads) {
      if (a.weight_sum) total = (double)*a.weight_sum;
      else { total = 0; for (int i = 0; i < kWeightBlocks; ++i) total += a.work[8 * kLossBlocks + i]; }
    }
    inv = total != 0 ? (float)((double)up / total) : 0.f;
  }
  const float ck = a.kl_coef, ce = a.entropy_coef;
  double acc[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < a.rows; row += (int64_t)gridDim.x * 4) {
    const T *z = (const T *)a.logits + row * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    T *dz = a.dlogits ? (T *)a.dlogits + row * a.kinds : nullptr;
    const float w = a.weight ? a.weight[row] : 1.f;
    acc[0] += (double)w;
    const int32_t kind = a.kind[row];
    const bool counts = w != 0.f && kind >= 0 && kind < a.kinds && (!ok || ok[kind]) && to_f(z[kind]) != -INFINITY;
    if (!counts) {
      if (dz) for (int64_t j = lane; j < a.kinds; j += 64) dz[j] = from_f<T>(0.f);
      if (lane < 2) {
        if (a.dmean) ((T *)a.dmean)[2 * row + lane] = from_f<T>(0.f);
        if (a.dlog_std && a.log_std_per_row) ((T *)a.dlog_std)[2 * row + lane] = from_f<T>(0.f);
      }
      continue;
    }
    float m, s, u;
    row_sums(z, ok, a.kinds, lane, m, s, u);
    const float log_s = logf(s), hcat = log_s - u / s;
    float lp = to_f(z[kind]) - m - log_s, ent = hcat;
    float dev[2] = {0, 0}, istd[2] = {0, 0};
    if (a.mean) for (int d = 0; d < 2; ++d) {
      const float ls = log_std_at<T>(a.log_std, a.log_std_per_row, row, d);
      istd[d] = expf(-ls);
      dev[d] = (a.move[2 * row + d] - to_f(((const T *)a.mean)[2 * row + d])) * istd[d];
      lp -= 0.5f * dev[d] * dev[d] + ls + kHalfLog2Pi;
      ent += ls + kHalfLog2PiE;
    }
    const float A = a.advantage[row], old = a.old_log_prob[row], ratio = expf(lp - old);
    const float low = A == 0.f ? 0.f : fminf(ratio * A, fminf(fmaxf(ratio, 1.f - a.clip_low), 1.f + a.clip_high) * A);
    const bool clipped = A >= 0.f ? ratio > 1.f + a.clip_high : ratio < 1.f - a.clip_low;
    const float back = (a.ref_log_prob ? a.ref_log_prob[row] : old) - lp, eb = expm1f(back), kl = eb - back;
    acc[1] += (double)w * low; acc[2] += (double)w * kl; acc[3] += (double)w * ent; acc[4] += clipped ? (double)w : 0.;
    float g = clipped || A == 0.f ? 0.f : -A * ratio;
    if (ck != 0.f) g -= ck * eb;
    if (shared_std) for (int d = 0; d < 2; ++d) acc[5 + d] += (double)w * (g * (dev[d] * dev[d] - 1.f) - ce);
    const float share = w * inv;
    if (dz) {
      const float rs = 1.f / s;
      for (int64_t j = lane; j < a.kinds; j += 64) {
        float v = 0.f;
        if (!ok || ok[j]) {
          const float d = to_f(z[j]) - m, p = __expf(d) * rs;
          v = g * ((j == kind ? 1.f : 0.f) - p);
          if (ce != 0.f && p > 0.f) v += ce * p * (d - log_s + hcat);
        }
        dz[j] = from_f<T>(share * v);
      }
    }
    if (lane < 2) {
      const float dv = lane ? dev[1] : dev[0], is = lane ? istd[1] : istd[0];
      if (a.dmean) ((T *)a.dmean)[2 * row + lane] = from_f<T>(share * g * dv * is);
      if (a.dlog_std && a.log_std_per_row) ((T *)a.dlog_std)[2 * row + lane] = from_f<T>(share * (g * (dv * dv - 1.f) - ce));
    }
  }
  if (!a.want_stats) return;
  if (lane == 0) for (int i = 0; i < 7; ++i) part[wave][i] = acc[i];
  __syncthreads();
  if (threadIdx.x < 7) a.work[8 * blockIdx.x + threadIdx.x] = part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
}

// the workgroups' sums in a fixed order: the same inputs give the same bits
__global__ __launch_bounds__(256) void k_loss_stats(const agarcl_policy_loss_args a, int blocks) {
  __shared__ double part[4][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double acc[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int b = threadIdx.x; b < blocks; b += 256) for (int i = 0; i < 7; ++i) acc[i] += a.work[8 * b + i];
  for (int i = 0; i < 7; ++i) { acc[i] = wave_sum(acc[i]); if (lane == 0) part[wave][i] = acc[i]; }
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 0; i < 7; ++i) acc[i] = part[0][i] + part[1][i] + part[2][i] + part[3][i];
  const double inv = acc[0] != 0 ? 1. / acc[0] : 0., by = a.mean_over_weight ? inv : 1.;
  const double kl = a.kl_coef != 0.f ? (double)a.kl_coef * acc[2] : 0., ent = a.entropy_coef != 0.f ? (double)a.entropy_coef * acc[3] : 0.;
  a.loss[0] = (float)((kl - acc[1] - ent) * by);
  for (int i = 1; i < 5; ++i) a.stats[i - 1] = (float)(acc[i] * inv);
  a.stats[4] = (float)acc[0]; a.stats[5] = a.stats[6] = a.stats[7] = 0.f;
  if (a.dlog_std && !a.log_std_per_row) for (int d = 0; d < 2; ++d) ((float *)a.dlog_std)[d] = (float)(acc[5 + d] * by);
}

template <class T>
__global__ __launch_bounds__(256) void k_sample(const agarcl_sample_args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < a.rows; row += (int64_t)gridDim.x * 4) {
    const T *z = (const T *)a.logits + row * a.logits_stride;
    const uint8_t *ok = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    const float *gum = a.gumbel ? a.gumbel + row * a.gumbel_stride : nullptr;
    float m, s, u;
    row_sums(z, ok, a.kinds, lane, m, s, u);
    float best = -INFINITY; int at = INT32_MAX;
    for (int64_t j = lane; j < a.kinds; j += 64) if ((!ok || ok[j]) && to_f(z[j]) != -INFINITY) {
      const float v = to_f(z[j]) + (gum ? gum[j] : 0.f);
      if (at == INT32_MAX || v > best) { best = v; at = (int)j; }
    }
    for (int d = 32; d; d >>= 1) {
      const float ob = __shfl_xor(best, d); const int oa = __shfl_xor(at, d);
      if (oa != INT32_MAX && (at == INT32_MAX || ob > best || (ob == best && oa < at))) { best = ob; at = oa; }
    }
    const bool any = at != INT32_MAX;
    if (lane == 0) {
      float lp = any ? to_f(z[at]) - m - logf(s) : 0.f;
      a.kind[row] = any ? at : 0;
      if (a.mean) for (int d = 0; d < 2; ++d) {
        const float ls = log_std_at<T>(a.log_std, a.log_std_per_row, row, d), n = a.normal ? a.normal[2 * row + d] : 0.f;
        const float raw = fmaf(expf(ls), n, to_f(((const T *)a.mean)[2 * row + d]));
        a.raw[2 * row + d] = raw; a.move[2 * row + d] = fminf(fmaxf(raw, -1.f), 1.f);
        lp -= 0.5f * n * n + ls + kHalfLog2Pi;
      }
      a.log_prob[row] = lp;
    }
  }
}
