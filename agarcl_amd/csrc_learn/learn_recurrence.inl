// learn_recurrence.inl -- gated linear recurrence and advantages: one thread per column, the steps one after the other

template <class T>
__global__ __launch_bounds__(256) void k_recurrence(const T *__restrict__ x, const T *__restrict__ gate, int64_t xs, int64_t gs, const float *__restrict__ state,
    const uint8_t *__restrict__ reset, int64_t rs, T *__restrict__ h, float *__restrict__ last, float *__restrict__ marks, int64_t steps, int64_t rows, int64_t width) {
  const int64_t K = rows * width;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < K; c += (int64_t)gridDim.x * 256) {
  const int64_t b = c / width;
  float s = state ? state[c] : 0.f;
  for (int64_t t = 0; t < steps; ++t) {
    if (marks && (t % AGARCL_MARK_STEPS) == 0) marks[t / AGARCL_MARK_STEPS * K + c] = s;
    const float p = reset && reset[t * rs + b] ? 0.f : s;
    float f, q; sigmoid2(to_f(gate[t * gs + c]), f, q);
    s = fmaf(f, p, q * to_f(x[t * xs + c]));
    h[t * K + c] = from_f<T>(s);
  }
  last[c] = s;
  }
}

// E[t] = the gradient that reaches h[t-1] = keep f (dh[t] + E[t+1]); G = dh[t] + E[t+1]
template <class T>
__global__ __launch_bounds__(256) void k_recurrence_grad(const T *__restrict__ x, const T *__restrict__ gate, int64_t xs, int64_t gs, const uint8_t *__restrict__ reset, int64_t rs,
    const float *__restrict__ marks, const T *__restrict__ dh, int64_t ds, const float *__restrict__ dlast, T *__restrict__ dx, T *__restrict__ dgate, float *__restrict__ dstate,
    int64_t steps, int64_t rows, int64_t width) {
  const int64_t K = rows * width;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < K; c += (int64_t)gridDim.x * 256) {
  const int64_t b = c / width;
  float E = dlast ? dlast[c] : 0.f;
  for (int64_t m = (steps + AGARCL_MARK_STEPS - 1) / AGARCL_MARK_STEPS - 1; m >= 0; --m) {
    const int64_t t0 = m * AGARCL_MARK_STEPS;
    float p[AGARCL_MARK_STEPS];      // what each step saw of the state before it, from the kept one
    float s = marks[m * K + c];
#pragma unroll
    for (int i = 0; i < AGARCL_MARK_STEPS; ++i) {
      const int64_t t = t0 + i;
      if (t >= steps) break;
      p[i] = reset && reset[t * rs + b] ? 0.f : s;
      float f, q; sigmoid2(to_f(gate[t * gs + c]), f, q);
      s = fmaf(f, p[i], q * to_f(x[t * xs + c]));
    }
#pragma unroll
    for (int i = AGARCL_MARK_STEPS - 1; i >= 0; --i) {
      const int64_t t = t0 + i;
      if (t >= steps) continue;
      const float G = (dh ? to_f(dh[t * ds + c]) : 0.f) + E;
      float f, q; sigmoid2(to_f(gate[t * gs + c]), f, q);
      dx[t * K + c] = from_f<T>(q * G);
      dgate[t * K + c] = from_f<T>(G * (p[i] - to_f(x[t * xs + c])) * f * q);
      E = reset && reset[t * rs + b] ? 0.f : f * G;
    }
  }
  dstate[c] = E;
  }
}

template <class T>
__global__ __launch_bounds__(256) void k_advantages(const float *__restrict__ reward, const T *__restrict__ value, const T *__restrict__ next_value,
    const uint8_t *__restrict__ terminated, const uint8_t *__restrict__ truncated, const T *__restrict__ final_value, int64_t rs, int64_t vs, int64_t es, int64_t us, int64_t fs,
    float gamma, float gl, float *__restrict__ advantage, float *__restrict__ returns, int64_t steps, int64_t rows) {
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < rows; b += (int64_t)gridDim.x * 256) {
  float next = to_f(next_value[b]), A = 0.f;
  for (int64_t t = steps - 1; t >= 0; --t) {
    const float v = to_f(value[t * vs + b]), r = reward[t * rs + b];
    const bool term = terminated[t * es + b], trunc = !term && truncated && truncated[t * us + b];
    float delta;
    if (term) delta = r - v;
    else if (!trunc) delta = fmaf(gamma, next, r) - v;
    else delta = final_value ? fmaf(gamma, to_f(final_value[t * fs + b]), r) - v : 0.f;
    A = term || trunc ? delta : fmaf(gl, A, delta);
    advantage[t * rows + b] = A; returns[t * rows + b] = A + v;
    next = v;
  }
  }
}
