// learn_common.inl -- element types and wave-wide sums of the learner's operators
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T> __device__ inline float to_f(T v) { return (float)v; }
template <class T> __device__ inline T from_f(float v) { return (T)v; }      // one rounding to nearest even

__device__ inline float wave_max(float v) { for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d)); return v; }
__device__ inline float wave_sum(float v) { for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d); return v; }
__device__ inline double wave_sum(double v) { for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d); return v; }

// f = sigmoid(g) and q = 1 - f, both to full relative accuracy at either end and without overflow; returns the lesser of them with g's sign
__device__ inline float sigmoid2(float g, float &f, float &q) {
  const float t = __expf(-fabsf(g)), r = __builtin_amdgcn_rcpf(1.f + t), s = t * r;
  f = g >= 0.f ? r : s; q = g >= 0.f ? s : r;
  return copysignf(s, g);
}
// f and q again from what that returned: 1 - the lesser is the greater to full accuracy (1 - the greater would keep nothing of a small one)
__device__ inline void sigmoid_again(float s, float &f, float &q) {
  const float less = fabsf(s), more = 1.f - less;
  const bool keeps = __float_as_int(s) >= 0;
  f = keeps ? more : less; q = keeps ? less : more;
}
