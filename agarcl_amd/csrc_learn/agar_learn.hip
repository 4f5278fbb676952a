// agar_learn.hip -- the operators of include/agarcl_learn.h: host side of the C ABI.  The kernels are in learn_recurrence.inl (gated recurrence,
// advantages) and learn_policy.inl (clipped policy loss, sampling); learn_common.inl holds what they share.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string>
#include <type_traits>

#include "../../include/agarcl_learn.h"
#include "learn_common.inl"
#include "learn_scan.inl"
#include "learn_recurrence.inl"
#include "learn_policy.inl"

static thread_local std::string g_learn_err;
static int fail(int code, const char *m, const char *more = nullptr) {
  try { g_learn_err = m; if (more) { g_learn_err += ": "; g_learn_err += more; } } catch (...) { }   // (no memory for a message is no reason to throw through a C entry)
  return code;
}
extern "C" const char *agarcl_learn_error(void) { return g_learn_err.c_str(); }

// the calling thread's device for the length of a call
struct DeviceScope {
  int before = -1; hipError_t err;
  explicit DeviceScope(int dev) { err = hipGetDevice(&before); if (err == hipSuccess && before != dev) err = hipSetDevice(dev); else before = -1; }
  ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
};
#define ON_DEVICE(dev) DeviceScope scope_(dev); if (scope_.err != hipSuccess) return fail(AGARCL_E_HIP, "device", hipGetErrorString(scope_.err))
static int launched(const char *what) { const hipError_t e = hipGetLastError(); return e == hipSuccess ? AGARCL_OK : fail(AGARCL_E_HIP, what, hipGetErrorString(e)); }
#define BY_TYPE(dt, ...) do { switch (dt) { case AGARCL_F32: { using T = float; __VA_ARGS__; break; } case AGARCL_BF16: { using T = bf16_t; __VA_ARGS__; break; } default: { using T = f16_t; __VA_ARGS__; break; } } } while (0)
// (4 bytes of columns per thread; the columns of one thread are always one row's where the width is a multiple of their number; a single column cannot be two)
#define BY_VEC(...) do { constexpr int W = 4 / sizeof(T); if (k < W) { constexpr int V = 1, R = 1; __VA_ARGS__; } else if (a->width % W == 0) { constexpr int V = W, R = 1; __VA_ARGS__; } \
                         else { constexpr int V = W, R = W; __VA_ARGS__; } } while (0)
static bool type_ok(int32_t dt) { return dt == AGARCL_F32 || dt == AGARCL_BF16 || dt == AGARCL_F16; }
static const int64_t kMost = (int64_t)1 << 40;      // no dimension, stride or product of dimensions above this: 64-bit index arithmetic cannot overflow
static bool sizes_ok(int64_t a, int64_t b, int64_t c) {
  if (a < 0 || b < 0 || c < 0 || a > kMost || b > kMost || c > kMost) return false;
  if (a == 0) a = 1;      // (the product of the others counts all the same)
  if (b == 0) b = 1;
  if (c == 0) c = 1;
  return a <= kMost / b && a * b <= kMost / c;
}
static bool stride_ok(int64_t s, int64_t steps, int64_t least) { return steps <= 1 || (s >= least && s <= kMost && s <= (kMost << 10) / steps); }
static int64_t reach(std::initializer_list<int64_t> strides, int64_t bytes) { int64_t m = 0; for (int64_t s : strides) if (s > m) m = s; return m * bytes; }      // from a step to the next, at most
static unsigned blocks_for(int64_t threads) { const int64_t n = (threads + 255) / 256; return (unsigned)(n < 65536 ? n : 65536); }   // (the kernels go on in strides of the grid)

// ---- recurrence -----------------------------------------------------------------------------------------------------------------------------
extern "C" int64_t agarcl_recurrence_work(int64_t steps, int64_t rows, int64_t width) { return sizes_ok(steps, rows, width) ? scan_work(steps, rows * width) : -1; }

static int recurrence_check(const agarcl_recurrence_args *a) {
  if (!a) return fail(AGARCL_E_INVALID, "null argument");
  if (!type_ok(a->dtype)) return fail(AGARCL_E_INVALID, "dtype");
  if (!sizes_ok(a->steps, a->rows, a->width)) return fail(AGARCL_E_INVALID, "steps, rows, width");
  if (a->steps * a->rows * a->width == 0) return AGARCL_OK;
  if (!a->x || !a->gate) return fail(AGARCL_E_INVALID, "x, gate");
  const int64_t k = a->rows * a->width;
  if (!stride_ok(a->x_stride, a->steps, k) || !stride_ok(a->gate_stride, a->steps, k) || (a->reset && !stride_ok(a->reset_stride, a->steps, a->rows)))
    return fail(AGARCL_E_INVALID, "a stride is smaller than a step");
  if (agarcl_recurrence_work(a->steps, a->rows, a->width) > 0 && !a->work) return fail(AGARCL_E_INVALID, "work");
  return AGARCL_OK;
}

extern "C" int agarcl_recurrence(const agarcl_recurrence_args *a) {
  if (const int rc = recurrence_check(a)) return rc;
  const int64_t k = a->rows * a->width;
  if (k == 0) return AGARCL_OK;
  if (!a->last || (a->steps && !a->h)) return fail(AGARCL_E_INVALID, "h, last");
  ON_DEVICE(a->device);
  const hipStream_t st = (hipStream_t)a->stream;
  if (a->steps == 0) {      // (the state as it is)
    k_copy_state<<<dim3(blocks_for(k)), 256, 0, st>>>(a->state, a->last, k);
  } else if (a->steps == 1) {
    BY_TYPE(a->dtype, {
      if (a->width % 4 == 0) k_recurrence_step<T, 4><<<dim3(blocks_for(k / 4)), 256, 0, st>>>((const T *)a->x, (const T *)a->gate, a->state, a->reset, (T *)a->h, a->last, a->marks, k, a->width);
      else k_recurrence_step<T, 1><<<dim3(blocks_for(k)), 256, 0, st>>>((const T *)a->x, (const T *)a->gate, a->state, a->reset, (T *)a->h, a->last, a->marks, k, a->width);
    });
  } else BY_TYPE(a->dtype, {
    BY_VEC({
      using Op = RecurrenceOp<T, V, R>;
      Op op;
      op.x = {(uintptr_t)a->x, a->x_stride}; op.gate = {(uintptr_t)a->gate, a->gate_stride}; op.resets.reset = {(uintptr_t)a->reset, a->reset_stride};
      op.resets.width = a->width; op.h = {(uintptr_t)a->h, k}; op.marks = {(uintptr_t)a->marks, k}; 
      scan_launch<Op, V>(op, scan_shape(a->steps, k, V, reach({a->x_stride, a->gate_stride, a->reset ? a->reset_stride : 0, k}, sizeof(T))), a->state, a->last, a->work, st);
    });
  });
  return launched("recurrence");
}

extern "C" int agarcl_recurrence_grad(const agarcl_recurrence_args *a) {
  if (const int rc = recurrence_check(a)) return rc;
  const int64_t k = a->rows * a->width;
  if (k == 0) return AGARCL_OK;
  if (!a->dstate || (a->steps && (!a->dx || !a->dgate || !a->marks))) return fail(AGARCL_E_INVALID, "marks, dx, dgate, dstate");
  if (a->steps && a->dh && !stride_ok(a->dh_stride, a->steps, k)) return fail(AGARCL_E_INVALID, "a stride is smaller than a step");
  ON_DEVICE(a->device);
  const hipStream_t st = (hipStream_t)a->stream;
  if (a->steps == 0) {
    k_copy_state<<<dim3(blocks_for(k)), 256, 0, st>>>(a->dlast, a->dstate, k);
  } else BY_TYPE(a->dtype, {
    BY_VEC({
      using Op = RecurrenceGradOp<T, V, R>;
      Op op;
      op.x = {(uintptr_t)a->x, a->x_stride}; op.gate = {(uintptr_t)a->gate, a->gate_stride}; op.dh = {(uintptr_t)a->dh, a->dh_stride};
      op.resets.reset = {(uintptr_t)a->reset, a->reset_stride}; op.resets.width = a->width; op.marks = {(uintptr_t)a->marks, k}; op.dx = {(uintptr_t)a->dx, k};
      op.dgate = {(uintptr_t)a->dgate, k}; 
      scan_launch<Op, V>(op, scan_shape(a->steps, k, V, reach({a->x_stride, a->gate_stride, a->dh ? a->dh_stride : 0, a->reset ? a->reset_stride : 0, k}, sizeof(T))), a->dlast, a->dstate, a->work, st);
    });
  });
  return launched("recurrence gradient");
}

// ---- advantages -----------------------------------------------------------------------------------------------------------------------------
extern "C" int64_t agarcl_advantages_work(int64_t steps, int64_t rows) { return sizes_ok(steps, rows, 1) ? scan_work(steps, rows) : -1; }

extern "C" int agarcl_advantages(const agarcl_advantages_args *a) {
  if (!a) return fail(AGARCL_E_INVALID, "null argument");
  if (!type_ok(a->dtype)) return fail(AGARCL_E_INVALID, "dtype");
  if (!sizes_ok(a->steps, a->rows, 1)) return fail(AGARCL_E_INVALID, "steps, rows");
  if (!(a->gamma >= 0.f && a->gamma <= 1.f && a->lambda >= 0.f && a->lambda <= 1.f)) return fail(AGARCL_E_INVALID, "gamma and lambda must be in [0, 1]");
  if (a->steps * a->rows == 0) return AGARCL_OK;
  if (!a->reward || !a->value || !a->next_value || !a->terminated || !a->advantage || !a->returns) return fail(AGARCL_E_INVALID, "null pointer");
  if (a->final_value && !a->truncated) return fail(AGARCL_E_INVALID, "final_value without truncated");
  if (!stride_ok(a->reward_stride, a->steps, a->rows) || !stride_ok(a->value_stride, a->steps, a->rows) || !stride_ok(a->terminated_stride, a->steps, a->rows) ||
      (a->truncated && !stride_ok(a->truncated_stride, a->steps, a->rows)) || (a->final_value && !stride_ok(a->final_stride, a->steps, a->rows)))
    return fail(AGARCL_E_INVALID, "a stride is smaller than a step");
  if (agarcl_advantages_work(a->steps, a->rows) > 0 && !a->work) return fail(AGARCL_E_INVALID, "work");
  ON_DEVICE(a->device);
  const hipStream_t st = (hipStream_t)a->stream;
  BY_TYPE(a->dtype, {
    AdvantageOp<T, 1> op;
    op.reward = {(uintptr_t)a->reward, a->reward_stride}; op.value = {(uintptr_t)a->value, a->value_stride}; op.final_value = {(uintptr_t)a->final_value, a->final_stride};
    op.next_value = {(uintptr_t)a->next_value, 0}; op.terminated = {(uintptr_t)a->terminated, a->terminated_stride};
    op.truncated = {(uintptr_t)a->truncated, a->truncated_stride};
    op.gamma = a->gamma; op.gl = a->gamma * a->lambda; op.advantage = {(uintptr_t)a->advantage, a->rows}; op.returns = {(uintptr_t)a->returns, a->rows}; op.steps = a->steps;
    scan_launch<AdvantageOp<T, 1>, 1>(op, scan_shape(a->steps, a->rows, 1, reach({a->reward_stride, a->value_stride, a->terminated_stride, a->truncated ? a->truncated_stride : 0, a->final_value ? a->final_stride : 0, a->rows}, 4)), nullptr, nullptr, a->work, st);
  });
  return launched("advantages");
}

// ---- policy ---------------------------------------------------------------------------------------------------------------------------------
static int policy_check(int64_t rows, int64_t kinds, int32_t dtype, const void *logits, int64_t logits_stride, const uint8_t *allowed, int64_t allowed_stride) {
  if (!type_ok(dtype)) return fail(AGARCL_E_INVALID, "dtype");
  if (kinds < 1 || kinds > INT32_MAX) return fail(AGARCL_E_INVALID, "kinds must be in [1, 2^31)");
  if (!sizes_ok(rows, kinds, 1)) return fail(AGARCL_E_INVALID, "rows");
  if (rows == 0) return AGARCL_OK;
  if (!logits) return fail(AGARCL_E_INVALID, "logits");
  if (!stride_ok(logits_stride, rows, kinds) || (allowed && !stride_ok(allowed_stride, rows, kinds))) return fail(AGARCL_E_INVALID, "a stride is smaller than a row");
  return AGARCL_OK;
}

extern "C" int agarcl_sample_actions(const agarcl_sample_args *a) {
  if (!a) return fail(AGARCL_E_INVALID, "null argument");
  if (const int rc = policy_check(a->rows, a->kinds, a->dtype, a->logits, a->logits_stride, a->allowed, a->allowed_stride)) return rc;
  if (a->rows == 0) return AGARCL_OK;
  if (!a->kind || !a->log_prob) return fail(AGARCL_E_INVALID, "kind, log_prob");
  if (a->gumbel && !stride_ok(a->gumbel_stride, a->rows, a->kinds)) return fail(AGARCL_E_INVALID, "a stride is smaller than a row");
  if (a->mean ? (!a->log_std || !a->raw || !a->move) : (a->log_std || a->normal)) return fail(AGARCL_E_INVALID, "mean, log_std, raw, move belong together");
  ON_DEVICE(a->device);
  BY_TYPE(a->dtype, sample_launch<T>(*a, (hipStream_t)a->stream));
  return launched("sample_actions");
}

extern "C" int64_t agarcl_policy_loss_work(void) { return kLossWork; }

extern "C" int agarcl_policy_loss(const agarcl_policy_loss_args *a) {
  if (!a) return fail(AGARCL_E_INVALID, "null argument");
  if (const int rc = policy_check(a->rows, a->kinds, a->dtype, a->logits, a->logits_stride, a->allowed, a->allowed_stride)) return rc;
  if (!(a->clip_low >= 0.f && a->clip_high >= 0.f) || !isfinite(a->kl_coef) || !isfinite(a->entropy_coef)) return fail(AGARCL_E_INVALID, "clip_low, clip_high >= 0 and finite coefficients");
  const bool row_grads = a->dlogits || a->dmean || (a->dlog_std && a->log_std_per_row);
  const bool sum_first = row_grads && a->weight && a->mean_over_weight && !a->weight_sum;
  if (a->want_stats && (!a->loss || !a->stats || !a->work)) return fail(AGARCL_E_INVALID, "loss, stats, work");
  if (sum_first && !a->work) return fail(AGARCL_E_INVALID, "work");
  if (a->rows && (!a->kind || !a->old_log_prob || !a->advantage)) return fail(AGARCL_E_INVALID, "kind, old_log_prob, advantage");
  if (a->rows && (a->mean ? (!a->log_std || !a->move) : (a->log_std || a->move || a->dmean || a->dlog_std))) return fail(AGARCL_E_INVALID, "mean, log_std, move belong together");
  if (!a->want_stats && a->dlog_std && !a->log_std_per_row && !a->dlog_std_one) return fail(AGARCL_E_INVALID, "dlog_std_one");
  if (a->skip_if_one && !a->upstream) return fail(AGARCL_E_INVALID, "skip_if_one without upstream");
  ON_DEVICE(a->device);
  const hipStream_t st = (hipStream_t)a->stream;
  if (sum_first && a->rows) {
    k_weight_sum<<<dim3(kWeightBlocks), 256, 0, st>>>(a->weight, a->rows, a->work + 8 * kLossBlocks);
    if (const int rc = launched("policy loss: weights")) return rc;
  }
  unsigned grid = 0;
  if (a->rows || (!a->want_stats && a->dlog_std)) {      // (of no rows at all the gradient of a shared log_std is still to be written)
    BY_TYPE(a->dtype, grid = loss_launch<T>(*a, st));
    if (const int rc = launched("policy loss")) return rc;
  }
  if (a->want_stats) {
    k_loss_stats<<<dim3(1), 512, 0, st>>>(*a, (int)grid);
    if (const int rc = launched("policy loss: sums")) return rc;
  }
  return AGARCL_OK;
}
