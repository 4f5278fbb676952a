/* agarcl_learn.h -- what a learner runs around agarcl_vec_step, on device tensors it already holds (libagarcl_hip.so; Python side:
 * agarcl_amd/learn.py).  The reference stops at the observation and the reward (/root/reference/gym_agario/AgarioEnv.py:85-132); these entry points
 * take up the buffers agarcl_vec_step writes (reward, done, truncated, ended) and produce the actions it reads (dxdy, act):
 *   agarcl_sample_actions   the next actions and their log-probability from a policy's outputs
 *   agarcl_advantages       advantages and returns of a rollout, over its reward / terminated / truncated
 *   agarcl_recurrence*      the memory of a policy over partially observed arenas, cleared where an episode ended
 *   agarcl_policy_loss      the clipped policy loss with its KL and entropy terms, and its gradients
 *
 * Conventions: rollouts are time major; "rows" is the number of arenas (x agents).  All pointers are device pointers of `device`; every call only
 * enqueues kernels on `stream` (a hipStream_t) -- no allocation, no synchronisation, no memset -- so it may be captured into a graph.  Scratch memory is the
 * caller's: two calls that may run at the same time need two.  Returns AGARCL_OK or AGARCL_E_*, never throws; agarcl_learn_error() is this thread's
 * message.  Each call leaves the calling thread's current device as it was.  Pointers need the alignment of their element type, no more.  States,
 * sums and statistics are held in f32 or f64 whatever the tensors' type; results are rounded once, to nearest even. */
#ifndef AGARCL_LEARN_H
#define AGARCL_LEARN_H
#include <stdint.h>
#include "agarcl_batch.h"
#ifdef __cplusplus
extern "C" {
#endif

#define AGARCL_F32 0
#define AGARCL_BF16 1
#define AGARCL_F16 2
#define AGARCL_MARK_STEPS 8    /* agarcl_recurrence keeps the state in front of every 8th step for its gradient */

const char *agarcl_learn_error(void);

/* f = sigmoid(gate[t]),  p = reset[t] ? 0 : h[t-1],  h[t] = f p + (1 - f) x[t],  h[-1] = state.
 * The gate comes before its sigmoid: a bf16 number near 1 could not say how long a memory lasts.  A reset drops whatever the state
 * holds, infinities and NaN included. */
typedef struct agarcl_recurrence_args {
  int64_t steps, rows, width;            /* T, B, C; any of them may be 0 */
  int32_t dtype, device;                 /* AGARCL_F32 / BF16 / F16 of x, gate, h, dh, dx, dgate */
  const void *x, *gate;                  /* [T] x [B][C]; a step's [B][C] is contiguous, steps are *_stride elements apart */
  int64_t x_stride, gate_stride;
  const float *state;                    /* [B][C] or NULL: zeros */
  const uint8_t *reset;                  /* [T][B] 0 / 1 or NULL: never; steps are reset_stride apart */
  int64_t reset_stride;
  void *h;                               /* out [T][B][C] (agarcl_recurrence) */
  float *last;                           /* out [B][C]: the state after the last step (agarcl_recurrence) */
  float *marks;                          /* [ceil(T / 8)][B][C]: written by agarcl_recurrence unless NULL, read by agarcl_recurrence_grad */
  const void *dh;                        /* [T] x [B][C] or NULL: zeros (agarcl_recurrence_grad), steps dh_stride apart */
  int64_t dh_stride;
  const float *dlast;                    /* [B][C] or NULL: zeros (agarcl_recurrence_grad) */
  void *dx, *dgate;                      /* out [T][B][C] (agarcl_recurrence_grad) */
  float *dstate;                         /* out [B][C] (agarcl_recurrence_grad) */
  float *work;                           /* agarcl_recurrence_work(steps, rows, width) floats, or NULL where that is 0 */
  void *stream;
} agarcl_recurrence_args;
int64_t agarcl_recurrence_work(int64_t steps, int64_t rows, int64_t width);
int agarcl_recurrence(const agarcl_recurrence_args *a);
int agarcl_recurrence_grad(const agarcl_recurrence_args *a);

/* next = terminated[t] ? 0 : truncated[t] ? final_value[t] : value[t+1]   (next_value behind the last step)
 * delta = reward[t] + gamma next - value[t];  a step that was truncated and has no final_value is left out: delta = 0
 * advantage[t] = delta + (terminated[t] || truncated[t] ? 0 : gamma lambda advantage[t+1]);  returns[t] = advantage[t] + value[t].
 * What stands behind the end of an episode is never looked at through it (NaN included). */
typedef struct agarcl_advantages_args {
  int64_t steps, rows;                   /* T, B; either may be 0 */
  int32_t dtype, device;                 /* of value, next_value, final_value */
  const float *reward;                   /* [T] x [B], steps reward_stride apart; likewise below */
  const void *value;
  const void *next_value;                /* [B] */
  const uint8_t *terminated;
  const uint8_t *truncated;              /* or NULL: never */
  const void *final_value;               /* or NULL: unknown */
  int64_t reward_stride, value_stride, terminated_stride, truncated_stride, final_stride;
  float gamma, lambda;
  float *advantage, *returns;            /* out [T][B] */
  float *work;                           /* agarcl_advantages_work(steps, rows) floats, or NULL where that is 0 */
  void *stream;
} agarcl_advantages_args;
int64_t agarcl_advantages_work(int64_t steps, int64_t rows);
int agarcl_advantages(const agarcl_advantages_args *a);

/* The env's action: a kind out of `kinds` (agarcl_vec_step's act has 3) by logits, and -- where mean is given -- a move by two independent normal
 * distributions.  A kind is allowed unless allowed[row][kind] is 0 or its logit is -inf; what stands in a place that is not allowed is never used.
 *   kind = the lowest index of the largest logit + gumbel among the allowed (gumbel NULL: of the largest logit); 0 where nothing is allowed
 *   raw = mean + exp(log_std) normal (normal NULL: mean);  move = raw limited to [-1, 1], what the engine takes; a NaN stays one, in log_prob too
 *   log_prob = log softmax(logits over the allowed)[kind] (0 where nothing is allowed) + the normal log-density of raw */
typedef struct agarcl_sample_args {
  int64_t rows, kinds;
  int32_t dtype, device;                 /* of logits, mean, and of log_std where it has a row's stride */
  const void *logits; int64_t logits_stride;
  const uint8_t *allowed; int64_t allowed_stride;      /* [rows][kinds] or NULL */
  const float *gumbel; int64_t gumbel_stride;          /* [rows][kinds] or NULL */
  const void *mean;                      /* [rows][2] or NULL: no move */
  const void *log_std; int32_t log_std_per_row;        /* f32 [2], or [rows][2] of dtype */
  int32_t reserved;
  const float *normal;                   /* [rows][2] or NULL */
  int32_t *kind;                         /* out [rows] */
  float *log_prob;                       /* out [rows] */
  float *raw, *move;                     /* out [rows][2], with mean */
  void *stream;
} agarcl_sample_args;
int agarcl_sample_actions(const agarcl_sample_args *a);

/* With lp = the log-probability of (kind, move) as above, r = exp(lp - old_log_prob), A = advantage, ref = ref_log_prob (old_log_prob without one):
 *   row loss = - min(r A, min(max(r, 1 - clip_low), 1 + clip_high) A) + kl_coef (exp(ref - lp) - (ref - lp) - 1) - entropy_coef H
 *   loss = sum of weight x row loss, over the sum of the weights where mean_over_weight (0 where that is 0)
 * H = the entropy of the kinds plus the move's.  A row is left out -- it adds nothing, has zero gradients, and nothing of it is used -- where its weight
 * is 0, its kind is outside 0 .. kinds - 1, or its kind is not allowed; its weight still counts in the mean.
 * At r = 1 - clip_low and r = 1 + clip_high the gradient is that of r A. */
typedef struct agarcl_policy_loss_args {
  int64_t rows, kinds;
  int32_t dtype, device;                 /* of logits, mean, dlogits, dmean, and of log_std, dlog_std where they have a row's stride */
  const void *logits; int64_t logits_stride;
  const uint8_t *allowed; int64_t allowed_stride;      /* [rows][kinds] or NULL */
  const int32_t *kind;                   /* [rows] */
  const void *mean;                      /* [rows][2] or NULL: no move */
  const void *log_std; int32_t log_std_per_row;
  int32_t mean_over_weight;              /* 0: the sum */
  const float *move;                     /* [rows][2]: raw of agarcl_sample_actions */
  const float *old_log_prob, *advantage; /* [rows] */
  const float *ref_log_prob, *weight;    /* [rows] or NULL (weight: ones) */
  const float *weight_sum;               /* NULL, or one number: stats[4] of an earlier call with these weights, which are then not summed again */
  float clip_low, clip_high, kl_coef, entropy_coef;
  const float *upstream;                 /* NULL, or one number that the gradients are multiplied by (the gradient of the loss itself) */
  int32_t skip_if_one;                   /* with upstream: leave the gradients as they are if it is 1 (they hold the ones for 1 already) */
  int32_t want_stats;                    /* write loss and stats (and with them dlog_std where log_std has no row's stride) */
  float *loss;                           /* out [1] */
  float *stats;                          /* out [8]: weighted means of min(..), the KL term, H, and "clipped" (0 / 1); the sum of the weights; 0, 0, 0 */
  void *dlogits;                         /* out [rows][kinds] contiguous, or NULL: no gradients */
  void *dmean, *dlog_std;                /* out, with mean; NULL: not wanted.  dlog_std: f32 [2], or [rows][2] of dtype */
  const float *dlog_std_one;             /* without want_stats and with f32 [2] dlog_std: its value for upstream = 1 */
  double *work;                          /* agarcl_policy_loss_work() doubles */
  void *stream;
} agarcl_policy_loss_args;
int64_t agarcl_policy_loss_work(void);
int agarcl_policy_loss(const agarcl_policy_loss_args *a);
#ifdef __cplusplus
}
#endif
#endif /* AGARCL_LEARN_H */
