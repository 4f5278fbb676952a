"""What a learner runs around `AgarioVectorEnv.step`, as HIP kernels on the tensors it already holds (include/agarcl_learn.h): nothing here copies to
the host or waits for the GPU, so all of it can be captured into a graph.

    memory  = torch.zeros(N, C, device=venv.device)
    ended   = None
    for t in range(T):                                                       # acting, under torch.no_grad()
        x, gate         = encoder(obs)                                       # [N, C] each, f32 / bf16 / f16
        h, memory       = learn.recurrence_step(x, gate, memory, ended)      # arenas are seen in part: the policy remembers
        logits, mean, v = heads(h)                                           # [N, 3], [N, 2], [N]
        actions         = learn.sample_actions(logits, mean, log_std, gumbel=gumbel[t], normal=normal[t])
        obs, reward, terminated, truncated, info = venv.step(actions)        # (move, kind, ...): what step() takes
        ended           = info["ended"].clone()                              # an ended arena restarts with an empty memory

    advantage, returns = learn.advantages(rewards, values, last_value, terminateds, truncateds)      # [T, N], the buffers of the loop above
    h, _ = learn.gated_recurrence(x, gate, memory_at_start, reset)           # [T, N, C]; reset[t] = ended of step t - 1
    loss = learn.policy_loss(logits, kinds, log_probs, advantage, mean, log_std, raws).loss           # + the value loss, then backward()

Conventions of every function: tensors live on one GPU; a rollout's first axis is time, then the arenas (and agents: venv's info["ended"] is per arena, so for
[N, agents] the resets are info["ended"][:, None].expand(N, agents)); `x`, `gate`, `logits`, `mean`,
`value` are float32, bfloat16 or float16, everything that counts, sums or carries a state is float32; flags are bool or uint8.  A wrong argument raises
ValueError, a failing call AgarclError.  Kernels run on the current stream of the tensors' device, also when that is not the current device.
Tensors of other strides than a kernel reads are copied first (a step's slice, a row, has to be contiguous; steps and rows may lie apart).  There are no
gradients of gradients: a backward pass with create_graph raises RuntimeError, a forward-mode gradient ValueError.  Forward and backward pass are captured
together, with no eager graph of the same leaves alive: autograd would tie its stream to the capture (such a call raises ValueError; a kept loss of a warm-up is
such a graph, and torch.cuda.make_graphed_callables keeps one).  An eager backward
pass is handed to a thread of autograd's and back, which takes longer than the kernels here: torch.autograd.set_multithreading_enabled(False) around it keeps
it in the calling thread (the loss of 32768 rows with its gradients 37 us instead of 64)."""
import collections

import torch  # noqa: F401   (its HIP runtime has to be the one that is loaded first)

from . import _capi

_capi.hip_lib()
try:
    from . import _learn
except ImportError as e:
    raise _capi.AgarclError(-4, "the module agarcl_amd._learn is missing or does not load (%s) -- build it with agarcl_amd/build.py (there is no other path)" % e)

Advantages = collections.namedtuple("Advantages", "advantage returns")
Actions = collections.namedtuple("Actions", "move kind log_prob raw")
PolicyLoss = collections.namedtuple("PolicyLoss", "loss surrogate kl entropy clipped")


def gated_recurrence(x, gate, state=None, reset=None):
    """The memory over a whole rollout: with f = sigmoid(gate[t]),

        h[t] = f * (0 if reset[t] else h[t-1]) + (1 - f) * x[t],      h[-1] = state

    x, gate [T, *rows, C] of one type; state float32 [*rows, C] or None (zeros); reset bool [T, *rows] or None: reset[t] says that the arena's episode
    began with step t (venv's info["ended"] of the step before).  Returns (h [T, *rows, C] of x's type, the state after the last step, float32 [*rows, C]).
    Differentiable in x, gate and state.  The state is carried in float32 through all steps; only h is rounded to x's type.  A reset drops whatever the
    state holds, infinities and NaN included."""
    return _learn.gated_recurrence(x, gate, state, reset)


def recurrence_step(x, gate, state, reset=None):
    """One acting step of gated_recurrence: x, gate [*rows, C], state float32 [*rows, C], reset bool [*rows] or None.  Returns (h of x's type, the new
    state, float32).  No gradients: train with gated_recurrence over the rollout."""
    return _learn.recurrence_step(x, gate, state, reset)


def advantages(reward, value, next_value, terminated, truncated=None, final_value=None, gamma=0.99, lam=0.95):
    """Advantages and returns of a rollout as AgarioVectorEnv writes it: reward float32 [T, *rows], value [T, *rows] (of the observation each step was
    taken in), next_value [*rows] (of the observation behind the last step), terminated / truncated bool [T, *rows].

        next      = 0 where terminated, final_value where truncated, else value[t+1]
        delta     = reward + gamma * next - value
        advantage = delta + gamma * lam * advantage[t+1]      (the last term only inside an episode);      returns = advantage + value

    The env resets an ended arena in the same step, so value[t+1] belongs to the next episode there.  final_value [T, *rows]: the value of the
    observation an episode was truncated in, for those who have one; without it a truncated step is left out (delta = 0), and the steps before
    it end in its own value.  Returns (advantage, returns), float32 [T, *rows], without gradients."""
    return Advantages._make(_learn.advantages(reward, value, next_value, terminated, truncated, final_value, gamma, lam))


def sample_actions(logits, mean=None, log_std=None, gumbel=None, normal=None, allowed=None):
    """The next actions from a policy's outputs: logits [*rows, kinds] and, for the env's move, mean [*rows, 2] with log_std float32 [2] (or per row, of
    mean's type).  The noise is the caller's, so that a seed repeats a rollout and one launch can make it for many steps: gumbel float32 [*rows, kinds]
    (-log(-log(u))), normal float32 [*rows, 2]; without them the likeliest kind and the mean.  allowed bool [*rows, kinds]: the kinds to choose among.

    Returns Actions(move, kind, log_prob, raw): `venv.step(actions)` takes it as it is.  kind int32 = the lowest index of the largest logits + gumbel
    among the allowed (0, "none", where nothing is allowed); raw = mean + exp(log_std) * normal; move = raw limited to [-1, 1]; log_prob of (kind, raw):
    what policy_loss divides by.  A NaN stays one in raw, move and log_prob (an arena that is stepped with it holds it until its next reset).  A logit of
    -inf is not allowed.  Without gradients.  log_prob, raw and move lie in one allocation (clone() what is to be kept alone)."""
    return Actions._make(_learn.sample_actions(logits, mean, log_std, gumbel, normal, allowed))


def policy_loss(logits, kind, old_log_prob, advantage, mean=None, log_std=None, move=None, ref_log_prob=None, allowed=None, weight=None, clip=0.2, kl_coef=0.0,
                entropy_coef=0.0, reduction="mean"):
    """The clipped policy loss on the env's action, with a KL term and an entropy bonus.  logits [*rows, kinds], mean [*rows, 2], log_std float32 [2] (or
    per row, of mean's type); kind int32 (or int64) [*rows] and move float32 [*rows, 2] = `kind` and `raw` of sample_actions, old_log_prob its `log_prob`;
    advantage, ref_log_prob, weight float32 [*rows] (weight also bool); allowed bool [*rows, kinds].  With r = exp(lp - old_log_prob):

        row loss = - min(r A, clamp(r, 1 - clip, 1 + clip) A) + kl_coef (exp(ref - lp) - (ref - lp) - 1) - entropy_coef H

    clip: a number, or (below, above).  ref_log_prob: the log-probability under a reference policy; old_log_prob without one.  reduction: "mean" (weighted;
    0 where the weights sum to 0) or "sum".  Returns PolicyLoss(loss, surrogate, kl, entropy, clipped): loss is differentiable in logits, mean and
    log_std; the others are weighted means of min(..), of the KL term, of H and of "the clip took the gradient"
    (r > 1 + above where A >= 0, r < 1 - below elsewhere), without gradients.

    A row is left out -- it adds nothing and its gradients are 0 -- where its weight is 0, its kind is outside 0 .. kinds - 1 (padding), or its kind is not
    allowed (a logit of -inf is not); except by its weight it still counts in the mean.  What stands in such rows and places is never used.
    Gradients in float16: scale the loss (the upstream gradient is applied in float32, before the one rounding).

    In float32 and bfloat16 the forward pass writes the gradients for an upstream gradient of 1 as well, and they are kept until the backward pass (the size of the
    logits).  Where the upstream gradient is another -- a loss that is divided or scaled after this call -- the backward pass works them out once more, twice the
    memory traffic in all: for many kinds let reduction="sum" and the weights hold the factor."""
    if reduction not in ("mean", "sum"):
        raise ValueError("reduction must be 'mean' or 'sum'")
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    return PolicyLoss._make(_learn.policy_loss(logits, kind, old_log_prob, advantage, mean, log_std, move, ref_log_prob, allowed, weight, low, high, kl_coef, entropy_coef,
                                               reduction == "mean"))
