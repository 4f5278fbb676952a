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

Conventions of every function: tensors live on one GPU; a rollout's first axis is time, then the arenas (and agents); `x`, `gate`, `logits`, `mean`,
`value` are float32, bfloat16 or float16, everything that counts, sums or carries a state is float32; flags are bool or uint8.  A wrong argument raises
ValueError, a failing call AgarclError.  Kernels run on the current stream of the tensors' device, also when that is not the current device.
Tensors of other strides than a kernel reads are copied first (a step's slice, a row, has to be contiguous; steps and rows may lie apart)."""
import collections
import ctypes
import math

import torch

from . import _capi

_TYPES = {torch.float32: _capi.F32, torch.bfloat16: _capi.BF16, torch.float16: _capi.F16}
_FLAGS = (torch.bool, torch.uint8)

Advantages = collections.namedtuple("Advantages", "advantage returns")
Actions = collections.namedtuple("Actions", "move kind log_prob raw")
PolicyLoss = collections.namedtuple("PolicyLoss", "loss surrogate kl entropy clipped")


# ---- arguments ----------------------------------------------------------------------------------------------------------------------------

def _first(t, name):
    """the tensor that says type and device for the others"""
    if not isinstance(t, torch.Tensor) or t.dtype not in _TYPES:
        raise ValueError("%s must be a float32, bfloat16 or float16 tensor" % name)
    return t


def _on_gpu(t):
    """(the last of the checks)"""
    if not t.is_cuda:
        raise ValueError("tensors must live on a GPU (there is no CPU path)")


def _like(t, name, ref, dtype, shape):
    if not isinstance(t, torch.Tensor):
        raise ValueError("%s must be a tensor" % name)
    if t.device != ref.device:
        raise ValueError("%s must live on %s" % (name, ref.device))
    if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError("%s must be %s, got %s" % (name, " or ".join(map(str, dtype)) if isinstance(dtype, tuple) else dtype, t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    return t


def _constant(**tensors):
    """gradients do not flow through these: better said than lost"""
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise ValueError("%s is taken as a constant here: detach() it, or call under torch.no_grad()" % name)


def _steps(t):
    """(tensor, elements from one index of the first axis to the next) with every t[i] contiguous; a copy only where it has to be one"""
    if t is None:
        return None, 0
    n = t.shape[0]
    if t.is_contiguous():
        return t, t.numel() // n if n else 0
    if n and t[0].is_contiguous() and t.stride(0) >= t[0].numel():
        return t, t.stride(0)
    t = t.contiguous()
    return t, t.numel() // n if n else 0


def _rows(t, width):
    """the same for [*rows, width] seen as rows: one stride has to lead from each row to the next"""
    if t is None or t.is_contiguous():
        return t, width
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= width:
        return t, t.stride(0)
    return t.contiguous(), width


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _call(fn, args):
    rc = fn(ctypes.byref(args))
    if rc != 0:
        raise _capi.AgarclError(rc, (_capi.hip_lib().agarcl_learn_error() or b"").decode())


# ---- the memory -----------------------------------------------------------------------------------------------------------------------------

def _recurrence_args(x, gate, state, reset, x_stride, gate_stride, reset_stride):
    shape = x.shape
    width = shape[-1]
    rows = math.prod(shape[1:-1])
    return _capi.RecurrenceArgs(steps=shape[0], rows=rows, width=width, dtype=_TYPES[x.dtype], device=x.device.index, x=_ptr(x), gate=_ptr(gate), x_stride=x_stride,
                                gate_stride=gate_stride, state=_ptr(state), reset=_ptr(reset), reset_stride=reset_stride, stream=_stream(x.device))


def _work(floats, ref):
    if floats < 0:
        raise ValueError("sizes out of range")
    return torch.empty(floats, dtype=torch.float32, device=ref.device) if floats else None


def _recurrence_forward(x, gate, state, reset, marked):
    L = _capi.hip_lib()
    (x, xs), (gate, gs), (reset, rs) = _steps(x), _steps(gate), _steps(reset)
    state = state if state is None else state.contiguous()
    a = _recurrence_args(x, gate, state, reset, xs, gs, rs)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    last = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
    marks = torch.empty((-(-x.shape[0] // _capi.MARK_STEPS),) + tuple(x.shape[1:]), dtype=torch.float32, device=x.device) if marked else None
    work = _work(L.agarcl_recurrence_work(a.steps, a.rows, a.width), x)
    a.h, a.last, a.marks, a.work = _ptr(h), _ptr(last), _ptr(marks), _ptr(work)
    _call(L.agarcl_recurrence, a)
    return h, last, marks


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, reset):
        ctx.set_materialize_grads(False)
        h, last, marks = _recurrence_forward(x, gate, state, reset, True)
        ctx.save_for_backward(x, gate, reset, marks)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        if dh is None and dlast is None:
            return None, None, None, None
        L = _capi.hip_lib()
        x, gate, reset, marks = ctx.saved_tensors
        (x, xs), (gate, gs), (reset, rs), (dh, ds) = _steps(x), _steps(gate), _steps(reset), _steps(dh)
        dlast = None if dlast is None else dlast.contiguous()
        a = _recurrence_args(x, gate, None, reset, xs, gs, rs)
        dx, dgate = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dstate = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
        work = _work(L.agarcl_recurrence_work(a.steps, a.rows, a.width), x)
        a.marks, a.dh, a.dh_stride, a.dlast, a.dx, a.dgate, a.dstate, a.work = _ptr(marks), _ptr(dh), ds, _ptr(dlast), _ptr(dx), _ptr(dgate), _ptr(dstate), _ptr(work)
        _call(L.agarcl_recurrence_grad, a)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dgate if need[1] else None, dstate if need[2] else None, None


def gated_recurrence(x, gate, state=None, reset=None):
    """The memory over a whole rollout: with f = sigmoid(gate[t]),

        h[t] = f * (0 if reset[t] else h[t-1]) + (1 - f) * x[t],      h[-1] = state

    x, gate [T, *rows, C] of one type; state float32 [*rows, C] or None (zeros); reset bool [T, *rows] or None: reset[t] says that the arena's episode
    began with step t (venv's info["ended"] of the step before).  Returns (h [T, *rows, C] of x's type, the state after the last step, float32 [*rows, C]).
    Differentiable in x, gate and state.  The state is carried in float32 through all steps; only h is rounded to x's type.  A reset drops whatever the
    state holds, infinities and NaN included."""
    _first(x, "x")
    if x.dim() < 2:
        raise ValueError("x must have shape [T, *rows, C], got %s" % (tuple(x.shape),))
    _like(gate, "gate", x, x.dtype, x.shape)
    if state is not None:
        _like(state, "state", x, torch.float32, x.shape[1:])
    if reset is not None:
        _like(reset, "reset", x, _FLAGS, x.shape[:-1])
    _on_gpu(x)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (state is not None and state.requires_grad)):
        return _Recurrence.apply(x, gate, state, reset)
    return _recurrence_forward(x, gate, state, reset, False)[:2]


def recurrence_step(x, gate, state, reset=None):
    """One acting step of gated_recurrence: x, gate [*rows, C], state float32 [*rows, C], reset bool [*rows] or None.  Returns (h of x's type, the new
    state, float32).  No gradients: train with gated_recurrence over the rollout."""
    _constant(x=x, gate=gate, state=state)
    _first(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have shape [*rows, C]")
    _like(gate, "gate", x, x.dtype, x.shape)
    _like(state, "state", x, torch.float32, x.shape)
    if reset is not None:
        _like(reset, "reset", x, _FLAGS, x.shape[:-1])
        reset = reset[None]
    _on_gpu(x)
    h, state, _ = _recurrence_forward(x[None], gate[None], state, reset, False)
    return h[0], state


# ---- the rollout ----------------------------------------------------------------------------------------------------------------------------

def advantages(reward, value, next_value, terminated, truncated=None, final_value=None, gamma=0.99, lam=0.95):
    """Advantages and returns of a rollout as AgarioVectorEnv writes it: reward float32 [T, *rows], value [T, *rows] (of the observation each step was
    taken in), next_value [*rows] (of the observation behind the last step), terminated / truncated bool [T, *rows].

        next      = 0 where terminated, final_value where truncated, else value[t+1]
        delta     = reward + gamma * next - value
        advantage = delta + gamma * lam * advantage[t+1]      (the last term only inside an episode);      returns = advantage + value

    The env resets an ended arena in the same step, so value[t+1] belongs to the next episode there.  final_value [T, *rows]: the value of the
    observation an episode was truncated in, for those who have one; without it a truncated step is left out (delta = 0), and the steps before
    it end in its own value.  Returns (advantage, returns), float32 [T, *rows], without gradients."""
    _constant(reward=reward, value=value, next_value=next_value, final_value=final_value)
    _first(value, "value")
    if value.dim() < 1:
        raise ValueError("value must have shape [T, *rows]")
    _like(reward, "reward", value, torch.float32, value.shape)
    _like(next_value, "next_value", value, value.dtype, value.shape[1:])
    _like(terminated, "terminated", value, _FLAGS, value.shape)
    if truncated is not None:
        _like(truncated, "truncated", value, _FLAGS, value.shape)
    if final_value is not None:
        if truncated is None:
            raise ValueError("final_value without truncated")
        _like(final_value, "final_value", value, value.dtype, value.shape)
    if not (0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0):
        raise ValueError("gamma and lam must be in [0, 1]")
    _on_gpu(value)
    L = _capi.hip_lib()
    (reward, r), (value, v), (terminated, e), (truncated, u), (final_value, f) = _steps(reward), _steps(value), _steps(terminated), _steps(truncated), _steps(final_value)
    next_value = next_value.contiguous()
    steps, rows = value.shape[0], math.prod(value.shape[1:])
    advantage, returns = torch.empty(value.shape, dtype=torch.float32, device=value.device), torch.empty(value.shape, dtype=torch.float32, device=value.device)
    work = _work(L.agarcl_advantages_work(steps, rows), value)
    a = _capi.AdvantagesArgs(steps, rows, _TYPES[value.dtype], value.device.index, _ptr(reward), _ptr(value), _ptr(next_value), _ptr(terminated), _ptr(truncated),
                             _ptr(final_value), r, v, e, u, f, gamma, lam, _ptr(advantage), _ptr(returns), _ptr(work), _stream(value.device))
    _call(L.agarcl_advantages, a)
    return Advantages(advantage, returns)


# ---- the policy -----------------------------------------------------------------------------------------------------------------------------

def _policy(logits, mean, log_std, allowed):
    """the checks that acting and training share; log_std's row stride (0 or 1)"""
    _first(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have shape [*rows, kinds] with at least one kind, got %s" % (tuple(logits.shape),))
    if allowed is not None:
        _like(allowed, "allowed", logits, _FLAGS, logits.shape)
    if (mean is None) != (log_std is None):
        raise ValueError("mean and log_std belong together")
    if mean is None:
        return 0
    _like(mean, "mean", logits, logits.dtype, logits.shape[:-1] + (2,))
    if isinstance(log_std, torch.Tensor) and log_std.shape == (2,) and log_std.dtype == torch.float32:
        _like(log_std, "log_std", logits, torch.float32, (2,))
        return 0
    _like(log_std, "log_std (float32 [2], or per row)", logits, logits.dtype, mean.shape)
    return 1


def sample_actions(logits, mean=None, log_std=None, gumbel=None, normal=None, allowed=None):
    """The next actions from a policy's outputs: logits [*rows, kinds] and, for the env's move, mean [*rows, 2] with log_std float32 [2] (or per row, of
    mean's type).  The noise is the caller's, so that a seed repeats a rollout and one launch can make it for many steps: gumbel float32 [*rows, kinds]
    (-log(-log(u))), normal float32 [*rows, 2]; without them the likeliest kind and the mean.  allowed bool [*rows, kinds]: the kinds to choose among.

    Returns Actions(move, kind, log_prob, raw): `venv.step(actions)` takes it as it is.  kind int32 = the lowest index of the largest logits + gumbel
    among the allowed (0, "none", where nothing is allowed); raw = mean + exp(log_std) * normal; move = raw limited to [-1, 1]; log_prob of (kind, raw):
    what policy_loss divides by.  A logit of -inf is not allowed.  Without gradients."""
    _constant(logits=logits, mean=mean, log_std=log_std, gumbel=gumbel, normal=normal)
    per_row = _policy(logits, mean, log_std, allowed)
    if gumbel is not None:
        _like(gumbel, "gumbel", logits, torch.float32, logits.shape)
    if normal is not None:
        if mean is None:
            raise ValueError("normal without mean")
        _like(normal, "normal", logits, torch.float32, mean.shape)
    _on_gpu(logits)
    kinds, lead, dev = logits.shape[-1], logits.shape[:-1], logits.device
    rows = math.prod(lead)
    (logits, zs), (allowed, ks), (gumbel, gs) = _rows(logits, kinds), _rows(allowed, kinds), _rows(gumbel, kinds)
    kind, log_prob = torch.empty(lead, dtype=torch.int32, device=dev), torch.empty(lead, dtype=torch.float32, device=dev)
    raw = move = None
    if mean is not None:
        mean, log_std, normal = mean.contiguous(), log_std.contiguous(), normal if normal is None else normal.contiguous()
        raw, move = torch.empty(mean.shape, dtype=torch.float32, device=dev), torch.empty(mean.shape, dtype=torch.float32, device=dev)
    a = _capi.SampleArgs(rows, kinds, _TYPES[logits.dtype], dev.index, _ptr(logits), zs, _ptr(allowed), ks, _ptr(gumbel), gs, _ptr(mean), _ptr(log_std), per_row, 0, _ptr(normal),
                         _ptr(kind), _ptr(log_prob), _ptr(raw), _ptr(move), _stream(dev))
    _call(_capi.hip_lib().agarcl_sample_actions, a)
    return Actions(move, kind, log_prob, raw)


def _loss_args(logits, mean, log_std, per_row, fixed, kept):
    """the arguments that both directions share; `kept` holds the tensors of other strides that were copied"""
    kind, old, adv, move, ref, allowed, weight, clip_low, clip_high, kl, ent, over = fixed
    (logits, zs), (allowed, ks) = _rows(logits, logits.shape[-1]), _rows(allowed, logits.shape[-1])
    kind, old, adv, move, ref, weight, mean, log_std = (t if t is None else t.contiguous() for t in (kind, old, adv, move, ref, weight, mean, log_std))
    kept.extend((logits, allowed, kind, old, adv, move, ref, weight, mean, log_std))
    return _capi.PolicyLossArgs(rows=math.prod(logits.shape[:-1]), kinds=logits.shape[-1], dtype=_TYPES[logits.dtype], device=logits.device.index, logits=_ptr(logits),
                                logits_stride=zs, allowed=_ptr(allowed), allowed_stride=ks, kind=_ptr(kind), mean=_ptr(mean), log_std=_ptr(log_std), log_std_per_row=per_row,
                                mean_over_weight=over, move=_ptr(move), old_log_prob=_ptr(old), advantage=_ptr(adv), ref_log_prob=_ptr(ref), weight=_ptr(weight),
                                clip_low=clip_low, clip_high=clip_high, kl_coef=kl, entropy_coef=ent, stream=_stream(logits.device))


def _loss_forward(logits, mean, log_std, per_row, fixed, std_grad, grads):
    """(loss, stats, the shared log_std's gradient); grads: the tensors (or None) that take the gradients of logits, mean and a log_std per row in the same pass"""
    L, dev, kept = _capi.hip_lib(), logits.device, []
    a = _loss_args(logits, mean, log_std, per_row, fixed, kept)
    loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(8, dtype=torch.float32, device=dev)
    work = torch.empty(L.agarcl_policy_loss_work(), dtype=torch.float64, device=dev)
    dstd = torch.empty(2, dtype=torch.float32, device=dev) if std_grad else None
    a.want_stats, a.loss, a.stats, a.work = 1, _ptr(loss), _ptr(stats), _ptr(work)
    a.dlogits, a.dmean, a.dlog_std = _ptr(grads[0]), _ptr(grads[1]), _ptr(dstd) if std_grad else _ptr(grads[2])
    _call(L.agarcl_policy_loss, a)
    return loss, stats, dstd


def _loss_grads(need, logits, mean, log_std, per_row):
    like = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)   # noqa: E731
    return [like(logits) if need[0] else None, like(mean) if need[1] else None, like(log_std) if need[2] and per_row else None]


class _PolicyLoss(torch.autograd.Function):
    """The gradients for an upstream gradient of 1 -- what loss.backward() brings -- are written by the forward pass, from the registers that hold the
    logits for the loss.  The first backward pass hands them out after its kernel has looked at the upstream gradient: it does nothing where that is
    1 and works the gradients out from the logits otherwise.  Every other backward pass (a second one through a kept graph, one that is captured: its replays
    may bring other upstream gradients) works them out, into tensors of its own.  In float16 a loss is scaled as a rule, so there the forward pass leaves them."""

    @staticmethod
    def forward(ctx, logits, mean, log_std, per_row, fixed):
        need = ctx.needs_input_grad
        ahead = logits.dtype != torch.float16 and not torch.cuda.is_current_stream_capturing()
        ctx.ahead = _loss_grads(need, logits, mean, log_std, per_row) if ahead else None
        loss, stats, dstd = _loss_forward(logits, mean, log_std, per_row, fixed, mean is not None and not per_row, ctx.ahead or (None, None, None))
        ctx.per_row, ctx.numbers = per_row, fixed[7:]
        ctx.save_for_backward(logits, mean, log_std, stats, dstd, *fixed[:7])
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream, _):
        L, kept = _capi.hip_lib(), []
        logits, mean, log_std, stats, dstd, *tensors = ctx.saved_tensors
        a = _loss_args(logits, mean, log_std, ctx.per_row, tuple(tensors) + ctx.numbers, kept)
        need = ctx.needs_input_grad
        upstream = upstream.to(torch.float32).contiguous()
        grads, ctx.ahead = (None if torch.cuda.is_current_stream_capturing() else ctx.ahead), None
        a.skip_if_one = int(grads is not None)
        grads = grads or _loss_grads(need, logits, mean, log_std, ctx.per_row)
        if need[2] and not ctx.per_row:
            grads[2] = torch.empty(2, dtype=torch.float32, device=logits.device)
        a.upstream, a.weight_sum, a.dlogits, a.dmean, a.dlog_std, a.dlog_std_one = _ptr(upstream), _ptr(stats) + 16, _ptr(grads[0]), _ptr(grads[1]), _ptr(grads[2]), _ptr(dstd)
        _call(L.agarcl_policy_loss, a)
        return grads[0], grads[1], grads[2], None, None


def policy_loss(logits, kind, old_log_prob, advantage, mean=None, log_std=None, move=None, ref_log_prob=None, allowed=None, weight=None, clip=0.2, kl_coef=0.0,
                entropy_coef=0.0, reduction="mean"):
    """The clipped policy loss on the env's action, with a KL term and an entropy bonus.  logits [*rows, kinds], mean [*rows, 2], log_std float32 [2] (or
    per row, of mean's type); kind int32 (or int64) [*rows] and move float32 [*rows, 2] = `kind` and `raw` of sample_actions, old_log_prob its `log_prob`;
    advantage, ref_log_prob, weight float32 [*rows] (weight also bool); allowed bool [*rows, kinds].  With r = exp(lp - old_log_prob):

        row loss = - min(r A, clamp(r, 1 - clip, 1 + clip) A) + kl_coef (exp(ref - lp) - (ref - lp) - 1) - entropy_coef H

    clip: a number, or (below, above).  ref_log_prob: the log-probability under a reference policy; old_log_prob without one.  reduction: "mean" (weighted;
    0 where the weights sum to 0) or "sum".  Returns PolicyLoss(loss, surrogate, kl, entropy, clipped): loss is differentiable in logits, mean and
    log_std; the others are weighted means of min(..), of the KL term, of H and of "the clip took the gradient", without gradients.

    A row is left out -- it adds nothing and its gradients are 0 -- where its weight is 0, its kind is outside 0 .. kinds - 1 (padding), or its kind is not
    allowed (a logit of -inf is not); except by its weight it still counts in the mean.  What stands in such rows and places is never used.
    Gradients in float16: scale the loss (the upstream gradient is applied in float32, before the one rounding)."""
    _constant(old_log_prob=old_log_prob, advantage=advantage, move=move, ref_log_prob=ref_log_prob, weight=weight)
    per_row = _policy(logits, mean, log_std, allowed)
    rows = logits.shape[:-1]
    _like(kind, "kind", logits, (torch.int32, torch.int64), rows)
    _like(old_log_prob, "old_log_prob", logits, torch.float32, rows)
    _like(advantage, "advantage", logits, torch.float32, rows)
    if (mean is None) != (move is None):
        raise ValueError("mean and move belong together")
    if move is not None:
        _like(move, "move", logits, torch.float32, mean.shape)
    if ref_log_prob is not None:
        _like(ref_log_prob, "ref_log_prob", logits, torch.float32, rows)
    if weight is not None:
        _like(weight, "weight", logits, (torch.float32, torch.bool), rows)
        weight = weight.to(torch.float32)
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (low >= 0 and high >= 0):
        raise ValueError("clip must not be negative")
    if not (math.isfinite(kl_coef) and math.isfinite(entropy_coef)):
        raise ValueError("kl_coef and entropy_coef must be finite")
    if reduction not in ("mean", "sum"):
        raise ValueError("reduction must be 'mean' or 'sum'")
    _on_gpu(logits)
    if kind.dtype != torch.int32:
        kind = kind.clamp(-1, logits.shape[-1]).to(torch.int32)      # (what 32 bits cannot hold is outside all the same)
    fixed = (kind, old_log_prob, advantage, move, ref_log_prob, allowed, weight, float(low), float(high), float(kl_coef), float(entropy_coef), int(reduction == "mean"))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (logits, mean, log_std)):
        loss, stats = _PolicyLoss.apply(logits, mean, log_std, per_row, fixed)
    else:
        loss, stats, _ = _loss_forward(logits, mean, log_std, per_row, fixed, False, (None, None, None))
    return PolicyLoss(loss, *stats[:4].unbind())
