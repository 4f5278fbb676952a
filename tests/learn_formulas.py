"""The operators of agarcl_amd.learn from their definitions, in 64 bits on the CPU, one step and one row at a time (tests only)."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # a rounding: half a step, relative to the value
SMALLEST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half of the smallest step
E = 2.0 ** -24


def d(t):
    return None if t is None else t.detach().cpu().double()


def flags(t):
    return t.cpu() != 0


def recurrence(x, gate, state, reset):
    x, f = d(x), torch.sigmoid(d(gate))
    q = torch.sigmoid(-d(gate))
    h = torch.zeros(x.shape[1:], dtype=torch.float64) if state is None else d(state)
    hs = []
    for t in range(x.shape[0]):
        p = h if reset is None else torch.where(flags(reset)[t][..., None], torch.zeros_like(h), h)
        h = f[t] * p + q[t] * x[t]
        hs.append(h)
    return (torch.stack(hs) if hs else x), h


def recurrence_grads(x, gate, state, reset, dh, dlast):
    """by autograd through the definition"""
    x, gate = d(x).requires_grad_(), d(gate).requires_grad_()
    s = (torch.zeros(x.shape[1:], dtype=torch.float64) if state is None else d(state)).requires_grad_()
    h, out = s, 0.0
    for t in range(x.shape[0]):
        p = h if reset is None else torch.where(flags(reset)[t][..., None], torch.zeros_like(h), h)
        h = torch.sigmoid(gate[t]) * p + torch.sigmoid(-gate[t]) * x[t]
        if dh is not None:
            out = out + (h * d(dh)[t]).sum()
    if dlast is not None:
        out = out + (h * d(dlast)).sum()
    return torch.autograd.grad(out, (x, gate, s), allow_unused=True, materialize_grads=True)


def advantages(reward, value, next_value, terminated, truncated, final_value, gamma, lam):
    r, v, nxt = d(reward), d(value), d(next_value)
    adv, A = torch.zeros_like(r), torch.zeros_like(nxt)
    for t in range(r.shape[0] - 1, -1, -1):
        for i in range(r.shape[1]):
            if terminated[t, i]:
                A[i] = r[t, i] - v[t, i]
            elif truncated is not None and truncated[t, i]:
                A[i] = 0.0 if final_value is None else r[t, i] + gamma * d(final_value)[t, i] - v[t, i]
            else:
                A[i] = r[t, i] + gamma * nxt[i] - v[t, i] + (gamma * lam * A[i] if gamma * lam else 0.0)
        adv[t], nxt = A, v[t]
    return adv, adv + v


def log_prob_entropy(logits, kind, mean, log_std, move, allowed):
    """per row, differentiable: log-probability and entropy; which rows have an allowed kind"""
    ok = logits != -math.inf
    if allowed is not None:
        ok = ok & flags(allowed)
    z = torch.where(ok, logits, torch.full_like(logits, -1e9))
    z = torch.where(ok.any(-1, keepdim=True), z, torch.zeros_like(z))
    lps = torch.log_softmax(z, -1)
    inside = (kind >= 0) & (kind < logits.shape[-1])
    at = kind.long().clamp(0, logits.shape[-1] - 1)[:, None]
    counts = inside & ok.gather(1, at)[:, 0]
    lp = lps.gather(1, at)[:, 0]
    ent = -torch.where(ok, lps.exp() * lps, torch.zeros_like(lps)).sum(-1)
    if mean is not None:
        u = (move - mean) * torch.exp(-log_std)
        lp = lp - (0.5 * u * u + log_std + 0.5 * math.log(2 * math.pi)).sum(-1)
        ent = ent + (log_std + 0.5 * math.log(2 * math.pi * math.e) + 0 * mean).sum(-1)
    return lp, ent, counts


def policy_loss(logits, kind, old, adv, mean=None, log_std=None, move=None, ref=None, allowed=None, weight=None, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0,
                reduction="mean"):
    """(loss, [surrogate, kl, entropy, clipped]); tensors in 64 bits, differentiable in logits, mean, log_std"""
    w = torch.ones_like(adv) if weight is None else weight.double()
    total = w.sum()
    junk = torch.zeros_like(logits)
    ok = torch.ones_like(logits, dtype=torch.bool) if allowed is None else flags(allowed)
    lp, ent, counts = log_prob_entropy(torch.where(ok, logits, junk), kind, mean, log_std, move, allowed)
    counts = counts & (w != 0)
    zero = torch.zeros_like(adv)
    ratio = torch.exp(torch.where(counts, lp - old, zero))
    A = torch.where(counts, adv, zero)
    low = torch.minimum(ratio * A, ratio.clamp(1 - clip[0], 1 + clip[1]) * A)
    back = torch.where(counts, (old if ref is None else ref) - lp, zero)
    kl = torch.expm1(back) - back
    clipped = counts & torch.where(A >= 0, ratio > 1 + clip[1], ratio < 1 - clip[0])
    mean_of = lambda q: torch.where(counts, w * q, zero).sum() / total if total != 0 else zero.sum()   # noqa: E731
    loss = mean_of(-low + kl_coef * kl - entropy_coef * ent)
    if reduction == "sum":
        loss = torch.where(counts, w * (-low + kl_coef * kl - entropy_coef * ent), zero).sum()
    loss = loss + 0 * torch.where(counts, lp, zero).sum()      # (stays differentiable where no weight is left)
    return loss, [mean_of(low), mean_of(kl), mean_of(ent), mean_of(clipped.double())]


def near(got, want, bound, what=""):
    """|got - want| <= bound + the one rounding to got's type, where want is finite; equal elsewhere.  bound: a number or a tensor"""
    dtype, got, want = got.dtype, d(got), d(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), (what, "finite elsewhere")
    off = (got - want).abs()
    room = bound + HALF[dtype] * (want.abs() + bound) + SMALLEST[dtype]
    bad = fine & ~(off <= room)
    if bad.any():
        i = torch.argmax(torch.where(bad, off / room, torch.zeros_like(off)).flatten())
        raise AssertionError("%s: %g instead of %g, %.1f x what rounding allows (%d of %d)" % (what, got.flatten()[i], want.flatten()[i], (off / room).flatten()[i], int(bad.sum()), bad.numel()))
