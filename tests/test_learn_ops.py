"""agarcl_amd.learn on the GPU against the definitions in 64 bits (learn_formulas.py): every type, sizes from one step and one row to many, strides,
resets, masks that leave nothing, rows left out, values that must not be looked at, streams and captured graphs.

Tolerances, derived, in units of E = 2^-24 (a rounding in 32 bits), before the one rounding to the output's type (learn_formulas.near):
  sigmoid: e^-|g| is off by (2 + 1.5 |g|) E or less (the product with log2 e is rounded: |g| 1.44 E; the hardware's exp2: 2 E), its sum, reciprocal and product by 4 E more:
    with |g| <= G both f and 1 - f are good to (6 + 1.5 G) E, relative.
  recurrence: a step adds (1 - f) (6 + 1.5 G) E (|x| + |p|) + 3 E |h| <= (1 - f) (12 + 3 G) E M + 3 E M, with M the largest magnitude of x and state; a step keeps f of the
    error before it, so the errors sum to (12 + 3 G) E M + 3 E M / min(1 - f).
  its gradient: the same bound with M the largest total gradient (Gr = (|dh| + |dlast|) / min(1 - f)); dgate multiplies by (p - x) f (1 - f): at most 2 M / 4, and its error has the
    factors' own, at most (30 + 6 G) E, once more.
Splitting the steps over threads reorders the same products: each join is a rounding of a product and a sum, at most 2 E more for every halving of the length, 64 E for any length."""
import gc
import math

import pytest
import torch

import learn_formulas as F
from learn_formulas import E, d, near

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def learn(hip_engine_cls):
    import os
    from agarcl_amd import build
    if not os.path.exists(build.learn_torch_out()):
        build.build_learn_torch()
    from agarcl_amd import learn as module
    return module


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def cuda(t, dtype=None):
    return None if t is None else t.to(device="cuda", dtype=dtype or t.dtype)


# ---- recurrence ---------------------------------------------------------------------------------------------------------------------------

def memory_inputs(T, rows, C, dtype, seed, resets, gmax=4.0):
    g = rng(seed)
    shape = (T,) + rows + (C,)
    x = cuda(torch.randn(shape, generator=g).clamp(-4, 4), dtype)
    gate = cuda((torch.randn(shape, generator=g) * 2).clamp(-gmax, gmax), dtype)
    state = cuda(torch.randn(rows + (C,), generator=g).clamp(-4, 4))
    dh = cuda(torch.randn(shape, generator=g).clamp(-4, 4), dtype)
    dlast = cuda(torch.randn(rows + (C,), generator=g).clamp(-4, 4))
    p = {"none": None, "some": 0.1, "all": 1.1, "first": 0.0}[resets]
    reset = None if p is None else cuda(torch.rand((T,) + rows, generator=g) < p)
    if resets == "first" and T:
        reset[0] = True
    return x, gate, state, reset, dh, dlast


def memory_bounds(gmax, biggest, steps):
    q = 1 / (1 + math.exp(gmax))                     # the smallest 1 - f
    lasting = min(1 / q, steps)                      # an error lasts for as many steps, at most
    h = (12 + 3 * gmax + 64 + 3 * lasting) * E * biggest
    top = 2 * biggest * min(1 / q, steps + 1)        # the largest total gradient
    grad = (12 + 3 * gmax + 64 + 3 * lasting) * E * top * 2
    return h, grad, grad * biggest / 2 + top * biggest / 2 * (30 + 6 * gmax) * E + top * h / 4


SHAPES = [(1, (1,), 1), (1, (5,), 3), (2, (1,), 7), (7, (3,), 5), (8, (2,), 8), (9, (1,), 64), (16, (4,), 32), (17, (33,), 77), (64, (4,), 256), (65, (2, 3), 12), (300, (2,), 4), (1000, (1,), 1),
          (31, (1000,), 8), (3, (4099,), 5), (2049, (3,), 20), (5000, (2,), 16),
          (1000, (5,), 13), (700, (1,), 65), (300, (3,), 43), (40, (171,), 3), (9, (1,), 4097), (2, (1,), 65537),      # (the last: 16-bit columns in pairs, one left over at the head of a workgroup)
          (1100, (1031,), 1), (24, (33000,), 4), (1500, (70,), 1), (2040, (9,), 5), (600, (1001,), 2)]      # (a shape of launch each)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape,resets", [(s, r) for s in SHAPES for r in ("none", "some", "all", "first") if s[0] <= 300 or r in ("none", "some")],
                         ids=lambda v: v if isinstance(v, str) else "x".join(map(str, (v[0],) + v[1] + (v[2],))))
def test_recurrence_and_its_gradients(learn, shape, resets, dtype):
    T, rows, C = shape
    x, gate, state, reset, dh, dlast = memory_inputs(T, rows, C, dtype, 1, resets)
    hb, gb, gateb = memory_bounds(4.0, 4.0, T)
    want_h, want_last = F.recurrence(x, gate, state, reset)
    h, last = learn.gated_recurrence(x, gate, state, reset)
    near(h, want_h, hb, "h"); near(last, want_last, hb, "last")
    assert h.dtype == dtype and last.dtype == torch.float32
    leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
    h2, last2 = learn.gated_recurrence(leaves[0], leaves[1], leaves[2], reset)
    assert torch.equal(h2, h) and torch.equal(last2, last)
    got = torch.autograd.grad((h2, last2), leaves, (dh, dlast))
    want = F.recurrence_grads(x, gate, state, reset, dh, dlast)
    for g, w, b, name in zip(got, want, (gb, gateb, gb), ("dx", "dgate", "dstate")):
        near(g, w, b, name)


def test_recurrence_step_is_one_step_and_many_make_a_rollout(learn):
    for dtype in TYPES:
        x, gate, state, reset, _, _ = memory_inputs(40, (37,), 19, dtype, 2, "some")
        want_h, want_last = learn.gated_recurrence(x, gate, state, reset)
        s = state
        for t in range(40):
            h, s = learn.recurrence_step(x[t], gate[t], s, reset[t])
            near(h, want_h[t], memory_bounds(4.0, 4.0, 40)[0] * 2 + F.HALF[dtype] * 4, "h")
        near(s, want_last, memory_bounds(4.0, 4.0, 40)[0] * 2, "state")
        h1, s1 = learn.gated_recurrence(x[:1], gate[:1], state, reset[:1])
        h0, s0 = learn.recurrence_step(x[0], gate[0], state, reset[0])
        near(h0, h1[0], memory_bounds(4.0, 4.0, 1)[0] * 2 + F.HALF[dtype] * 4, "h"); near(s0, s1, memory_bounds(4.0, 4.0, 1)[0] * 2, "state")
        h0, s0 = learn.recurrence_step(x[0], gate[0], state)
        near(s0, F.recurrence(x[:1], gate[:1], state, None)[1], memory_bounds(4.0, 4.0, 1)[0], "state")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_recurrence_strides_offsets_and_flag_types(learn, dtype):
    """a slice of arenas of a larger rollout, tensors that start in the middle of a vector load, transposed tensors, flags as uint8"""
    T, B, C = 45, 6, 13
    x, gate, state, reset, dh, dlast = memory_inputs(T, (B,), C, dtype, 3, "some")
    want = learn.gated_recurrence(x, gate, state, reset)
    big = torch.full((T, B + 5, C), float("nan"), dtype=dtype, device="cuda")
    big[:, 2:2 + B] = x
    odd = torch.full((T * B * C + 3,), float("nan"), dtype=dtype, device="cuda")
    odd[3:] = gate.flatten()
    turned = gate.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    wide = torch.ones(T, B + 3, dtype=torch.uint8, device="cuda")
    wide[:, 1:1 + B] = reset
    for xx, gg, rr in ((big[:, 2:2 + B], gate, reset), (x, odd[3:].view(T, B, C), reset), (x, turned, reset), (x, gate, wide[:, 1:1 + B]), (x, gate, reset.to(torch.uint8) * 7)):
        assert all(torch.equal(a, b) for a, b in zip(learn.gated_recurrence(xx, gg, state, rr), want))
        lx, lg, ls = xx.detach().requires_grad_(), gg.detach().requires_grad_(), state.clone().requires_grad_()
        got = torch.autograd.grad(learn.gated_recurrence(lx, lg, ls, rr), (lx, lg, ls), (dh, dlast))
        for g, w, b in zip(got, F.recurrence_grads(x, gate, state, reset, dh, dlast), (1, 2, 1)):
            near(g, w, memory_bounds(4.0, 4.0, T)[b])
    every = x[:1].expand(T, B, C)
    near(learn.gated_recurrence(every, gate, state.expand(B, C), None)[0], F.recurrence(every, gate, state, None)[0], memory_bounds(4.0, 4.0, T)[0])


def test_recurrence_looks_at_nothing_behind_a_reset(learn):
    for T in (3, 20, 700):
        x, gate, state, reset, dh, dlast = memory_inputs(T, (9,), 6, torch.float32, 4, "first")
        bad = state.clone(); bad[:3] = float("nan"); bad[3:6] = float("inf"); bad[6:] = -float("inf")
        cut = T // 2
        reset[cut] = True
        x2 = x.clone(); x2[:cut] = float("nan")                                    # an episode that went wrong ends with it
        h, last = learn.gated_recurrence(x2, gate, bad, reset)
        near(h[cut:], F.recurrence(x, gate, state, reset)[0][cut:], memory_bounds(4.0, 4.0, T)[0]); assert torch.isfinite(last).all()
        dh2 = dh.clone(); dh2[cut:] = float("nan")                                 # nor does a gradient pass it backwards
        leaves = [t.detach().requires_grad_() for t in (x, gate, bad)]
        dx, dgate, dstate = torch.autograd.grad(learn.gated_recurrence(*leaves, reset), leaves, (dh2, dlast))
        want = F.recurrence_grads(x[:cut], gate[:cut], state, reset[:cut], dh[:cut], None)
        near(dx[:cut], want[0], memory_bounds(4.0, 4.0, T)[1]); near(dgate[:cut], want[1], memory_bounds(4.0, 4.0, T)[2])
        assert torch.equal(dstate, torch.zeros_like(dstate))


def test_recurrence_gates_without_end(learn):
    """a gate of +inf keeps the state, one of -inf takes x, and neither loses the other's finite value"""
    inf = float("inf")
    x = torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda").view(4, 1, 1).repeat(1, 1, 5).contiguous()
    gate = torch.tensor([inf, -inf, 200.0, -200.0], device="cuda").view(4, 1, 1).repeat(1, 1, 5).contiguous()
    h, last = learn.gated_recurrence(x, gate, torch.full((1, 5), 9.0, device="cuda"))
    assert h[:, 0, 0].tolist() == [9.0, 2.0, 2.0, 4.0]
    leaves = [t.detach().requires_grad_() for t in (x, gate)]
    grads = torch.autograd.grad(learn.gated_recurrence(*leaves)[0].sum(), leaves)
    assert all(torch.isfinite(g).all() for g in grads)
    assert grads[0][:, 0, 0].tolist() == [0.0, 2.0, 0.0, 1.0]


def test_recurrence_long_memories_keep_their_length(learn):
    """1 - f of a few 1e-4 over thousands of steps: the relative error of 1 - f must not grow with 1 / (1 - f)"""
    T = 6000
    gate = torch.full((T, 2, 4), 8.0, device="cuda")
    x = torch.randn((T, 2, 4), generator=rng(5)).clamp(-4, 4).cuda()
    h, last = learn.gated_recurrence(x, gate)
    near(h, F.recurrence(x, gate, None, None)[0], memory_bounds(8.0, 4.0, T)[0])
    const, _ = learn.gated_recurrence(torch.ones_like(x), gate)
    near(const, F.recurrence(torch.ones_like(x), gate, None, None)[0], memory_bounds(8.0, 1.0, T)[0])


def test_recurrence_parts_of_the_gradient(learn):
    x, gate, state, reset, dh, dlast = memory_inputs(21, (4,), 6, torch.float32, 6, "some")
    for use_h, use_last in ((True, False), (False, True)):
        leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
        h, last = learn.gated_recurrence(*leaves, reset)
        got = torch.autograd.grad([t for t, u in ((h, use_h), (last, use_last)) if u], leaves, [t for t, u in ((dh, use_h), (dlast, use_last)) if u])
        for g, w, b in zip(got, F.recurrence_grads(x, gate, state, reset, dh if use_h else None, dlast if use_last else None), (1, 2, 1)):
            near(g, w, memory_bounds(4.0, 4.0, 21)[b])
    leaves = [t.detach().requires_grad_() for t in (x, gate)]
    (learn.gated_recurrence(*leaves)[0] * 2).sum().backward()                     # an expanded gradient, no state, no reset
    want = F.recurrence_grads(x, gate, None, None, torch.full_like(dh, 2.0), None)
    near(leaves[0].grad, want[0], memory_bounds(4.0, 4.0, 21)[1]); near(leaves[1].grad, want[1], memory_bounds(4.0, 4.0, 21)[2])
    only = x.detach().requires_grad_()
    h, _ = learn.gated_recurrence(only, gate, state)
    a, b = torch.autograd.grad(h.sum(), only, retain_graph=True)[0], torch.autograd.grad(h.sum(), only)[0]
    assert torch.equal(a, b)
    # against differences of the definition in 64 bits, along random directions
    for i in range(3):
        v = torch.randn(x.shape, generator=rng(70 + i), dtype=torch.float64)
        f = lambda s: (F.recurrence(d(x) + s * v, d(gate) + s * v, d(state), reset)[0] * d(dh)).sum()   # noqa: E731
        leaves = [t.detach().requires_grad_() for t in (x, gate)]
        got = torch.autograd.grad(learn.gated_recurrence(*leaves, state, reset)[0], leaves, dh)
        along = sum((d(g) * v).sum() for g in got)
        n = v.numel()
        assert abs(along - (f(1e-4) - f(-1e-4)) / 2e-4) < n * 4 * sum(memory_bounds(4.0, 4.0, 21)[1:]) + 1e-4


def test_recurrence_of_nothing(learn):
    for shape in ((0, 3, 4), (5, 0, 4), (5, 3, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True); state = torch.randn(shape[1:], device="cuda").requires_grad_()
        h, last = learn.gated_recurrence(x, torch.zeros(shape, device="cuda"), state)
        assert h.shape == shape and last.shape == shape[1:]
        gx, gs = torch.autograd.grad((h.sum() + (last * 3).sum()), (x, state))
        if shape[0] == 0:
            assert torch.equal(last, state) and torch.equal(gs, torch.full_like(gs, 3.0))
        assert gx.shape == shape
    h, s = learn.recurrence_step(torch.zeros(0, 4, device="cuda"), torch.zeros(0, 4, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert h.shape == s.shape == (0, 4)


# ---- advantages: delta sums three rounded terms (3 E (|r| + 2 |v|)), a step keeps gamma lam of the error before it and adds 2 roundings of A: <= (6 V + 2 A) E / (1 - gamma lam),
# ---- or times the steps; 64 E A for the joins of a split length ----------------------------------------------------------------------------------------------------------

def rollout(T, B, dtype, seed, p_term, p_trunc):
    g = rng(seed)
    reward, value = cuda(torch.randn(T, B, generator=g).clamp(-4, 4) * 2), cuda(torch.randn(T, B, generator=g).clamp(-4, 4) + 5, dtype)
    nxt = cuda(torch.randn(B, generator=g).clamp(-4, 4) + 5, dtype)
    term, trunc = cuda(torch.rand(T, B, generator=g) < p_term), cuda(torch.rand(T, B, generator=g) < p_trunc)
    final = cuda(torch.randn(T, B, generator=g).clamp(-4, 4) + 5, dtype)
    return reward, value, nxt, term, trunc, final


def adv_bound(T, gl):
    last = min(T, 1 / (1 - gl) if gl < 1 else T)
    top = 26 * last
    return (64 + 2 * last) * E * top + 80 * E * last


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,B", [(1, 1), (1, 70), (2, 3), (7, 5), (8, 8), (9, 64), (32, 64), (33, 257), (129, 16), (300, 4), (257, 1030), (2000, 1), (9001, 3), (1100, 1031), (520, 4100), (2040, 45), (600, 2003)])
def test_advantages(learn, T, B, dtype):
    for seed, (p_term, p_trunc, with_trunc, with_final, gamma, lam) in enumerate([(0.0, 0, False, False, 0.99, 0.95), (0.1, 0.1, True, False, 0.99, 0.95), (0.1, 0.1, True, True, 0.999, 1.0),
                                                                                  (1.1, 0.5, True, True, 0.9, 0.9), (0.05, 1.1, True, False, 0.9, 0.9), (0.1, 0.1, True, True, 0.9, 0.0),
                                                                                  (0.1, 0.1, True, True, 0.0, 0.9), (0.0, 0.0, True, True, 1.0, 1.0)]):
        if T > 1000 and seed not in (1, 2):
            continue
        if T * B > 100000 and seed != 2:
            continue
        reward, value, nxt, term, trunc, final = rollout(T, B, dtype, 100 * seed + T, p_term, p_trunc)
        trunc, final = trunc if with_trunc else None, final if with_final else None
        got = learn.advantages(reward, value, nxt, term, trunc, final, gamma=gamma, lam=lam)
        cpu = [None if t is None else t.cpu() for t in (reward, value, nxt, term, trunc, final)]
        want = F.advantages(*cpu, float(torch.tensor(gamma)), float(torch.tensor(lam))) if T * B <= 40000 else fast_advantages(*cpu, float(torch.tensor(gamma)), float(torch.tensor(lam)))
        near(got.advantage, want[0], adv_bound(T, gamma * lam), "advantage"); near(got.returns, want[1], adv_bound(T, gamma * lam) + 20 * E, "returns")


def fast_advantages(r, v, nxt, term, trunc, final, gamma, lam):
    """F.advantages with the rows at once"""
    r, v, nxt = r.double(), v.double(), nxt.double()
    adv, A = torch.zeros_like(r), torch.zeros_like(nxt)
    trunc = torch.zeros_like(term) if trunc is None else trunc & ~term
    for t in range(r.shape[0] - 1, -1, -1):
        on = r[t] + gamma * nxt - v[t] + gamma * lam * A
        cut = (r[t] + gamma * final[t].double() - v[t]) if final is not None else torch.zeros_like(on)
        A = torch.where(term[t], r[t] - v[t], torch.where(trunc[t], cut, on))
        adv[t], nxt = A, v[t]
    return adv, adv + v


def test_advantages_look_at_nothing_behind_an_end(learn):
    for T in (6, 40, 900):
        reward, value, nxt, term, trunc, final = rollout(T, 8, torch.float32, 9, 0, 0)
        cut = T // 2
        term[cut, :4] = True; trunc[cut, 4:] = True
        want = learn.advantages(reward, value, nxt, term, trunc, final)
        value2, reward2, nxt2, final2 = value.clone(), reward.clone(), torch.full_like(nxt, float("nan")), torch.full_like(final, float("nan"))
        value2[cut + 1:] = float("nan"); reward2[cut + 1:] = float("inf"); final2[cut, 4:] = final[cut, 4:]
        got = learn.advantages(reward2, value2, nxt2, term, trunc, final2)
        assert torch.equal(got.advantage[:cut + 1], want.advantage[:cut + 1]) and torch.equal(got.returns[:cut + 1], want.returns[:cut + 1])
        both = learn.advantages(reward, value, nxt, term | trunc, trunc, final)          # terminated and truncated: terminated
        near(both.advantage[cut], d(reward[cut] - value[cut]), 4 * E * 16)


def test_advantages_strides_agents_and_env_flags(learn):
    T, B = 37, 11
    reward, value, nxt, term, trunc, final = rollout(T, B, torch.bfloat16, 10, 0.1, 0.1)
    want = learn.advantages(reward, value, nxt, term, trunc, final)
    wide = lambda t: torch.cat((t, t, t), 1)[:, B - 3:2 * B - 3 + 3][:, 3:]               # noqa: E731  (rows of a wider buffer)
    got = learn.advantages(wide(reward), wide(value), nxt, wide(term).to(torch.uint8), wide(trunc), wide(final))
    assert torch.equal(got.advantage, want.advantage) and torch.equal(got.returns, want.returns)
    agents = lambda t: t.view(T, 1, B) if t.dim() == 2 else t.view(1, B)                  # noqa: E731
    got = learn.advantages(*(agents(t) for t in (reward, value, nxt, term, trunc, final)))
    assert got.advantage.shape == (T, 1, B) and torch.equal(got.advantage.view(T, B), want.advantage)
    turned = lambda t: t.t().contiguous().t()                                             # noqa: E731
    got = learn.advantages(turned(reward), turned(value), nxt, turned(term), turned(trunc), turned(final))
    assert torch.equal(got.advantage, want.advantage)
    for shape in ((0, 4), (4, 0)):
        got = learn.advantages(torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda"), torch.zeros(shape[1], device="cuda"), torch.zeros(shape, dtype=torch.bool, device="cuda"))
        assert got.advantage.shape == got.returns.shape == shape


# ---- policy: a log-probability is off by at most lp_err: z - max and the log of the sum are rounded (3 E (Z + log V + 1), Z the largest |z| difference), each exp of the sum by
# ---- (2 + 1.5 Z) E and the sum itself by V / 64 + 8 additions; the move adds its own terms' roundings, 8 E each -----------------------------------------------------------

def lp_err(Z, V, lp_move=0.0):
    return (3 * (Z + math.log(V) + 1) + 2 + 1.5 * Z + V / 64 + 8) * E + 16 * E * (1 + lp_move)


def policy_inputs(R, V, dtype, seed, move=True, per_row=False, mask=0.0, junk=True, lead=None):
    g = rng(seed)
    z = torch.randn(R, V, generator=g).clamp(-4, 4)
    allowed = None
    if mask:
        allowed = torch.rand(R, V, generator=g) >= mask
        if R > 2:
            allowed[1] = False                                       # nothing is allowed
            allowed[2] = False; allowed[2, V // 2] = True            # one kind is
    p = dict(logits=cuda(z, dtype), allowed=cuda(allowed))
    if mask and junk:
        bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min])[torch.randint(0, 4, (R, V), generator=g)]
        p["logits"] = torch.where(p["allowed"], p["logits"], cuda(bad, dtype))
    if move:
        p["mean"] = cuda(torch.randn(R, 2, generator=g).clamp(-2, 2), dtype)
        p["log_std"] = cuda(torch.randn(R, 2, generator=g).clamp(-1, 1), dtype) if per_row else cuda(torch.randn(2, generator=g).clamp(-1, 1))
    return p, g


SIZES = [(1, 1), (1, 3), (5, 2), (70, 3), (257, 4), (33, 5), (64, 8), (31, 9), (130, 24), (9, 63), (9, 64), (9, 65), (17, 129), (6, 511), (6, 513), (5, 1000), (4, 2049), (3, 5001), (3, 9000),
         (3, 33000), (2, 70001), (4, 1300), (4, 1800), (3, 7001)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("R,V", SIZES)
def test_sample_actions(learn, R, V, dtype):
    for seed, (move, per_row, mask, noise) in enumerate([(True, False, 0.0, True), (False, False, 0.4, True), (True, True, 0.4, True), (True, False, 0.4, False)]):
        p, g = policy_inputs(R, V, dtype, seed * 1000 + V, move, per_row, mask)
        gumbel = cuda(-torch.log(-torch.log(torch.rand(R, V, generator=g).clamp(1e-7, 1 - 1e-6)))) if noise else None
        if mask and noise:
            gumbel = torch.where(p["allowed"], gumbel, torch.full_like(gumbel, float("nan")))
        normal = cuda(torch.randn(R, 2, generator=g).clamp(-3, 3)) if move and noise else None
        a = learn.sample_actions(gumbel=gumbel, normal=normal, **p)
        ok = torch.ones(R, V, dtype=torch.bool) if p["allowed"] is None else p["allowed"].cpu()
        score = (p["logits"].cpu().float() + (0 if gumbel is None else gumbel.cpu())).masked_fill(~ok, -math.inf)      # the one rounding that the definition has
        kind = torch.tensor([int((row == row.max()).nonzero()[0]) if okr.any() else 0 for row, okr in zip(score, ok)], dtype=torch.int32)
        assert torch.equal(a.kind.cpu(), kind) and a.kind.dtype == torch.int32
        mean, ls = d(p.get("mean")), d(p.get("log_std"))
        raw = None
        if move:
            raw = mean + ls.exp() * (0 if normal is None else d(normal))
            near(a.raw, raw.expand(R, 2), 12 * E * (2 + 3 * math.e)); assert torch.equal(a.move, a.raw.clamp(-1, 1))
        else:
            assert a.raw is None and a.move is None
        lp, _, counts = F.log_prob_entropy(torch.where(ok, d(p["logits"]), torch.zeros(R, V, dtype=torch.float64)), kind, mean, ls, raw, p["allowed"])
        if move:
            alone = F.log_prob_entropy(torch.zeros(R, 1, dtype=torch.float64), torch.zeros(R), mean, ls, raw, None)[0]
        want = torch.where(counts, lp, alone if move else torch.zeros_like(lp))
        near(a.log_prob, want, lp_err(8, V, 16 if move else 0), "log_prob")


def test_sampling_follows_the_policy(learn):
    """200000 draws from one row: each kind's share within 5 standard deviations, the move's mean and spread too"""
    n = 200000
    z = torch.tensor([0.5, -1.0, 1.2], device="cuda").expand(n, 3)
    g = torch.Generator(device="cuda"); g.manual_seed(5)
    gumbel = -torch.log(-torch.log(torch.rand(n, 3, generator=g, device="cuda").clamp(1e-7, 1 - 1e-6)))
    a = learn.sample_actions(z, torch.zeros(n, 2, device="cuda") + 0.3, torch.zeros(2, device="cuda") - 0.5, gumbel=gumbel, normal=torch.randn(n, 2, generator=g, device="cuda"))
    p = torch.softmax(z[0].double().cpu(), 0)
    share = torch.bincount(a.kind.long(), minlength=3).double().cpu() / n
    assert ((share - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()
    s = math.exp(-0.5)
    assert (a.raw.mean(0) - 0.3).abs().max() < 5 * s / math.sqrt(n) and (a.raw.std(0) - s).abs().max() < 5 * s / math.sqrt(2 * n)


def test_sample_ties_and_infinities(learn):
    z = torch.zeros(3, 300, device="cuda"); z[0, 100] = z[0, 7] = z[0, 299] = 2.0
    z[1] = -float("inf"); z[2] = torch.finfo(torch.float32).min; z[2, 250] = -float("inf")
    a = learn.sample_actions(z)
    assert a.kind.tolist() == [7, 0, 0]
    near(a.log_prob, torch.tensor([2 - math.log(3 * math.exp(2) + 297), 0.0, -math.log(299)], dtype=torch.float64), lp_err(8, 300))
    assert learn.sample_actions(torch.zeros(0, 3, device="cuda")).kind.shape == (0,)
    one = learn.sample_actions(torch.full((2, 2, 1), 5.0, device="cuda", dtype=torch.float16))
    assert one.kind.shape == (2, 2) and (one.log_prob == 0).all()


def loss_inputs(R, V, dtype, seed, move, per_row, mask, ref, weight):
    p, g = policy_inputs(R, V, dtype, seed, move, per_row, mask)
    ok = torch.ones(R, V, dtype=torch.bool) if p["allowed"] is None else p["allowed"].cpu()
    kind = torch.where(ok, torch.rand(R, V, generator=g), torch.full((R, V), -1.0)).argmax(1).int()
    if R > 8:
        kind[3], kind[4], kind[5] = -1, V, -2147483648
        if mask:
            kind[6] = int((~ok[6]).int().argmax())                  # (not allowed, where anything is not)
    p["kind"] = cuda(kind)
    raw = None
    if move:
        p["move"] = cuda(d(p["mean"]).float() + d(p["log_std"]).exp().float() * torch.randn(R, 2, generator=g).clamp(-2, 2))
        raw = d(p["move"])
    lp, _, counts = F.log_prob_entropy(torch.where(ok, d(p["logits"]), torch.zeros(R, V, dtype=torch.float64)), kind, d(p.get("mean")), d(p.get("log_std")), raw, p["allowed"])
    drift = torch.randn(R, generator=g).double().clamp(-2, 2) * 0.2
    for border in (0.8, 1.3):                                        # (no row on a border of the clip, where one rounding would decide its side)
        drift = torch.where((drift.exp() - border).abs() < 1e-3, drift + 4e-3, drift)
    p["old_log_prob"] = cuda((lp - drift).float())
    p["advantage"] = cuda(torch.randn(R, generator=g).clamp(-3, 3))
    if R > 1:
        p["advantage"][R - 1] = 0.0
    p["ref_log_prob"] = cuda((lp - torch.randn(R, generator=g).double().clamp(-2, 2) * 0.3).float()) if ref else None
    w = None
    if weight:
        w = torch.rand(R, generator=g) + 0.5
        w[::5] = 0.0
        p["advantage"][::5] = float("nan"); p["old_log_prob"][::5] = float("inf")       # what a weight of 0 leaves out is not looked at
        if R > 11:
            p["logits"][10] = float("nan")
    p["weight"] = cuda(w)
    skip = ~counts
    if skip.any():
        p["advantage"][cuda(skip)] = float("nan")
        if move:
            p["move"][cuda(skip)] = float("nan")
    return p


def check_loss(learn, p, V, dtype, kw, upstream=None):
    R = p["kind"].numel()
    move = p.get("mean") is not None
    names = [n for n in ("logits", "mean", "log_std") if p.get(n) is not None]
    leaves = {n: p[n].detach().requires_grad_() for n in names}
    out = learn.policy_loss(**dict(p, **leaves), **kw)
    up = torch.tensor(1.0 if upstream is None else upstream, device="cuda")
    got = torch.autograd.grad(out.loss, list(leaves.values()), up)
    with torch.no_grad():
        plain = learn.policy_loss(**p, **kw)
    assert all(torch.equal(a, b) for a, b in zip(plain, out))        # (with and without gradients)
    q = {n: d(t) for n, t in p.items() if n not in ("kind", "allowed")}
    zeroed = q["weight"] == 0 if q["weight"] is not None else torch.zeros(R, dtype=torch.bool)
    q["logits"] = torch.where(zeroed[:, None], torch.zeros_like(q["logits"]), q["logits"])
    ok = torch.ones_like(q["logits"], dtype=torch.bool) if p["allowed"] is None else p["allowed"].cpu()
    q["logits"] = torch.where(ok, q["logits"], torch.zeros_like(q["logits"]))
    if move:
        q["move"] = torch.where(torch.isfinite(q["move"]), q["move"], torch.zeros_like(q["move"]))
    for n in names:
        q[n].requires_grad_()
    clip = kw.get("clip", 0.2)
    clip = clip if isinstance(clip, tuple) else (clip, clip)
    ck, ce = kw.get("kl_coef", 0.0), kw.get("entropy_coef", 0.0)
    loss, stats = F.policy_loss(q["logits"], p["kind"].cpu(), q["old_log_prob"], q["advantage"], q.get("mean"), q.get("log_std"), q.get("move"), q["ref_log_prob"], p["allowed"],
                                q["weight"], clip, ck, ce, kw.get("reduction", "mean"))
    want = torch.autograd.grad(loss, [q[n] for n in names], torch.tensor(float(up), dtype=torch.float64), allow_unused=True, materialize_grads=True)
    # the ratio is at most e^0.45, |advantage| <= 3, |ref - lp| <= 0.65: a row's terms and their slopes in lp are at most 6 + 2 ck; the entropy is at most log V + 8
    le = lp_err(8, V, 16 if move else 0)
    weight_top, denom = (1.5, float(q["weight"].sum())) if q["weight"] is not None else (1.0, float(R))
    by = (1.0 / denom if denom else 0.0) if kw.get("reduction", "mean") == "mean" else 1.0
    term = 6 * (le + 4 * E) + ck * 2 * (le + 4 * E) + ce * (le * 4 + 8 * E * (math.log(V) + 8))
    near(out.loss, loss.detach(), term * (1 if by < 1 or R == 1 else 1.5 * R), "loss")
    for g, w, b, n in zip((out.surrogate, out.kl, out.entropy, out.clipped), stats, (6 * (le + 4 * E), 2 * (le + 4 * E), le * 4 + 8 * E * (math.log(V) + 8), 4 * E), ("surrogate", "kl", "entropy", "clipped")):
        near(g, w.detach(), b, n)
    share = weight_top * by * float(up)
    slope = 6 + 2 * ck
    row = share * (slope * (2 * le + 12 * E) + 6 * le + ce * (math.log(V) + 4) * (2 * le + 12 * E))
    near(got[0], want[0], row, "dlogits")
    if move:     # a deviation is at most 2 (2.1 with the roundings), a reciprocal spread e; both good to 8 E times the magnitudes
        near(got[1], want[1], 6 * row + share * slope * 200 * E, "dmean")
        near(got[2], want[2], (6 * row + share * slope * 200 * E) * (1 if p["log_std"].dim() > 1 else R), "dlog_std")
    return out, got


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("R,V", SIZES)
def test_policy_loss_and_its_gradients(learn, R, V, dtype):
    for seed, (move, per_row, mask, ref, weight, kw) in enumerate([
            (False, False, 0.0, False, False, dict()),
            (True, False, 0.0, False, False, dict(clip=(0.2, 0.3), entropy_coef=0.01)),
            (True, True, 0.4, True, True, dict(clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.02)),
            (True, False, 0.4, True, True, dict(clip=(0.2, 0.3), kl_coef=0.1, reduction="sum")),
            (False, False, 0.4, True, False, dict(clip=(0.2, float("inf")), kl_coef=0.3, entropy_coef=-0.02))]):
        p = loss_inputs(R, V, dtype, seed * 77 + V, move, per_row, mask, ref, weight)
        check_loss(learn, p, V, dtype, kw, upstream=None if seed % 2 else 1024.0 if dtype == torch.float16 else 0.5)


def test_policy_loss_over_many_rows(learn):
    for R, V, dtype in ((20011, 3, torch.float32), (20011, 24, torch.bfloat16), (15001, 511, torch.bfloat16), (1601, 5001, torch.bfloat16), (1301, 8001, torch.float32)):
        p = loss_inputs(R, V, dtype, 8, True, False, 0.2, True, True)
        check_loss(learn, p, V, dtype, dict(clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.01))


def test_policy_loss_forms_of_its_arguments(learn):
    R, V = 60, 7
    p = loss_inputs(R, V, torch.float32, 11, True, False, 0.3, True, False)
    kw = dict(clip=0.2, kl_coef=0.1, entropy_coef=0.01)

    def both(p, **more):
        leaves = [p[n].detach().requires_grad_() for n in ("logits", "mean", "log_std")]
        out = learn.policy_loss(**dict(p, logits=leaves[0], mean=leaves[1], log_std=leaves[2]), **dict(kw, **more))
        return list(out) + list(torch.autograd.grad(out.loss, leaves))

    want = both(p)
    same = lambda got: all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))     # noqa: E731
    assert same(both(dict(p, kind=p["kind"].long())))
    assert same(both(dict(p, allowed=p["allowed"].to(torch.uint8) * 3)))
    assert same(both(dict(p, weight=torch.ones(R, dtype=torch.bool, device="cuda"))))
    wide = torch.full((R, V + 3), float("nan"), device="cuda"); wide[:, 2:2 + V] = p["logits"]
    assert same(both(dict(p, logits=wide[:, 2:2 + V])))
    assert same(both(dict(p, logits=p["logits"].t().contiguous().t(), mean=p["mean"].t().contiguous().t())))
    lead = lambda t: None if t is None else t if t.shape == (2,) else t.reshape((4, 15) + t.shape[1:])   # noqa: E731
    assert same(both({n: lead(t) for n, t in p.items()}))
    huge = p["kind"].long(); huge[3] = 1 << 40; huge[4] = -(1 << 40)
    assert same(both(dict(p, kind=huge)))
    zero = both(dict(p, weight=torch.zeros(R, device="cuda")))
    assert all((t == 0).all() for t in zero)
    none = learn.policy_loss(torch.zeros(0, 3, device="cuda", requires_grad=True), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"))
    std = torch.zeros(2, device="cuda", requires_grad=True)
    moved = learn.policy_loss(torch.zeros(0, 3, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"),
                              torch.zeros(0, 2, device="cuda"), std, torch.zeros(0, 2, device="cuda"))
    assert torch.autograd.grad(moved.loss, std)[0].tolist() == [0.0, 0.0]
    assert none.loss.item() == 0 and torch.autograd.grad(none.loss, none.loss)[0].item() == 1
    none.loss.backward()


def test_policy_loss_gradient_twice_and_with_other_upstreams(learn):
    p = loss_inputs(50, 5, torch.bfloat16, 12, True, False, 0.0, False, True)
    names = ("logits", "mean", "log_std")
    leaves = [p[n].detach().requires_grad_() for n in names]
    out = learn.policy_loss(**dict(p, **dict(zip(names, leaves))))
    first = torch.autograd.grad(out.loss, leaves, retain_graph=True)
    kept = [g.clone() for g in first]
    half = torch.autograd.grad(out.loss, leaves, torch.tensor(0.5, device="cuda"), retain_graph=True)
    again = torch.autograd.grad(out.loss, leaves)
    for f, k, h, a in zip(first, kept, half, again):
        assert torch.equal(f, k) and torch.equal(f, a) and torch.equal(h, (f.float() * 0.5).to(f.dtype))       # (halving is exact)
    only = p["mean"].detach().requires_grad_()
    g = torch.autograd.grad(learn.policy_loss(**dict(p, mean=only)).loss, only)[0]
    assert torch.equal(g, first[1])
    accumulated = p["logits"].detach().requires_grad_()
    for _ in range(2):
        learn.policy_loss(**dict(p, logits=accumulated)).loss.backward()
    assert torch.equal(accumulated.grad, first[0] + first[0])
    p["old_log_prob"].add_(0)                                                        # the graph above is gone; a live one notices a rewritten buffer
    out = learn.policy_loss(**dict(p, logits=accumulated))
    p["old_log_prob"].add_(1)
    with pytest.raises(RuntimeError):
        out.loss.backward()


def test_no_gradients_of_gradients(learn):
    x = torch.randn(3, 2, 4, device="cuda", requires_grad=True)
    h, _ = learn.gated_recurrence(x, torch.randn(3, 2, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(h.sum(), x, create_graph=True)
    z = torch.randn(5, 3, device="cuda", requires_grad=True)
    out = learn.policy_loss(z, torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, device="cuda"), torch.ones(5, device="cuda"))
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(out.loss, z, create_graph=True)


def test_policy_loss_gradient_against_differences(learn):
    p = loss_inputs(40, 6, torch.float32, 13, True, True, 0.0, True, False)
    kw = dict(clip=(0.2, 0.3), kl_coef=0.1, entropy_coef=0.02)
    _, got = check_loss(learn, p, 6, torch.float32, kw)
    q = {n: d(t) for n, t in p.items() if n not in ("kind", "allowed")}
    q["move"] = torch.where(torch.isfinite(q["move"]), q["move"], torch.zeros_like(q["move"]))
    for seed in range(3):
        g = rng(seed)
        v = [torch.randn(q[n].shape, generator=g, dtype=torch.float64) for n in ("logits", "mean", "log_std")]
        f = lambda s: F.policy_loss(q["logits"] + s * v[0], p["kind"].cpu(), q["old_log_prob"], q["advantage"], q["mean"] + s * v[1], q["log_std"] + s * v[2], q["move"],   # noqa: E731
                                    q["ref_log_prob"], None, None, (0.2, 0.3), 0.1, 0.02)[0]
        along = sum((d(a) * b).sum() for a, b in zip(got, v))
        assert abs(along - (f(1e-5) - f(-1e-5)) / 2e-5) < 1e-4


def test_sampled_actions_start_with_a_ratio_of_one(learn):
    """what sample_actions says of an action is what policy_loss finds for it: before any update the surrogate is the mean advantage and nothing is clipped"""
    for dtype in TYPES:
        p, g = policy_inputs(500, 3, dtype, 14)
        gumbel = cuda(-torch.log(-torch.log(torch.rand(500, 3, generator=g).clamp(1e-7, 1 - 1e-6))))
        a = learn.sample_actions(gumbel=gumbel, normal=cuda(torch.randn(500, 2, generator=g).clamp(-3, 3)), **p)
        adv = cuda(torch.randn(500, generator=g))
        out = learn.policy_loss(p["logits"], a.kind, a.log_prob, adv, p["mean"], p["log_std"], a.raw, clip=0.001)
        near(out.surrogate, adv.double().mean(), 4 * 4 * lp_err(8, 3, 60)); assert out.clipped.item() == 0 and abs(out.kl.item()) < 1e-9


# ---- streams, graphs, repetition ------------------------------------------------------------------------------------------------------------

def everything(learn, seed=0, T=70, B=24, C=10):
    """one call of each operator, as closures over their inputs: () -> list of outputs"""
    x, gate, state, reset, dh, dlast = memory_inputs(T, (B,), C, torch.bfloat16, seed, "some")
    reward, value, nxt, term, trunc, final = rollout(T, B, torch.float32, seed, 0.1, 0.1)
    p = loss_inputs(300, 9, torch.float32, seed, True, False, 0.3, True, True)
    s, g = policy_inputs(300, 9, torch.float32, seed)
    gumbel = cuda(torch.randn(300, 9, generator=g))
    data = [x, gate, state, reward, value, s["logits"], gumbel]

    def memory():
        leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
        h, last = learn.gated_recurrence(*leaves, reset)
        return [h.detach(), last.detach()] + list(torch.autograd.grad((h, last), leaves, (dh, dlast))) + list(learn.recurrence_step(x[0], gate[0], state, reset[0]))

    def adv():
        return list(learn.advantages(reward, value, nxt, term, trunc, final))

    def sample():
        return list(learn.sample_actions(gumbel=gumbel, **s))

    def loss():
        leaves = [p[n].detach().requires_grad_() for n in ("logits", "mean", "log_std")]
        out = learn.policy_loss(**dict(p, logits=leaves[0], mean=leaves[1], log_std=leaves[2]), kl_coef=0.1, entropy_coef=0.01)
        return [t.detach() for t in out] + list(torch.autograd.grad(out.loss, leaves))

    return dict(memory=memory, adv=adv, sample=sample, loss=loss), data


@pytest.mark.parametrize("name", ["memory", "adv", "sample", "loss"])
def test_same_bits_again_and_on_another_stream(learn, name):
    ops, _ = everything(learn)
    first = [t.clone() for t in ops[name]()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops[name]()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, ops[name]())) and all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.parametrize("name", ["memory", "adv", "sample", "loss"])
def test_captured_and_replayed(learn, name):
    """two graphs of the same call, replayed in turn with new inputs and eager calls between the replays"""
    ops, data = everything(learn)
    ops[name]()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops[name]())
        graphs.append(graph)
    for i in range(5):
        for t in data:
            t.mul_(0.9)
        want = [t.clone() for t in ops[name]()]
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs[i % 2])), i
        both = [t.clone() for t in outs[i % 2]]
        graphs[1 - i % 2].replay(); graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(both, outs[i % 2])) and all(torch.equal(a, b) for a, b in zip(both, outs[1 - i % 2]))


def training(learn, name):
    """a leaf and a training pass over it that leaves the gradient in leaf.grad: () -> the loss"""
    if name == "memory":
        x, gate, state, reset, dh, _ = memory_inputs(20, (6,), 5, torch.float32, 3, "some")
        leaf = x.requires_grad_()
        return leaf, lambda: (learn.gated_recurrence(leaf * 2, gate, state, reset)[0] * dh).sum()
    p = loss_inputs(40, 5, torch.float32, 3, True, False, 0.3, True, True)
    leaf = p["logits"].detach().requires_grad_()
    return leaf, lambda: learn.policy_loss(**dict(p, logits=leaf), kl_coef=0.1).loss


@pytest.mark.parametrize("name", ["memory", "loss"])
def test_capture_of_a_backward_pass_beside_an_eager_graph(learn, name):
    """a leaf's node belongs to the stream of the graph that is alive: the capture refuses the call, and takes it once that graph is gone"""
    leaf, run = training(learn, name)
    want = torch.autograd.grad(run(), leaf)[0]
    alive = run()
    torch.cuda.synchronize()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        dummy = torch.zeros(4, device="cuda")
        with pytest.raises(ValueError, match="another stream"):
            run()
    assert dummy is not None
    alive.backward()                                   # (the eager graph is as it was)
    assert torch.equal(leaf.grad, want)
    del alive
    gc.collect()
    leaf.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run().backward()
    for _ in range(3):
        leaf.grad.fill_(7)                             # (the captured pass writes leaf.grad: it was None when it was captured)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad, want)


def test_calls_from_several_threads_at_once(learn):
    """every thread with a stream of its own, all calling all operators at the same time"""
    import threading
    jobs = [everything(learn, seed=s)[0] for s in range(4)]
    want = [{n: [t.clone() for t in op()] for n, op in job.items()} for job in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                for n, op in jobs[i].items():
                    got = [t.clone() for t in op()]
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i][n])):
                        wrong.append((i, n))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_views_that_negate(learn):
    """the imaginary part of a conjugate lies in memory with the other sign"""
    base = torch.randn(20, 6, 1, dtype=torch.complex64, generator=rng(1)).cuda()
    x = base.conj().imag
    assert x.is_neg()
    gate = torch.randn(20, 6, 1, generator=rng(2)).cuda()
    got, want = learn.gated_recurrence(x, gate), learn.gated_recurrence(x.clone(), gate)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- long arrays --------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
def test_steps_that_lie_far_apart(learn, dtype):
    """20 steps of few columns, 256 MB apart: more than the 32 bits of an offset hold"""
    T, B, C = 20, 3, 40

    def apart(t):
        step = (1 << 28) // t.element_size()
        size = t[0].numel()
        out = torch.empty((T - 1) * step + size, dtype=t.dtype, device="cuda").as_strided(t.shape, (step,) + t[0].stride())
        return out.copy_(t)

    x, gate, state, reset, dh, dlast = memory_inputs(T, (B,), C, dtype, 5, "some")
    leaves = [apart(x).requires_grad_(), gate.clone().requires_grad_(), state.clone().requires_grad_()]
    h, last = learn.gated_recurrence(*leaves, apart(reset))
    want = F.recurrence(x, gate, state, reset)
    hb, gb, gateb = memory_bounds(4.0, 4.0, T)
    near(h, want[0], hb, "h"); near(last, want[1], hb, "last")
    got = torch.autograd.grad((h, last), leaves, (apart(dh), dlast))
    for g, w, bound, name in zip(got, F.recurrence_grads(x, gate, state, reset, dh, dlast), (gb, gateb, gb), ("dx", "dgate", "dstate")):
        near(g, w, bound, name)
    r, v, nxt, term, trunc, final = rollout(T, B, dtype, 5, 0.1, 0.1)
    got = learn.advantages(r, apart(v), nxt, apart(term), trunc, apart(final))
    want = F.advantages(*(t.cpu() for t in (r, v, nxt, term, trunc, final)), float(torch.tensor(0.99)), float(torch.tensor(0.95)))
    near(got.advantage, want[0], adv_bound(T, 0.99 * 0.95), "advantage"); near(got.returns, want[1], adv_bound(T, 0.99 * 0.95) + 20 * E, "returns")


def test_arrays_beyond_32_bits_of_elements(learn):
    """more than 2^31 elements and 4 GB in every array of a rollout, an odd number of columns.  Against the formulas in torch's float32: both are off by less than 1e-4"""
    T, B, C = 9, 53687093, 5                           # 268435465 columns
    x = torch.empty(T, B, C, dtype=torch.bfloat16, device="cuda").normal_()
    gate = torch.empty_like(x).normal_()
    reset = torch.empty(T, B, device="cuda").uniform_() < 0.1
    h, last = learn.gated_recurrence(x.requires_grad_(), gate.requires_grad_(), None, reset)
    dlast = torch.ones_like(last)
    dx, dgate = torch.autograd.grad(last, (x, gate), dlast)
    off = lambda got, want: ((got.float() - want).abs() - want.abs() * torch.finfo(torch.bfloat16).eps / 2).max().item()      # noqa: E731
    with torch.no_grad():
        s, seen = torch.zeros(B, C, device="cuda"), []
        for t in range(T):
            f = torch.sigmoid(gate[t].float())
            seen.append(torch.where(reset[t][:, None], 0, s))
            s = f * seen[t] + (1 - f) * x[t].float()
            assert off(h[t], s) < 1e-4, t
        assert (last - s).abs().max().item() < 1e-4
        G = dlast
        for t in reversed(range(T)):
            f = torch.sigmoid(gate[t].float())
            assert off(dx[t], (1 - f) * G) < 1e-4 and off(dgate[t], G * (seen[t] - x[t].float()) * f * (1 - f)) < 1e-4, t
            G = torch.where(reset[t][:, None], 0, f * G)
    del x, gate, h, last, dx, dgate, s, f, G, seen
    torch.cuda.empty_cache()


def test_logits_beyond_32_bits_of_elements(learn):
    R, V = 66000, 65543
    z = torch.empty(R, V, dtype=torch.bfloat16, device="cuda")
    z.normal_()
    z.requires_grad_()
    zeros = torch.zeros(R, device="cuda")
    weight = zeros.clone()
    weight[-5:] = 1
    kind = torch.full((R,), V - 1, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        a = learn.sample_actions(z)
        old = a.log_prob
        assert torch.equal(a.kind[-50:], torch.stack([(row == row.max()).nonzero()[0, 0] for row in z[-50:].float()]).int())
        lp = torch.log_softmax(d(z[-5:]), -1)
        near(old[-5:], lp.max(-1).values, lp_err(16.0, V))
    out = learn.policy_loss(z, kind, torch.cat([zeros[:-5], lp[:, -1].float().cuda()]), torch.ones(R, device="cuda"), weight=weight)
    (dz,) = torch.autograd.grad(out.loss, z)
    want = (lp.exp() - torch.eye(V, dtype=torch.float64)[V - 1]) / 5
    near(dz[-5:], want, 0.2 * 2 * lp_err(16.0, V))      # (the ratio and a probability are each off by as much)
    assert dz[:-5].count_nonzero().item() == 0
    del z, dz, out
    torch.cuda.empty_cache()


def test_the_rollout_example_learns_from_its_rollouts(learn):
    """examples/vector_rollout.py --learn runs to its end: acting, advantages, loss and an update, twice (what it computes is the next test's)"""
    import os
    import subprocess
    import sys
    from conftest import ROOT
    p = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "vector_rollout.py"), "--learn", "--updates", "2", "--envs", "256", "--steps", "40", "--number-steps", "15"],
                       capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr[-2000:]
    lines = [l for l in p.stdout.splitlines() if l.startswith("update ")]
    assert len(lines) == 2 and "nan" not in p.stdout and "clipped 0.000" in lines[0]        # (the first update looks at the policy that acted)


# ---- a run of them together ---------------------------------------------------------------------------------------------------------------------

def test_act_collect_and_learn_on_the_env(learn):
    """the loop of the module's text on AgarioVectorEnv, several episodes long: what was remembered while acting is what the rollout's recurrence
    remembers, the log-probabilities are the loss's, and the gradients are the definition's"""
    from agarcl_amd.vector_env import AgarioVectorEnv
    N, T, C = 24, 40, 16
    venv = AgarioVectorEnv(N, obs_type="ram", arena_size=200, num_pellets=300, num_viruses=4, number_steps=9)
    D = venv.single_observation_shape[-1]
    g = torch.Generator(device="cuda"); g.manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")                          # noqa: E731
    w_x, w_g, w_z, w_m, w_v = rand(D, C) * 0.02, rand(D, C) * 0.02, rand(C, 3) * 0.5, rand(C, 2) * 0.5, rand(C) * 0.5
    log_std = torch.full((2,), -0.5, device="cuda")
    gumbel, normal = -torch.log(-torch.log(torch.rand((T, N, 3), generator=g, device="cuda").clamp(1e-7, 1 - 1e-6))), rand(T, N, 2)
    obs, _ = venv.reset(seed=3)
    state, ended, buf = torch.zeros(N, C, device="cuda"), None, {k: [] for k in "obs reset h kind raw lp reward term trunc value".split()}
    with torch.no_grad():
        for t in range(T):
            o = torch.tanh(obs * 0.05)
            h, state = learn.recurrence_step(o @ w_x, o @ w_g, state, ended)
            a = learn.sample_actions(h @ w_z, h @ w_m, log_std, gumbel=gumbel[t], normal=normal[t])
            buf["obs"].append(o); buf["reset"].append(torch.zeros(N, dtype=torch.bool, device="cuda") if ended is None else ended)
            for k, v in (("h", h), ("kind", a.kind), ("raw", a.raw), ("lp", a.log_prob), ("value", h @ w_v)):
                buf[k].append(v)
            obs, reward, term, trunc, info = venv.step(a)
            ended = info["ended"].clone()
            for k, v in (("reward", reward), ("term", term), ("trunc", trunc)):
                buf[k].append(v.clone())
        b = {k: torch.stack(v) for k, v in buf.items()}
        assert b["reset"].sum() >= 3 * N and b["term"].any()          # (an episode of number_steps = 9 ends with its tenth step)
        adv, ret = learn.advantages(b["reward"], b["value"], state @ w_v, b["term"], b["trunc"])
    leaves = [t.clone().requires_grad_() for t in (w_x, w_g, w_z, w_m, log_std)]
    h, _ = learn.gated_recurrence(b["obs"] @ leaves[0], b["obs"] @ leaves[1], None, b["reset"])
    near(h.detach(), d(b["h"]), 2e-4)                                                     # (other products: torch's matmul over T x N rows and over N)
    out = learn.policy_loss(h @ leaves[2], b["kind"], b["lp"], adv, h @ leaves[3], leaves[4], b["raw"], clip=0.2, kl_coef=0.05, entropy_coef=0.01)
    assert out.clipped.item() == 0 and abs(out.kl.item()) < 1e-7
    got = torch.autograd.grad(out.loss, leaves)
    q = [d(t).requires_grad_() for t in leaves]
    want_adv, want_ret = F.advantages(*(b[k].cpu() for k in ("reward", "value")), d(state @ w_v), b["term"].cpu(), b["trunc"].cpu(), None, float(torch.tensor(0.99)), float(torch.tensor(0.95)))
    near(adv, want_adv, 1e-4); near(ret, want_ret, 1e-4)
    hh = torch.zeros(N, C, dtype=torch.float64); hs = []
    for t in range(T):
        p = torch.where(b["reset"][t].cpu()[:, None], torch.zeros_like(hh), hh)
        f = torch.sigmoid(d(b["obs"][t]) @ q[1])
        hh = f * p + (1 - f) * (d(b["obs"][t]) @ q[0]); hs.append(hh)
    hs = torch.stack(hs).view(T * N, C)
    loss, _ = F.policy_loss(hs @ q[2], b["kind"].cpu().flatten(), d(b["lp"]).flatten(), d(adv).flatten(), hs @ q[3], q[4], d(b["raw"]).view(-1, 2), kl_coef=0.05, entropy_coef=0.01)
    want = torch.autograd.grad(loss, q)
    for a, w in zip(got, want):      # sums of 960 rows' terms over chains of up to 9 steps, in 32 bits with torch's own products around: 960 x 9 x 6 roundings of 6e-8, at worst
        assert ((d(a) - w).norm() / w.norm()) < 3e-3
    venv.close()
