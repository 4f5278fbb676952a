"""agarcl_amd.learn on the GPU where an error would hide: policies that are NaN, small forget factors, upstream gradients that are not plain numbers in memory, what becomes
of the outputs afterwards.  Tolerances in units of E = 2^-24, on top of those of test_learn_ops.py."""
import ctypes
import io

import pytest
import torch

import learn_formulas as F
from learn_formulas import E, d, near

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
KINDS = [1, 3, 8, 9, 63, 500, 1000, 1300, 1800, 2049, 5001, 7001, 9000]      # every kernel of the loss and of sampling
nan, inf = float("nan"), float("inf")


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


# ---- policies that are NaN ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", KINDS)
def test_a_nan_logit_shows_in_the_loss(learn, V, dtype):
    R = 12
    for A in (1.5, -1.5, 0.0):
        for at in {V // 2, V - 1}:                           # the row's own kind, and another one
            z = torch.randn(R, V, generator=rng(V)).to("cuda", dtype)
            kind = torch.full((R,), V // 2, dtype=torch.int32, device="cuda")
            old, adv = torch.full((R,), -1.0, device="cuda"), torch.ones(R, device="cuda")
            z[7, at], adv[7] = nan, A
            leaf = z.clone().requires_grad_()
            out = learn.policy_loss(leaf, kind, old, adv)
            (dz,) = torch.autograd.grad(out.loss, leaf)
            assert out.loss.isnan() and out.surrogate.isnan() and out.kl.isnan() and out.entropy.isnan(), (A, at)
            assert torch.isfinite(torch.cat((dz[:7], dz[8:]))).all()
            weight = torch.ones(R, device="cuda")
            weight[7] = 0                                    # a row that is left out is not looked at
            assert all(torch.isfinite(t) for t in learn.policy_loss(z, kind, old, adv, weight=weight))
            allowed = torch.ones(R, V, dtype=torch.bool, device="cuda")
            allowed[7, at] = False                           # nor is a kind that is not allowed
            assert all(torch.isfinite(t) for t in learn.policy_loss(z, kind, old, adv, allowed=allowed))


@pytest.mark.parametrize("what", ["mean", "log_std", "move", "old_log_prob"])
def test_any_nan_shows_in_the_loss(learn, what):
    for A in (2.0, -2.0, 0.0):
        p = dict(logits=torch.zeros(9, 3), kind=torch.zeros(9, dtype=torch.int32), old_log_prob=torch.full((9,), -3.0), advantage=torch.full((9,), A), mean=torch.zeros(9, 2),
                 log_std=torch.zeros(9, 2), move=torch.zeros(9, 2))
        p[what][4 if p[what].dim() == 1 else (4, 1)] = nan
        out = learn.policy_loss(**{k: t.cuda() for k, t in p.items()})
        assert out.loss.isnan() and out.surrogate.isnan(), A


def test_infinite_ratios_are_still_clipped(learn):
    """a ratio that overflows: clipped where that is the lesser, and nothing of it with an advantage of 0"""
    z, kind, old = torch.zeros(1, 1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), -200.0, device="cuda")
    for A, want in ((1.0, -1.2), (-1.0, inf), (0.0, 0.0)):
        leaf = z.clone().requires_grad_()
        out = learn.policy_loss(leaf, kind, old, torch.full((1,), A, device="cuda"))
        assert out.loss.item() == torch.tensor(want).item()


@pytest.mark.parametrize("V", [3, 24, 5000])
@pytest.mark.parametrize("what", ["mean", "log_std", "normal"])
def test_a_nan_move_is_not_a_move(learn, V, what):
    p = dict(logits=torch.randn(9, V, generator=rng(V)), mean=torch.randn(9, 2, generator=rng(1)) * 2, log_std=torch.zeros(9, 2), normal=torch.randn(9, 2, generator=rng(2)))
    good = learn.sample_actions(**{k: t.cuda() for k, t in p.items()})
    p[what][4, 1] = nan
    a = learn.sample_actions(**{k: t.cuda() for k, t in p.items()})
    assert a.raw[4, 1].isnan() and a.move[4, 1].isnan() and a.log_prob[4].isnan()
    assert torch.equal(a.move[4, 0], good.move[4, 0]) and torch.equal(a.kind, good.kind)
    rest = [i for i in range(9) if i != 4]
    assert all(torch.equal(s[rest], t[rest]) for s, t in zip(a, good))
    p["mean"], p["log_std"], p["normal"] = torch.tensor([[inf, -inf]]).repeat(9, 1), torch.zeros(9, 2), torch.zeros(9, 2)
    assert learn.sample_actions(**{k: t.cuda() for k, t in p.items()}).move.tolist() == [[1.0, -1.0]] * 9


# ---- small forget factors -------------------------------------------------------------------------------------------------------------------------
# All gradients that come in are >= 0, so no sum cancels: every step a gradient crosses multiplies it by f, relative error (6 + 1.5 G) E with G = 16, and adds the next, 3 E more: 33 E.
# Every 21 steps a gradient comes in anew, and what is older has crossed three factors of e^-8 or less since: it is not seen beside it.  So a total gradient has crossed at most 21
# steps with its own step's, 22 x 33 E, and the joins' 64 E of any length: 790 E, relative.  dx multiplies by 1 - f (30 E + 1 rounding), dgate by f, 1 - f and p - x; p is good to
# (12 + 3 G + 64 + 3 / min(1 - f)) E <= 150 E (gates are 2 at most) with x <= 1.

def small_factors(T, rows, C, dtype, dh_too):
    g = rng(T + C)
    t, c = torch.arange(T)[:, None], torch.arange(C)[None]
    gate = torch.where((t + c // 5) % 7 == 3, -(8.0 + 2 * (c % 5)), torch.full((), 2.0))
    gate = gate[:, None, :].expand(T, rows, C).contiguous()
    x = ((torch.rand(T, rows, C, generator=g) + 1) / 2) * torch.where(torch.rand(T, rows, C, generator=g) < 0.5, -1.0, 1.0)
    dh = torch.zeros(T, rows, C)
    if dh_too:
        dh[T % 21::21] = torch.rand(dh[T % 21::21].shape, generator=g) + 0.5
    return x.to(dtype), gate.to(dtype), torch.rand(rows, C, generator=g), dh.to(dtype), torch.rand(rows, C, generator=g) + 0.5


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("C", [35, 70])
@pytest.mark.parametrize("T,rows,resets", [(5, 1, False), (13, 3, False), (21, 1, True), (7, 2000, False), (20, 4000, True), (2003, 1, False), (3001, 2, True)])
def test_gradients_through_small_forget_factors(learn, T, rows, C, resets, dtype):
    x, gate, state, dh, dlast = (t.cuda() for t in small_factors(T, rows, C, dtype, T > 21))
    reset = None
    if resets:
        reset = torch.zeros(T, rows, dtype=torch.bool)
        reset[T // 2::10] = True
        reset = reset.cuda()
    leaves = [t.clone().requires_grad_() for t in (x, gate, state)]
    h, last = learn.gated_recurrence(*leaves, reset)
    dx, dgate, dstate = torch.autograd.grad((h, last), leaves, (dh, dlast))
    x, gate, G, dh = d(x), d(gate), d(dlast), d(dh)
    f, q = torch.sigmoid(gate), torch.sigmoid(-gate)
    seen, s = [], d(state)
    for t in range(T):
        p = s if reset is None else torch.where(F.flags(reset)[t][:, None], 0.0, s)
        seen.append(p)
        s = f[t] * p + q[t] * x[t]
    want = [torch.empty_like(x), torch.empty_like(x)]
    room = torch.empty_like(x)
    for t in range(T - 1, -1, -1):
        G = G + dh[t]
        want[0][t], want[1][t] = q[t] * G, G * (seen[t] - x[t]) * f[t] * q[t]
        room[t] = G * f[t] * q[t] * ((seen[t] - x[t]).abs() * 860 + 160) * E
        G = f[t] * G
        if reset is not None:
            G = torch.where(F.flags(reset)[t][:, None], 0.0, G)
    near(dx, want[0], want[0] * 830 * E, "dx")
    near(dgate, want[1], room, "dgate")
    near(dstate, G, G * 800 * E, "dstate")


# ---- the gradient of the loss itself ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("per_row", [0, 1])
@pytest.mark.parametrize("weighted", [False, True])
def test_c_entry_multiplies_every_gradient_by_upstream(learn, per_row, weighted):
    """one call for loss and gradients (the autograd node makes two): a power of two as the upstream gradient is exact in all of them"""
    from agarcl_amd import _capi
    lib = _capi.hip_lib()
    R, V, g = 300, 5, rng(4)
    t = dict(logits=torch.randn(R, V, generator=g), mean=torch.randn(R, 2, generator=g), log_std=torch.randn(R, 2, generator=g) * 0.3 if per_row else torch.tensor([-0.5, 0.2]),
             move=torch.randn(R, 2, generator=g), old_log_prob=torch.full((R,), -4.0), advantage=torch.randn(R, generator=g), kind=torch.randint(0, V, (R,), generator=g).int())
    if weighted:
        t["weight"] = torch.rand(R, generator=g)
    t = {k: v.cuda() for k, v in t.items()}
    results = []
    for up in (None, 1.0, 0.25, 1024.0):
        out = dict(loss=torch.zeros(1), stats=torch.zeros(8), dlogits=torch.zeros(R, V), dmean=torch.zeros(R, 2), dlog_std=torch.zeros(R, 2) if per_row else torch.zeros(2))
        out = {k: v.cuda() for k, v in out.items()}
        upstream = None if up is None else torch.tensor([up], device="cuda")
        work = torch.empty(lib.agarcl_policy_loss_work(), dtype=torch.float64, device="cuda")
        a = _capi.PolicyLossArgs(rows=R, kinds=V, dtype=0, device=0, logits_stride=V, log_std_per_row=per_row, mean_over_weight=1, clip_low=0.2, clip_high=0.2, kl_coef=0.1, entropy_coef=0.01,
                                 want_stats=1, work=work.data_ptr(), upstream=None if up is None else upstream.data_ptr(), stream=torch.cuda.current_stream().cuda_stream,
                                 **{k: v.data_ptr() for k, v in dict(t, **out).items()})
        assert lib.agarcl_policy_loss(ctypes.byref(a)) == 0, lib.agarcl_learn_error()
        torch.cuda.synchronize()
        results.append((up or 1.0, out))
    one = results[0][1]
    assert one["dlog_std"].abs().min() > 0
    for up, out in results[1:]:
        assert torch.equal(out["loss"], one["loss"]) and torch.equal(out["stats"], one["stats"])
        for k in ("dlogits", "dmean", "dlog_std"):
            assert torch.equal(out[k], one[k] * up), (k, up)


def loss_call(learn, R=40, V=5):
    g = rng(6)
    t = [torch.randn(R, V, generator=g), torch.randint(0, V, (R,), generator=g).int(), torch.full((R,), -4.0), torch.randn(R, generator=g), torch.randn(R, 2, generator=g), torch.tensor([-0.5, 0.2]),
         torch.randn(R, 2, generator=g)]
    t = [k.cuda() for k in t]
    for i in (0, 4, 5):
        t[i].requires_grad_()
    return [t[0], t[4], t[5]], lambda: learn.policy_loss(*t).loss


def negated(t):
    """t's numbers in a tensor that lies in memory with the other sign"""
    t = torch._neg_view(-t)
    assert t.is_neg()
    return t


def test_an_upstream_gradient_that_negates(learn):
    leaves, loss = loss_call(learn)
    for up in (1.0, 0.5):
        up = torch.tensor(up, device="cuda")
        want = torch.autograd.grad(loss(), leaves, up)
        out = loss()
        for _ in range(2):                                   # the gradients made ahead, and those of a second pass
            got = torch.autograd.grad(out, leaves, negated(up), retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    out = loss()
    through = (torch.complex(torch.zeros_like(out), out).conj() * 1j).real      # = out: autograd hands on a view that negates by itself
    got, want = torch.autograd.grad(through, leaves), torch.autograd.grad(loss(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_an_upstream_gradient_of_the_memory_that_negates(learn):
    g = rng(7)
    x, gate, state, dh, dlast = (torch.randn(*s, generator=g).cuda() for s in ((30, 4, 6), (30, 4, 6), (4, 6), (30, 4, 6), (4, 6)))
    leaves = [t.requires_grad_() for t in (x, gate, state)]
    want = torch.autograd.grad(learn.gated_recurrence(*leaves), leaves, (dh, dlast))
    for a, b in ((negated(dh), dlast), (dh, negated(dlast)), (negated(dh), negated(dlast))):
        got = torch.autograd.grad(learn.gated_recurrence(*leaves), leaves, (a, b))
        assert all(torch.equal(s, t) for s, t in zip(got, want))


# ---- tensors without memory -------------------------------------------------------------------------------------------------------------------------

def zeros_unstored(*shape, dtype=torch.float32):
    """zeros as autograd makes them where it need not store them: their address is null"""
    t = torch._efficientzerotensor(shape, dtype=dtype, device="cuda")
    assert t._is_zerotensor()
    return t


def test_zeros_that_are_not_stored(learn):
    leaves, loss = loss_call(learn)
    for _ in range(2):
        out = loss()
        for _ in range(2):
            got = torch.autograd.grad(out, leaves, zeros_unstored(), retain_graph=True)
            assert all((t == 0).all() for t in got)
    g = rng(8)
    x, gate, state = (torch.randn(*s, generator=g).cuda().requires_grad_() for s in ((9, 4, 6), (9, 4, 6), (4, 6)))
    want = torch.autograd.grad(learn.gated_recurrence(x, gate, state), (x, gate, state), (torch.ones(9, 4, 6, device="cuda"), torch.zeros(4, 6, device="cuda")))
    got = torch.autograd.grad(learn.gated_recurrence(x, gate, state), (x, gate, state), (torch.ones(9, 4, 6, device="cuda"), zeros_unstored(4, 6)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    z, kind, old, adv = torch.randn(9, 3, generator=g).cuda(), torch.zeros(9, dtype=torch.int32, device="cuda"), torch.full((9,), -1.0, device="cuda"), torch.randn(9, generator=g).cuda()
    for name, dtype, shape in (("ref_log_prob", torch.float32, (9,)), ("weight", torch.float32, (9,)), ("allowed", torch.bool, (9, 3))):
        a = learn.policy_loss(z, kind, old, adv, kl_coef=0.1, **{name: zeros_unstored(*shape, dtype=dtype)})
        b = learn.policy_loss(z, kind, old, adv, kl_coef=0.1, **{name: torch.zeros(*shape, dtype=dtype, device="cuda")})
        assert all(torch.equal(s, t) for s, t in zip(a, b)), name
    got = learn.sample_actions(z, allowed=zeros_unstored(9, 3, dtype=torch.bool))
    assert (got.kind == 0).all() and (got.log_prob == 0).all()


class Wrapper(torch.Tensor):
    """a tensor that is a tensor only to Python, as tensor subclasses that hold others are"""
    @staticmethod
    def __new__(cls, like):
        return torch.Tensor._make_wrapper_subclass(cls, like.shape, dtype=like.dtype, device=like.device)

    @classmethod
    def __torch_dispatch__(cls, *args):
        raise AssertionError("nothing is computed with it")


def test_tensors_without_memory_are_refused(learn):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")        # noqa: E731
    loss = dict(logits=z(4, 3), kind=z(4, dtype=torch.int32), old_log_prob=z(4), advantage=z(4), ref_log_prob=z(4), allowed=z(4, 3, dtype=torch.bool), weight=z(4))
    memory = dict(x=z(5, 4, 3), gate=z(5, 4, 3), state=z(4, 3), reset=z(5, 4, dtype=torch.bool))
    rollout = dict(reward=z(5, 4), value=z(5, 4), next_value=z(4), terminated=z(5, 4, dtype=torch.bool), truncated=z(5, 4, dtype=torch.bool), final_value=z(5, 4))
    acting = dict(logits=z(4, 3), gumbel=z(4, 3), allowed=z(4, 3, dtype=torch.bool), mean=z(4, 2), log_std=z(2), normal=z(4, 2))
    for name, args in (("policy_loss", loss), ("gated_recurrence", memory), ("advantages", rollout), ("sample_actions", acting)):
        getattr(learn, name)(**args)
        for k in args:
            with pytest.raises((ValueError, RuntimeError), match="memory of its own"):
                getattr(learn, name)(**dict(args, **{k: Wrapper(args[k])}))


# ---- what becomes of the outputs ----------------------------------------------------------------------------------------------------------------------

def test_actions_are_saved_and_copied_together(learn):
    import copy
    a = learn.sample_actions(torch.randn(50, 3, generator=rng(9)).cuda(), torch.zeros(50, 2, device="cuda"), torch.zeros(2, device="cuda"))
    f = io.BytesIO()
    torch.save(dict(a._asdict()), f)
    f.seek(0)
    back = torch.load(f, weights_only=True)
    assert all(torch.equal(back[k], t) and back[k].dtype == t.dtype for k, t in a._asdict().items())
    twin = copy.deepcopy(dict(a._asdict()))
    assert all(torch.equal(twin[k], t) and twin[k].dtype == t.dtype for k, t in a._asdict().items())
    alone = learn.sample_actions(torch.zeros(4, 3, device="cuda"))
    f = io.BytesIO()
    torch.save([alone.kind, alone.log_prob], f)


# ---- several agents -----------------------------------------------------------------------------------------------------------------------------------

def test_acting_with_several_agents(learn):
    """rows are arenas x agents; info["ended"] is the arenas' and goes to their agents"""
    from agarcl_amd.vector_env import AgarioVectorEnv
    N, n, T, C = 6, 2, 14, 8
    venv = AgarioVectorEnv(N, obs_type="ram", arena_size=200, num_pellets=200, num_viruses=4, num_agents=n, multi_agent=True, number_steps=5)
    D = venv.single_observation_shape[-1]
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    w = [torch.randn(s, generator=g, device="cuda") * 0.05 for s in ((D, C), (D, C), (C, 3), (C, 2), (C,))]
    obs, _ = venv.reset(seed=1)
    state, ended, xs, gs, hs, resets, rew, term, trunc, value = torch.zeros(N, n, C, device="cuda"), torch.zeros(N, dtype=torch.bool, device="cuda"), [], [], [], [], [], [], [], []
    for t in range(T):
        o = torch.tanh(obs * 0.05)
        x, gate, reset = o @ w[0], o @ w[1], ended[:, None].expand(N, n)
        h, state = learn.recurrence_step(x, gate, state, reset)
        a = learn.sample_actions(h @ w[2], h @ w[3], torch.full((2,), -0.5, device="cuda"), normal=torch.randn(N, n, 2, generator=g, device="cuda"))
        assert a.move.shape == (N, n, 2) and a.kind.shape == (N, n)
        obs, reward, terminated, truncated, info = venv.step(a)
        ended = info["ended"].clone()
        for buf, v in ((xs, x), (gs, gate), (hs, h), (resets, reset), (rew, reward), (term, terminated), (trunc, truncated), (value, h @ w[4])):
            buf.append(v.clone())
    assert torch.stack(resets).any()
    h, last = learn.gated_recurrence(torch.stack(xs), torch.stack(gs), None, torch.stack(resets))
    M = max(t.abs().max().item() for t in xs)
    assert max(t.abs().max().item() for t in gs) <= 4          # (what the bound assumes: (12 + 3 G + 64 + 3 T) E M, twice)
    near(h, d(torch.stack(hs)), 2 * (12 + 12 + 64 + 3 * T) * E * M)
    near(last, d(state), 2 * (12 + 12 + 64 + 3 * T) * E * M)
    args = [torch.stack(t) for t in (rew, value)] + [state @ w[4], torch.stack(term), torch.stack(trunc)]
    got = learn.advantages(*args)
    flat = [t.cpu().reshape(t.shape[0], N * n) if t.dim() == 3 else t.cpu().reshape(N * n) for t in args]
    want = F.advantages(*flat, None, float(torch.tensor(0.99)), float(torch.tensor(0.95)))
    top = T * (args[0].abs().max().item() + 2 * args[1].abs().max().item() + args[2].abs().max().item())      # the largest advantage there can be
    near(got.advantage.reshape(T, N * n), want[0], (6 + 2 * T + 64) * E * top)
    venv.close()


# ---- the gradient against differences -----------------------------------------------------------------------------------------------------------------

def test_recurrence_gradient_against_differences(learn):
    """each gradient for itself, along random directions, with room for what the formulas lose and no more: a gradient of 0 is farther off, which is asserted.
    Crossing a step costs a total gradient (6 + 1.5 x 4 + 3) E of the sum of its terms' magnitudes: (21 x 15 + 64) E = 379 E in all (64 E for the joins); dx multiplies by 1 - f,
    dgate by f, 1 - f and p - x (12 E and a rounding each), with p good to (12 + 12 + 64 + 3 x 21) E x 4 = 604 E.  Central differences with steps of 1e-6 in 64 bits: the third derivative
    along v, |v| <= 4, of a product of 21 sigmoids is at most (21 x 4)^3 of the value's magnitude, 500: off by 5e-5; rounding by 1e-6."""
    g = rng(11)
    T, B, C = 21, 4, 6
    x, gate, dh = (torch.randn(T, B, C, generator=g).clamp(-4, 4) for _ in range(3))
    state, dlast = torch.randn(B, C, generator=g), torch.randn(B, C, generator=g)
    reset = torch.rand(T, B, generator=g) < 0.1
    leaves = [t.cuda().requires_grad_() for t in (x, gate, state)]
    got = torch.autograd.grad(learn.gated_recurrence(*leaves, reset.cuda()), leaves, (dh.cuda(), dlast.cuda()))

    def value(at):
        h, last = F.recurrence(*at, reset)
        return (h * d(dh)).sum() + (last * d(dlast)).sum()

    f, q = torch.sigmoid(d(gate)), torch.sigmoid(-d(gate))
    h, _ = F.recurrence(x, gate, state, reset)
    G, off = d(dlast).abs(), [torch.empty_like(f), torch.empty_like(f), None]
    for t in reversed(range(T)):
        G = G + d(dh)[t].abs()
        p = torch.where(reset[t][:, None], 0.0, h[t - 1] if t else d(state))
        off[0][t], off[1][t] = q[t] * G * 392 * E, G * f[t] * q[t] * ((p - d(x)[t]).abs() * 410 + 604) * E
        G = torch.where(reset[t][:, None], 0.0, f[t] * G)
    off[2] = G * 380 * E
    for i, name in enumerate(("dx", "dgate", "dstate")):
        for k in range(3):
            v = torch.randn(leaves[i].shape, generator=g, dtype=torch.float64).clamp(-4, 4)
            shifted = [[d(t) + (s * v if j == i else 0) for j, t in enumerate((x, gate, state))] for s in (1e-6, -1e-6)]
            want = (value(shifted[0]) - value(shifted[1])) / 2e-6
            room = (off[i] * v.abs()).sum() + 1e-4
            assert abs((d(got[i]) * v).sum() - want) < room, (name, k)
            assert abs(want) > room, (name, k, "a gradient of 0 would pass")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("per_row", [False, True])
def test_gradients_of_some_of_the_leaves(learn, per_row, dtype):
    """whatever is differentiated, each gradient is what it is beside the others, for an upstream gradient of 1 and another, the first time and the second"""
    R, V, g = 70, 9, rng(12)
    t = dict(logits=torch.randn(R, V, generator=g).to(dtype), mean=torch.randn(R, 2, generator=g).to(dtype),
             log_std=(torch.randn(R, 2, generator=g) * 0.3).to(dtype) if per_row else torch.tensor([-0.5, 0.2]))
    fixed = dict(kind=torch.randint(-1, V + 1, (R,), generator=g).int(), old_log_prob=torch.full((R,), -4.0), advantage=torch.randn(R, generator=g), move=torch.randn(R, 2, generator=g),
                 weight=torch.rand(R, generator=g))
    t, fixed = ({k: v.cuda() for k, v in s.items()} for s in (t, fixed))
    for up in (1.0, 8.0):
        up = torch.tensor(up, device="cuda")
        results = {}
        for wanted in (("logits", "mean", "log_std"), ("logits",), ("mean",), ("log_std",), ("logits", "log_std"), ("mean", "log_std"), ("logits", "mean")):
            leaves = {k: v.detach().requires_grad_(k in wanted) for k, v in t.items()}
            out = learn.policy_loss(**leaves, **fixed, kl_coef=0.1, entropy_coef=0.01)
            for again in (False, True):
                for k, got in zip(wanted, torch.autograd.grad(out.loss, [leaves[k] for k in wanted], up, retain_graph=True)):
                    want = results.setdefault(k, got)
                    if again:      # (the weights' sum is rounded to 32 bits between the passes, a shared log_std's gradient before it is multiplied)
                        near(got, d(want), d(want).abs() * (4 * E + F.HALF[got.dtype]), k)
                    else:
                        assert torch.equal(got, want), (k, wanted)
