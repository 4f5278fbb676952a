"""What agarcl_amd.learn and include/agarcl_learn.h refuse -- on any machine: every check of an argument comes before the first GPU call."""
import ctypes
import os
import re

import pytest
import torch

from agarcl_amd import _capi, build
from conftest import ROOT

if not os.path.exists(_capi.HIP_SO):
    build.build()
if not os.path.exists(build.learn_torch_out()):
    build.build_learn_torch()
from agarcl_amd import learn  # noqa: E402

f32, bf16 = torch.float32, torch.bfloat16
z = torch.zeros


@pytest.fixture(scope="module")
def lib():
    return _capi.hip_lib()


def test_header_and_binding_agree(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "agarcl_learn.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(agarcl_[a-z_0-9]+)\s*\(", src)))
    assert names == sorted(n for n, _, _ in _capi.LEARN_SYMBOLS)
    for name in names:
        assert hasattr(lib, name), name
    sizes = {"int64_t": 8, "int32_t": 4, "float": 4}
    for cname, cls in (("agarcl_recurrence_args", _capi.RecurrenceArgs), ("agarcl_advantages_args", _capi.AdvantagesArgs), ("agarcl_sample_args", _capi.SampleArgs),
                       ("agarcl_policy_loss_args", _capi.PolicyLossArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), src, flags=re.S).group(1)
        fields = []
        for decl in re.findall(r"([^;{}]+);", body):
            base = decl.replace("const ", "").split()[0]
            for part in decl.replace("const ", "").strip()[len(base):].split(","):
                fields.append((part.strip().lstrip("*").strip(), 8 if "*" in part else sizes[base]))
        assert fields == [(n, ctypes.sizeof(t)) for n, t in cls._fields_], cname


T, B, C = 3, 2, 4
GOOD = {
    "gated_recurrence": dict(x=z(T, B, C), gate=z(T, B, C), state=z(B, C), reset=z(T, B, dtype=torch.bool)),
    "recurrence_step": dict(x=z(B, C), gate=z(B, C), state=z(B, C), reset=z(B, dtype=torch.bool)),
    "advantages": dict(reward=z(T, B), value=z(T, B), next_value=z(B), terminated=z(T, B, dtype=torch.bool), truncated=z(T, B, dtype=torch.bool), final_value=z(T, B)),
    "sample_actions": dict(logits=z(B, C), mean=z(B, 2), log_std=z(2), gumbel=z(B, C), normal=z(B, 2), allowed=z(B, C, dtype=torch.bool)),
    "policy_loss": dict(logits=z(B, C), kind=z(B, dtype=torch.int32), old_log_prob=z(B), advantage=z(B), mean=z(B, 2), log_std=z(2), move=z(B, 2), ref_log_prob=z(B),
                        allowed=z(B, C, dtype=torch.bool), weight=z(B)),
}


@pytest.mark.parametrize("name", sorted(GOOD))
def test_good_arguments_reach_the_device_check(name):
    with pytest.raises(ValueError, match="GPU"):
        getattr(learn, name)(**GOOD[name])


def grad(*shape, dtype=f32):
    return torch.zeros(*shape, dtype=dtype, requires_grad=True)


BAD = [
    ("gated_recurrence", dict(x=z(T, B, C, dtype=torch.float64)), "x must be a float32"),
    ("gated_recurrence", dict(x=[[1.0]]), "x must be a float32"),
    ("gated_recurrence", dict(x=z(C)), "T, "),
    ("gated_recurrence", dict(gate=z(T, B, C, dtype=bf16)), "gate"),
    ("gated_recurrence", dict(gate=z(T, B, C + 1)), "gate"),
    ("gated_recurrence", dict(state=z(B, C, dtype=bf16)), "state"),
    ("gated_recurrence", dict(state=z(C)), "state"),
    ("gated_recurrence", dict(reset=z(T, B)), "reset"),
    ("gated_recurrence", dict(reset=z(T, B, C, dtype=torch.bool)), "reset"),
    ("gated_recurrence", dict(gate=z(T, B, C, device="meta")), "gate must live on"),
    ("recurrence_step", dict(x=z(())), "rows"),
    ("recurrence_step", dict(state=None), "state"),
    ("recurrence_step", dict(x=grad(B, C)), "x is taken as a constant"),
    ("recurrence_step", dict(reset=z(B, C, dtype=torch.bool)), "reset"),
    ("advantages", dict(value=z(T, B, dtype=torch.int32)), "value"),
    ("advantages", dict(value=z(())), "value"),
    ("advantages", dict(value=grad(T, B)), "value is taken as a constant"),
    ("advantages", dict(reward=z(T, B, dtype=torch.float64)), "reward"),
    ("advantages", dict(next_value=z(T, B)), "next_value"),
    ("advantages", dict(next_value=z(B, dtype=bf16)), "next_value"),
    ("advantages", dict(terminated=z(T, B)), "terminated"),
    ("advantages", dict(truncated=None), "final_value without truncated"),
    ("advantages", dict(final_value=z(B)), "final_value"),
    ("advantages", dict(gamma=1.5), "gamma"),
    ("advantages", dict(lam=float("nan")), "gamma"),
    ("sample_actions", dict(logits=z(B, 0), gumbel=None, allowed=None), "at least one kind"),
    ("sample_actions", dict(logits=z(())), "at least one kind"),
    ("sample_actions", dict(logits=grad(B, C)), "logits is taken as a constant"),
    ("sample_actions", dict(mean=None, normal=None), "belong together"),
    ("sample_actions", dict(log_std=None), "belong together"),
    ("sample_actions", dict(mean=None, log_std=None), "normal without mean"),
    ("sample_actions", dict(mean=z(B, 3)), "mean"),
    ("sample_actions", dict(mean=z(B, 2, dtype=bf16)), "mean"),
    ("sample_actions", dict(log_std=z(2, dtype=bf16)), "log_std"),
    ("sample_actions", dict(log_std=z(3)), "log_std"),
    ("sample_actions", dict(log_std=0.5), "log_std"),
    ("sample_actions", dict(gumbel=z(B)), "gumbel"),
    ("sample_actions", dict(gumbel=z(B, C, dtype=bf16)), "gumbel"),
    ("sample_actions", dict(normal=z(B, 3)), "normal"),
    ("sample_actions", dict(allowed=z(C, dtype=torch.bool)), "allowed"),
    ("policy_loss", dict(kind=z(B)), "kind"),
    ("policy_loss", dict(kind=z(B, 1, dtype=torch.int32)), "kind"),
    ("policy_loss", dict(old_log_prob=z(B, 1)), "old_log_prob"),
    ("policy_loss", dict(advantage=grad(B)), "advantage is taken as a constant"),
    ("policy_loss", dict(old_log_prob=grad(B)), "old_log_prob is taken as a constant"),
    ("policy_loss", dict(move=None), "mean and move"),
    ("policy_loss", dict(mean=None, log_std=None), "mean and move"),
    ("policy_loss", dict(weight=z(B, dtype=torch.int32)), "weight"),
    ("policy_loss", dict(ref_log_prob=z(B, dtype=bf16)), "ref_log_prob"),
    ("policy_loss", dict(clip=-0.1), "clip"),
    ("policy_loss", dict(clip=(0.1, float("nan"))), "clip"),
    ("policy_loss", dict(kl_coef=float("inf")), "finite"),
    ("policy_loss", dict(entropy_coef=float("nan")), "finite"),
    ("policy_loss", dict(reduction="none"), "reduction"),
]


@pytest.mark.parametrize("name,change,says", BAD, ids=["%s-%s" % (n, "-".join(c)) for n, c, _ in BAD])
def test_refused(name, change, says):
    with pytest.raises(ValueError, match=says):
        getattr(learn, name)(**dict(GOOD[name], **change))


# the C entries, with pointers that are never followed: 64 stands for a device address
def rec(**kw):
    return _capi.RecurrenceArgs(**dict(dict(steps=4, rows=2, width=3, x=64, gate=64, x_stride=6, gate_stride=6, h=64, last=64, marks=64, dx=64, dgate=64, dstate=64, work=64), **kw))


def adv(**kw):
    return _capi.AdvantagesArgs(**dict(dict(steps=4, rows=2, reward=64, value=64, next_value=64, terminated=64, reward_stride=2, value_stride=2, terminated_stride=2, gamma=0.9,
                                            advantage=64, returns=64, work=64), **{"lambda": 0.9}, **kw))


def sam(**kw):
    return _capi.SampleArgs(**dict(dict(rows=4, kinds=3, logits=64, logits_stride=3, kind=64, log_prob=64), **kw))


def los(**kw):
    return _capi.PolicyLossArgs(**dict(dict(rows=4, kinds=3, logits=64, logits_stride=3, kind=64, old_log_prob=64, advantage=64, clip_low=0.2, clip_high=0.2, want_stats=1, loss=64,
                                            stats=64, work=64), **kw))


C_BAD = [
    ("agarcl_recurrence", rec(dtype=3)), ("agarcl_recurrence", rec(steps=-1)), ("agarcl_recurrence", rec(rows=1 << 39, width=1 << 39)), ("agarcl_recurrence", rec(x=None)),
    ("agarcl_recurrence", rec(x_stride=5)), ("agarcl_recurrence", rec(gate_stride=-6)), ("agarcl_recurrence", rec(reset=64, reset_stride=1)), ("agarcl_recurrence", rec(h=None)),
    ("agarcl_recurrence", rec(steps=0, rows=1 << 39, width=1 << 39)), ("agarcl_recurrence", rec(last=None)), ("agarcl_recurrence", rec(x_stride=1 << 62)),
    ("agarcl_recurrence_grad", rec(marks=None)), ("agarcl_recurrence_grad", rec(dx=None)), ("agarcl_recurrence_grad", rec(dstate=None)), ("agarcl_recurrence_grad", rec(dh=64, dh_stride=1)),
    ("agarcl_advantages", adv(dtype=-1)), ("agarcl_advantages", adv(gamma=2.0)), ("agarcl_advantages", adv(gamma=float("nan"))), ("agarcl_advantages", adv(returns=None)),
    ("agarcl_advantages", adv(final_value=64, final_stride=2)), ("agarcl_advantages", adv(truncated=64, truncated_stride=1)), ("agarcl_advantages", adv(value_stride=1)),
    ("agarcl_sample_actions", sam(kinds=0)), ("agarcl_sample_actions", sam(kinds=1 << 31)), ("agarcl_sample_actions", sam(rows=-1)), ("agarcl_sample_actions", sam(logits=None)),
    ("agarcl_sample_actions", sam(logits_stride=2)), ("agarcl_sample_actions", sam(allowed=64, allowed_stride=1)), ("agarcl_sample_actions", sam(gumbel=64, gumbel_stride=1)),
    ("agarcl_sample_actions", sam(kind=None)), ("agarcl_sample_actions", sam(mean=64, log_std=64)), ("agarcl_sample_actions", sam(normal=64)),
    ("agarcl_policy_loss", los(clip_low=-1.0)), ("agarcl_policy_loss", los(clip_high=float("nan"))), ("agarcl_policy_loss", los(kl_coef=float("inf"))), ("agarcl_policy_loss", los(loss=None)),
    ("agarcl_policy_loss", los(work=None)), ("agarcl_policy_loss", los(kind=None)), ("agarcl_policy_loss", los(mean=64)), ("agarcl_policy_loss", los(dmean=64)),
    ("agarcl_policy_loss", los(skip_if_one=1)), ("agarcl_policy_loss", los(want_stats=0, mean=64, log_std=64, move=64, dlog_std=64)),
    ("agarcl_policy_loss", los(want_stats=0, weight=64, mean_over_weight=1, dlogits=64, work=None)),
]


@pytest.mark.parametrize("i", range(len(C_BAD)), ids=["%s-%d" % (n, i) for i, (n, _) in enumerate(C_BAD)])
def test_c_entry_refuses(lib, i):
    name, args = C_BAD[i]
    assert getattr(lib, name)(ctypes.byref(args)) == -1
    assert lib.agarcl_learn_error()


def test_c_entries_refuse_null_and_fail_loudly_without_a_gpu(lib):
    for name in ("agarcl_recurrence", "agarcl_recurrence_grad", "agarcl_advantages", "agarcl_sample_actions", "agarcl_policy_loss"):
        assert getattr(lib, name)(None) == -1
    assert lib.agarcl_recurrence_work(-1, 1, 1) == -1 and lib.agarcl_recurrence_work(1 << 30, 1 << 30, 1) == -1 and lib.agarcl_advantages_work(1, -1) == -1
    if not torch.cuda.is_available():
        for name, args in (("agarcl_recurrence", rec()), ("agarcl_recurrence_grad", rec()), ("agarcl_advantages", adv()), ("agarcl_sample_actions", sam()), ("agarcl_policy_loss", los())):
            assert getattr(lib, name)(ctypes.byref(args)) == -4, name


def test_nothing_to_do_is_no_error(lib):
    assert lib.agarcl_recurrence_work(0, 3, 4) == lib.agarcl_recurrence_work(3, 0, 4) == lib.agarcl_recurrence_work(3, 4, 0) == lib.agarcl_advantages_work(0, 5) == 0
    assert all(lib.agarcl_recurrence_work(t, b, c) >= 0 for t in (1, 8, 9, 100, 30000) for b in (1, 3, 5000) for c in (1, 2, 7, 256))
    for name, args in (("agarcl_recurrence", rec(rows=0)), ("agarcl_recurrence_grad", rec(width=0)), ("agarcl_advantages", adv(steps=0)), ("agarcl_sample_actions", sam(rows=0))):
        assert getattr(lib, name)(ctypes.byref(args)) == 0, name


@pytest.mark.parametrize("name,arg", [("gated_recurrence", "gate"), ("recurrence_step", "x"), ("advantages", "value"), ("policy_loss", "logits"), ("policy_loss", "mean")])
def test_forward_mode_gradients_are_refused(name, arg):
    with torch.autograd.forward_ad.dual_level():
        args = dict(GOOD[name])
        args[arg] = torch.autograd.forward_ad.make_dual(args[arg].clone(), torch.ones_like(args[arg]))
        with pytest.raises(ValueError, match=arg + " carries a forward-mode gradient"):
            getattr(learn, name)(**args)
