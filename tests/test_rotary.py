"""Rotary plans and refusals (CPU; no kernel runs)."""
import math

import pytest
import torch

from lockstep_b200 import _lib
from lockstep_b200 import rotary as R


def test_frequencies_follow_their_formulas():
    th, m = R.frequencies(8, 10000.0)
    assert m == 1.0 and th == [10000.0 ** (-i / 8) for i in (0, 2, 4, 6)]
    assert R.frequencies(8, 10000.0, {"kind": "linear", "factor": 4.0})[0] == [t / 4 for t in th]
    ntk = R.frequencies(8, 10000.0, {"kind": "ntk", "factor": 3.0})[0]
    # the slowest pair is slowed by the whole factor, the fastest not at all
    assert ntk[0] == 1.0 and math.isclose(ntk[3], th[3] / 3, rel_tol=1e-12)
    th, _ = R.frequencies(128)
    sc = {"kind": "bands", "factor": 32.0, "original": 8192}
    b, m = R.frequencies(128, scaling=sc)
    assert math.isclose(m, 0.1 * math.log(32) + 1)
    for t, x in zip(th, b):
        turns = 8192 * t / (2 * math.pi)
        if turns >= 32:
            assert x == t
        elif turns <= 1:
            assert math.isclose(x, t / 32, rel_tol=1e-15)
        else:
            assert t / 32 < x < t
    assert R.frequencies(128, scaling=dict(sc, attention=2.0))[1] == 2.0


def test_plan_holds_turns():
    p = R.make_plan(64, rotary_dim=32, device="cpu")
    assert p.freq.dtype == torch.int64 and p.freq.numel() == 16 and p.rotary_dim == 32
    assert p.freq[0].item() == round(1 / (2 * math.pi) * 2.0 ** 64)


@pytest.mark.parametrize("kw", [dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=7), dict(head_dim=0),
                                dict(head_dim=514), dict(head_dim=64, layout="x"), dict(head_dim=64, rotary_dim=0),
                                dict(head_dim=64, scaling={"kind": "other", "factor": 2.0}),
                                dict(head_dim=64, scaling={"kind": "linear", "factor": 0.0}),
                                dict(head_dim=64, base=-1.0),
                                dict(head_dim=64, scaling={"kind": "bands", "factor": 2.0, "original": 0})])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        R.make_plan(device="cpu", **kw)


def test_rotate_refusals():
    p = R.make_plan(64, device="cpu")
    x = torch.zeros(2, 3, 5, 64)
    with pytest.raises(ValueError, match="CUDA"):
        R.rotate(x, torch.arange(5), p)
    for bad_x, pos in ((x[..., :32], torch.arange(5)), (x[0, 0], torch.arange(5)), (x, torch.arange(4)),
                       (x[0], torch.arange(3))):
        with pytest.raises(ValueError):
            R.rotate(bad_x, pos, p)
    with pytest.raises(TypeError):
        R.rotate(x, torch.arange(5.0), p)
    with pytest.raises(TypeError):
        R.rotate(x.double(), torch.arange(5), p)
    with pytest.raises(ValueError, match="share memory"):
        R.rotate(x, torch.arange(5), p, out=torch.zeros(2, 3, 1, 64).expand(2, 3, 5, 64))
    with pytest.raises(ValueError, match="gradient"):
        R.rotate(x.clone().requires_grad_(True), torch.arange(5), p, out=torch.zeros_like(x))
    with pytest.raises(ValueError, match="CUDA"):
        R.rotate_append(x[0], x[0], x[0], torch.arange(3), torch.arange(3), x, x, p)


def test_c_entry_refusals():
    L = _lib.load()
    s4, s2, f = _lib.i64x([1, 1, 1, 1]), _lib.i64x([1, 1]), 256
    ok = dict(rot=64, layout=0, dh=64, B=1)
    for change in (dict(rot=65), dict(rot=66), dict(rot=0), dict(layout=2), dict(dh=0), dict(dh=1024), dict(B=0)):
        a = dict(ok, **change)
        assert L.lssab8_rotate(f, 2, a["B"], 1, 1, a["dh"], s4, f, 1, s2, f, 1.0, a["rot"], a["layout"], 0, f, s4, None) == 1
    assert L.lssab8_rotate(None, 2, 1, 1, 1, 64, s4, f, 1, s2, f, 1.0, 64, 0, 0, f, s4, None) == 1
    neg = _lib.i64x([1, -1, 1, 1])
    assert L.lssab8_rotate(f, 2, 1, 1, 1, 64, neg, f, 1, s2, f, 1.0, 64, 0, 0, f, s4, None) == 1
