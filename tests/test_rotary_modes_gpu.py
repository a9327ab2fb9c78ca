"""Rotary positions under the ways torch differentiates and rewrites tensors, on the kernel: forward mode, gradients that
arrive as negative views, and in-place writes.  The map is linear and each element's rounding depends on its own pair
alone, so every tangent and gradient equals the same call on its own, bit for bit."""
import pytest
import torch
from torch.autograd import forward_ad as fwd

from lockstep_b200 import rotary as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,rot", [("half", 64), ("interleaved", 30)])
def test_tangents(layout, rot, dtype):
    plan = R.make_plan(64, rot, layout=layout)
    pos = torch.randint(0, 100000, (2, 9), device="cuda")
    x, t = (torch.randn(2, 3, 9, 64, device="cuda").to(dtype) for _ in range(2))
    with fwd.dual_level():
        y = fwd.unpack_dual(R.rotate(fwd.make_dual(x, t), pos, plan))
        assert torch.equal(y.primal, R.rotate(x, pos, plan)) and torch.equal(y.tangent, R.rotate(t, pos, plan))
        wide = torch.randn(2, 9, 3, 65, device="cuda").to(dtype)[..., :64].transpose(1, 2)      # a strided tangent
        y = fwd.unpack_dual(R.rotate(fwd.make_dual(x, wide), pos, plan, inverse=True))
        assert torch.equal(y.tangent, R.rotate(wide, pos, plan, inverse=True))


def test_gradients_that_arrive_as_negative_views():
    plan, pos = R.make_plan(64), torch.arange(9, device="cuda")
    x, zero = torch.randn(2, 3, 9, 64, device="cuda", requires_grad=True), torch.zeros(2, 3, 9, 64, device="cuda")
    w = torch.randn(2, 3, 9, 64, device="cuda", dtype=torch.complex64)
    torch.autograd.backward(torch.complex(zero, R.rotate(x, pos, plan)), w.conj())
    assert torch.equal(x.grad, R.rotate((-w.imag).contiguous(), pos, plan, inverse=True))
    view = w.conj().imag
    assert view.is_neg() and torch.equal(R.rotate(view, pos, plan), R.rotate(view.clone(), pos, plan))


def test_in_place_writes_are_seen_by_autograd():
    plan, pos = R.make_plan(64), torch.arange(9, device="cuda")
    x, w = torch.randn(9, 3, 64, device="cuda"), torch.randn(9, 3, 64, device="cuda", requires_grad=True)
    y = (w * x).sum()
    R.rotate(x, pos, plan, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():                                # where torch keeps no versions
        z = torch.randn(9, 3, 64, device="cuda")
        want = R.rotate(z, pos, plan)
        assert torch.equal(R.rotate(z, pos, plan, out=z), want)
    assert torch.equal(R.rotate(z, pos, plan, out=z), R.rotate(want, pos, plan))
