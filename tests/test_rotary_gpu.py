"""Rotary positions on the GPU against complex rotation in 64 bits.

Tolerance, u = 2^-24: the angle's remainder (at most pi / 4) is rounded once (pi / 4 u), sincospif errs by at most
2 ulp (2 u, values below 1), the factor and the product with it round once each (2 u): a coefficient is off by
less than 5 m u.  A result sums two products, (|x1| + |x2|) 5 m u, rounds one product and the fused sum (2 u m (|x1| +
|x2|)), and is rounded once to its type (eps / 2 |y|)."""
import math

import pytest
import torch

from lockstep_b200 import decode as D
from lockstep_b200 import rotary as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BANDS = {"kind": "bands", "factor": 32.0, "original": 8192}


def reference(x, pos, rot, layout, scaling=None, sign=1.0):
    """x [..., dh] float64 (channels last), pos broadcast against x's leading dims -> (y, |x1| + |x2| per channel)."""
    th, m = R.frequencies(rot, scaling=scaling)
    ang = pos.double()[..., None] * torch.tensor(th, dtype=torch.float64, device=x.device) * sign
    i1 = torch.arange(rot // 2, device=x.device) if layout == "half" else torch.arange(0, rot, 2, device=x.device)
    i2 = i1 + (rot // 2 if layout == "half" else 1)
    a, b = x[..., i1], x[..., i2]
    z = torch.complex(a, b) * torch.polar(torch.full_like(ang, m), ang)
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., i1], y[..., i2] = z.real, z.imag
    mag[..., i1] = mag[..., i2] = (a.abs() + b.abs()) * m
    return y, mag


def check(got, want, mag):
    tol = 7 * U * mag + torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 1e-6) + torch.finfo(got.dtype).tiny
    passed = mag == 0
    assert (got.double() - want).abs().le(tol).all()
    assert torch.equal(got.double()[passed], want[passed].to(got.dtype).double())


CASES = [  # B, H, T, dh, rot, layout, scaling, start
    (1, 1, 1, 64, 64, "half", None, 0),
    (2, 5, 33, 128, 128, "half", BANDS, 250000),
    (1, 3, 300, 64, 64, "interleaved", {"kind": "ntk", "factor": 8.0}, 1 << 20),
    (2, 2, 17, 128, 64, "half", {"kind": "linear", "factor": 4.0}, 77),
    (1, 4, 19, 128, 50, "interleaved", None, 1000),      # a vector half rotated, half passed
    (1, 4, 19, 128, 50, "half", None, 1000),             # no whole vectors a half
    (2, 1, 5, 80, 2, "half", None, 5),
    (1, 1, 3, 7, 6, "interleaved", None, (1 << 31) - 2), # odd head dim, positions past 2^31
    (1, 40, 2, 512, 512, "half", None, 31),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,T,dh,rot,layout,scaling,start", CASES)
def test_rotate(B, H, T, dh, rot, layout, scaling, start, dtype):
    g = torch.Generator("cuda").manual_seed(T)
    x = torch.randn((B, H, T, dh), generator=g, device="cuda").to(dtype)
    pos = torch.arange(start, start + T, device="cuda")
    plan = R.make_plan(dh, rot, layout=layout, scaling=scaling)
    for inverse in (False, True):
        want, mag = reference(x.double(), pos, rot, layout, scaling, -1.0 if inverse else 1.0)
        check(R.rotate(x, pos, plan, inverse=inverse), want, mag)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_strides_and_places(layout):
    plan = R.make_plan(64, 32, layout=layout)
    base = torch.randn(4, 9, 7, 3, 65, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 9000, (4, 9), device="cuda", dtype=torch.int32)
    views = [base[:, :, 0, :, :64].transpose(1, 2),           # [B, H, T, dh], unaligned rows
             base[:, :, :3, 0, :64].transpose(1, 2),
             torch.randn(4, 64, 9, 3, device="cuda").permute(0, 3, 2, 1),        # channels not contiguous
             torch.randn(4, 1, 9, 64, device="cuda").expand(4, 3, 9, 64)]        # one head's memory for all
    for x in views:
        want, mag = reference(x.double(), pos[:, None], 32, layout)
        y = R.rotate(x, pos, plan)
        check(y, want, mag)
        out = torch.full((4, 9, 3, 64), 7.0, device="cuda", dtype=x.dtype).transpose(1, 2)
        assert R.rotate(x, pos, plan, out=out) is out and torch.equal(out, y)
        if 0 not in x.stride():
            keep = base.clone()
            assert R.rotate(x, pos, plan, out=x) is x and torch.equal(x, y)      # in place
            base.copy_(keep)
    x3 = torch.randn(9, 3, 64, device="cuda")
    want, mag = reference(x3.double(), pos[1, :, None], 32, layout)
    check(R.rotate(x3, pos[1], plan), want, mag)
    assert R.rotate(x3[:0], pos[1, :0], plan).shape == (0, 3, 64)
    one = pos[0, :1].expand(9)                                 # one position for all tokens
    want, mag = reference(x3.double(), one[:, None], 32, layout)
    check(R.rotate(x3, one, plan), want, mag)


def test_passed_channels_keep_their_bits():
    plan = R.make_plan(64, 32, layout="interleaved")
    x = torch.zeros(3, 2, 64, device="cuda")
    x[..., 40], x[..., 41], x[..., 33] = float("nan"), float("inf"), -0.0
    x[..., 63] = 1e-40
    y = R.rotate(x, torch.arange(3, device="cuda"), plan)
    assert torch.equal(y[..., 32:].view(torch.int32), x[..., 32:].view(torch.int32))
    assert torch.equal(y[..., :32], torch.zeros_like(y[..., :32]))


@pytest.mark.parametrize("layout,scaling", [("half", BANDS), ("interleaved", None)])
def test_gradient(layout, scaling):
    """The gradient against the formula's (the transposed map) and against differences (the map is linear)."""
    plan = R.make_plan(64, 48, layout=layout, scaling=scaling)
    x = torch.randn(2, 3, 21, 64, device="cuda", requires_grad=True)
    pos = torch.randint(0, 100000, (2, 21), device="cuda")
    g = torch.randn_like(x)
    y = R.rotate(x, pos, plan)
    gx, = torch.autograd.grad(y, x, g, create_graph=True)
    want, mag = reference(g.double(), pos[:, None], 48, layout, scaling, -1.0)
    check(gx.detach(), want, mag)
    with torch.no_grad():
        d = torch.randn_like(x)
        lhs = ((R.rotate(x + d, pos, plan) - y).double() * g.double()).sum()
        rhs = (gx.double() * ((x + d) - x).double()).sum()
        # every element of either sum is off by at most 16 u of its terms' magnitudes (bound above, and the
        # difference's cancellation)
        m = R.frequencies(48, scaling=scaling)[1]
        scale = (g.abs().sum() * 2 * m * (x.abs().max() + d.abs().max()) * 16 * U).double()
        assert (lhs - rhs).abs() <= scale
    h = x.detach().expand(2, 3, 21, 64)[:, :1].expand(2, 3, 21, 64).clone().requires_grad_(True)
    shared = torch.randn(2, 1, 21, 64, device="cuda", requires_grad=True)          # one key head for three
    gs, = torch.autograd.grad(R.rotate(shared.expand(2, 3, 21, 64), pos, plan), shared, g)
    want, mag = reference(g.double(), pos[:, None], 48, layout, scaling, -1.0)
    assert (gs.double() - want.sum(1, keepdim=True)).abs().le(
        (7 * U * mag + U * want.abs()).sum(1, keepdim=True) + 3 * U * want.abs().sum(1, keepdim=True)).all()
    assert R.rotate(h, pos, plan).requires_grad
    with torch.no_grad():
        assert not R.rotate(h, pos, plan).requires_grad


@pytest.mark.parametrize("dtype,cdtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                          (torch.float16, torch.float32), (torch.float32, torch.float16),
                                          (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("N,H,KVH,dh,rot,layout", [(1, 8, 2, 128, 128, "half"), (45, 7, 1, 64, 64, "interleaved"),
                                                   (200, 4, 4, 128, 30, "half"), (3, 2, 1, 24, 10, "interleaved")])
def test_rotate_append(N, H, KVH, dh, rot, layout, dtype, cdtype):
    g = torch.Generator("cuda").manual_seed(N + dh)
    qkv = torch.randn((N, H + 2 * KVH, dh), generator=g, device="cuda").to(dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
    pages = N // 16 + 2
    cache = torch.randn((pages, 2, 16, KVH, dh), generator=g, device="cuda").to(cdtype)
    slots = torch.randperm(pages * 16, generator=g, device="cuda")[:N]
    if N > 5:
        slots[[1, N - 1]] = -1
    pos = torch.randint(0, 1 << 18, (N,), generator=g, device="cuda")
    plan = R.make_plan(dh, rot, layout=layout, scaling=BANDS if dh == 128 else None)
    sc = BANDS if dh == 128 else None
    before = cache.clone()
    out = R.rotate_append(q, k, v, pos, slots, cache[:, 0], cache[:, 1], plan)
    check(out, *reference(q.double(), pos[:, None], rot, layout, sc))
    ok = slots >= 0
    s = slots[ok]
    want, mag = reference(k.double(), pos[:, None], rot, layout, sc)
    check(cache[s // 16, 0, s % 16], want[ok], mag[ok])
    assert torch.equal(cache[s // 16, 1, s % 16], v[ok].to(cdtype))
    after = cache.clone()
    after[s // 16, :, s % 16] = before[s // 16, :, s % 16]
    assert torch.equal(after, before)                          # every other row as it was
    assert torch.equal(R.rotate(q.contiguous(), pos, plan), out)           # the same rotation
    q2 = q.clone()
    assert R.rotate_append(q2, k, v, pos, slots, cache[:, 0], cache[:, 1], plan, out=q2) is q2
    assert torch.equal(q2, out)


def test_rotate_append_bad_slot_is_flagged_and_skipped():
    plan = R.make_plan(64)
    x = torch.randn(3, 2, 64, device="cuda")
    kc, vc = torch.zeros(2, 16, 2, 64, device="cuda"), torch.zeros(2, 16, 2, 64, device="cuda")
    pos = torch.arange(3, device="cuda")
    for bad in (32, -2, 1 << 40):
        with pytest.raises(RuntimeError, match="bits 0x4 "):
            R.rotate_append(x, x, x, pos, torch.tensor([bad, -1, -1], device="cuda"), kc, vc, plan)
        assert not kc.any() and not vc.any()
    with pytest.raises(TypeError):
        R.rotate_append(x, x, x, pos, torch.zeros(3, dtype=torch.int32, device="cuda"), kc, vc, plan)
    with pytest.raises(ValueError):
        R.rotate_append(x, x, x, pos, pos, kc[:, :8], vc[:, :8], plan)
    with pytest.raises(ValueError, match="gradient"):
        R.rotate_append(x.clone().requires_grad_(True), x, x, pos, pos, kc, vc, plan)


def test_streams_and_graph():
    """On a side stream, and captured and replayed with new inputs in the same buffers."""
    plan = R.make_plan(128)
    x = torch.randn(8, 4, 128, device="cuda").to(torch.bfloat16)
    pos = torch.arange(8, device="cuda")
    want = R.rotate(x, pos, plan)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = R.rotate(x, pos, plan)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = R.rotate(x, pos, plan)
        z = R.rotate(y, pos, plan, inverse=True)
    x.copy_(torch.randn_like(x))
    pos += 1000
    graph.replay()
    assert torch.equal(y, R.rotate(x, pos, plan)) and torch.equal(z, R.rotate(y, pos, plan, inverse=True))
    # a captured backward pass, and the gradient captured directly while an eager graph of the leaf lives
    leaf, g = x.float().requires_grad_(True), torch.randn(8, 4, 128, device="cuda")
    want = R.rotate(g, pos, plan, inverse=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(R.rotate(leaf, pos, plan), leaf, g)
    graph.replay()
    assert torch.equal(got, want)
    alive = R.rotate(leaf, pos, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = R.rotate(g, pos, plan, inverse=True)
    graph.replay()
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(alive, leaf, g)[0], want)
    assert D.PAGE == R.PAGE and math.isfinite(float(z.float().sum()))
