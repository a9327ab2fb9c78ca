"""Rotary positions (host layer over the C ABI): the rotation of queries and keys before the contract's
quantisers, its inverse (the gradient), and a serving step's fused form that also stores the new keys and
values in the engine's paged float cache.

    plan = make_plan(128, scaling={"kind": "bands", "factor": 32.0, "original": 8192})
    q = rotate(q, positions, plan)                      # [B, H, T, dh] or [N, H, dh]
    q = rotate_append(q, k, v, positions, slot_mapping, k_cache, v_cache, plan)

theta_i = base^(-2 i / rotary_dim) for pair i, scaled for long contexts by one of
    {"kind": "linear", "factor": s}         theta / s
    {"kind": "ntk", "factor": s}            base s^(d / (d - 2)), d = rotary_dim
    {"kind": "bands", "factor": s, "original": L0, "fast": 32.0, "slow": 1.0, "attention": m}
        pairs that turn more than `fast` times over L0 positions keep theta, those below `slow` turns take
        theta / s, in between linearly in the turns; cosine and sine times m (default 0.1 ln s + 1)
The angle of position p is p theta_i, kept as an exact fraction of a turn (64-bit integer arithmetic), so it
is as good at position 10^6 as at 1.
"""
import functools
import math
from dataclasses import dataclass

import torch

from . import _lib
from . import attention as _A

PAGE = 16
_LAYOUTS = {"half": 0, "interleaved": 1}


@dataclass
class RotaryPlan:
    """freq [rotary_dim / 2] int64 on the device: theta_i / (2 pi) in 2^-64 turns."""
    freq: torch.Tensor
    factor: float
    head_dim: int
    rotary_dim: int
    layout: str


def frequencies(rotary_dim, base=10000.0, scaling=None):
    """(theta_i as Python floats, the factor on cosine and sine)."""
    d, factor = int(rotary_dim), 1.0
    kind = None if scaling is None else scaling.get("kind")
    if scaling is not None and kind not in ("linear", "ntk", "bands"):
        raise ValueError("scaling kind must be linear, ntk or bands, got %r" % (kind,))
    s = 1.0 if scaling is None else float(scaling["factor"])
    if not (s > 0.0 and math.isfinite(s)) or not (base > 0.0 and math.isfinite(base)):
        raise ValueError("base and scaling factor must be positive")
    if kind == "ntk" and d > 2:
        base = base * s ** (d / (d - 2))
    theta = [base ** (-i / d) for i in range(0, d, 2)]
    if kind == "linear":
        theta = [t / s for t in theta]
    if kind == "bands":
        L0, fast, slow = float(scaling["original"]), float(scaling.get("fast", 32.0)), float(scaling.get("slow", 1.0))
        if not (L0 > 0 and fast > slow):
            raise ValueError("bands need original > 0 and fast > slow")
        keep = [min(1.0, max(0.0, (L0 * t / (2 * math.pi) - slow) / (fast - slow))) for t in theta]
        theta = [t * k + t / s * (1 - k) for t, k in zip(theta, keep)]
        m = scaling.get("attention")
        factor = float(m) if m is not None else (0.1 * math.log(s) + 1.0 if s > 1 else 1.0)
    return theta, factor


def make_plan(head_dim, rotary_dim=None, base=10000.0, layout="half", scaling=None, device=None):
    """The plan of a model's rotary positions: made once, kept by the caller, shared by its layers."""
    rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
    if not 0 < head_dim <= 512 or not 0 < rotary_dim <= head_dim or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at most head_dim, head_dim at most 512")
    if layout not in _LAYOUTS:
        raise ValueError("layout must be half or interleaved, got %r" % (layout,))
    theta, factor = frequencies(rotary_dim, base, scaling)
    turns = [int(round(t / (2 * math.pi) * 2.0 ** 64)) % (1 << 64) for t in theta]
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    freq = torch.tensor([u - (1 << 64) if u >= 1 << 63 else u for u in turns], dtype=torch.int64).to(dev)
    return RotaryPlan(freq=freq, factor=factor, head_dim=int(head_dim), rotary_dim=rotary_dim, layout=layout)


def _check_positions(positions):
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be int32 or int64, got %s" % positions.dtype)


def _launch(x, positions, plan, inverse, out):
    dev = _A._require_cuda(x, positions, plan.freq, out)
    if x.numel() == 0:
        return out
    x = x.resolve_neg()                          # (gradients through the imaginary part of a conjugate come as views)
    x4, y4 = (x, out) if x.dim() == 4 else (x.transpose(0, 1)[None], out.transpose(0, 1)[None])
    B, H, T, dh = x4.shape
    ps = (0, positions.stride(0)) if positions.dim() == 1 else positions.stride()
    with _A._on(dev):
        _lib.check(_lib.load().lssab8_rotate(
            x4.data_ptr(), _A.dtype_code(x.dtype), B, H, T, dh, _lib.i64c(x4.stride()), positions.data_ptr(),
            int(positions.dtype == torch.int64), _lib.i64c(ps), plan.freq.data_ptr(), plan.factor, plan.rotary_dim,
            _LAYOUTS[plan.layout], int(bool(inverse)), y4.data_ptr(), _lib.i64c(y4.stride()), _A._stream_handle(dev)),
            "lssab8_rotate")
    return out


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, plan, inverse):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.plan, ctx.inverse = plan, inverse
        return _launch(x, positions, plan, inverse, torch.empty_like(x))

    @staticmethod
    def backward(ctx, g):
        positions, = ctx.saved_tensors
        if torch.is_grad_enabled():                              # a gradient of the gradient is wanted
            return rotate(g, positions, ctx.plan, inverse=not ctx.inverse), None, None, None
        return _launch(g, positions, ctx.plan, not ctx.inverse, torch.empty_like(g)), None, None, None

    @staticmethod
    def jvp(ctx, t, *_):                                         # the map is linear: the tangent is rotated as x is
        positions, = ctx.saved_tensors
        return rotate(t, positions, ctx.plan, inverse=ctx.inverse)


def rotate(x, positions, plan, inverse=False, out=None):
    """x [B, H, T, dh] with positions [T] or [B, T], or x [N, H, dh] with positions [N] -> rotated x, same type
    and shape (any strides; float32, float16, bfloat16).  inverse=True: the transposed map (it undoes
    the rotation when the plan's factor is 1); differentiable in x, the gradient being the other direction
    (forward mode: the tangent is rotated too).
    out: written instead (out=x rotates in place, else apart from x); not with a gradient.  In a captured graph: torch
    refuses to capture a backward pass while an eager graph of the same leaf is alive; rotate(g, positions, plan,
    inverse=True) is the same gradient and needs no graph of the leaf."""
    shape, ps = x.shape, positions.shape
    if len(shape) not in (3, 4) or shape[-1] != plan.head_dim:
        raise ValueError("x must be [B, H, T, %d] or [N, H, %d], got %s" % (plan.head_dim, plan.head_dim, tuple(shape)))
    _check_positions(positions)
    if ps != (shape[0] if len(shape) == 3 else shape[2],) and (len(shape) == 3 or ps != (shape[0], shape[2])):
        raise ValueError("positions must be [N], [T] or [B, T] for x %s, got %s" % (tuple(shape), tuple(ps)))
    _A.dtype_code(x.dtype)
    if _A._differentiable(x):
        if out is not None:
            raise ValueError("out= has no gradient: rotate a detached tensor, or leave out away")
        return _Rotate.apply(x, positions, plan, bool(inverse))
    if out is None:
        return _launch(x, positions, plan, inverse, torch.empty_like(x))
    if out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("out must have x's shape and dtype")
    if not _A._written_once(out) or out.is_neg():
        raise ValueError("out has elements that share memory, or is a negative view")
    if _A._differentiable(out):
        raise ValueError("out= has no gradient: rotate into a tensor that requires none")
    if not _A._same_places(x, out) and _A._share(x, out):
        raise ValueError("out must be x itself or lie apart from it")
    _launch(x, positions, plan, inverse, out)
    _A._wrote(out)
    return out


def rotate_append(query, key, value, positions, slot_mapping, k_cache, v_cache, plan, out=None, check=True):
    """A serving step's new tokens: query [N, H, dh] rotated (returned, or written to out, which may be the query and
    else lies apart from the inputs), key [N, KVH, dh] rotated and value [N, KVH, dh] stored in k_cache / v_cache
    [num_pages, 16, KVH, dh], which lie apart from the inputs and each other (any page, row and head strides; the cache's
    own dtype, one rounding), at slot_mapping [N] int64, page * 16 + row.  Slot -1 stores nothing; the other slots must differ (two tokens in one slot leave a mix of both).  Inference
    only: no gradient flows through it."""
    dev = _A._require_cuda(query, key, value, positions, slot_mapping, k_cache, v_cache, plan.freq)
    if _A._differentiable(query, key, value, k_cache, v_cache):
        raise ValueError("rotate_append has no gradient (use rotate)")
    qdt, kcdt = query.dtype, k_cache.dtype
    if qdt is not torch.bfloat16 and (query.is_neg() or key.is_neg() or value.is_neg()):     # (bfloat16 has no complex type)
        query, key, value = query.resolve_neg(), key.resolve_neg(), value.resolve_neg()
    if kcdt is not torch.bfloat16 and (k_cache.is_neg() or v_cache.is_neg()):
        raise ValueError("the caches must not be negative views")
    fresh = out is None
    if fresh:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        like = None
    else:
        like = out.shape, out.stride(), out.dtype
        if out.device != dev:
            raise ValueError("out must be on the query's device")
        if out.is_neg() or _A._differentiable(out):
            raise ValueError("out must not be a negative view, nor require a gradient")
    qp, kp, vp, kcp, vcp = (query.data_ptr(), key.data_ptr(), value.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr())
    args = _append_args(query.shape, query.stride(), qdt, key.shape, key.stride(), key.dtype, value.shape,
                        value.stride(), value.dtype, k_cache.shape, k_cache.stride(), kcdt, v_cache.shape,
                        v_cache.stride(), v_cache.dtype, like, positions.shape, positions.dtype, slot_mapping.shape,
                        slot_mapping.dtype, plan.head_dim)
    dims, qs, ks, vs, pos64, os_, cdt, kcs, vcs, (nq, nk, nv, nkc, nvc, _), dims_of, in_place = args
    if dims[1] == 0:
        return out
    op = out.data_ptr()
    # what is written lies apart from what is read (out may be the query) and from each other: by address ranges,
    # then exactly where these meet
    if kcp < vcp + nvc and vcp < kcp + nkc and _A._meet(vcp - kcp, dims_of[3], dims_of[4]):
        raise ValueError("the caches must lie apart from each other")
    lo, hi = min(kcp, vcp), max(kcp + nkc, vcp + nvc)
    if not fresh or (qp < hi and qp + nq > lo) or (kp < hi and kp + nk > lo) or (vp < hi and vp + nv > lo):
        _check_places((qp, kp, vp, kcp, vcp, op), args[9], dims_of, in_place)
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    with _A._on(dev):
        _lib.check(_lib.load().lssab8_rotate_append(
            qp, kp, vp, *dims, qs, ks, vs, positions.data_ptr(), pos64, positions.stride(0), plan.freq.data_ptr(),
            plan.factor, plan.rotary_dim, _LAYOUTS[plan.layout], op, os_, kcp, vcp, cdt, kcs, vcs, k_cache.shape[0],
            slot_mapping.data_ptr(), _A._stream_handle(dev)), "lssab8_rotate_append")
    if fresh:
        _A._wrote(k_cache, v_cache)
    else:
        _A._wrote(k_cache, v_cache, out)
    if check:
        _A.check_device_errors(dev)
    return out


@functools.lru_cache(maxsize=1024)
def _append_args(q, qst, qdt, k, kst, kdt, v, vst, vdt, kc, kcst, kcdt, vc, vcst, vcdt, like, pos, pdt, sl, sdt,
                 head_dim):
    """The checks of rotate_append's shapes, strides and types, and the arguments made from them; kept, since a
    model's steps repeat them.  like: out's shape, strides and type (None: a new contiguous one)."""
    if len(q) != 3 or len(k) != 3 or k != v or k[0] != q[0]:
        raise ValueError("query must be [N, H, dh], key and value [N, KVH, dh]")
    if not qdt == kdt == vdt or kcdt != vcdt:
        raise TypeError("query, key and value must share one dtype, and so must the caches")
    N, H, dh = q
    KVH = k[1]
    o, ost, odt = (q, (H * dh, dh, 1), qdt) if like is None else like
    if dh != head_dim or k[2] != dh:
        raise ValueError("the plan is for head dim %d" % head_dim)
    if len(kc) != 4 or kc != vc or tuple(kc[1:]) != (PAGE, KVH, dh):
        raise ValueError("caches must be [num_pages, 16, %d, %d]" % (KVH, dh))
    if pdt not in (torch.int32, torch.int64):
        raise TypeError("positions must be int32 or int64, got %s" % pdt)
    if tuple(pos) != (N,) or tuple(sl) != (N,):
        raise ValueError("positions and slot_mapping must be [%d]" % N)
    if sdt != torch.int64:
        raise TypeError("slot_mapping must be int64")
    if o != q or odt != qdt:
        raise ValueError("out must have the query's shape and dtype")
    if dh > 1 and any(st[-1] != 1 for st in (qst, kst, vst, kcst, vcst, ost)):
        raise ValueError("channels must be contiguous")
    if not (_A._apart(ost, o) and _A._apart(kcst, kc) and _A._apart(vcst, vc)):
        raise ValueError("out and the caches must not have elements that share memory")
    reach, dims_of = zip(*(_A._reach(*x) for x in ((qst, q, qdt), (kst, k, kdt), (vst, v, vdt), (kcst, kc, kcdt),
                                                   (vcst, vc, vcdt), (ost, o, odt))))
    return ((_A.dtype_code(qdt), N, H, KVH, dh), _lib.i64c(qst[:2]), _lib.i64c(kst[:2]), _lib.i64c(vst[:2]),
            int(pdt == torch.int64), _lib.i64c(ost[:2]), _A.dtype_code(kcdt), _lib.i64c(kcst[:3]), _lib.i64c(vcst[:3]),
            reach, dims_of, all(x == y for x, y, n in zip(qst, ost, q) if n > 1))


def _check_places(at, reach, dims_of, in_place):
    """query, key, value, key cache, value cache, out, each an address, the bytes reached and its dimensions: the caches
    and out lie apart from the inputs and out from the caches, except out in the query's own places."""
    for w, others in ((3, (0, 1, 2)), (4, (0, 1, 2)), (5, (0, 1, 2, 3, 4))):
        for x in others:
            d = at[x] - at[w]
            if -reach[x] < d < reach[w] and not (w == 5 and x == 0 and d == 0 and in_place) and \
                    _A._meet(d, dims_of[w], dims_of[x]):
                raise ValueError("out and the caches must lie apart from the inputs (out may be the query) and from each "
                                 "other")
