"""The host layer of the serving-step operators without a GPU: the library is a stand-in that records its calls, so what
is tested is everything around the kernels (workspaces, checks, gradients, versions), on CPU tensors."""
import ctypes
import itertools
import random

import pytest
import torch
from torch.autograd import forward_ad as fwd

from lockstep_b200 import _lib
from lockstep_b200 import attention as A
from lockstep_b200 import decode as D
from lockstep_b200 import engine as E
from lockstep_b200 import paging as P
from lockstep_b200 import rotary as R


class Recorder:
    """Every entry point succeeds and is recorded as (name, arguments); a size query answers 4096."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 4096 if name.endswith("workspace_size") else 0
        return entry

    def names(self):
        return [n for n, _ in self.calls if not n.endswith("workspace_size")]


class Here:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


@pytest.fixture
def lib(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(A, "_require_cuda", lambda *ts: ts[0].device)
    monkeypatch.setattr(A, "_on", lambda dev: Here())
    monkeypatch.setattr(A, "_stream_handle", lambda dev: 0)
    monkeypatch.setattr(A, "check_device_errors", lambda dev=None: None)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: Here())
    return rec


def lattice(B=2, KVH=2, dh=64, blocks=4, pages=40, sink=False):
    kv = D.empty_paged_kv(B, KVH, dh, blocks * 128, torch.zeros((B, blocks * 8), dtype=torch.int32), pages, sink=sink)
    kv.seq_lens.fill_(300)
    return kv


def test_every_call_has_a_workspace_of_its_own():
    """Two calls in flight (two streams, or two captured graphs) never write one buffer."""
    a = A.workspace(torch.device("cpu"), 64)
    b = A.workspace(torch.device("cpu"), 32)
    assert a.numel() >= 64 and b.numel() >= 32 and a.data_ptr() != b.data_ptr()


@pytest.mark.parametrize("shared", [0, 100, 200])
def test_decode_shared_checks_its_arguments_at_every_prefix_length(lib, shared):
    q, kv = torch.zeros(2, 4, 64), lattice()
    D.decode_shared(q, kv, shared)
    assert lib.names() == ["lssab8_decode" if shared < 128 else "lssab8_decode_shared"]
    del lib.calls[:]
    for out in (torch.zeros(2, 4, 32), torch.zeros(1, 4, 64), torch.zeros(2, 1, 64).expand(2, 4, 64)):
        with pytest.raises(ValueError):
            D.decode_shared(q, kv, shared, out=out)
    wide = lattice()
    wide.block_table = torch.zeros((2, 64), dtype=torch.int32)[:, :32]           # rows that are not next to each other
    cut = lattice()
    cut.ek = torch.zeros((2, 2, 8), dtype=torch.int32)[..., ::2]
    half = lattice()
    half.ev = half.ev.to(torch.int16)
    for bad in (wide, cut, half, lattice(B=3), lattice(dh=128), lattice(KVH=3)):
        with pytest.raises((ValueError, TypeError)):
            D.decode_shared(q, bad, shared)
    assert not lib.names()


def plain_rotation(x, positions, plan, inverse, out):
    """rotary._launch in elementary operations, half layout."""
    n = plan.rotary_dim // 2
    theta = torch.tensor(R.frequencies(plan.rotary_dim)[0], dtype=torch.float64)
    a = positions.double()[:, None] * theta * (-1.0 if inverse else 1.0)
    with torch.no_grad():
        x = x.detach()
        c, s, x1, x2 = a.cos(), a.sin(), x[..., :n].double(), x[..., n:2 * n].double()
        out[..., :n], out[..., n:2 * n], out[..., 2 * n:] = x1 * c - x2 * s, x2 * c + x1 * s, x[..., 2 * n:]
    return out


@pytest.fixture
def rotation(monkeypatch):
    monkeypatch.setattr(R, "_launch", plain_rotation)
    plan = R.make_plan(8, 6, device="cpu")
    pos = torch.tensor([0, 3, 70000, 5, 1])
    return plan, pos, lambda x: plain_rotation(x, pos, plan, False, torch.empty_like(x))


def test_rotate_carries_tangents(rotation):
    plan, pos, want = rotation
    x, t, g = (torch.randn(2, 3, 5, 8, dtype=torch.float32) for _ in range(3))
    with fwd.dual_level():
        for grad in (False, True):
            dual = fwd.make_dual(x.clone().requires_grad_(grad), t)
            y = fwd.unpack_dual(R.rotate(dual, pos, plan))
            assert torch.equal(y.primal, want(x)) and torch.equal(y.tangent, want(t))
        with torch.no_grad():                                   # no_grad stops gradients, not tangents
            assert torch.equal(fwd.unpack_dual(R.rotate(dual, pos, plan)).tangent, want(t))
        assert fwd.unpack_dual(R.rotate(x, pos, plan)).tangent is None
        with pytest.raises(ValueError, match="gradient"):
            R.rotate(fwd.make_dual(x, t), pos, plan, out=torch.empty_like(x))
    with fwd.dual_level():                                      # forward over reverse: the gradient's tangent
        x0 = x.clone().requires_grad_(True)
        y = R.rotate(x0, pos, plan)
        gx, = torch.autograd.grad(y, x0, fwd.make_dual(g, t), create_graph=True)
        inv = lambda z: plain_rotation(z, pos, plan, True, torch.empty_like(z))          # noqa: E731
        gx = fwd.unpack_dual(gx)
        assert torch.equal(gx.primal, inv(g)) and torch.equal(gx.tangent, inv(t))


def test_rotate_append_refuses_tangents(lib):
    x, c = torch.randn(3, 2, 8), torch.zeros(2, 16, 2, 8)
    plan, pos = R.make_plan(8, device="cpu"), torch.arange(3)
    with fwd.dual_level():
        for i in range(3):
            qkv = [fwd.make_dual(x, x) if i == j else x for j in range(3)]
            with pytest.raises(ValueError, match="gradient"):
                R.rotate_append(*qkv, pos, pos, c, c.clone(), plan)
    assert not lib.names()


def neg(x):
    """-x as a negative view: x in memory, a bit that says the sign is the other one."""
    y = torch.complex(torch.zeros_like(x), x).conj().imag
    assert y.is_neg() and torch.equal(y, -x)
    return y


def test_negative_views_are_read_as_their_values(lib):
    """The kernels read memory: a view whose sign is pending is resolved, as an input; written, it is refused."""
    first = lambda t: t.reshape(-1)[0].item()                   # noqa: E731
    plan, pos = R.make_plan(64, device="cpu"), torch.arange(3)
    x, c = torch.randn(3, 2, 64), torch.zeros(2, 16, 2, 64)
    kv, cu = lattice(), torch.tensor([0, 2, 3], dtype=torch.int32)
    for n, call in ((3, lambda q, k, v: R.rotate_append(q, k, v, pos, pos, c, c.clone(), plan)),
                    (1, lambda q, k, v: R.rotate(q, pos, plan)), (1, lambda q, k, v: D.decode_shared(q[:2], kv, 256)),
                    (1, lambda q, k, v: D.prefill_paged(q, kv, cu))):
        got, qkv = [], [neg(torch.randn(3, 2, 64)) for i in range(3)]
        for name in ("lssab8_rotate", "lssab8_rotate_append", "lssab8_prefill_paged", "lssab8_decode_shared"):
            setattr(lib, name, lambda *a: got.extend(ctypes.c_float.from_address(p).value for p in a[:n]) or 0)
        call(*qkv)
        assert got == [first(t) for t in qkv[:n]]
    for call in (lambda o: R.rotate(x, pos, plan, out=o), lambda o: R.rotate_append(x, x, x, pos, pos, c, c, plan, out=o),
                 lambda o: R.rotate_append(x, x, x, pos, pos, o, c, plan)):
        with pytest.raises(ValueError, match="negative view"):
            call(neg(torch.randn(3, 2, 64)))


def test_gradients_that_arrive_as_negative_views(rotation, monkeypatch):
    """The gradient of an imaginary part is a negative view of complex memory."""
    plan, pos, _ = rotation
    seen = []
    monkeypatch.setattr(R, "_launch", lambda x, *a: seen.append(x.is_neg()) or plain_rotation(x, *a))
    x, w = torch.randn(1, 1, 5, 8, requires_grad=True), torch.randn(1, 1, 5, 8, dtype=torch.complex64)
    torch.autograd.backward(torch.complex(torch.zeros(1, 1, 5, 8), R.rotate(x, pos, plan)), w.conj())
    assert seen == [False, True]                                # it does arrive so, and _launch resolves it (above)
    assert torch.equal(x.grad, plain_rotation(-w.imag, pos, plan, True, torch.empty(1, 1, 5, 8)))


def version_of(*ts):
    return [t._version for t in ts]


def test_writes_raise_versions(lib):
    """What a kernel writes in place, autograd sees: a tensor saved for a backward pass and rewritten raises there."""
    plan, pos = R.make_plan(64, device="cpu"), torch.arange(3)
    x, kc, vc = torch.randn(3, 2, 64), torch.zeros(2, 16, 2, 64), torch.zeros(2, 16, 2, 64)
    kv, cu = lattice(), torch.tensor([0, 2, 3], dtype=torch.int32)
    i32 = torch.zeros(2, dtype=torch.int32)
    t, bt = P.alloc_step_tables(2, 3, "cpu"), torch.zeros(2, 4, dtype=torch.int32)
    fields = [getattr(t, f) for f in P.StepTables.__dataclass_fields__]
    q = torch.randn(3, 4, 64)
    for ts, call in (([x], lambda: R.rotate(x, pos, plan, out=x)),
                     ([x, kc, vc], lambda: R.rotate_append(x, x.clone(), x.clone(), pos, pos, kc, vc, plan, out=x)),
                     ([kc, vc], lambda: R.rotate_append(x, x.clone(), x.clone(), pos, pos, kc, vc, plan)),
                     ([q], lambda: D.prefill_paged(q.clone(), kv, cu, out=q)),
                     ([q], lambda: D.decode_shared(q[:2].clone(), kv, 256, out=q[:2])),
                     ([q], lambda: D.decode_shared(q[:2].clone(), kv, 100, out=q[:2])),
                     ([bt] + fields, lambda: P.step_tables(i32, i32.clone(), bt, i32, 3, out=t)),
                     ([bt], lambda: P.step_tables(i32, i32.clone(), bt, i32, 3))):
        before = version_of(*ts)
        call()
        assert all(a > b for a, b in zip(version_of(*ts), before))
    keep = version_of(x, q)
    R.rotate(x, pos, plan)
    D.prefill_paged(q, kv, cu)
    assert version_of(x, q) == keep                             # what is only read keeps its version
    w = torch.randn(3, 2, 64, requires_grad=True)
    y = (w * x).sum()
    R.rotate(x, pos, plan, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_outputs_that_require_a_gradient_are_refused(lib):
    plan, pos = R.make_plan(64, device="cpu"), torch.arange(3)
    x, c = torch.randn(3, 2, 64), torch.zeros(2, 16, 2, 64)
    kv, cu = lattice(), torch.tensor([0, 2, 3], dtype=torch.int32)
    leaf = lambda *s: torch.zeros(s, requires_grad=True)        # noqa: E731
    for call in (lambda: R.rotate(x, pos, plan, out=leaf(3, 2, 64)),
                 lambda: R.rotate_append(x, x, x, pos, pos, c, c.clone(), plan, out=leaf(3, 2, 64)),
                 lambda: R.rotate_append(x, x, x, pos, pos, c, leaf(2, 16, 2, 64), plan),
                 lambda: D.prefill_paged(x, kv, cu, out=leaf(3, 2, 64)),
                 lambda: D.decode_shared(x[:2], kv, 256, out=leaf(2, 2, 64)),
                 lambda: D.decode_shared(x[:2], kv, 100, out=leaf(2, 2, 64))):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():                                   # as torch's own out=
            call()


def test_shared_memory_is_found_exactly():
    r = random.Random(3)
    buf, found = torch.zeros(1000), [0, 0]

    def draw():
        n = r.randint(1, 4)
        shape, stride = [r.randint(1, 4) for _ in range(n)], [r.choice([0, 1, 2, 3, 4, 5, 6, 8, 12, 24]) for _ in range(n)]
        return torch.as_strided(buf.view(r.choice([torch.float32, torch.float16])), shape, stride, r.randint(0, 60))

    def places(t):
        return {t.data_ptr() + sum(i * s for i, s in zip(ix, t.stride())) * t.element_size() + b
                for ix in itertools.product(*map(range, t.shape)) for b in range(t.element_size())}
    for _ in range(1500):
        a, b = draw(), draw()
        want = bool(places(a) & places(b))
        found[want] += 1
        assert A._share(a, b) == want, (a.shape, a.stride(), b.shape, b.stride())
    assert min(found) > 300 and not A._share(buf[:0], buf) and not A._share(buf, torch.zeros(1000))


def test_outputs_over_other_inputs_are_refused(lib):
    plan, pos = R.make_plan(64, device="cpu"), torch.arange(3)
    wide = torch.randn(4, 2, 130)
    x = wide[:3, :, :64]
    for out in (x, wide[:3, :, 64:128], torch.empty(3, 2, 64)):          # itself, between its rows, elsewhere
        R.rotate(x, pos, plan, out=out)
    buf = torch.randn(400)
    for a, out in ((x, wide[1:, :, :64]), (x, wide[:3, :, 1:65]), (buf[:384].view(3, 2, 64), buf[1:385].view(3, 2, 64)),
                   (wide[:3, :, :64], wide.view(-1)[2:].as_strided((3, 2, 64), (260, 130, 1)))):
        with pytest.raises(ValueError, match="apart"):
            R.rotate(a, pos, plan, out=out)
    del lib.calls[:]
    qkv = torch.randn(3, 6, 64)                                          # one projection, cut
    q, k, v = qkv[:, :2], qkv[:, 2:4], qkv[:, 4:]
    c = torch.zeros(4, 2, 16, 2, 64)                                     # one cache, keys and values page by page
    go = lambda out=None, kc=c[:, 0], vc=c[:, 1]: R.rotate_append(q, k, v, pos, pos, kc, vc, plan, out=out)   # noqa: E731
    for out in (None, q, torch.empty(3, 2, 64)):
        go(out)
    n = len(lib.names())
    for kw in (dict(out=k), dict(out=v), dict(out=qkv[:, 1:3]), dict(out=c[0, 0, :3]), dict(vc=c[:, 0]),
               dict(kc=torch.zeros(4, 16, 2, 64), vc=c[:, 0], out=c[3, 0, 13:]),
               dict(vc=c.view(-1)[1:].as_strided((4, 16, 2, 64), (4096, 128, 64, 1)))):
        with pytest.raises(ValueError, match="apart"):
            go(**kw)
    store = torch.zeros(2, 16, 2, 64)                                    # keys that lie in the cache they go to
    with pytest.raises(ValueError, match="apart"):
        R.rotate_append(q, store[1, :3], v, pos, pos, store, c[:2, 1], plan)
    assert len(lib.names()) == n


def test_tables_over_their_inputs_are_refused(lib):
    """Every CTA of the kernel reads all lengths while the first writes the new ones."""
    buf = torch.zeros(64, dtype=torch.int32)
    lens, new, free, bt = buf[0:4], buf[8:12], buf[16:20], buf[24:40].view(4, 4)
    t = P.alloc_step_tables(4, 3, "cpu")
    P.step_tables(lens, new, bt, free, 3, out=t)
    for at in (1, 3, 9, 11, 17, 25, 39):
        for name, n in (("seq_lens", 4), ("query_start_loc", 5), ("pages_used", 1)):
            u = P.alloc_step_tables(4, 3, "cpu")
            setattr(u, name, buf[at:at + n])
            with pytest.raises(ValueError):
                P.step_tables(lens, new, bt, free, 3, out=u)
    u = P.alloc_step_tables(4, 3, "cpu")
    u.seq_lens = buf[4:8]                                       # next to the lengths, not over them
    P.step_tables(lens, new, bt, free, 3, out=u)
    assert lib.names() == ["lssab8_step_tables"] * 2


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("pool", ["k8p", "v8p"])
def test_page_pools_of_another_type_are_refused(lib, pool, dtype):
    kv = lattice()
    setattr(kv, pool, getattr(kv, pool).to(dtype))
    for call in (lambda: D.prefill_paged(torch.zeros(3, 4, 64), kv, torch.tensor([0, 2, 3], dtype=torch.int32)),
                 lambda: D.decode_shared(torch.zeros(2, 4, 64), kv, 256),
                 lambda: D.decode_shared(torch.zeros(2, 4, 64), kv, 0)):
        with pytest.raises(TypeError, match="int8"):
            call()
    assert not lib.names()


def test_attention_refuses_queries_with_a_gradient(lib):
    kv, cu = lattice(), torch.tensor([0, 2, 3], dtype=torch.int32)
    q = torch.randn(3, 4, 64)
    calls = (lambda x: D.prefill_paged(x, kv, cu), lambda x: D.decode_shared(x[:2], kv, 256),
             lambda x: D.decode_shared(x[:2], kv, 5))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(q.clone().requires_grad_(True))
        with fwd.dual_level(), pytest.raises(ValueError, match="gradient"):
            call(fwd.make_dual(q, q))
        assert not lib.names()
        with torch.no_grad():
            call(q.clone().requires_grad_(True))
        call(q)
        del lib.calls[:]


@pytest.mark.parametrize("prefill", [True, False])
def test_engine_takes_projections_that_require_a_gradient(lib, prefill):
    """An engine in a program that records gradients: its attention is cut off from them, as ever."""
    att = E.Lssab8Attention(4, 2, 64, 40, max_len=512, max_seqs=2, device="cpu")
    c = torch.zeros(2, 40, 16, 2, 64)
    table = torch.arange(32, dtype=torch.int32)[None]
    meta = E.StepMeta([0, 1], [1], table, torch.zeros(1, dtype=torch.long), [prefill])
    q, k, v = (torch.randn(1, h, 64, requires_grad=True) for h in (4, 2, 2))
    out = att.forward(0, q, k.detach(), v.detach(), c[0], c[1], meta)
    assert not out.requires_grad and lib.names()[-1] == ("lssab8_prefill_paged" if prefill else "lssab8_decode")


@pytest.mark.parametrize("nq,nout", [(3, 8), (8, 3), (8, 8), (6, 9)])
def test_engine_takes_buffers_longer_than_the_step(lib, nq, nout):
    att = E.Lssab8Attention(4, 2, 64, 40, max_len=512, max_seqs=2, device="cpu")
    c, table = torch.zeros(2, 40, 16, 2, 64), torch.arange(64, dtype=torch.int32).view(2, 32)
    meta = E.StepMeta([0, 2, 3], [2, 1], table, torch.tensor([0, 1, 512]), [True, False])
    out = torch.zeros(nout, 4, 64)
    att.forward(0, torch.randn(nq, 4, 64), torch.randn(3, 2, 64), torch.randn(3, 2, 64), c[0], c[1], meta, out=out)
    (_, args), = [x for x in lib.calls if x[0] == "lssab8_prefill_paged"]
    assert args[3] == 3 and args[22] == out.data_ptr()


def test_sequences_on_one_first_page_are_refused(lib):
    """Lattice slots are kept by first page: forks would take one slot, an idle row takes none."""
    att = E.Lssab8Attention(4, 2, 64, 40, max_len=512, max_seqs=3, device="cpu")
    st, c = att.layers[0], torch.zeros(2, 40, 16, 2, 64)

    def step(first, before, new):
        table = torch.full((len(first), 4), -1, dtype=torch.int32)
        table[:, 0] = torch.tensor(first, dtype=torch.int32)
        qsl = [sum(new[:i]) for i in range(len(new) + 1)]
        n = qsl[-1]
        meta = E.StepMeta(qsl, [a + b for a, b in zip(before, new)], table, torch.zeros(n, dtype=torch.long),
                          [x == 0 for x in before])
        lib.lssab8_kv_append = lambda *a: att_exponents(a) or 0
        att.forward(0, torch.randn(n, 4, 64), torch.randn(n, 2, 64), torch.randn(n, 2, 64), c[0], c[1], meta)

    def att_exponents(args):                                    # the append writes its sequences' exponents
        n = args[3]
        ek = (ctypes.c_int32 * (n * 2 * st.max_blocks)).from_address(args[20])
        for b in range(n):
            ek[b * 2 * st.max_blocks] += 1

    step([5, 9], [0, 0], [1, 1])
    assert st.ek[st.slot_of[5], 0, 0] == 1 and st.ek[st.slot_of[9], 0, 0] == 1
    with pytest.raises(RuntimeError, match="start on page 5"):
        step([5, 5], [1, 1], [1, 1])
    with pytest.raises(RuntimeError, match="start on page 7"):
        step([7, 9, 7], [0, 1, 0], [1, 1, 1])
    with pytest.raises(RuntimeError, match="holds 1 tokens"):
        step([5], [2], [1])
    keep = dict(st.slot_of)
    step([5, -1, 9, -1, 5], [1, 0, 1, 0, 0], [1, 0, 1, 0, 0])   # idle rows, one over a live sequence's first page
    assert st.slot_of == keep and st.lens[keep[5]] == st.lens[keep[9]] == 2
    assert st.ek[keep[5], 0, 0] == 2 and st.ek[keep[9], 0, 0] == 2 and int((st.ek != 0).sum()) == 2


def test_token_counters_stay_in_range(lib):
    """The kernel's 32-bit counters step by a grid's threads: capacities from which they could wrap are refused, by the
    host layer and by the library itself."""
    i32 = torch.zeros(2, dtype=torch.int32)
    for cap in (2 ** 31 - 1, 2 ** 30 + 1):
        with pytest.raises(ValueError, match="2\\^30"):
            P.step_tables(i32, i32.clone(), torch.zeros(2, 4, dtype=torch.int32), i32, cap)
    assert not lib.names()


def test_token_counters_stay_in_range_at_the_c_entry():
    L, f = _lib.load(), 256
    call = lambda cap: L.lssab8_step_tables(f, f, 2, f, 4, 4, f, 3, cap, f, f, f, f, f, f, None)     # noqa: E731
    assert call(2 ** 31 - 1) == call(2 ** 30 + 1) == 2


def test_outputs_without_room_are_refused(lib):
    kv, q = lattice(), torch.zeros(2, 4, 64)
    x = torch.zeros(1, 4, 200, 64)
    for out in (torch.zeros(2, 4, 64), torch.zeros(3, 5, 64)):
        D.decode(q, kv, out=out)
    A.prefill(x, x[:, :2], x[:, :2], out=torch.zeros(1, 300, 4, 64))
    n = len(lib.names())
    for out in (torch.zeros(1, 4, 64), torch.zeros(2, 3, 64), torch.zeros(2, 4, 32), torch.zeros(2 * 4 * 64),
                torch.zeros(2, 4, 64, device="meta")):
        with pytest.raises(ValueError):
            D.decode(q, kv, out=out)
    for out in (torch.zeros(1, 199, 4, 64), torch.zeros(1, 4, 200, 64), torch.zeros(200, 4, 64)):
        with pytest.raises(ValueError):
            A.prefill(x, x[:, :2], x[:, :2], out=out)
    assert len(lib.names()) == n
