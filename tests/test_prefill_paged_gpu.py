"""Packed prompt rows over the paged lattice (decode.prefill_paged): every row bit for bit against the oracle
on its own sequence (document mask), with bidirectional prefixes (the oracle's key_valid rows), chunks, sinks, and
the exponent-jump and flush fixtures; strides, idle sequences, refusals, streams and graphs."""
import numpy as np
import pytest
import torch

import oracle as O
from fixtures import all_cases
from lockstep_b200 import _lib
from lockstep_b200 import attention as A
from lockstep_b200 import decode as D
from lockstep_b200 import workloads as W

DEV = "cuda"
BITS = {torch.float32: torch.int32, torch.float16: torch.int16, torch.bfloat16: torch.int16}


def same_bits(a, b):
    return torch.equal(a.contiguous().view(BITS[a.dtype]), b.contiguous().view(BITS[b.dtype]))


def lattice(ks, vs, sink, seed=0, extra_blocks=0):
    """A lattice of sequences ks[b] / vs[b] [KVH, L, dh] float32 numpy, on a random page table."""
    lens = [k.shape[1] for k in ks]
    bt, total = W.page_table([max(x, 1) for x in lens], 16, seed)
    nb = max(-(-max(x, 1) // 128) for x in lens) + extra_blocks
    btp = np.full((len(lens), nb * 8), -1, np.int32)
    btp[:, :bt.shape[1]] = bt
    KVH, dh = ks[0].shape[0], ks[0].shape[2]
    flat = lambda xs: torch.from_numpy(np.concatenate([x.transpose(1, 0, 2) for x in xs] +     # noqa: E731
                                                      [np.zeros((1, KVH, dh), np.float32)])).to(DEV)
    cu = np.concatenate([[0], np.cumsum(lens)])
    kv = D.build_paged_kv(flat(ks), flat(vs), torch.tensor(lens, dtype=torch.int32, device=DEV),
                          torch.from_numpy(btp).to(DEV), total, sink=sink, cu_seqlens=cu)
    if kv.max_blocks < nb:
        kv0 = D.empty_paged_kv(len(lens), KVH, dh, nb * 128, kv.block_table, total, sink=sink)
        for n in ("ek", "ev"):
            getattr(kv0, n)[:, :, :kv.max_blocks] = getattr(kv, n)
        kv0.k8p, kv0.v8p, kv0.ev0, kv0.seq_lens = kv.k8p, kv.v8p, kv.ev0, kv.seq_lens
        kv = kv0
    return kv


def oracle_rows(q, k, v, T0, P, sink):
    """Rows [T0, L) of one sequence: q [n, H, dh], k / v [KVH, L, dh] -> float32 [n, H, dh]."""
    L, (n, H, dh) = k.shape[1], q.shape
    full = np.zeros((H, L, dh), np.float32)
    full[:, T0:] = q.transpose(1, 0, 2)
    rows = np.arange(T0, L)
    out = O.attention(full, k, v, sink=sink, rows=rows)
    if P > T0:
        two = O.attention(full, k, v, sink=sink, causal=False, key_valid=np.arange(L) < P, rows=rows)
        out = out.copy()
        out[:, T0:P] = two[:, T0:P]
    return out[:, T0:].transpose(1, 0, 2)


def draw(lens, T0, H, KVH, dh, seed):
    r = np.random.default_rng(seed)
    f = lambda *s: W.bf16_round(r.standard_normal(s).astype(np.float32))          # noqa: E731
    ks, vs = [f(KVH, L, dh) for L in lens], [f(KVH, L, dh) for L in lens]
    qs = [f(L - t, H, dh) for L, t in zip(lens, T0)]
    return qs, ks, vs


def cu_of(qs):
    return torch.tensor(np.concatenate([[0], np.cumsum([x.shape[0] for x in qs])]), dtype=torch.int32, device=DEV)


CASES = [  # lens, T0, P, H, KVH, dh
    ([1], [0], [0], 1, 1, 64),
    ([127, 128, 129, 1, 2], [0] * 5, [0] * 5, 4, 2, 128),
    ([300, 513, 64], [256, 0, 0], [0] * 3, 8, 2, 64),
    ([300, 700, 1, 260], [128, 0, 0, 256], [300, 450, 1, 100], 4, 1, 128),
    ([256, 200, 640], [0, 0, 384], [129, 128, 640], 7, 7, 64),
    ([4300, 130], [4096, 0], [0, 0], 2, 1, 128),               # more than one fold segment
    ([4400, 90], [128 * 33, 0], [4300, 90], 12, 1, 64),        # a prefix across segments; a group of 12
]


@pytest.mark.gpu
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("lens,T0,P,H,KVH,dh", CASES)
def test_rows_equal_oracle(lens, T0, P, H, KVH, dh, sink):
    qs, ks, vs = draw(lens, T0, H, KVH, dh, sum(lens))
    kv = lattice(ks, vs, sink)
    q = torch.from_numpy(np.concatenate(qs)).to(DEV)
    pl = torch.tensor(P, dtype=torch.int32, device=DEV) if any(P) else None
    out = D.prefill_paged(q, kv, cu_of(qs), prefix_lens=pl)
    want = np.concatenate([oracle_rows(*x, sink) for x in zip(qs, ks, vs, T0, P)])
    assert same_bits(out, torch.from_numpy(want).to(DEV))
    for dt in (torch.bfloat16, torch.float16):                 # one rounding at the end
        assert same_bits(D.prefill_paged(q, kv, cu_of(qs), prefix_lens=pl, out_dtype=dt), out.to(dt))
    qb = q.to(torch.bfloat16)                                  # bf16 values already: the same rows
    assert same_bits(D.prefill_paged(qb, kv, cu_of(qs), prefix_lens=pl, out_dtype=torch.float32), out)


@pytest.mark.gpu
def test_fixture_sequences_packed():
    """The exponent jumps, flush ladders, ties and dead blocks of the contract's selftest, packed into one step."""
    cases = [c for c in all_cases() if c["q"].shape[0] in (1, 2) and c["k"].shape[0] == 1]
    for H in (1, 2):
        cs = [c for c in cases if c["q"].shape[0] == H]
        kv = lattice([c["k"] for c in cs], [c["v"] for c in cs], False, seed=H)
        qs = [c["q"].transpose(1, 0, 2) for c in cs]
        out = D.prefill_paged(torch.from_numpy(np.concatenate(qs)).to(DEV), kv, cu_of(qs))
        want = np.concatenate([O.attention(c["q"], c["k"], c["v"]).transpose(1, 0, 2) for c in cs])
        assert same_bits(out, torch.from_numpy(want).to(DEV))


@pytest.mark.gpu
def test_equals_the_prefill_of_each_sequence_alone():
    lens = [1000, 77, 4200]
    qs, ks, vs = draw(lens, [0] * 3, 8, 2, 128, 5)
    t = lambda x: torch.from_numpy(x).to(torch.bfloat16).to(DEV)              # noqa: E731
    out = D.prefill_paged(t(np.concatenate(qs)), lattice(ks, vs, True), cu_of(qs))
    at = 0
    for q, k, v in zip(qs, ks, vs):
        alone = A.prefill(t(q.transpose(1, 0, 2)[None].copy()), t(k[None]), t(v[None]), sink=True)[0]
        assert same_bits(out[at:at + q.shape[0]], alone)
        at += q.shape[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_queries_that_are_not_finite(dtype):
    qs, ks, vs = draw([150], [0], 4, 2, 64, 6)
    qs[0][3, 1, 2], qs[0][4, 0, 0], qs[0][5], qs[0][6, 3, 63] = np.inf, np.nan, 0.0, -np.inf
    qs[0][7] *= np.float32(2.0 ** 60)                          # past the exponent's clamp (infinite in float16)
    qs[0][8] *= np.float32(2.0 ** -130)                        # subnormal (zero in float16)
    qs[0][9, 2, 5:9] = np.nan
    qs[0][9, 2, 9] = -300.0
    q = torch.from_numpy(qs[0]).to(DEV).to(dtype)
    t = lambda x: torch.from_numpy(x[None]).to(DEV).to(dtype)                 # noqa: E731
    alone = A.prefill(q.transpose(0, 1)[None], t(ks[0]), t(vs[0]))[0]
    assert same_bits(D.prefill_paged(q, lattice(ks, vs, False), cu_of(qs)), alone)


@pytest.mark.gpu
def test_many_short_sequences():
    """More sequences than the plan's threads, most of them idle or of a single row."""
    r = np.random.default_rng(3)
    lens = [int(x) for x in r.choice([1, 2, 17, 128, 130, 257], size=700)]
    qs, ks, vs = draw(lens, [0] * 700, 2, 1, 64, 12)
    act = torch.from_numpy(r.random(700) < 0.6).to(DEV)
    kv, cu = lattice(ks, vs, False), cu_of(qs)
    q = torch.from_numpy(np.concatenate(qs)).to(DEV)
    out = D.prefill_paged(q, kv, cu, active=act, out=torch.full_like(q, 4.0))
    for b in range(0, 700, 23):
        rows = out[cu[b]:cu[b + 1]]
        if act[b]:
            assert same_bits(rows, torch.from_numpy(oracle_rows(qs[b], ks[b], vs[b], 0, 0, False).copy()).to(DEV)), b
        else:
            assert (rows == 4.0).all()


@pytest.mark.gpu
def test_strides_idle_sequences_and_untouched_rows():
    lens, T0 = [200, 140, 90, 300], [128, 0, 0, 256]
    qs, ks, vs = draw(lens, T0, 4, 2, 64, 9)
    kv = lattice(ks, vs, False, extra_blocks=40)               # a lattice with room for long rows
    cu = cu_of(qs)
    n = int(cu[-1])
    q = torch.from_numpy(np.concatenate(qs)).to(DEV)
    want = D.prefill_paged(q, kv, cu)
    big = torch.randn(n + 30, 6, 2, 64, device=DEV)            # rows behind the last sequence, strided heads
    big[:n, :4, 0] = q
    store = torch.full((n + 30, 64, 4), 3.5, device=DEV)       # channels outermost in memory
    out = store.transpose(1, 2)
    act = torch.tensor([True, False, True, True], device=DEV)
    got = D.prefill_paged(big[:, :4, 0], kv, cu, active=act, out=out)
    assert got is out
    keep = torch.ones(n + 30, dtype=torch.bool, device=DEV)
    for b in (0, 2, 3):
        keep[cu[b]:cu[b + 1]] = False
        assert same_bits(out[cu[b]:cu[b + 1]], want[cu[b]:cu[b + 1]])
    assert (out[keep] == 3.5).all()
    none = torch.zeros(4, dtype=torch.bool, device=DEV)
    out.fill_(2.0)
    D.prefill_paged(big[:, :4, 0], kv, cu, active=none, out=out)
    assert (out == 2.0).all()
    assert D.prefill_paged(q[:0], kv, torch.zeros_like(cu)).shape == (0, 4, 64)


@pytest.mark.gpu
def test_lengths_that_break_the_rules_are_flagged():
    lens = [300, 128]
    qs, ks, vs = draw(lens, [0, 0], 2, 1, 64, 3)
    kv = lattice(ks, vs, False)
    q = torch.from_numpy(np.concatenate(qs)).to(DEV)
    good = D.prefill_paged(q, kv, cu_of(qs))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)           # noqa: E731
    for cu, P in ((i32(0, 200, 328), None),                    # sequence 0 would start at 100
                  (i32(0, 301, 428), None), (i32(0, 300, 429), None), (i32(300, 0, 128), None),
                  (i32(0, 300, 428), i32(301, 0)), (i32(0, 300, 428), i32(0, -1))):
        out = torch.full_like(q, 9.0)
        with pytest.raises(RuntimeError, match="bits 0x10 "):
            D.prefill_paged(q, kv, cu, prefix_lens=P, out=out)
    assert same_bits(D.prefill_paged(q, kv, cu_of(qs)), good)
    kv.block_table[1, 0] = 10 ** 6                             # a page outside the pool: flagged, page 0 read
    with pytest.raises(RuntimeError):
        D.prefill_paged(q, kv, cu_of(qs))


@pytest.mark.gpu
def test_streams_and_graphs_do_not_share_a_workspace():
    """Two captured calls and two streams at once, each with its own workspace; replayed on new lengths."""
    lens = [400, 129]
    qs, ks, vs = draw(lens, [0, 0], 4, 2, 128, 4)
    kv = lattice(ks, vs, False)
    q = torch.from_numpy(np.concatenate(qs)).to(DEV)
    q2, cu = q.flip(0).contiguous(), cu_of(qs)
    w1, w2 = D.prefill_paged(q, kv, cu), D.prefill_paged(q2, kv, cu)
    graphs, outs = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(D.prefill_paged(x, kv, cu, check=False))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert same_bits(outs[0], w1) and same_bits(outs[1], w2)
    eager = []
    for x, s in zip((q, q2), streams):
        with torch.cuda.stream(s):
            eager.append(D.prefill_paged(x, kv, cu, check=False))
    torch.cuda.synchronize()
    assert same_bits(eager[0], w1) and same_bits(eager[1], w2)
    cu.copy_(torch.tensor([0, 16, 145], dtype=torch.int32))    # sequence 0's last 16 rows, then all of sequence 1
    graphs[0].replay()
    torch.cuda.synchronize()
    assert same_bits(outs[0][:145], D.prefill_paged(q, kv, cu)[:145])


@pytest.mark.gpu
def test_argument_refusals():
    lens = [130]
    qs, ks, vs = draw(lens, [0], 4, 2, 64, 1)
    kv = lattice(ks, vs, False)
    q, cu = torch.from_numpy(qs[0]).to(DEV), cu_of(qs)
    for args, kw in (((q[None], kv, cu), {}), ((q, kv, cu.long()), {}), ((q, kv, cu[:1]), {}), ((q[:, :3], kv, cu), {}),
                     ((q[..., :32], kv, cu), {}), ((q, kv, cu), dict(prefix_lens=cu)),
                     ((q, kv, cu), dict(active=cu[:1])), ((q, kv, cu), dict(out=q[:5].clone())), ((q, kv, cu.cpu()), {})):
        with pytest.raises(ValueError):
            D.prefill_paged(*args, **kw)
    with pytest.raises(TypeError):
        D.prefill_paged(q.double(), kv, cu)


def test_c_entry_refusals():
    L = _lib.load()
    s, f = _lib.i64x([1, 1, 1]), 256

    def call(N=10, H=4, KVH=2, dh=64, B=1, mb=1, mp=8, npg=8, sink=0, ev0=f, q=f, ws=1 << 30, k8=f, v8=f):
        return L.lssab8_prefill_paged(q, 2, s, N, H, KVH, dh, f, f, None, None, B, f, mp, npg, k8, v8, f, f, ev0, mb, sink, f,
                                      2, s, f, ws, None)
    for kw in (dict(N=0), dict(H=3), dict(B=0), dict(mb=0), dict(mp=0), dict(npg=0), dict(npg=1 << 27), dict(q=None),
               dict(sink=1, ev0=None), dict(k8=f + 8), dict(v8=f + 1)):
        assert call(**kw) == 1, kw
    assert call(dh=96) == 2 and call(ws=100) == 4
    assert L.lssab8_prefill_paged_workspace_size(0, 4, 2, 64, 1) == 0
