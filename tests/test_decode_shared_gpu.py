"""Decode over a prefix that the batch shares (decode.decode_shared): bit for bit the plain decode of the same
lattice, and the oracle's rows; groups of 1 to 8 heads, tiles with rows to spare, prefixes that end inside a block,
at a sequence's end, and across fold segments; idle, short and foreign sequences; streams and graphs."""
import numpy as np
import pytest
import torch

import oracle as O
from fixtures import ftz_cases, jump_cases
from lockstep_b200 import _lib
from lockstep_b200 import attention as A
from lockstep_b200 import decode as D
from lockstep_b200 import workloads as W

DEV = "cuda"
BITS = {torch.float32: torch.int32, torch.float16: torch.int16, torch.bfloat16: torch.int16}


def same_bits(a, b):
    return torch.equal(a.contiguous().view(BITS[a.dtype]), b.contiguous().view(BITS[b.dtype]))


def shared_lattice(pk, pv, ks, vs, sink):
    """Sequences prefix + own tokens (float32 numpy [KVH, L, dh]), whose whole shared blocks are one set of pages."""
    KVH, Lp, dh = pk.shape
    pages = Lp // 128 * 8
    lens = [Lp + k.shape[1] for k in ks]
    nb = max(-(-L // 128) for L in lens)
    total = pages + sum(-(-L // 16) - pages for L in lens)
    perm = np.random.default_rng(7).permutation(total).astype(np.int32)
    bt, o = np.full((len(ks), nb * 8), -1, np.int32), pages
    for b, L in enumerate(lens):
        n = -(-L // 16) - pages
        bt[b, :pages], bt[b, pages:pages + n] = perm[:pages], perm[o:o + n]
        o += n
    dense = lambda p, own: torch.from_numpy(np.stack([np.concatenate(    # noqa: E731
        [p, x, np.zeros((KVH, nb * 128 - Lp - x.shape[1], dh), np.float32)], 1) for x in own])).to(DEV)
    return D.build_paged_kv(dense(pk, ks), dense(pv, vs), torch.tensor(lens, dtype=torch.int32, device=DEV),
                            torch.from_numpy(bt).to(DEV), total, sink=sink)


def draw(B, H, KVH, dh, Lp, own, seed):
    r = np.random.default_rng(seed)
    f = lambda *s: W.bf16_round(r.standard_normal(s).astype(np.float32))          # noqa: E731
    return (f(B, H, dh), f(KVH, Lp, dh), f(KVH, Lp, dh), [f(KVH, x, dh) for x in own], [f(KVH, x, dh) for x in own])


CASES = [  # H, KVH, dh, shared, own lengths
    (1, 1, 128, 128, [0]),                                     # nothing of its own
    (4, 4, 64, 200, [1]),
    (8, 2, 128, 256, [0, 1, 127, 128, 129]),
    (14, 2, 64, 300, [5, 200, 84, 1]),
    (6, 2, 128, 1000, [30, 0, 24, 25, 700]),                   # groups of 3: 126 rows a tile
    (8, 1, 128, 640, list(range(1, 40))),                      # 16 sequences a tile, the last one short
    (5, 5, 64, 384, list(range(0, 135))),                      # 128 sequences a tile
    (10, 2, 128, 515, [3] * 26),                               # groups of 5: 25 sequences a tile
    (4, 1, 128, 4096, [100, 0]),                               # a whole fold segment
    (8, 1, 128, 4300, [0, 4000, 60]),                          # across segments, shared and own
    (4, 2, 64, 8400, [10, 100, 300]),
    (64, 64, 64, 4300, [0, 5]),                                # enough kv heads that whole segments are folded
    (128, 64, 128, 4100, [0, 200, 60]),
    (384, 48, 128, 8500, [30, 1]),                             # two folded segments, then partials
]


@pytest.mark.gpu
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("H,KVH,dh,shared,own", CASES)
def test_rows_equal_decode_and_oracle(H, KVH, dh, shared, own, sink):
    q, pk, pv, ks, vs = draw(len(own), H, KVH, dh, shared, own, shared + H)
    kv = shared_lattice(pk, pv, ks, vs, sink)
    qt = torch.from_numpy(q).to(DEV)
    want = D.decode(qt, kv)
    got = D.decode_shared(qt, kv, shared)
    assert same_bits(got, want)
    for dt in (torch.bfloat16, torch.float16):
        assert same_bits(D.decode_shared(qt, kv, shared, out_dtype=dt), want.to(dt))
    assert same_bits(D.decode_shared(qt.to(torch.bfloat16), kv, shared, out_dtype=torch.float32), want)
    if shared >= 384:                                          # any number of shared blocks gives the same rows
        assert same_bits(D.decode_shared(qt, kv, 130), want) and same_bits(D.decode_shared(qt, kv, 300), want)
    assert same_bits(D.decode_shared(qt, kv, 127), want)       # less than a block: the plain decode
    for b in (0, len(own) - 1):
        ref = O.decode_rows(q[b], np.concatenate([pk, ks[b]], 1), np.concatenate([pv, vs[b]], 1), sink=sink)
        assert same_bits(got[b], torch.from_numpy(ref).to(DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("cut", [128, 256, 384])
def test_fixture_rows(cut):
    """The exponent jumps and flush ladders of the contract's selftest, cut into shared and own blocks."""
    for c in jump_cases() + ftz_cases():
        T = c["k"].shape[1]
        if T <= cut:
            continue
        H, k, v = c["q"].shape[0], c["k"], c["v"]
        own = [T - cut, 1, T - cut]
        q = np.stack([c["q"][:, T - 1], c["q"][:, cut], c["q"][:, T - 1] * np.float32(0.5)])
        kv = shared_lattice(k[:, :cut], v[:, :cut], [k[:, cut:cut + x] for x in own], [v[:, cut:cut + x] for x in own],
                            False)
        got = D.decode_shared(torch.from_numpy(q).to(DEV), kv, cut)
        for b, x in enumerate(own):
            ref = O.decode_rows(q[b], k[:, :cut + x], v[:, :cut + x])
            assert same_bits(got[b], torch.from_numpy(ref).to(DEV)), (c["tag"], b)
        assert H == got.shape[1]


@pytest.mark.gpu
def test_folded_segments_of_fixture_rows():
    """The same jumps and ladders, tiled past a fold segment over enough kv heads that the segment is folded whole."""
    for c in jump_cases()[::3] + ftz_cases()[::2]:
        reps = -(-4200 // c["k"].shape[1])
        k, v = (np.tile(x, (48, reps, 1))[:, :4200] for x in (c["k"], c["v"]))
        q = np.tile(c["q"][:1, -1], (48, 1))
        q = np.stack([q, q * np.float32(0.25)])
        kv = shared_lattice(k[:, :4100], v[:, :4100], [k[:, 4100:], k[:, 4100:4101]], [v[:, 4100:], v[:, 4100:4101]], False)
        qt = torch.from_numpy(q).to(DEV)
        assert same_bits(D.decode_shared(qt, kv, 4100), D.decode(qt, kv)), c["tag"]


@pytest.mark.gpu
def test_queries_that_are_not_finite():
    q, pk, pv, ks, vs = draw(2, 8, 2, 128, 300, [9, 1], 8)
    kv = shared_lattice(pk, pv, ks, vs, False)
    q[0, 1, 3], q[0, 2, 5], q[1, 0], q[1, 7, 64] = np.inf, np.nan, 0.0, -np.inf
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        qt = torch.from_numpy(q).to(DEV).to(dt)
        assert same_bits(D.decode_shared(qt, kv, 300), D.decode(qt, kv))


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [300, 8300])
def test_idle_short_and_foreign_sequences(shared):
    own = [20, 40, 60, 80]
    q, pk, pv, ks, vs = draw(4, 8, 2, 128, shared, own, 11)
    kv = shared_lattice(pk, pv, ks, vs, True)
    qt = torch.from_numpy(q).to(DEV)
    want = D.decode(qt, kv)
    lens = kv.seq_lens.clone()
    for idle in ([0], [1, 3], [0, 1, 2, 3]):                   # idle sequences, the first of the batch among them
        kv.seq_lens = lens.clone()
        kv.seq_lens[idle] = 0
        out = torch.full_like(qt, 5.0)
        assert D.decode_shared(qt, kv, shared, out=out) is out
        for b in range(4):
            assert (out[b] == 5.0).all() if b in idle else same_bits(out[b], want[b])
    kv.seq_lens = lens.clone()
    kv.seq_lens[2] = shared // 128 * 128 - 1                   # does not hold the shared blocks
    out = torch.full_like(qt, 5.0)
    with pytest.raises(RuntimeError, match="bits 0x10 "):
        D.decode_shared(qt, kv, shared, out=out)
    assert (out[2] == 5.0).all() and same_bits(out[[0, 1, 3]], want[[0, 1, 3]])
    kv.seq_lens = lens
    keep = kv.block_table.clone()
    kv.block_table[1, shared // 128 * 8 - 1] = kv.block_table[1, shared // 128 * 8]      # one page is not the shared one
    with pytest.raises(RuntimeError, match="bits 0x10 "):
        D.decode_shared(qt, kv, shared)
    kv.block_table.copy_(keep)
    for name in ("ek", "ev"):
        getattr(kv, name)[3, 1, shared // 128 - 1] += 1        # nor is an exponent
        with pytest.raises(RuntimeError, match="bits 0x10 "):
            D.decode_shared(qt, kv, shared)
        getattr(kv, name)[3, 1, shared // 128 - 1] -= 1
    kv.block_table[:, 0] = kv.num_pages                        # a page outside the pool: flagged, page 0 read
    with pytest.raises(RuntimeError, match="bits 0x4 "):
        D.decode_shared(qt, kv, shared)
    kv.block_table.copy_(keep)
    assert same_bits(D.decode_shared(qt, kv, shared), want)


@pytest.mark.gpu
def test_strided_queries_and_outputs():
    q, pk, pv, ks, vs = draw(3, 8, 2, 128, 260, [9, 1, 140], 2)
    kv = shared_lattice(pk, pv, ks, vs, False)
    qt = torch.from_numpy(q).to(DEV)
    want = D.decode(qt, kv)
    wide = torch.randn(3, 12, 130, device=DEV)
    wide[:, 2:10, 1:129] = qt
    out = torch.zeros(128, 3, 8, device=DEV).permute(1, 2, 0)
    D.decode_shared(wide[:, 2:10, 1:129], kv, 260, out=out)
    assert same_bits(out, want)
    with pytest.raises(ValueError):
        D.decode_shared(qt, kv, 260, out=torch.zeros(3, 8, 64, device=DEV))
    with pytest.raises(ValueError):
        D.decode_shared(qt, kv, 260, out=torch.zeros(3, 1, 128, device=DEV).expand(3, 8, 128))
    for dev in (None, "cuda", torch.device("cuda"), qt.device):        # every way to name the device
        A.check_device_errors(dev)
    with pytest.raises(ValueError):
        D.decode_shared(qt, kv, 128 * (kv.max_blocks + 1))
    with pytest.raises(ValueError):
        D.decode_shared(qt, kv, -1)
    with pytest.raises(ValueError):
        D.decode_shared(qt[:2], kv, 260)
    with pytest.raises(ValueError):
        D.decode_shared(qt[..., :64], kv, 260)


@pytest.mark.gpu
@pytest.mark.parametrize("dh,shared", [(128, 4300), (64, 500)])
def test_streams_and_graphs_do_not_share_a_workspace(dh, shared):
    q, pk, pv, ks, vs = draw(5, 8, 2, dh, shared, [9, 1, 140, 0, 33], 6)
    kv = shared_lattice(pk, pv, ks, vs, False)
    q1 = torch.from_numpy(q).to(DEV)
    q2 = q1.flip(0).contiguous()
    w1, w2 = D.decode(q1, kv), D.decode(q2, kv)
    graphs, outs = [], []
    for x in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(D.decode_shared(x, kv, shared, check=False))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert same_bits(outs[0], w1) and same_bits(outs[1], w2)
    kv.seq_lens[2] -= 7                                        # replayed on another length
    graphs[0].replay()
    torch.cuda.synchronize()
    assert same_bits(outs[0][[0, 1, 3, 4]], w1[[0, 1, 3, 4]])
    eager = []
    for x, s in zip((q1, q2), streams):
        with torch.cuda.stream(s):
            eager.append(D.decode_shared(x, kv, shared, check=False))
    torch.cuda.synchronize()
    assert same_bits(eager[0], outs[0]) and same_bits(eager[1][[0, 1, 3, 4]], w2[[0, 1, 3, 4]])


def test_c_entry_refusals():
    L = _lib.load()
    s, f = _lib.i64x([1, 1, 1]), 256

    def call(B=2, H=4, KVH=2, dh=64, shared=128, mp=8, npg=8, mb=1, sink=0, ev0=f, q=f, k8=f, v8=f):
        return L.lssab8_decode_shared(q, 2, s, B, H, KVH, dh, f, shared, f, mp, npg, k8, v8, f, f, ev0, mb, sink, f, 2, s, f,
                                      1 << 40, None)
    for kw in (dict(B=0), dict(H=3), dict(shared=127), dict(shared=256), dict(mb=0), dict(mp=0), dict(npg=0),
               dict(npg=1 << 27), dict(q=None), dict(sink=1, ev0=None), dict(B=70000), dict(k8=f + 8),
               dict(v8=f + 1)):
        assert call(**kw) == 1, kw
    assert call(dh=96) == 2 and call(H=18, KVH=2) == 2
    assert L.lssab8_decode_shared_workspace_size(2, 4, 2, 64, 1, 127) == 0
