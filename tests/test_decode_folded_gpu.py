"""decode_shared where whole segments of the prefix are folded in the shared-prefix kernel, over several row tiles: rows
bit for bit the plain decode and the oracle, idle first sequences, short and foreign ones, streams and graphs.  Every
case asserts that its segments are folded (the workspace then holds no partials for them)."""
import numpy as np
import pytest
import torch

import oracle as O
from lockstep_b200 import _lib
from lockstep_b200 import decode as D

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def make(H, KVH, dh, shared, own, sink, seed=0):
    """Queries bf16 [B, H, dh], and a lattice of B sequences on one set of pages for the whole shared blocks."""
    g = torch.Generator("cuda").manual_seed(seed + H)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)       # noqa: E731
    B, pages, nb = len(own), shared // 128 * 8, -(-(shared + max(own)) // 128)
    k, v = (torch.cat([draw(KVH, shared, dh).expand(B, -1, -1, -1), draw(B, KVH, nb * 128 - shared, dh)], 2)
            for _ in range(2))
    lens = [shared + n for n in own]
    total = pages + sum(-(-x // 16) - pages for x in lens)
    perm, at = torch.randperm(total, generator=g, device="cuda").to(torch.int32), pages
    bt = torch.full((B, nb * 8), -1, dtype=torch.int32, device="cuda")
    for b, x in enumerate(lens):
        n = -(-x // 16) - pages
        bt[b, :pages], bt[b, pages:pages + n] = perm[:pages], perm[at:at + n]
        at += n
    kv = D.build_paged_kv(k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), bt, total, sink=sink)
    size = _lib.load().lssab8_decode_shared_workspace_size(B, H, KVH, dh, kv.max_blocks, shared)
    assert size < B * H * kv.max_blocks * dh * 4, "this case folds no segment"
    return draw(B, H, dh), k, v, kv


CASES = [  # H, KVH, dh, shared, own lengths
    (256, 32, 64, 4300, [(7 * b) % 150 for b in range(40)]),           # 3 tiles of 16 sequences, the last of 8
    (128, 16, 128, 8500, [b % 3 for b in range(33)]),                  # 2 segments, then partials; a tile of one sequence
    (96, 32, 128, 4100, [5 * b % 131 for b in range(90)]),             # groups of 3: tiles of 42 sequences and 2 rows to spare
    (48, 48, 64, 4096, [b % 2 for b in range(129)]),                   # the segment is the whole prefix
]


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("H,KVH,dh,shared,own", CASES)
def test_folded_rows_over_several_tiles(H, KVH, dh, shared, own, sink):
    q, k, v, kv = make(H, KVH, dh, shared, own, sink)
    got = D.decode_shared(q, kv, shared)
    assert same(got, D.decode(q, kv))
    f = lambda x: x.float().cpu().numpy()                              # noqa: E731
    group = H // KVH
    for b, g in ((0, 0), (len(own) - 1, KVH - 1), (len(own) // 2, 1)):
        L, hs = shared + own[b], slice(g * group, (g + 1) * group)
        ref = O.decode_rows(f(q[b, hs]), f(k[b, g:g + 1, :L]), f(v[b, g:g + 1, :L]), sink=sink)
        assert np.array_equal(O.f32_to_bf16_bits(ref), got[b, hs].cpu().view(torch.int16).numpy().view(np.uint16)), (b, g)


@pytest.mark.parametrize("H,KVH,dh,shared,own", CASES[:3])
def test_folded_idle_short_and_foreign_sequences(H, KVH, dh, shared, own):
    q, k, v, kv = make(H, KVH, dh, shared, own, True, seed=1)
    B, want, lens = len(own), D.decode(q, kv), kv.seq_lens.clone()
    for idle in (list(range(17)), [1, B - 1], list(range(B - 1)), list(range(B))):     # a whole first tile among them
        kv.seq_lens = lens.clone()
        kv.seq_lens[idle] = 0
        out = torch.full_like(q, 5.0)
        D.decode_shared(q, kv, shared, out=out)
        live = [b for b in range(B) if b not in idle]
        assert (out[idle] == 5.0).all() and same(out[live], want[live])
    kv.seq_lens = lens.clone()
    kv.seq_lens[0], kv.seq_lens[20] = shared // 128 * 128 - 1, 4000                    # the first one too: not the leader
    out = torch.full_like(q, 5.0)
    with pytest.raises(RuntimeError, match="bits 0x10 "):
        D.decode_shared(q, kv, shared, out=out)
    live = [b for b in range(B) if b not in (0, 20)]
    assert (out[[0, 20]] == 5.0).all() and same(out[live], want[live])
    kv.seq_lens = lens
    b, last = B - 1, shared // 128 - 1
    for x, at in ((kv.block_table, (b, 8)), (kv.ek, (b, KVH - 1, 0)), (kv.ev, (b, 0, last)), (kv.ev0, (b, KVH - 1))):
        keep = x[at].item()
        x[at] = keep + 1 if x is not kv.block_table else kv.block_table[b, 9].item()   # (a page of the pool)
        out = torch.full_like(q, 5.0)
        with pytest.raises(RuntimeError, match="bits 0x10 "):
            D.decode_shared(q, kv, shared, out=out)
        assert same(out[:b], want[:b])
        x[at] = keep
    assert same(D.decode_shared(q, kv, shared), want)


@pytest.mark.parametrize("H,KVH,dh,shared,own", CASES[:2])
def test_folded_calls_side_by_side(H, KVH, dh, shared, own):
    q1, k, v, kv = make(H, KVH, dh, shared, own, False, seed=2)
    q2 = q1.flip(0).contiguous()
    want, graphs, outs = [D.decode(q1, kv), D.decode(q2, kv)], [], []
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
        assert same(outs[0], want[0]) and same(outs[1], want[1])
        eager = []
        for x, s in zip((q1, q2), streams):
            with torch.cuda.stream(s):
                eager.append(D.decode_shared(x, kv, shared, check=False))
        torch.cuda.synchronize()
        assert same(eager[0], want[0]) and same(eager[1], want[1])
    kv.seq_lens[0] = 0                                                 # replayed with another leader
    graphs[0].replay()
    torch.cuda.synchronize()
    assert same(outs[0][1:], want[0][1:])
