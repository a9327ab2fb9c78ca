"""The engine seam with steps as schedulers pad them: idle rows (one over a live sequence's first page), query and out
longer than the step, projections that require a gradient.  Every step equals the same step without the padding, run by
another engine."""
import pytest
import torch

from lockstep_b200 import engine as E

pytestmark = pytest.mark.gpu
H, KVH, DH, PAGES = 8, 2, 128, 64


def bits(x):
    return x.detach().contiguous().view(torch.int16)


@pytest.mark.parametrize("sink", [False, True])
def test_padded_steps_equal_plain_ones(sink):
    g = torch.Generator("cuda").manual_seed(9)
    draw = lambda n, h: torch.randn((n, h, DH), generator=g, device="cuda").to(torch.bfloat16)       # noqa: E731
    atts = [E.Lssab8Attention(H, KVH, DH, PAGES, max_len=512, max_seqs=2, sink=sink) for _ in range(2)]
    caches = [torch.zeros(2, PAGES, 16, KVH, DH, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    pages = [list(range(0, 30)), list(range(30, 60))]
    lens = [0, 0]
    for new, prefill in (([256, 70], [True, True]), ([30, 1], [True, False]), ([1, 1], [False, False]), ([1, 1], [False, False])):
        n = sum(new)
        q, k, v = draw(n, H), draw(n, KVH), draw(n, KVH)
        slots = torch.tensor([pages[i][t // 16] * 16 + t % 16 for i in range(2) for t in range(lens[i], lens[i] + new[i])],
                             device="cuda")
        lens = [a + b for a, b in zip(lens, new)]
        table = torch.tensor(pages, dtype=torch.int32, device="cuda")
        meta = E.StepMeta([0, new[0], n], lens, table, slots, prefill)
        want = atts[0].forward(0, q, k, v, caches[0][0], caches[0][1], meta)
        idle = torch.full((1, 30), -1, dtype=torch.int32, device="cuda")
        over = idle.clone()
        over[0, 0] = pages[0][0]                                 # a stale row: the first sequence's first page
        meta = E.StepMeta([0, 0, new[0], new[0], n, n], [0, lens[0], 0, lens[1], 0],
                          torch.cat([idle, table[:1], over, table[1:], idle]), slots,
                          [False, prefill[0], True, prefill[1], True])
        out = torch.full((n + 5, H, DH), 7.0, device="cuda", dtype=torch.bfloat16)
        qpad = torch.cat([q, draw(3, H)]).requires_grad_(True)
        got = atts[1].forward(0, qpad, k, v, caches[1][0], caches[1][1], meta, out=out)
        assert got is out and torch.equal(bits(out[:n]), bits(want)) and (out[n:] == 7.0).all()
    a, b = (x.layers[0] for x in atts)
    for s in range(2):
        sa, sb = a.slot_of[pages[s][0]], b.slot_of[pages[s][0]]
        assert torch.equal(a.ek[sa], b.ek[sb]) and torch.equal(a.ev[sa], b.ev[sb]) and torch.equal(a.ev0[sa], b.ev0[sb])
    with pytest.raises(RuntimeError, match="start on page 0"):
        twice = E.StepMeta([0, 1, 2], [lens[0] + 1] * 2, table[[0, 0]], torch.zeros(2, dtype=torch.long, device="cuda"),
                           [False, False])
        atts[0].forward(0, q, k, v, caches[0][0], caches[0][1], twice)
