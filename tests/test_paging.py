"""Step tables: refusals on the CPU, and on the GPU against a plain loop."""
import random

import pytest
import torch

from lockstep_b200 import _lib
from lockstep_b200 import paging as P


def reference(lens, new, table, free, cap):
    table = [list(r) for r in table]
    qsl, slots, pos, seq, used = [0], [], [], [], 0
    for i, (a, m) in enumerate(zip(lens, new)):
        for p in range(-(-a // 16), -(-(a + m) // 16)):
            table[i][p] = free[used]
            used += 1
        for t in range(a, a + m):
            slots.append(table[i][t // 16] * 16 + t % 16)
            pos.append(t)
            seq.append(i)
        qsl.append(qsl[-1] + m)
    pad = cap - len(slots)
    return qsl, [a + m for a, m in zip(lens, new)], slots + [-1] * pad, pos + [0] * pad, seq + [-1] * pad, [used], table


def make(n, lo, hi, max_len, seed, spare=3):
    r = random.Random(seed)
    new = [r.randint(lo, hi) for _ in range(n)]
    lens = [r.choice([0, 15, 16, 17, r.randint(0, max_len)]) for _ in range(n)]
    have = [-(-a // 16) for a in lens]
    need = [-(-(a + m) // 16) - h for a, m, h in zip(lens, new, have)]
    pages = list(range(1000, 1000 + sum(have) + sum(need) + spare))
    r.shuffle(pages)
    width = max(max(h + x for h, x in zip(have, need)), 1)
    table, o = [], 0
    for h in have:
        table.append(pages[o:o + h] + [-1] * (width - h))
        o += h
    return lens, new, table, pages[o:]


def gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def got(t, table):
    return tuple(x.tolist() for x in (t.query_start_loc, t.seq_lens, t.slot_mapping, t.positions, t.seq_index,
                                      t.pages_used, table))


@pytest.mark.gpu
@pytest.mark.parametrize("n,lo,hi,max_len,pad", [(1, 1, 1, 40, 0), (1, 0, 0, 40, 0), (1, 700, 700, 40, 5), (64, 1, 1, 500, 0),
                                                 (33, 0, 60, 300, 7), (1000, 0, 3, 90, 1), (1025, 0, 40, 90, 100),
                                                 (16384, 0, 2, 30, 9), (5, 0, 5000, 20000, 1)])
def test_tables(n, lo, hi, max_len, pad):
    lens, new, table, free = make(n, lo, hi, max_len, n)
    cap = sum(new) + pad
    want = reference(lens, new, table, free, cap)
    bt = gpu(table)
    t = P.step_tables(gpu(lens), gpu(new), bt, gpu(free), cap)
    assert got(t, bt) == want
    bt2 = gpu([r + [5, 6] for r in table])                     # a wider table, a column slice of it
    P.step_tables(gpu(lens), gpu(new), bt2[:, :len(table[0])], gpu(free), cap, out=t)
    assert got(t, bt2[:, :len(table[0])]) == want and bt2[:, -2:].tolist() == [[5, 6]] * n


@pytest.mark.gpu
def test_replayed_with_new_lengths():
    lens, new, table, free = make(20, 0, 30, 100, 1)
    a, m, bt, f = gpu(lens), gpu(new), gpu(table), gpu(free)
    graph = torch.cuda.CUDAGraph()
    keep = bt.clone()
    with torch.cuda.graph(graph):
        t = P.step_tables(a, m, bt, f, 640, check=False)
    graph.replay()
    assert got(t, bt) == reference(lens, new, table, free, 640)
    new2 = [x // 2 for x in new]
    m.copy_(gpu(new2))
    bt.copy_(keep)
    graph.replay()
    assert got(t, bt) == reference(lens, new2, table, free, 640)


@pytest.mark.gpu
def test_lengths_that_do_not_fit_are_flagged():
    """Each fault raises, writes nothing out of place, and the next call is clean."""
    free = gpu([7, 8, 9])
    for lens, new, cap, width, nfree in (([0, -1], [1, 1], 9, 4, 3), ([0, 3], [1, -5], 9, 4, 3),       # negative
                                         ([0, 0], [40, 40], 80, 4, 3),                               # too few pages
                                         ([0, 0], [40, 1], 80, 2, 3),                                # table too narrow
                                         ([0, 0], [9, 9], 10, 4, 3),                                 # too few token slots
                                         ([1 << 30, 0], [5, 0], 9, 4, 3), ([20, 0], [1, 0], 9, 4, 3)):  # missing pages
        guard = torch.full((4, width + 2), -1, dtype=torch.int32, device="cuda")
        bt = guard[1:3, 1:width + 1]
        with pytest.raises(RuntimeError, match="bits 0x10 "):
            P.step_tables(gpu(lens), gpu(new), bt, free[:nfree], cap)
        inner = guard.clone()
        inner[1:3, 1:width + 1] = -1
        assert (inner == -1).all()
    t = P.step_tables(gpu([0, 0]), gpu([40, 1]), gpu([[-1] * 4] * 2), gpu([3, 4]), 41, check=False)   # one page short
    assert t.slot_mapping.tolist() == list(range(48, 80)) + [-1] * 9 and t.pages_used.item() == 2
    from lockstep_b200 import attention as A
    with pytest.raises(RuntimeError, match="bits 0x10 "):
        A.check_device_errors(t.seq_lens.device)
    P.step_tables(gpu([0]), gpu([1]), gpu([[-1]]), free, 1)


@pytest.mark.gpu
def test_refusals_gpu():
    a, bt, f = gpu([0, 0]), gpu([[-1], [-1]]), gpu([1])
    t = P.step_tables(a, a, bt, f, 0)
    assert t.query_start_loc.tolist() == [0, 0, 0]
    for args in ((a, a[:1], bt, f, 1), (a, a, bt[:1], f, 1), (a, a, bt[0], f, 1), (a, a, bt.expand(2, 1), f, -1),
                 (a, a, bt[:1].expand(2, 1), f, 1), (a[:0], a[:0], bt[:0], f, 1)):
        with pytest.raises(ValueError):
            P.step_tables(*args)
    with pytest.raises(TypeError):
        P.step_tables(a.long(), a, bt, f, 1)
    with pytest.raises(ValueError):
        P.step_tables(a, a, bt, f, 1, out=t)                   # another token capacity
    t1 = P.alloc_step_tables(2, 1, a.device)
    t1.seq_lens = a
    with pytest.raises(ValueError):
        P.step_tables(a, a.clone(), bt, f, 1, out=t1)


def test_refusals_cpu():
    a = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        P.step_tables(a, a, torch.zeros(2, 1, dtype=torch.int32), a, 4)
    L = _lib.load()
    f = 256
    args = lambda n=2, mp=4, ts=4, nf=3, cap=5: (f, f, n, f, ts, mp, f, nf, cap, f, f, f, f, f, f, None)   # noqa: E731
    for kw in (dict(n=0), dict(mp=0), dict(ts=3), dict(nf=-1), dict(cap=-1)):
        assert L.lssab8_step_tables(*args(**kw)) == 1
    assert L.lssab8_step_tables(*args(n=16385)) == 2
    bad = list(args())
    bad[0] = None
    assert L.lssab8_step_tables(*bad) == 1
