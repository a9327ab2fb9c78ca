"""The serving-step operators as an engine uses them together: step tables on the device, rotary positions fused with
the float-cache store, the lattice append, packed prompt rows and generated rows (engine.Lssab8Attention), then
sequences forked from one prompt decoded over their shared pages -- every row against the oracle on keys and queries
rotated by the same kernel."""
import numpy as np
import pytest
import torch

import oracle as O
from lockstep_b200 import decode as D
from lockstep_b200 import engine as E
from lockstep_b200 import rotary as R

pytestmark = pytest.mark.gpu
H, KVH, DH, PAGES, WIDTH = 8, 2, 128, 160, 64


def bits(x):
    return x.cpu().view(torch.int16).numpy().view(np.uint16)


def rows(q, k, v, n, sink):
    """The last n rows of a sequence, q / k / v [L, heads, dh] bf16."""
    f = lambda x: x.float().cpu().numpy().transpose(1, 0, 2)                  # noqa: E731
    L = k.shape[0]
    full = np.zeros((H, L, DH), np.float32)
    full[:, L - n:] = f(q[-n:])
    return O.f32_to_bf16_bits(O.attention(full, f(k), f(v), sink=sink, rows=np.arange(L - n, L)).transpose(1, 0, 2)[L - n:])


@pytest.mark.parametrize("sink", [False, True])
def test_engine_steps_with_tables_and_rotary(sink):
    plan = R.make_plan(DH, layout="interleaved", scaling={"kind": "bands", "factor": 4.0, "original": 128})
    att = E.Lssab8Attention(H, KVH, DH, PAGES, max_len=WIDTH * 16, max_seqs=4, sink=sink, rotary=plan)
    cache = torch.zeros(PAGES, 2, 16, KVH, DH, dtype=torch.bfloat16, device="cuda")
    free = torch.randperm(PAGES, device="cuda").to(torch.int32)
    table = torch.full((3, WIDTH), -1, dtype=torch.int32, device="cuda")
    lens, hist = [0, 0, 0], [[], [], []]
    g = torch.Generator("cuda").manual_seed(3)
    # three sequences from the start: prompts in 128-aligned chunks beside generated rows
    for new, prefill in (([256, 100, 1], [True] * 3), ([44, 1, 1], [True, False, False]), ([1, 1, 1], [False] * 3)):
        meta, used = E.StepMeta.build(lens, new, prefill, table, free)
        free = free[used:]
        qkv = torch.randn((sum(new), H + 2 * KVH, DH), generator=g, device="cuda").to(torch.bfloat16)
        q, k, v = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
        out = att.forward(0, q, k, v, cache[:, 0], cache[:, 1], meta)
        at = 0
        for i, n in enumerate(new):
            pos = torch.arange(lens[i], lens[i] + n, device="cuda")
            s = slice(at, at + n)
            hist[i].append((R.rotate(q[s].contiguous(), pos, plan), R.rotate(k[s].contiguous(), pos, plan), v[s]))
            lens[i] += n
            at += n
            qq, kk, vv = (torch.cat(x) for x in zip(*hist[i]))
            assert np.array_equal(bits(out[s]), rows(qq, kk, vv, n, sink)), (new, i)
    with pytest.raises(ValueError, match="free"):
        E.StepMeta.build(lens, [16 * PAGES, 0, 0], [True] * 3, table, free)
    meta, _ = E.StepMeta.build(lens, [1, 1, 1], [False] * 3, table, free)
    meta.positions = None
    with pytest.raises(ValueError, match="positions"):
        att.forward(0, q[:3], k[:3], v[:3], cache[:, 0], cache[:, 1], meta)


@pytest.mark.parametrize("sink", [False, True])
def test_forked_sequences_over_their_shared_prompt(sink):
    B, shared = 6, 300
    plan = R.make_plan(DH)
    cache = torch.zeros(PAGES, 2, 16, KVH, DH, dtype=torch.bfloat16, device="cuda")
    free = torch.randperm(PAGES, device="cuda").to(torch.int32)
    g = torch.Generator("cuda").manual_seed(5)
    draw = lambda n: torch.randn((n, H + 2 * KVH, DH), generator=g, device="cuda").to(torch.bfloat16)    # noqa: E731
    split = lambda x: (x[:, :H], x[:, H:H + KVH], x[:, H + KVH:])             # noqa: E731

    def store(meta, qkv, kv, lens):
        q = R.rotate_append(*split(qkv), meta.positions, meta.slot_mapping, cache[:, 0], cache[:, 1], plan)
        D.append_kv(kv, cache[:, 0], cache[:, 1], torch.tensor(lens, dtype=torch.int32, device="cuda"),
                    src_block_table=kv.block_table)
        return q

    # the prompt, once
    t1 = torch.full((1, WIDTH), -1, dtype=torch.int32, device="cuda")
    meta, used = E.StepMeta.build([0], [shared], [True], t1, free)
    free = free[used:]
    kv1 = D.empty_paged_kv(1, KVH, DH, WIDTH * 16, t1, PAGES, sink=sink)
    prompt = draw(shared)
    qp = store(meta, prompt, kv1, [shared])
    out = D.prefill_paged(qp, kv1, torch.tensor([0, shared], dtype=torch.int32, device="cuda"))
    kp, vp = cache[:, 0], cache[:, 1]
    pg = t1[0, :-(-shared // 16)].long()
    kr, vr = (x[pg].reshape(-1, KVH, DH)[:shared] for x in (kp, vp))
    assert np.array_equal(bits(out), rows(qp, kr, vr, shared, sink))
    # forks: whole shared blocks by page, the open block's tokens stored again in pages of their own
    whole = shared // 128 * 128
    table = torch.full((B, WIDTH), -1, dtype=torch.int32, device="cuda")
    table[:, :whole // 16] = t1[:, :whole // 16]
    kv = D.PagedKV(k8p=kv1.k8p, v8p=kv1.v8p, ek=kv1.ek.repeat(B, 1, 1), ev=kv1.ev.repeat(B, 1, 1), ev0=kv1.ev0.repeat(B, 1),
                   block_table=table, seq_lens=torch.full((B,), whole, dtype=torch.int32, device="cuda"),
                   max_blocks=kv1.max_blocks, num_pages=PAGES, sink=sink)
    new = [shared - whole + i * 9 for i in range(B)]
    meta, used = E.StepMeta.build([whole] * B, new, [True] * B, table, free)
    free = free[used:]
    own = [torch.cat([prompt[whole:], draw(i * 9)]) for i in range(B)]
    lens = [whole + n for n in new]
    store(meta, torch.cat(own), kv, lens)
    for _ in range(2):                                         # generated rows
        meta, used = E.StepMeta.build(lens, [1] * B, [False] * B, table, free)
        free, lens = free[used:], [x + 1 for x in lens]
        q = store(meta, draw(B), kv, lens)
        got = D.decode_shared(q, kv, shared)
        assert torch.equal(got.view(torch.int16), D.decode(q, kv).view(torch.int16))
        for b in range(B):
            pg = table[b, :-(-lens[b] // 16)].long()
            k, v = (x[pg].reshape(-1, KVH, DH)[:lens[b]] for x in (kp, vp))
            assert np.array_equal(bits(got[b:b + 1]), rows(q[b:b + 1], k, v, 1, sink)), b
