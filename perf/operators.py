"""The serving-step operators, as they are measured: their cases, inputs, plain forms and 64-bit values.

Four operators of one engine step around the contract attention (lockstep_b200):

  rotate / append   rotary positions: the rotation and its gradient (rotary.rotate), and the step's fused form that
                    rotates queries and keys and stores keys and values in the paged float cache (rotary.rotate_append)
  tables            block tables, slots and positions of a step from its request lengths (paging.step_tables)
  prefill           all prompt rows of a step over the paged int8 lattice in one call, each sequence apart (document
                    mask), with an optional bidirectional prefix (prefix mask) (decode.prefill_paged)
  shared            one decode step of a batch whose sequences share their first pages (decode.decode_shared)

`run` computes the plain forms from elementary torch operations when `own` is false, and calls the framework when it is
true.  Shapes follow the repository's benchmark configurations (32 or 64 query heads, 4 or 8 kv heads of 128 channels,
8 heads of 64, 16-token pages, 8,192 and 32,768 positions) and odd sizes around them.
"""
import math
import random

import torch

own = False

PAGE, KB, SEG, SKIP = 16, 128, 32, 32      # tokens a page, keys a block, blocks a fold segment, skip window
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step's tokens (one per sequence of the paged-decode configuration): latency
        dict(name="append_step", op="append", tokens=64, H=32, KVH=4, dh=128, rot=128, layout="half", scaling="none",
             dtype="bf16", cache="bf16", max_pos=32768, pad=0),
        # a step that prefills two 8,192-token prompts of the 64-head model with a long-context scaling
        dict(name="append_prompt", op="append", tokens=16384, H=64, KVH=8, dh=128, rot=128, layout="half",
             scaling="bands", dtype="bf16", cache="bf16", max_pos=262144, pad=0),
        # training rows: rotation and gradient, part of each head, interleaved pairs
        dict(name="rotate_grad", op="rotate", B=4, H=32, T=2047, dh=128, rot=64, layout="interleaved", scaling="linear",
             dtype="f32", max_pos=131072),
        # a decode step of 64 sequences
        dict(name="tables_step", op="tables", n=64, max_len=32768, new_lo=1, new_hi=1, lseed=1),
        # a mixed step: 1,000 sequences, prompts of up to 250 tokens among them, idle ones too
        dict(name="tables_mixed", op="tables", n=1000, max_len=4096, new_lo=0, new_hi=250, lseed=2),
        # three short prompts of the 8-head model, one of a single token
        dict(name="prefill_short", op="prefill", lens="1 77 260", T0="0 0 0", P="", H=8, KVH=8, dh=64,
             dtype="f32", sink=False),
        # ragged prompts packed into one step (32 heads on 8)
        dict(name="prefill_packed", op="prefill", lens="8192 2048 511 1300 90 4096 129 333",
             T0="0 0 0 0 0 0 0 0", P="", H=32, KVH=8, dh=128, dtype="bf16", sink=False),
        # chunks of longer prompts with bidirectional prefixes, sink on
        dict(name="prefill_prefix", op="prefill", lens="5000 2500 700 1", T0="2048 0 512 0",
             P="2600 1000 0 1", H=32, KVH=4, dh=128, dtype="f16", sink=True),
        # a few sequences on a short common instruction, 64-channel heads
        dict(name="shared_small", op="shared", B=3, H=8, KVH=8, dh=64, shared=640, own_lo=0, own_hi=70, dtype="f16",
             sink=False, lseed=3),
        # the decode configuration's batch on one 8,192-token prefix
        dict(name="shared_batch", op="shared", B=32, H=32, KVH=8, dh=128, shared=8192, own_lo=1, own_hi=1024,
             dtype="bf16", sink=False, lseed=4),
        # the paged-decode configuration's batch on one 32,768-token prefix, sink on
        dict(name="shared_long", op="shared", B=64, H=32, KVH=4, dh=128, shared=32768, own_lo=1, own_hi=2048,
             dtype="bf16", sink=True, lseed=5),
        # a group of 7 heads, a prefix that ends inside a block, several rows a tile short
        dict(name="shared_odd", op="shared", B=21, H=28, KVH=4, dh=128, shared=5000, own_lo=3, own_hi=300, dtype="f32",
             sink=True, lseed=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "rotate", "tables", "prefill", "prefill", "shared", "shared"])
    dt = rng.choice(["bf16", "f16", "f32"])
    if op in ("append", "rotate"):
        dh = rng.choice([64, 128])
        c = dict(op=op, dh=dh, rot=rng.choice([dh, dh // 2, 2 * rng.randint(1, dh // 2)]), dtype=dt,
                 layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "bands"]),
                 max_pos=_log(rng, 64, 1 << 20))
        if op == "append":
            kvh = rng.choice([1, 2, 4, 8])
            c.update(tokens=_log(rng, 1, 8192), H=kvh * rng.choice([1, 4, 7, 8]), KVH=kvh,
                     cache=rng.choice(["bf16", "f16", dt]), pad=rng.choice([0, 0, rng.randint(1, 20)]))
        else:
            c.update(B=rng.randint(1, 4), H=rng.choice([1, 5, 8, 32]), T=_log(rng, 1, 2000))
        return c
    if op == "tables":
        lo = rng.choice([0, 1])
        return dict(op=op, n=_log(rng, 1, 1000), max_len=_log(rng, 64, 8192), new_lo=lo,
                    new_hi=max(lo, _log(rng, 1, 200)), lseed=rng.randrange(1 << 30))
    dh = rng.choice([64, 128, 128])
    kvh = rng.choice([1, 2, 4, 8])
    H = kvh * rng.choice([1, 2, 4, 7, 8] if kvh < 8 or op == "shared" else [1, 2, 4])
    sink = rng.random() < 0.5
    if op == "prefill":
        lens, T0, P = [], [], []
        prefixes = rng.random() < 0.5
        for _ in range(rng.randint(1, 6)):
            L = _log(rng, 1, 2500)
            lens.append(L)
            T0.append(KB * rng.randrange(0, (L - 1) // KB + 1) if rng.random() < 0.4 else 0)
            P.append(rng.randint(0, L) if prefixes else 0)
        text = lambda v: " ".join(map(str, v))                                  # noqa: E731
        return dict(op=op, lens=text(lens), T0=text(T0), P=text(P) if prefixes else "", H=H, KVH=kvh, dh=dh, dtype=dt, sink=sink)
    hi = _log(rng, 1, 1500)
    return dict(op=op, B=_log(rng, 1, 64), H=H, KVH=kvh, dh=dh, shared=_log(rng, 20, 14000), own_lo=rng.randint(1, hi),
                own_hi=hi, dtype=dt, sink=sink, lseed=rng.randrange(1 << 30))


def _spec(case):
    """(length, first row, bidirectional prefix) of each sequence of a prefill case."""
    ints = lambda t: [int(x) for x in t.split()]                                # noqa: E731
    lens = ints(case["lens"])
    return list(zip(lens, ints(case["T0"]), ints(case["P"]) or [0] * len(lens)))


def _own_lens(case):
    r = random.Random(case["lseed"])
    return [r.randint(case["own_lo"], case["own_hi"]) for _ in range(case["B"])]


def _table_lens(case):
    r = random.Random(case["lseed"])
    before, new = [], []
    for _ in range(case["n"]):
        m = r.randint(case["new_lo"], case["new_hi"])
        if case["new_hi"] > 1 and r.random() < 0.6:      # most sequences of a mixed step generate one token
            m = min(1, case["new_hi"])
        before.append(r.choice([0, r.randint(0, case["max_len"])]) if m > 1 else r.randint(0, case["max_len"]))
        new.append(m)
    return before, new


def _pairs(case):
    """Visible (row, key) pairs of one query head."""
    if case["op"] == "shared":
        return sum(case["shared"] + x for x in _own_lens(case))
    return sum(max(i + 1, P) for L, T0, P in _spec(case) for i in range(T0, L))


def work(case):
    op = case["op"]
    if op == "append":
        e = SIZE[case["dtype"]]
        n, H, KVH, dh = case["tokens"], case["H"], case["KVH"], case["dh"]
        return {"bytes": n * dh * (2 * H * e + 2 * KVH * (e + SIZE[case["cache"]])) + 16 * n,
                "flops": 3 * n * (H + KVH) * case["rot"]}
    if op == "rotate":
        el = case["B"] * case["H"] * case["T"] * case["dh"]
        return {"bytes": 4 * el * SIZE[case["dtype"]] + 8 * case["T"], "flops": 6 * el * case["rot"] // case["dh"]}
    if op == "tables":
        before, new = _table_lens(case)
        pages = sum(-(-(b + m) // PAGE) - -(-b // PAGE) for b, m in zip(before, new))
        return {"bytes": 16 * case["n"] + 20 * _cap(new) + 8 * pages, "flops": 4 * _cap(new)}
    H, KVH, dh, e = case["H"], case["KVH"], case["dh"], SIZE[case["dtype"]]
    if op == "prefill":
        rows = sum(L - T0 for L, T0, _ in _spec(case))
        keys = sum(L for L, _, _ in _spec(case))
    else:
        rows = case["B"]
        keys = case["shared"] + sum(_own_lens(case))
    return {"bytes": 2 * keys * KVH * dh + 2 * rows * H * dh * e, "flops": 4 * dh * H * _pairs(case)}


def _cap(new):
    """Token slots of a step: its tokens rounded up, as a captured step keeps them."""
    return (sum(new) // 64 + 1) * 64


# ------------------------------------------------------------------------------------------------ the inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    return g


def _scaling(case):
    s = case["scaling"]
    if s == "none":
        return None
    if s == "linear":
        return {"kind": "linear", "factor": 4.0}
    if s == "ntk":
        return {"kind": "ntk", "factor": 8.0}
    return {"kind": "bands", "factor": 32.0, "original": 8192}


def _lattice(pieces, KVH, dh, sink, gen, dev):
    """The paged int8 lattice of sequences given as [(K, V)] pieces, K/V [KVH, L, dh] float: a list per sequence, whose
    first piece may be the same object for several sequences (their pages are then the same too)."""
    T = [sum(k.shape[1] for k, _ in p) for p in pieces]
    nb = max(-(-t // KB) for t in T)
    npages, page_of, tables = 0, {}, []
    for p, t in zip(pieces, T):
        row, pos = [], 0
        shared = p[0][0].shape[1] // KB * (KB // PAGE) if len(p) > 1 else 0
        if shared:
            key = id(p[0][0])
            if key not in page_of:
                page_of[key] = list(range(npages, npages + shared))
                npages += shared
            row += page_of[key]
        n = -(-t // PAGE) - shared
        row += list(range(npages, npages + n))
        npages += n
        tables.append(row)
    perm = torch.randperm(npages, generator=gen, device=dev).to(torch.int32)
    bt = torch.full((len(T), nb * (KB // PAGE)), -1, dtype=torch.int32)
    for b, row in enumerate(tables):
        bt[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    bt = bt.to(dev)
    bt = torch.where(bt >= 0, perm[bt.clamp(min=0).long()], bt)
    k8p = torch.zeros((npages, KVH, PAGE, dh), dtype=torch.int8, device=dev)
    v8p = torch.zeros((npages, KVH, dh, PAGE), dtype=torch.int8, device=dev)
    ek = torch.zeros((len(T), KVH, nb), dtype=torch.int32, device=dev)
    ev = torch.zeros_like(ek)
    ev0 = torch.zeros((len(T), KVH), dtype=torch.int32, device=dev)
    done = {}
    for b, (p, t) in enumerate(zip(pieces, T)):
        first = p[0][0].shape[1] // KB * KB if len(p) > 1 else 0
        key = id(p[0][0])
        rest_k = torch.cat([p[0][0][:, first:]] + [k for k, _ in p[1:]], 1)
        rest_v = torch.cat([p[0][1][:, first:]] + [v for _, v in p[1:]], 1)
        parts = [(0, p[0][0][:, :first], p[0][1][:, :first], key)] if first else []
        parts.append((first, rest_k, rest_v, None))
        for pos, k, v, key in parts:
            if k.shape[1] == 0:
                continue
            if key is None or key not in done:
                sk = sink and pos == 0 and t > 1
                q = _quant_blocks(k, 40, False) + _quant_blocks(v, 48 if sink else 40, sk)
                n = -(-k.shape[1] // PAGE)
                pg = bt[b, pos // PAGE:pos // PAGE + n].long()
                k8p[pg] = q[0].view(KVH, -1, PAGE, dh)[:, :n].transpose(0, 1)
                v8p[pg] = q[3].view(KVH, -1, PAGE, dh)[:, :n].permute(1, 0, 3, 2)
                if key is not None:
                    done[key] = q
            else:
                q = done[key]
            j, m = pos // KB, q[1].shape[1]
            ek[b, :, j:j + m], ev[b, :, j:j + m] = q[1], q[4]
            if pos == 0:
                ev0[b] = q[5]
    return dict(k8p=k8p, v8p=v8p, ek=ek, ev=ev, ev0=ev0, block_table=bt, max_blocks=nb, num_pages=npages,
                seq_lens=torch.tensor(T, dtype=torch.int32, device=dev), sink=sink)


def _exponent(m, hi):
    e = 7 - torch.frexp(m)[1]
    e = e - (torch.ldexp(m, e) > 127).to(e.dtype)
    return torch.where(m == 0, torch.zeros_like(e), e.clamp(-32, hi))


def _quant_blocks(x, hi, split0):
    """x [G, T, dh] -> int8 [G, Tpad, dh] on one power-of-two grid a 128-row block, its exponents, row 0's own."""
    G, T, dh = x.shape
    nb = -(-T // KB)
    f = torch.zeros((G, nb * KB, dh), dtype=torch.float32, device=x.device)
    f[:, :T] = x.float()
    a = f.abs().amax(2)
    m0 = a[:, 0].clone()
    if split0:
        a[:, 0] = 0
    e = _exponent(a.view(G, nb, KB).amax(2), hi)
    er = e.repeat_interleave(KB, 1)
    e0 = _exponent(m0, hi) if split0 else e[:, 0]
    er[:, 0] = e0
    q = torch.ldexp(f, er[:, :, None]).round().clamp(-127, 127)
    return q.to(torch.int8), e.to(torch.int32), e0.to(torch.int32)


def _normal(shape, gen, dev, dt):
    return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dt)


def _kv(KVH, L, dh, gen, dev):
    """Keys with one channel in a hundred eight times as large, as the prefill configuration has them, and values."""
    k = _normal((KVH, L, dh), gen, dev, torch.bfloat16)
    ch = torch.randperm(dh, generator=gen, device=dev)[:-(-dh // 100)]
    k[:, :, ch] *= 8
    return k, _normal((KVH, L, dh), gen, dev, torch.bfloat16)


def prepare(case, seed):
    dev, op = _device(), case["op"]
    gen = _gen(seed, dev)
    st = {"case": case}
    if op in ("append", "rotate"):
        dt, dh = DTYPES[case["dtype"]], case["dh"]
        if op == "append":
            n, H, KVH = case["tokens"], case["H"], case["KVH"]
            qkv = _normal((n, H + 2 * KVH, dh), gen, dev, dt)          # the projection's output, split in place
            st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
            pages = -(-n // PAGE) + 3
            st["kv"] = _normal((pages, 2, PAGE, KVH, dh), gen, dev, DTYPES[case["cache"]])
            slots = torch.randperm(pages * PAGE, generator=gen, device=dev)[:n]
            if case["pad"] and n > 1:                                  # the padded end of a captured step
                slots[-min(case["pad"], n - 1):] = -1
            st["slots"] = slots
            st["pos"] = torch.randint(0, case["max_pos"], (n,), generator=gen, device=dev)
        else:
            B, H, T = case["B"], case["H"], case["T"]
            st["x"] = _normal((B, T, H, dh), gen, dev, dt).transpose(1, 2).requires_grad_(True)
            st["g"] = _normal((B, T, H, dh), gen, dev, dt).transpose(1, 2)
            start = int(torch.randint(0, max(1, case["max_pos"] - T), (1,), generator=gen, device=dev))
            st["pos"] = torch.arange(start, start + T, device=dev)
        if own:
            from lockstep_b200 import rotary
            st["plan"] = rotary.make_plan(dh, rotary_dim=case["rot"], base=10000.0, layout=case["layout"],
                                          scaling=_scaling(case), device=dev)
        else:
            st["freq"], st["factor"] = _frequencies(case, dev)
        return st
    if op == "tables":
        before, new = _table_lens(case)
        r = random.Random(seed)
        have = [-(-b // PAGE) for b in before]
        need = [-(-(b + m) // PAGE) - h for b, m, h in zip(before, new, have)]
        pages = list(range(sum(have) + sum(need) + 7))
        r.shuffle(pages)
        bt = torch.full((case["n"], max(h + x for h, x in zip(have, need)) + 2), -1, dtype=torch.int32)
        o = 0
        for i, h in enumerate(have):
            bt[i, :h] = torch.tensor(pages[o:o + h], dtype=torch.int32)
            o += h
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)          # noqa: E731
        st.update(before=i32(before), new=i32(new), table=bt.to(dev), free=i32(pages[o:]), cap=_cap(new))
        return st
    dt, H, KVH, dh = DTYPES[case["dtype"]], case["H"], case["KVH"], case["dh"]
    if op == "prefill":
        pieces = [[_kv(KVH, L, dh, gen, dev)] for L, _, _ in _spec(case)]
        n = [L - T0 for L, T0, _ in _spec(case)]
        st["q"] = _normal((sum(n), H, dh), gen, dev, dt)
        cu = [0]
        for x in n:
            cu.append(cu[-1] + x)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        st["prefix"] = (torch.tensor([P for _, _, P in _spec(case)], dtype=torch.int32, device=dev)
                        if case["P"] else None)
    else:
        common = _kv(KVH, case["shared"], dh, gen, dev)
        pieces = [[common, _kv(KVH, L, dh, gen, dev)] for L in _own_lens(case)]
        st["q"] = _normal((case["B"], H, dh), gen, dev, dt)
    lat = _lattice(pieces, KVH, dh, case["sink"], gen, dev)
    if own:
        from lockstep_b200 import decode
        st["kv"] = decode.PagedKV(**lat)
    else:
        st["kv"] = lat
        st["t2"] = _t2(dev)
        st["p2"] = _powers(dev)
    return st


# ------------------------------------------------------------------------------------------------ run
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    case = st["case"]
    op = case["op"]
    if op == "append":
        from lockstep_b200 import rotary
        out = rotary.rotate_append(st["q"], st["k"], st["v"], st["pos"], st["slots"], st["kv"][:, 0], st["kv"][:, 1],
                                   st["plan"], check=False)
        return out, st["kv"]
    if op == "rotate":
        from lockstep_b200 import rotary
        y = rotary.rotate(st["x"], st["pos"], st["plan"])
        return y, torch.autograd.grad(y, st["x"], st["g"])[0]
    if op == "tables":
        from lockstep_b200 import paging
        t = paging.step_tables(st["before"], st["new"], st["table"], st["free"], st["cap"], check=False)
        return t.query_start_loc, t.seq_lens, t.slot_mapping, t.positions, t.seq_index, st["table"]
    from lockstep_b200 import decode
    if op == "prefill":
        return decode.prefill_paged(st["q"], st["kv"], st["cu"], prefix_lens=st["prefix"], check=False)
    return decode.decode_shared(st["q"], st["kv"], case["shared"], check=False)


def _run_plain(st):
    op = st["case"]["op"]
    if op == "append":
        return _plain_append(st)
    if op == "rotate":
        y = _plain_rotate(st["x"], st["pos"], st, 1.0)
        return y, torch.autograd.grad(y, st["x"], st["g"])[0]
    if op == "tables":
        return _plain_tables(st)
    return _plain_prefill(st) if op == "prefill" else _plain_shared(st)


# ---- rotary
def _frequencies(case, dev):
    """theta_i of the rotated pairs, and the factor on cosine and sine."""
    d = case["rot"]
    i = torch.arange(0, d, 2, dtype=torch.float64, device=dev)
    s = _scaling(case)
    base = 10000.0
    if s and s["kind"] == "ntk" and d > 2:
        base *= s["factor"] ** (d / (d - 2))
    th = base ** (-i / d)
    if s and s["kind"] == "linear":
        th = th / s["factor"]
    if s and s["kind"] == "bands":
        turns = s["original"] * th / (2 * math.pi)                     # turns over the original context
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return th * keep + th / s["factor"] * (1 - keep), 0.1 * math.log(s["factor"]) + 1.0
    return th, 1.0


def _plain_rotate(x, pos, st, sign):
    """x [..., T, dh] (or [T, heads, dh] with pos shaped to it)."""
    case = st["case"]
    d = case["rot"]
    ang = pos.double()[..., None] * st["freq"]
    c, s = (ang.cos() * st["factor"]).float(), (ang.sin() * (st["factor"] * sign)).float()
    f = x.float()
    if case["layout"] == "half":
        a, b = f[..., :d // 2], f[..., d // 2:d]
        y = torch.cat([a * c - b * s, b * c + a * s, f[..., d:]], -1)
    else:
        a, b = f[..., 0:d:2], f[..., 1:d:2]
        y = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), f[..., d:]], -1)
    return y.to(x.dtype)


def _plain_append(st):
    pos = st["pos"][:, None]
    q = _plain_rotate(st["q"], pos, st, 1.0)
    case = st["case"]
    kf = _plain_rotate(st["k"].float(), pos, st, 1.0)
    ok = st["slots"] >= 0
    if case["pad"]:                          # skipped tokens repeat the first stored one
        idx = torch.where(ok, torch.arange(ok.numel(), device=ok.device), ok.to(torch.int32).argmax())
    else:
        idx = torch.arange(ok.numel(), device=ok.device)
    slots = st["slots"][idx]
    page, row = slots // PAGE, slots % PAGE
    st["kv"][page, 0, row] = kf[idx].to(st["kv"].dtype)
    st["kv"][page, 1, row] = st["v"][idx].to(st["kv"].dtype)
    return q, st["kv"]


# ---- tables
def _plain_tables(st):
    before, new, table, free, cap = st["before"], st["new"], st["table"], st["free"], st["cap"]
    dev, n = before.device, before.numel()
    after = before + new
    qsl = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), new.cumsum(0).to(torch.int32)])
    have, want = (before + PAGE - 1) // PAGE, (after + PAGE - 1) // PAGE
    cnt = want - have
    first = cnt.cumsum(0) - cnt
    j = torch.arange(table.shape[1], device=dev)
    take = (j >= have[:, None]) & (j < want[:, None])
    src = (first[:, None] + j - have[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(take, free[src], table))
    t = torch.arange(cap, device=dev)
    i = (t[:, None] >= qsl[1:]).sum(1).clamp(max=n - 1)
    pos = before[i] + t - qsl[i]
    slot = table[i, (pos // PAGE).clamp(max=table.shape[1] - 1)].long() * PAGE + pos % PAGE
    live = t < qsl[n]
    none = torch.full_like(t, -1)
    return (qsl, after, torch.where(live, slot, none), torch.where(live, pos, torch.zeros_like(pos)),
            torch.where(live, i, none).to(torch.int32), table)


# ---- contract attention: exact integers up to the block sums, then the ordered binary32 fold
def _t2(dev):
    """Weights 255 2^(-k/128), rounded half up, for k < 1152; 0 from there on."""
    return torch.tensor([math.floor(255 * 2.0 ** (-k / 128) + 0.5) for k in range(9 * 128)] + [0], device=dev)


def _powers(dev):
    return torch.tensor([2.0 ** e for e in range(-600, 601)], dtype=torch.float64, device=dev)


def _base(dh):
    return round(2.0 ** 26 / (math.sqrt(dh) * math.log(2.0)))


def _fold_g(dh, sh):
    """round-half-up(base 2^-sh), the chain's step a score, in [1, 2^30]."""
    sh = sh.clamp(-7, 23)
    right = sh.clamp(min=0)
    half = torch.where(right > 0, 1 << (right - 1).clamp(min=0), torch.zeros_like(right))
    g = torch.where(sh >= 0, (_base(dh) + half) >> right, _base(dh) << (-sh).clamp(min=0))
    return g.clamp(1, 1 << 30)


def _rescale(x, D, p2):
    """x 2^-D, flushed to zero below the smallest normal binary32."""
    y = x.double() * p2[600 - D.clamp(0, 600)]
    return torch.where(y.abs() < 2.0 ** -126, torch.zeros_like(y), y).float()


def _attend(st, q8, eq, nblk, block, visible, split, ev0, v0):
    """Rows q8 [G, R, dh] (binary32 integers), eq [G, R] against blocks 0 .. nblk-1 of G key sets.  block(j) gives
    (K, V, ek, ev); visible(j) the first row that may see block j and a mask over its rows and keys."""
    p2, t2 = st["p2"], st["t2"]
    G, R, dh = q8.shape
    dev = q8.device
    f = lambda *s: torch.zeros(s, dtype=torch.float32, device=dev)              # noqa: E731
    z = lambda: torch.zeros((G, R), dtype=torch.int64, device=dev)              # noqa: E731
    O, l, run, have = f(G, R, dh), f(G, R), z(), z().bool()
    Or, lr, rrun, haver = f(G, R, dh), f(G, R), z(), z().bool()
    low = -(1 << 40)
    for j in range(nblk):
        K, V, ek, ev = block(j)
        r0, vis = visible(j)
        S = (q8[:, r0:] @ K.transpose(1, 2)).long()
        g = _fold_g(dh, eq[:, r0:] + ek[:, None])
        m = (S if vis is None else torch.where(vis, S, low)).amax(2)
        live = m > low
        m = torch.where(live, m, 0)
        nb = -((-(m * g)) >> 26)
        w = t2[(((nb << 26)[:, :, None] - S * g[:, :, None]) >> 19).clamp(0, 9 * 128)]
        if vis is not None:
            w = torch.where(vis, w, 0)
        lb = w.sum(2).float()
        w0 = None
        if j == 0 and split is not None:
            w0 = w[:, :, 0] * split[:, None]
            w[:, :, 0] -= w0
        A = w.float() @ V
        run_, have_ = run[:, r0:], have[:, r0:]
        before = torch.where(have_, run_, nb)
        D = torch.where(live, nb - before, 0)
        o, ll = O[:, r0:], l[:, r0:]
        if j % SEG:
            o, ll = _rescale(o, D[:, :, None], p2), _rescale(ll, D, p2)
        s = (-D).clamp(min=0)
        add = live & (s <= SKIP)
        sc = lambda e: torch.where(add, p2[(600 - s - e).clamp(0, 1200)], 0.0).float()[:, :, None]   # noqa: E731
        if w0 is not None:
            o = o + w0.float()[:, :, None] * v0[:, None] * sc(ev0[:, None])
        O[:, r0:] = o + A * sc(ev[:, None])
        l[:, r0:] = ll + lb * sc(0)[:, :, 0]
        run[:, r0:] = torch.where(live, torch.maximum(before, nb), run_)
        have[:, r0:] = have_ | live
        if j % SEG == SEG - 1 or j == nblk - 1:
            before = torch.where(haver, rrun, run)
            D = torch.where(have, run - before, 0)
            s = (-D).clamp(min=0)
            add = have & (s <= SKIP)
            zero = torch.zeros((), device=dev)
            Or = _rescale(Or, D[:, :, None], p2) + torch.where(add[:, :, None], _rescale(O, s[:, :, None], p2), zero)
            lr = _rescale(lr, D, p2) + torch.where(add, _rescale(l, s, p2), zero)
            rrun = torch.where(have, torch.maximum(before, run), rrun)
            haver = haver | have
            O, l, run, have = f(G, R, dh), f(G, R), z(), z().bool()
    return torch.where(lr[:, :, None] != 0, Or / lr[:, :, None], torch.zeros_like(Or))


def _quant_queries(q):
    """q [..., dh] -> binary32 integers and exponents, one grid a row."""
    f = q.float()
    e = _exponent(f.abs().amax(-1), 40)
    return torch.ldexp(f, e[..., None]).round().clamp(-127, 127), e.long()


def _plain_prefill(st):
    case, kv = st["case"], st["kv"]
    H, KVH, dh = case["H"], case["KVH"], case["dh"]
    gq, dev = H // KVH, st["q"].device
    out = torch.empty_like(st["q"])
    q8, eq = _quant_queries(st["q"])
    at = 0
    for b, (L, T0, P) in enumerate(_spec(case)):
        n = L - T0
        rows = lambda x: x[at:at + n].reshape(n, KVH, gq, -1).transpose(0, 1).reshape(KVH, n * gq, -1)   # noqa: E731
        pg = kv["block_table"][b, :-(-L // PAGE)].long()
        nblk = -(-L // KB)
        K = torch.zeros((KVH, nblk * KB, dh), device=dev)
        V = torch.zeros_like(K)
        K[:, :pg.numel() * PAGE] = kv["k8p"][pg].transpose(0, 1).reshape(KVH, -1, dh).float()
        V[:, :pg.numel() * PAGE] = kv["v8p"][pg].permute(1, 0, 3, 2).reshape(KVH, -1, dh).float()
        ek, ev = kv["ek"][b].long(), kv["ev"][b].long()
        i = torch.arange(T0, L, device=dev).repeat_interleave(gq)

        def visible(j):
            r0 = 0 if j * KB < P else max(0, j * KB - T0)
            c = torch.arange(j * KB, (j + 1) * KB, device=dev)
            full = (j + 1) * KB <= P or (j * KB < T0 and P <= j * KB)
            seen = (c <= i[r0 * gq:, None]) | (c < P)
            return r0 * gq, None if full else seen[None]

        split = torch.full((KVH,), L > 1, dtype=torch.int64, device=dev) if case["sink"] else None
        o = _attend(st, rows(q8), rows(eq[..., None])[..., 0], nblk,
                    lambda j: (K[:, j * KB:(j + 1) * KB], V[:, j * KB:(j + 1) * KB], ek[:, j], ev[:, j]), visible, split,
                    kv["ev0"][b].long(), V[:, 0])
        out[at:at + n] = o.view(KVH, n, gq, dh).transpose(0, 1).reshape(n, H, dh).to(out.dtype)
        at += n
    return out


def _plain_shared(st):
    case, kv, q = st["case"], st["kv"], st["q"]
    B, H, KVH, dh = case["B"], case["H"], case["KVH"], case["dh"]
    gq = H // KVH
    q8, eq = _quant_queries(q)
    L = kv["seq_lens"].long()
    pp = KB // PAGE

    def block(j):
        pg = kv["block_table"][:, j * pp:(j + 1) * pp].long().clamp(min=0)
        K = kv["k8p"][pg].transpose(1, 2).reshape(B * KVH, KB, dh).float()
        V = kv["v8p"][pg].permute(0, 2, 1, 4, 3).reshape(B * KVH, KB, dh).float()
        return K, V, kv["ek"][:, :, j].reshape(-1).long(), kv["ev"][:, :, j].reshape(-1).long()

    def visible(j):
        c = torch.arange(j * KB, (j + 1) * KB, device=q.device)
        return 0, (c < L[:, None]).repeat_interleave(KVH, 0)[:, None]

    split = (L > 1).long().repeat_interleave(KVH) if case["sink"] else None
    v0 = kv["v8p"][kv["block_table"][:, 0].long(), :, :, 0].reshape(B * KVH, dh).float()
    o = _attend(st, q8.view(B * KVH, gq, dh), eq.view(B * KVH, gq), kv["max_blocks"], block, visible, split,
                kv["ev0"].reshape(-1).long(), v0)
    return o.view(B, H, dh).to(q.dtype)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    op = case["op"]
    if op == "append":
        q = _exact_rotate(case, st["q"], st["pos"][:, None])
        kv = st["kv"].double()
        ok = st["slots"] >= 0
        s = st["slots"][ok]
        kv[s // PAGE, 0, s % PAGE] = _exact_rotate(case, st["k"], st["pos"][:, None])[ok]
        kv[s // PAGE, 1, s % PAGE] = st["v"].double()[ok]
        return q, kv
    if op == "rotate":
        return (_exact_rotate(case, st["x"].detach(), st["pos"]),
                _exact_rotate(case, st["g"], -st["pos"]))
    if op == "tables":
        return _exact_tables(st)
    return _exact_prefill(case, st) if op == "prefill" else _exact_shared(case, st)


def _exact_rotate(case, x, pos):
    """Each pair as a complex number times m exp(i pos theta)."""
    d = case["rot"]
    s = _scaling(case) or {"kind": "none", "factor": 1.0}
    th, m = [], 1.0
    for i in range(d // 2):
        w = -2.0 * i / d * math.log(10000.0)
        if s["kind"] == "ntk" and d > 2:
            w -= 2.0 * i / (d - 2) * math.log(s["factor"])
        t = math.exp(w)
        if s["kind"] == "linear":
            t /= s["factor"]
        if s["kind"] == "bands":
            r = min(1.0, max(0.0, (s["original"] * t / (2 * math.pi) - 1.0) / 31.0))
            t = (1.0 - r) * t / s["factor"] + r * t
            m = 1.0 + 0.1 * math.log(s["factor"])
        th.append(t)
    th = torch.tensor(th, dtype=torch.float64, device=x.device)
    ang = pos.double().unsqueeze(-1) * th
    turn = torch.polar(torch.full_like(ang, m), ang)
    f = x.double()
    half = case["layout"] == "half"
    a, b = (f[..., :d // 2], f[..., d // 2:d]) if half else (f[..., 0:d:2], f[..., 1:d:2])
    y = torch.complex(a.contiguous(), b.contiguous()) * turn
    out = f.clone()
    if half:
        out[..., :d // 2], out[..., d // 2:d] = y.real, y.imag
    else:
        out[..., 0:d:2], out[..., 1:d:2] = y.real, y.imag
    return out


def _exact_tables(st):
    before, new, table, free = (st[k].tolist() for k in ("before", "new", "table", "free"))
    qsl, slot, posn, idx, take = [0], [], [], [], 0
    for i, (b, m) in enumerate(zip(before, new)):
        for p in range(-(-b // PAGE), -(-(b + m) // PAGE)):
            table[i][p] = free[take]
            take += 1
        for p in range(b, b + m):
            slot.append(table[i][p // PAGE] * PAGE + p % PAGE)
            posn.append(p)
            idx.append(i)
        qsl.append(qsl[-1] + m)
    pad = st["cap"] - len(slot)
    t = lambda v, dt=torch.int64: torch.tensor(v, dtype=dt, device=st["before"].device)      # noqa: E731
    i32 = torch.int32
    return (t(qsl, i32), t([b + m for b, m in zip(before, new)], i32), t(slot + [-1] * pad), t(posn + [0] * pad),
            t(idx + [-1] * pad, i32), t(table, i32))


def _exact_rows(q, kv, b, g, hi, dh, sink):
    """Rows q [R, dh] of one kv head against sequence b's keys: row r sees keys 0 .. hi[r]-1.  Weights on the 8-bit
    exponential grid below each block's rounded maximum; sums and the quotient in 64 bits."""
    dev = q.device
    L = int(kv["seq_lens"][b])
    nb = -(-L // KB)
    pg = kv["block_table"][b, :-(-L // PAGE)].long()
    k = torch.zeros((nb * KB, dh), dtype=torch.float64, device=dev)
    v = torch.zeros_like(k)
    k[:pg.numel() * PAGE] = kv["k8p"][pg, g].reshape(-1, dh).double()
    v[:pg.numel() * PAGE] = kv["v8p"][pg, g].transpose(1, 2).reshape(-1, dh).double()
    ev = kv["ev"][b, g, :nb].repeat_interleave(KB).double()
    if sink and L > 1:
        ev[0] = float(kv["ev0"][b, g])
    v = v * torch.exp2(-ev)[:, None]
    ek = kv["ek"][b, g, :nb].long()
    out = torch.empty((q.shape[0], dh), dtype=torch.float64, device=dev)
    weights = torch.tensor([float(math.floor(0.5 + 255 * math.exp(-k * math.log(2) / 128))) for k in range(1152)] + [0.0],
                           dtype=torch.float64, device=dev)
    f = q.double()
    top = f.abs().amax(1)
    eq = 6 - torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    eq = torch.where(top * torch.exp2(eq) > 127, eq - 1, eq)
    eq = torch.where(top * torch.exp2(eq) > 127, eq - 1, eq)
    eq = torch.where(top > 0, eq.clamp(-32, 40), torch.zeros_like(eq))
    f = (f * torch.exp2(eq)[:, None]).round().clamp(-127, 127)
    step = max(1, (1 << 25) // (nb * KB))
    col = torch.arange(nb * KB, device=dev)
    for r in range(0, q.shape[0], step):
        s = (f[r:r + step] @ k.T).view(-1, nb, KB)
        seen = (col < hi[r:r + step, None]).view(-1, nb, KB)
        sh = (eq[r:r + step, None].long() + ek).clamp(-7, 23).double()
        unit = torch.floor(_base(dh) * torch.exp2(-sh) + 0.5).clamp(1, 2.0 ** 30)
        z = s * unit[:, :, None]                                     # below 2^52: exact
        top = torch.where(seen, z, torch.full_like(z, -2.0 ** 60)).amax(2)
        lift = torch.ceil(top / 2.0 ** 26)
        w = weights[torch.floor((lift[:, :, None] * 2.0 ** 26 - z) / 2.0 ** 19).clamp(0, 1152).long()] * seen
        lift = torch.where(seen.any(2), lift, torch.full_like(lift, -2.0 ** 30))
        w = (w * torch.exp2((lift - lift.amax(1, keepdim=True)).clamp(min=-1000))[:, :, None]).view(-1, nb * KB)
        out[r:r + step] = (w @ v) / w.sum(1, keepdim=True)
    return out


def _exact_prefill(case, st):
    H, KVH, dh = case["H"], case["KVH"], case["dh"]
    gq, q = H // KVH, st["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    at = 0
    for b, (L, T0, P) in enumerate(_spec(case)):
        n = L - T0
        hi = torch.arange(T0 + 1, L + 1, device=q.device).clamp(min=P)
        for h in range(H):
            out[at:at + n, h] = _exact_rows(q[at:at + n, h], st["kv"], b, h // gq, hi, dh, case["sink"])
        at += n
    return out


def _exact_shared(case, st):
    H, KVH, dh = case["H"], case["KVH"], case["dh"]
    gq, q = H // KVH, st["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for b in range(case["B"]):
        hi = st["kv"]["seq_lens"][b].long().expand(gq)
        for g in range(KVH):
            out[b, g * gq:(g + 1) * gq] = _exact_rows(q[b, g * gq:(g + 1) * gq], st["kv"], b, g, hi, dh, case["sink"])
    return out
