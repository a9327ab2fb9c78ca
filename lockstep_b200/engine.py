"""The serving-engine seam: one attention call per layer and engine step, over a paged float KV
cache, with prompt rows and generated rows routed by the scheduler's flag.

The reference's engine is a vLLM plugin that registers a custom attention backend
(paper/main.tex:846-860): the scheduler's is_prefilling flag -- never the number of query rows --
decides whether a sequence's rows in a step are prompt rows (docs/SPEC.md:88-93), prompt chunks
start on 128-token boundaries (a scheduler hook; the 128-aligned chunk invariance,
reference/lssab8_selftest.py:292-317, makes each chunk's rows equal the whole prefill's), and
generated rows are LSSA-B8 rows too (contract v2).  This module is that backend's forward pass on
this library, in the engine's own terms:

  * the engine keeps its float K/V cache in 16-token pages, [num_pages, 16, KVH, dh], addressed
    by its block table [nseq, max_pages] and written at slot_mapping (page * 16 + row);
  * LatticeLayer keeps the int8 lattice that shadows that cache for one layer: pages with the same
    ids as the engine's (so the engine's block table addresses both), and per-sequence block
    exponents in slots keyed by the sequence's first page, the identity a sequence keeps across
    steps (as the reference's row verifier keys it, tools/verify_rows.py:63-104);
  * Lssab8Attention.forward(layer, query, key, value, k_cache, v_cache, meta) stores the step's new
    keys and values in the float cache, appends them to the lattice (lssab8_kv_append: only the
    open block and new blocks are quantised), then runs the prompt rows of every sequence through one
    packed prefill over the lattice (decode.prefill_paged) and every generated row through one
    split-KV decode call;
  * with a rotary plan (lockstep_b200.rotary) the queries and keys come unrotated and the float-cache
    store rotates them (one launch); StepMeta.build makes a step's block table, slots and positions
    on the device (lockstep_b200.paging) for an engine that keeps only request lengths.

lockstep_b200.vllm_backend wraps this forward pass as a vLLM attention backend: its metadata
builder supplies query_start_loc, seq_lens, block_table, slot_mapping and the scheduler's prefill
flags; the 128-aligned chunk boundaries are the scheduler's to keep.
"""
from dataclasses import dataclass

import torch

from . import decode as D
from . import paging as P
from . import rotary as R

PAGE = 16
KB = 128


@dataclass
class StepMeta:
    """One engine step: nseq sequences, ntok new tokens in sequence order.

    query_start_loc [nseq + 1] (host ints): sequence i's new tokens are rows [qsl[i], qsl[i+1]);
    seq_lens [nseq] (host ints): each sequence's length after this step; block_table
    [nseq, max_pages] int32 (CUDA): the pages of each sequence; slot_mapping [ntok] int64 (CUDA):
    page * 16 + row of each new token; is_prefill [nseq] (host bools): the scheduler's flag;
    positions [ntok] (CUDA, int32 or int64): each new token's position, for an engine with a rotary
    plan."""
    query_start_loc: list
    seq_lens: list
    block_table: torch.Tensor
    slot_mapping: torch.Tensor
    is_prefill: list
    positions: torch.Tensor = None

    @classmethod
    def build(cls, lens, new_tokens, is_prefill, block_table, free_pages):
        """The step in which sequence i grows from lens[i] by new_tokens[i] tokens (host ints).  The new pages
        are the first entries of free_pages (int32, CUDA) in sequence order, written to block_table [nseq,
        max_pages] (int32, CUDA) in place; returns (meta, number of free pages taken)."""
        lens, new = [int(x) for x in lens], [int(x) for x in new_tokens]
        if len(new) != len(lens) or len(is_prefill) != len(lens) or min(lens + new, default=0) < 0:
            raise ValueError("lens, new_tokens and is_prefill must match, lengths must not be negative")
        pages = lambda x: -(-x // PAGE)                      # noqa: E731
        used = sum(pages(a + b) - pages(a) for a, b in zip(lens, new))
        if used > free_pages.numel():
            raise ValueError("the step needs %d pages, %d are free" % (used, free_pages.numel()))
        dev = block_table.device
        t = P.step_tables(torch.tensor(lens, dtype=torch.int32, device=dev),
                          torch.tensor(new, dtype=torch.int32, device=dev), block_table, free_pages, sum(new))
        qsl = [0]
        for x in new:
            qsl.append(qsl[-1] + x)
        return cls(query_start_loc=qsl, seq_lens=[a + b for a, b in zip(lens, new)], block_table=block_table,
                   slot_mapping=t.slot_mapping, is_prefill=list(is_prefill), positions=t.positions), used


class LatticeLayer:
    """The int8 lattice of one layer: pages shared with the engine's float cache page ids, block
    exponents per sequence slot (keyed by the sequence's first page)."""

    def __init__(self, num_pages, KVH, dh, max_len, max_seqs, sink, device):
        self.KVH, self.dh, self.sink = KVH, dh, bool(sink)
        self.max_blocks = (max_len + KB - 1) // KB
        self.max_pages = self.max_blocks * 8
        self.num_pages = num_pages
        self.k8p = torch.zeros((num_pages, KVH, PAGE, dh), dtype=torch.int8, device=device)
        self.v8p = torch.zeros((num_pages, KVH, dh, PAGE), dtype=torch.int8, device=device)
        self.ek = torch.zeros((max_seqs, KVH, self.max_blocks), dtype=torch.int32, device=device)
        self.ev = torch.zeros_like(self.ek)
        self.ev0 = torch.zeros((max_seqs, KVH), dtype=torch.int32, device=device)
        self.lens = [0] * max_seqs
        self.slot_of = {}                                 # first page -> slot
        self.last_use = [0] * max_seqs                    # step of the slot's last use
        self.step = 0

    def slots(self, first_pages, lens_before):
        """Slots of the step's sequences.  A sequence seen for the first time (its length before
        the step is 0) takes a free slot, or the least recently used one of a sequence not in this
        step (an engine that never calls release() reuses its finished sequences' slots this way).
        A sequence that continues (length before > 0) must still hold its slot: if it was taken,
        its block exponents are gone and the step is refused.  So is one that continues past what
        its slot holds, and a step in which two sequences start on one page (forks of a prompt that
        share its pages): they would keep their exponents in one slot."""
        if len(set(first_pages)) != len(first_pages):
            twice = next(fp for i, fp in enumerate(first_pages) if fp in first_pages[:i])
            raise RuntimeError("two sequences of the step start on page %d: sequences that share pages keep their own "
                               "lattice and decode with decode_shared" % twice)
        self.step += 1
        out = []
        for fp, l0 in zip(first_pages, lens_before):
            s = self.slot_of.get(fp)
            if s is None:
                if l0 != 0:
                    raise RuntimeError("the sequence with first page %d continues at length %d, but its lattice "
                                       "slot was reused (more live sequences than slots)" % (fp, l0))
                s = self._take_slot()
                self.slot_of[fp] = s
            elif l0 > self.lens[s]:
                raise RuntimeError("the sequence with first page %d continues at length %d, but its lattice holds %d "
                                   "tokens" % (fp, l0, self.lens[s]))
            if l0 == 0:
                self.lens[s] = 0                          # a new sequence (possibly on a reused first page)
            self.last_use[s] = self.step
            out.append(s)
        return out

    def _take_slot(self):
        used = set(self.slot_of.values())
        for i in range(len(self.lens)):
            if i not in used:
                return i
        idle = [i for i in range(len(self.lens)) if self.last_use[i] < self.step]
        if not idle:
            raise RuntimeError("more sequences in one step than lattice slots")
        victim = min(idle, key=lambda i: self.last_use[i])
        for fp, s in list(self.slot_of.items()):
            if s == victim:
                del self.slot_of[fp]
        return victim

    def release(self, first_page):
        """Forget a finished sequence (the engine frees its pages)."""
        s = self.slot_of.pop(first_page, None)
        if s is not None:
            self.lens[s] = 0


class Lssab8Attention:
    """LSSA-B8 (sink=False) / B9.1 sink_alone (sink=True) attention for a paged serving engine."""

    def __init__(self, num_heads, num_kv_heads, head_size, num_pages, max_len, max_seqs, num_layers=1, sink=False,
                 device=None, rotary=None):
        if num_heads % num_kv_heads:
            raise ValueError("query heads must be a multiple of kv heads")
        self.H, self.KVH, self.dh = num_heads, num_kv_heads, head_size
        self.sink = bool(sink)
        self.rotary = rotary                              # a rotary plan: queries and keys come unrotated
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        self.layers = [LatticeLayer(num_pages, num_kv_heads, head_size, max_len, max_seqs, sink, dev)
                       for _ in range(num_layers)]

    def forward(self, layer, query, key, value, k_cache, v_cache, meta, out=None):
        """query [ntok, H, dh], key / value [ntok, KVH, dh] (this step's new tokens), k_cache /
        v_cache [num_pages, 16, KVH, dh] (the engine's float cache; rows and channels contiguous,
        any page stride) -> out [ntok, H, dh] in
        query.dtype.  Prompt chunks must start on a multiple of 128 tokens."""
        st = self.layers[layer]
        dev = query.device
        nseq = len(meta.seq_lens)
        qsl = [int(x) for x in meta.query_start_loc]
        lens = [int(x) for x in meta.seq_lens]
        qlen = [qsl[i + 1] - qsl[i] for i in range(nseq)]
        before = [lens[i] - qlen[i] for i in range(nseq)]
        if out is None:
            out = torch.empty_like(query)
        # 1. the step's keys and values into the engine's float cache (by page and row, so a cache
        #    whose pages are strided -- K and V interleaved per page -- is written in place)
        if self.rotary is not None:
            if meta.positions is None:
                raise ValueError("an engine with a rotary plan needs the step's positions")
            query = R.rotate_append(query, key, value, meta.positions, meta.slot_mapping, k_cache, v_cache, self.rotary)
        else:
            page, row = meta.slot_mapping // PAGE, meta.slot_mapping % PAGE
            k_cache[page, row] = key.to(k_cache.dtype)
            v_cache[page, row] = value.to(v_cache.dtype)
        # 2. the lattice: the open block and new blocks of every sequence, from the float cache
        bt = meta.block_table.to(device=dev, dtype=torch.int32)
        if bt.shape[1] < st.max_pages:
            bt = torch.cat([bt, bt.new_full((nseq, st.max_pages - bt.shape[1]), -1)], 1)
        bt = bt[:, :st.max_pages].contiguous()
        first = [int(x) for x in bt[:, 0].tolist()]
        held = [i for i in range(nseq) if lens[i] > 0]     # (an idle row has no slot: its first page may be anyone's)
        slots = st.slots([first[i] for i in held], [before[i] for i in held])
        rows = [0] * nseq
        for i, s in zip(held, slots):
            rows[i] = s
        sidx = torch.tensor(rows, dtype=torch.long, device=dev)
        kv = D.PagedKV(k8p=st.k8p, v8p=st.v8p, ek=st.ek[sidx].contiguous(), ev=st.ev[sidx].contiguous(),
                       ev0=st.ev0[sidx].contiguous(), block_table=bt,
                       seq_lens=torch.tensor(before, dtype=torch.int32, device=dev), max_blocks=st.max_blocks,
                       num_pages=st.num_pages, sink=self.sink)
        D.append_kv(kv, k_cache, v_cache, torch.tensor(lens, dtype=torch.int32, device=dev), src_block_table=bt)
        if len(held) == nseq:
            st.ek[sidx], st.ev[sidx], st.ev0[sidx] = kv.ek, kv.ev, kv.ev0
        else:
            hi = torch.tensor(held, dtype=torch.long, device=dev)
            st.ek[sidx[hi]], st.ev[sidx[hi]], st.ev0[sidx[hi]] = kv.ek[hi], kv.ev[hi], kv.ev0[hi]
        for i, s in zip(held, slots):
            st.lens[s] = lens[i]
        # 3. prompt rows: every sequence's block-aligned chunk in one packed prefill over the lattice
        prompts = [bool(meta.is_prefill[i]) and qlen[i] > 0 for i in range(nseq)]
        for i in range(nseq):
            if prompts[i] and before[i] % KB:
                raise ValueError("prompt chunk of sequence %d starts at %d, not a multiple of %d (the scheduler's "
                                 "chunk alignment)" % (i, before[i], KB))
        if any(prompts):
            cu = torch.tensor(qsl, dtype=torch.int32, device=dev)
            act = torch.tensor(prompts, dtype=torch.bool, device=dev)
            query = query.detach()                        # (the contract's integers have no gradient)
            q = query[:qsl[-1]]                           # (query and out may be longer than the step's rows)
            if out.dtype == query.dtype:
                D.prefill_paged(q, kv, cu, active=act, out=out[:qsl[-1]])
            else:
                rows = D.prefill_paged(q, kv, cu, active=act)
                for i in range(nseq):
                    if prompts[i]:
                        out[qsl[i]:qsl[i + 1]] = rows[qsl[i]:qsl[i + 1]]
        # 4. generated rows: one split-KV decode over the lattice for every one-row sequence
        gen = [i for i in range(nseq) if not meta.is_prefill[i] and qlen[i] > 0]
        if any(qlen[i] != 1 for i in gen):
            raise NotImplementedError("generated steps of more than one row (speculative tokens) are not routed")
        if gen:
            gi = torch.tensor(gen, dtype=torch.long, device=dev)
            rows = torch.tensor([qsl[i] for i in gen], dtype=torch.long, device=dev)
            dkv = D.PagedKV(k8p=st.k8p, v8p=st.v8p, ek=kv.ek[gi].contiguous(), ev=kv.ev[gi].contiguous(),
                            ev0=kv.ev0[gi].contiguous(), block_table=bt[gi].contiguous(),
                            seq_lens=torch.tensor([lens[i] for i in gen], dtype=torch.int32, device=dev),
                            max_blocks=st.max_blocks, num_pages=st.num_pages, sink=self.sink)
            out[rows] = D.decode(query[rows].contiguous(), dkv, out_dtype=query.dtype)
        return out
