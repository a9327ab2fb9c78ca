"""A serving step's tables, built on the device from its request lengths (host layer over the C ABI): query
starts, lengths, the pages that new tokens need (from a free list, in sequence order), slots and positions.
Nothing is read back, so a step can be captured in a CUDA graph and replayed with new lengths in the same
buffers."""
from dataclasses import dataclass

import torch

from . import _lib
from . import attention as _A

PAGE = 16
MAX_SEQS = 16384
MAX_TOKENS = 1 << 30


@dataclass
class StepTables:
    """query_start_loc [n + 1] int32, seq_lens [n] int32 (after the step), slot_mapping [cap] int64, positions
    [cap] int64, seq_index [cap] int32 (entries past the last token: -1, 0, -1), pages_used [1] int32 (entries
    of the free list taken)."""
    query_start_loc: torch.Tensor
    seq_lens: torch.Tensor
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    seq_index: torch.Tensor
    pages_used: torch.Tensor


def alloc_step_tables(n, cap, device):
    # two buffers, cut: a step's call pays for two allocations instead of six
    qsl, lens, seq, used = torch.unsafe_split_with_sizes(
        torch.empty(2 * n + 2 + cap, dtype=torch.int32, device=device), (n + 1, n, cap, 1))
    slots, pos = torch.empty((2, cap), dtype=torch.int64, device=device).unbind(0)
    return StepTables(qsl, lens, slots, pos, seq, used)


def step_tables(lens, new_tokens, block_table, free_pages, max_tokens, out=None, check=True):
    """Tables of a step in which sequence i grows from lens[i] by new_tokens[i] tokens (both [n] int32, CUDA).

    block_table [n, max_pages] int32 is updated in place with the new pages, which are the first entries of
    free_pages [F] int32 in sequence order; its other entries stay.  max_tokens: length of the token arrays
    (at least the step's tokens, at most 2^30).  out: tables of an earlier call with the same n and max_tokens, rewritten
    (apart from the inputs: lens is not its own seq_lens).
    Lengths that do not fit raise RuntimeError (device error 16) when checked."""
    dev = _A._require_cuda(lens, new_tokens, block_table, free_pages)
    n = lens.numel()
    i32 = torch.int32
    if lens.dtype != i32 or new_tokens.dtype != i32 or block_table.dtype != i32 or free_pages.dtype != i32:
        raise TypeError("lens, new_tokens, block_table and free_pages must be int32")
    if lens.dim() != 1 or new_tokens.shape != lens.shape or not 0 < n <= MAX_SEQS:
        raise ValueError("lens and new_tokens must be [n], n from 1 to %d" % MAX_SEQS)
    if block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("block_table must be [n, max_pages], free_pages [F]")
    rows, width = block_table.shape
    pitch, step = block_table.stride()
    if rows != n or width == 0:
        raise ValueError("block_table must be [n, max_pages], free_pages [F]")
    if (step != 1 and width > 1) or (pitch < width and n > 1):
        raise ValueError("block_table rows must be contiguous and apart")
    cap, nfree = int(max_tokens), free_pages.numel()
    if not 0 <= cap <= MAX_TOKENS:
        raise ValueError("max_tokens must be from 0 to 2^30")
    lens, new_tokens, free_pages = lens.contiguous(), new_tokens.contiguous(), free_pages.contiguous()
    wrote = [block_table]
    if out is None:
        out = alloc_step_tables(n, cap, dev)
    else:
        i64 = torch.int64
        for f, t, size, dt in (("query_start_loc", out.query_start_loc, n + 1, i32), ("seq_lens", out.seq_lens, n, i32),
                               ("slot_mapping", out.slot_mapping, cap, i64), ("positions", out.positions, cap, i64),
                               ("seq_index", out.seq_index, cap, i32), ("pages_used", out.pages_used, 1, i32)):
            if t.shape != (size,) or t.dtype != dt or t.device != dev or not t.is_contiguous():
                raise ValueError("out: tables of another step shape (%s)" % f)
            wrote.append(t)
        ins = [(x.data_ptr(), x.data_ptr() + 4 * size, x) for x, size in (
            (lens, n), (new_tokens, n), (block_table, (n - 1) * pitch + width), (free_pages, nfree))]
        outs = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), t) for t in wrote[1:]]
        if any(p < e2 and p2 < e and _A._share(t, x) for p, e, t in outs for p2, e2, x in ins):
            raise ValueError("out must lie apart from the step's own lengths, table and free pages")
    with _A._on(dev):
        _lib.check(_lib.load().lssab8_step_tables(
            lens.data_ptr(), new_tokens.data_ptr(), n, block_table.data_ptr(), max(pitch, width), width,
            free_pages.data_ptr() if nfree else None, nfree, cap,
            out.query_start_loc.data_ptr(), out.seq_lens.data_ptr(), out.slot_mapping.data_ptr(), out.positions.data_ptr(),
            out.seq_index.data_ptr(), out.pages_used.data_ptr(), _A._stream_handle(dev)), "lssab8_step_tables")
    _A._wrote(*wrote)
    if check:
        _A.check_device_errors(dev)
    return out
