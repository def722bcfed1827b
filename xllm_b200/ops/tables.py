"""Tables of a step built on the device from request lengths (csrc/kernels/step_tables.cu): what `AttentionMetadata` and the
model's forward pass read of a batch, for steps whose lengths or blocks are known on the device only, or whose host side
should not pack them.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _count, _debug, _lib
from ._lib import I, L, P, check, ptr, stream_on

_lib.register_signature("xllm_step_tables", [P, L, I, I, P, P, I, I, P, I, P, P, P, P, P, P, P])

MAX_REQUESTS = 8192


class StepTables(NamedTuple):
    cu_q: torch.Tensor         # int32 [requests + 1]: token rows of request b are cu_q[b] .. cu_q[b + 1]
    kv_lens: torch.Tensor      # int32 [requests]: tokens in the cache after the step; 0 for a refused request
    positions: torch.Tensor    # int64 [n_rows]
    slots: torch.Tensor        # int32 [n_rows]: block * page + offset, -1 where nothing is written
    last_rows: torch.Tensor    # int64 [requests]: the request's last token row (where its next token is read)
    taken: torch.Tensor        # int32 []: blocks handed out, the first `taken` of free_blocks


def step_tables_reference(block_table, ctx_lens, q_lens, page, n_rows, free_blocks):
    B, width = block_table.shape
    dev = block_table.device
    ctx, new = ctx_lens.long().clamp(min=0), q_lens.long().clamp(min=0)
    end = torch.cumsum(new, 0)
    have, need = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    fits = (need <= width) & (end <= n_rows) & (ctx + new < 1 << 31)
    added = torch.where(fits, need - have, 0)
    upto = torch.cumsum(added, 0)
    ok = fits & ((added == 0) | (upto <= free_blocks.shape[0]))
    for b in torch.nonzero(ok & (added > 0)).flatten().tolist():
        at = int(upto[b] - added[b])
        block_table[b, int(have[b]):int(need[b])] = free_blocks[at:at + int(added[b])]
    row = torch.arange(n_rows, device=dev)
    seq = torch.searchsorted(end, row, right=True).clamp(max=B - 1)
    live = (row < end[-1]) & ok[seq]
    positions = torch.where(live, ctx[seq] + row - (end - new)[seq], 0)
    entry = block_table[seq, (positions // page).clamp(max=max(width - 1, 0))].long()
    slots = entry * page + positions % page
    slots = torch.where(live & (entry >= 0) & (slots < 1 << 31), slots, -1)
    cu_q = torch.cat([end.new_zeros(1), end.clamp(max=n_rows)])
    return StepTables(cu_q.int(), torch.where(ok, ctx + new, 0).int(), positions, slots.int(), (cu_q[1:] - 1).clamp(min=0),
                      torch.where(ok, added, 0).sum().int())


def step_tables(block_table, ctx_lens, q_lens, page, n_rows, free_blocks=None):
    """Request b has ctx_lens[b] tokens in the cache, whose blocks are the first ceil(ctx / page) entries of its row of
    block_table (int32 [requests, width], rows at any stride), and q_lens[b] tokens in this step (0 and more; 1: decoding).  The
    blocks that the new tokens need beyond those are taken from free_blocks (int32) in the order of the requests and written into block_table; its
    other entries are left as they are.  Token rows follow one another by request; n_rows of them are filled in (the
    padded size of a captured step), rows behind the last request with position 0 and slot -1.

    A request that does not fit takes no blocks and becomes inert like a padding row (kv_len 0, its rows position 0 and slot -1):
    when block_table is too narrow for it, when its rows end behind n_rows, or when free_blocks ends before its new blocks do
    (then no later request takes any either).  A row whose block is negative, or whose slot
    passes 31 bits, has slot -1.  Nothing is read back: whoever may run short compares kv_lens later.

    ctx_lens, q_lens: int32 [requests], negative ones count as 0.  Returns StepTables."""
    if block_table.dim() != 2 or block_table.dtype is not torch.int32 or block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise TypeError(f"step_tables: block_table is int32 [requests, width] with adjacent entries, got {block_table.dtype} "
                        f"{tuple(block_table.shape)} strides {block_table.stride()}")
    B, width = block_table.shape
    dev = block_table.device
    if not (ctx_lens.dtype is q_lens.dtype is torch.int32 and ctx_lens.shape == q_lens.shape == (B,) and ctx_lens.device == q_lens.device == dev):
        raise TypeError(f"step_tables: ctx_lens and q_lens are int32 [{B}] on {dev}, got {ctx_lens.dtype} {tuple(ctx_lens.shape)} on "
                        f"{ctx_lens.device}, {q_lens.dtype} {tuple(q_lens.shape)} on {q_lens.device}")
    if free_blocks is not None and (free_blocks.dtype is not torch.int32 or free_blocks.dim() != 1 or free_blocks.device != dev
                                    or free_blocks.shape[0] >= 1 << 31):
        raise TypeError(f"step_tables: free_blocks is int32 [blocks] on {dev}, fewer than 2^31")
    if block_table.stride(0) < width and B > 1:
        raise ValueError(f"step_tables: rows of block_table that lie apart, got strides {block_table.stride()} for {width} entries")
    if not 1 <= B <= MAX_REQUESTS or not 1 <= width < 1 << 31 or not 1 <= page < 1 << 31 or not 0 <= n_rows < 1 << 31:
        raise ValueError(f"step_tables: 1 to {MAX_REQUESTS} requests, a width and a page of 1 or more and 0 or more rows, all below 2^31, got "
                         f"{B}, {width}, {page}, {n_rows}")
    if _debug.enabled():
        _debug.check_range(ctx_lens, 0, 1 << 31, "step_tables ctx_lens")
        _debug.check_range(q_lens, 0, 1 << 31, "step_tables q_lens")
    if not block_table.is_cuda:
        free = free_blocks if free_blocks is not None else torch.empty(0, dtype=torch.int32)
        return step_tables_reference(block_table, ctx_lens, q_lens, page, n_rows, free)
    index = dev.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return step_tables(block_table, ctx_lens, q_lens, page, n_rows, free_blocks)
    ctx_lens, q_lens = ctx_lens.contiguous(), q_lens.contiguous()
    n_free = 0
    if free_blocks is not None:
        free_blocks, n_free = free_blocks.contiguous(), free_blocks.shape[0]
    # one allocation: a short step's time is the host's
    i64 = 2 * (n_rows + B)
    buf = ctx_lens.new_empty(i64 + n_rows + 2 * B + 2)
    positions, last_rows, slots, cu_q, kv_lens, taken = buf.split_with_sizes([2 * n_rows, 2 * B, n_rows, B + 1, B, 1])
    at = buf.data_ptr()
    rest = at + 4 * i64
    check(_lib.load().xllm_step_tables(ptr(block_table), block_table.stride(0), B, width, ptr(ctx_lens), ptr(q_lens), int(page),
                                       int(n_rows), ptr(free_blocks), n_free, rest + 4 * n_rows, rest + 4 * (n_rows + B + 1), at, rest,
                                       at + 8 * n_rows, rest + 4 * (n_rows + 2 * B + 1), stream_on(index)), "step_tables")
    _count()
    return StepTables(cu_q, kv_lens, positions.view(torch.int64), slots, last_rows.view(torch.int64), taken.view(()))
