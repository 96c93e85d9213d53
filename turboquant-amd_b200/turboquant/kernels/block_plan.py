"""Block tables and slot maps of a paged cache, kept on the GPU.

The two paged caches take a slot for every new token and a table of blocks for every sequence.  `plan_step` makes both from
the requests' lengths in one launch, taking blocks from a stack of free ones; `release_blocks` puts the blocks of ended
requests back.  Nothing comes back to the host, so a captured step can build its own tables.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from turboquant.kernels import _native


class StepPlan(NamedTuple):
    """slot_mapping, positions: int64 [num_rows]; seq_lens: int32 [n]; query_start_loc: int32 [n + 1]; free_count: int32 [1].
    They may lie in one allocation."""

    slot_mapping: torch.Tensor
    positions: torch.Tensor
    seq_lens: torch.Tensor
    query_start_loc: torch.Tensor
    free_count: torch.Tensor


def plan_step(query_lens: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor,
              free_count: torch.Tensor, block_size: int, num_rows: int) -> StepPlan:
    """Tables of a step in which request i brings query_lens[i] new tokens to the context_lens[i] it has (int32 [n]).

    block_tables int32 [n, width] is extended in place: further blocks come from the top of the stack free_blocks[:free_count]
    (int32 [F] and [1]) in the order of the requests.  num_rows: rows of the step's tensors; those behind the last request
    get slot -1 and position 0.  free_blocks and free_count are not changed: the plan's free_count is the stack's new
    height, to be handed to the next call, and a call that is repeated gives the same tables.
    A request for which the free blocks do not suffice (STATUS_NO_BLOCKS), or whose rows or blocks do not fit (STATUS_TOO_LONG),
    takes none; its rows get slot -1 and its seq_lens entry stays the context.
    """
    if not torch.compiler.is_compiling():
        res = _native.host().plan_step(query_lens, context_lens, block_tables, free_blocks, free_count, block_size, num_rows)
        if res is not None:
            return StepPlan._make(res)
    return StepPlan._make(torch.ops.tq_b200.plan_step(query_lens, context_lens, block_tables, free_blocks, free_count, int(block_size),
                                                     int(num_rows)))


def release_blocks(ended: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor,
                   free_count: torch.Tensor, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Put the blocks of the requests with ended[i] (bool [n]) back on the stack; returns (context_lens, free_count) afterwards.

    The first ceil(context_lens[i] / block_size) entries of their rows are appended to free_blocks at free_count, request after
    request (in place; free_count itself is not changed).  The returned lengths are 0 for them.  Blocks that other requests
    share must not be released twice: this keeps no counts.  What exceeds free_blocks is dropped and sets STATUS_TOO_LONG.
    """
    if not torch.compiler.is_compiling():
        res = _native.host().release_blocks(ended, context_lens, block_tables, free_blocks, free_count, block_size)
        if res is not None:
            return res
    return torch.ops.tq_b200.release_blocks(ended, context_lens, block_tables, free_blocks, free_count, int(block_size))
