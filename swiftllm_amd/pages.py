"""Pages of the cache where sequences come of one another, on the device.

    fork_pages       rows that go on from others: tables, references, copies of
                     blocks that are about to be written, the free list
    compact_pages    the blocks in use moved to the pool's front

Reference (paths relative to the swiftllm repository): the host routines these
stand for are
  crates/swiftllm-core/src/memory/block_manager.rs
                                               reference counts, copy-on-write fork
A pool's state is device memory: ref_counts int32 [num_blocks], how many rows
hold each block, and free_blocks int32 [num_blocks] with num_free, which
attention_step.plan_step takes blocks from. Device tensors are DeviceArrays or raw
device pointers (ints). Nothing here synchronises or allocates.
"""

from __future__ import annotations

from typing import Optional

from . import _lib
from ._hip import Stream
from .paged_attention import CudaError, Ptr, _p, _s, check_status


def pages_workspace_size(num_seqs: int, num_blocks: int) -> int:
    n = _lib.lib().swiftllm_hip_pages_workspace_size(num_seqs, num_blocks)
    if n == 0:
        check_status(_lib.lib().swiftllm_hip_last_error() or CudaError.code)
    return int(n)


def fork_pages(block_tables_out: Ptr, context_lens_out: Ptr, block_tables: Ptr, context_lens: Ptr,
               parents: Ptr, ref_counts: Ptr, free_blocks: Ptr, num_free: Ptr, copy_pairs: Ptr,
               counts: Ptr, workspace: Ptr, workspace_bytes: int, num_seqs: int,
               max_num_blocks_per_seq: int, block_size: int, num_blocks: int, taken: Ptr = None,
               new_lens: Ptr = None, stream: Optional[Stream] = None) -> None:
    """Row i of the new tables goes on from row parents[i] of the old ones, -1
    from none (swiftllm_hip_fork_pages). ref_counts, free_blocks and num_free are
    brought up to date in place; copy_pairs int64 [num_seqs, 2] is for
    paged_attention.copy_blocks, -1 behind the last pair; counts int32 [2] =
    (copies, rows cut short because no block was free). taken: the counts of the
    plan_step since the last fork, whose blocks get their first reference here.
    new_lens int32 [num_seqs]: 1 for rows that go on, for the next plan_step.
    With parents[i] = i for every row but those that end, this frees pages."""
    check_status(_lib.lib().swiftllm_hip_fork_pages(
        _p(block_tables_out), _p(context_lens_out), _p(block_tables), _p(context_lens),
        _p(parents), _p(ref_counts), _p(free_blocks), _p(num_free), _p(taken), _p(copy_pairs),
        _p(new_lens), _p(counts), _p(workspace), workspace_bytes, num_seqs, max_num_blocks_per_seq, block_size,
        num_blocks, _s(stream)))


def compact_pages(block_tables_out: Ptr, ref_counts_out: Ptr, block_tables: Ptr,
                  context_lens: Ptr, ref_counts: Ptr, free_blocks: Ptr, num_free: Ptr,
                  copy_pairs: Ptr, new_ids: Ptr, counts: Ptr, workspace: Ptr,
                  workspace_bytes: int, num_seqs: int, max_num_blocks_per_seq: int,
                  block_size: int, num_blocks: int, max_moves: int,
                  stream: Optional[Stream] = None) -> None:
    """Moves the highest blocks in use to the lowest free ones, at most max_moves
    (swiftllm_hip_compact_pages): copy_pairs int64 [max_moves, 2] for
    paged_attention.copy_blocks, new_ids int32 [num_blocks], tables and
    references by the new ids, the free list, and counts int32 [2] = (moves,
    blocks in use). block_tables_out may be block_tables."""
    check_status(_lib.lib().swiftllm_hip_compact_pages(
        _p(block_tables_out), _p(ref_counts_out), _p(block_tables), _p(context_lens),
        _p(ref_counts), _p(free_blocks), _p(num_free), _p(copy_pairs), _p(new_ids), _p(counts),
        _p(workspace), workspace_bytes, num_seqs, max_num_blocks_per_seq, block_size, num_blocks,
        max_moves, _s(stream)))
