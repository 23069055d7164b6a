"""Beam search over the paged cache, all of it on the device.

    beam_select    the best continuations of every request's beams
    BeamSearch     a search's state, and its step: selection, fork, plan

The reference has no beam search; its samplers are on the host
(crates/swiftllm-core/src/sampling/mod.rs, whose order of ties, the lower index
first, is kept). Device tensors are DeviceArrays or raw device pointers (ints).
beam_select and a search's steps neither synchronise nor allocate, so they may be
captured in a graph.
"""

from __future__ import annotations

from typing import Optional, Sequence

import numpy as np

from . import _lib
from ._hip import HIP_MEMCPY_D2D, DeviceArray, Stream, check, hip
from .attention_step import AttentionStep
from .pages import compact_pages, fork_pages, pages_workspace_size
from .paged_attention import (CudaError, InvalidParameter, NotSupported, Ptr, _p, _s, check_status,
                              copy_blocks)

LOGIT_DTYPES = {"f16": 0, "bf16": 1, "f32": 2}   # SWIFTLLM_HIP_F16, _BF16, _F32


def beam_select_workspace_size(num_requests: int, beam_width: int, vocab: int,
                               num_candidates: int) -> int:
    n = _lib.lib().swiftllm_hip_beam_select_workspace_size(num_requests, beam_width, vocab,
                                                           num_candidates)
    if n == 0:
        check_status(_lib.lib().swiftllm_hip_last_error() or CudaError.code)
    return int(n)


def beam_select(logits: Ptr, beam_scores: Ptr, cand_scores: Ptr, cand_rows: Ptr, cand_tokens: Ptr,
                next_scores: Ptr, next_rows: Ptr, next_tokens: Ptr, workspace: Ptr,
                workspace_bytes: int, num_requests: int, beam_width: int, vocab: int,
                num_candidates: int, dtype: str = "f32", logits_stride: Optional[int] = None,
                eos_id: int = -1, stream: Optional[Stream] = None, query_offsets: Ptr = None) -> None:
    """The num_candidates largest of beam_scores[row] + log softmax(logits[row])
    over the rows request * beam_width + beam of every request and their tokens,
    in descending order, and the first beam_width of them that do not end with
    eos_id (swiftllm_hip_beam_select): scores float32, rows and tokens int32,
    -inf, -1 and -1 where there is none. next_rows are the parents of
    pages.fork_pages; next_scores may be beam_scores. query_offsets int32 [rows + 1],
    as plan_step writes them: rows without a token in them have no logits, and their
    beams no score (swiftllm_hip_beam_select_rows)."""
    if dtype not in LOGIT_DTYPES:
        raise NotSupported(f"dtype {dtype!r} (supported: {', '.join(LOGIT_DTYPES)})")
    check_status(_lib.lib().swiftllm_hip_beam_select_rows(
        _p(logits), _p(beam_scores), _p(query_offsets), _p(cand_scores), _p(cand_rows), _p(cand_tokens),
        _p(next_scores), _p(next_rows), _p(next_tokens), _p(workspace), workspace_bytes,
        LOGIT_DTYPES[dtype], num_requests, beam_width, vocab, num_candidates,
        vocab if logits_stride is None else logits_stride, eos_id, _s(stream)))


class BeamSearch:
    """A beam search over a paged pool: the scores, tables, references and free list
    of num_requests requests of beam_width rows each, and what a step does with
    them. Row r * beam_width + w is beam w of request r; until a request's first
    selection its prompt is the first of its rows.

        search = BeamSearch(R, W, vocab, max_blocks, num_blocks, eos_id=2)
        step = AttentionStep(R * W, R * W, max_blocks, H, Hkv, D, score, inv_freq, num_groups=R)
        search.start(prompt_tables, prompt_lens)           # prompts that are in the cache
        search.select(logits)                              # of every row's last token
        search.fork(key_caches, value_caches, Hkv, D)      # tables and copies for the chosen
        search.plan(step)                                  # a block for each row's next token
        step.layer(q, k, v, key_cache, value_cache, out, decode=True)   # every layer

    next_tokens and scores are the rows' choice, cand_* all of a request's
    candidates, among them those that end with eos_id. A row whose score is -inf
    (a request's other rows at first; one that the caller gives up) ends, and its
    blocks are free again. A row that ended, that fork() cut or that plan() refused
    because no block was free (counts[1], step.counts[2]) brings no token, and the
    tokens of the rows behind it move up: row s's is token step.query_offsets[s] of the
    step. select() takes its logits in row s; one without a token has none to give, and
    ends there.

    From plan() to the next fork() the step's arrays hold what the search goes on from:
    select() and fork() refuse one that was planned again meanwhile, by another search
    or otherwise. Searches with one step between them change over after a fork(); one
    that is captured has a step of its own.

    The calls are asynchronous on `stream`, in that order; all but start() and
    compact() may be captured. fork() changes between two sets of tables, and what it
    counts is of the plan() before: a graph holds an even number of steps, is captured
    after the first step behind start(), and is replayed as many steps behind a start()
    as it was captured, or an even number more."""

    def __init__(self, num_requests: int, beam_width: int, vocab: int,
                 max_num_blocks_per_seq: int, num_blocks: int,
                 num_candidates: Optional[int] = None, eos_id: int = -1, dtype: str = "f32",
                 block_size: int = 16):
        if min(num_requests, beam_width, max_num_blocks_per_seq, num_blocks) <= 0:
            raise InvalidParameter(f"num_requests {num_requests} beam_width {beam_width} "
                                   f"max_num_blocks_per_seq {max_num_blocks_per_seq} num_blocks {num_blocks}")
        if dtype not in LOGIT_DTYPES:
            raise NotSupported(f"dtype {dtype!r} (supported: {', '.join(LOGIT_DTYPES)})")
        if block_size != 16:
            raise NotSupported(f"block_size {block_size} (supported: 16)")
        R, W, S = num_requests, beam_width, num_requests * beam_width
        C = max(W, min(2 * W, 64)) if num_candidates is None else num_candidates
        select_bytes = beam_select_workspace_size(R, W, vocab, C)
        pages_bytes = pages_workspace_size(S, num_blocks)
        self.num_requests, self.beam_width, self.vocab, self.num_candidates = R, W, vocab, C
        self.max_num_blocks_per_seq, self.num_blocks = max_num_blocks_per_seq, num_blocks
        self.eos_id, self.dtype, self.block_size, self.num_seqs = eos_id, dtype, block_size, S
        i32 = np.int32
        self._select_space = DeviceArray((select_bytes,), np.uint8)
        self._pages_space = DeviceArray((pages_bytes,), np.uint8)
        self.scores = DeviceArray((R, W), np.float32)
        self.next_rows, self.next_tokens = DeviceArray((R, W), i32), DeviceArray((R, W), i32)
        self.cand_scores = DeviceArray((R, C), np.float32)
        self.cand_rows, self.cand_tokens = DeviceArray((R, C), i32), DeviceArray((R, C), i32)
        self._tables = [DeviceArray.zeros((S, max_num_blocks_per_seq), i32) for _ in range(2)]
        self._lens = [DeviceArray.zeros((S,), i32) for _ in range(2)]
        self.new_lens = DeviceArray.zeros((S,), i32)
        self.ref_counts = DeviceArray.zeros((num_blocks,), i32)
        self.free_blocks, self.num_free = DeviceArray.zeros((num_blocks,), i32), DeviceArray.zeros((1,), i32)
        self.copy_pairs, self.counts = DeviceArray((S, 2), np.int64), DeviceArray((2,), i32)
        self.compact_counts = DeviceArray.zeros((2,), i32)
        self.group_offsets = DeviceArray.from_numpy(np.arange(R + 1, dtype=i32) * W)
        self._now, self._planned, self._plan_number = 0, None, 0

    @property
    def block_tables(self) -> DeviceArray:
        """[num_seqs, max_num_blocks_per_seq], as of the last fork() or start()."""
        return self._tables[self._now]

    @property
    def context_lens(self) -> DeviceArray:
        """[num_seqs]: after plan() with the token that the step brings."""
        step = self._its_step()
        return self._lens[self._now] if step is None else step.context_lens

    def _its_step(self) -> Optional[AttentionStep]:
        """What the last plan() planned, where there was no fork() since."""
        if self._planned is not None and self._planned.plans != self._plan_number:
            raise InvalidParameter("the step of the last plan() was planned again before fork()")
        return self._planned

    def start(self, block_tables: np.ndarray, context_lens: np.ndarray) -> None:
        """Tables [num_requests, at most max_num_blocks_per_seq] and lengths of the
        prompts; requests may share blocks, as prompts that begin alike do. Every
        other block of the pool is free. Synchronous."""
        R, W, BS, MB = self.num_requests, self.beam_width, self.block_size, self.max_num_blocks_per_seq
        # (64 bits until ids and lengths are known to fit 32)
        bt, lens = np.asarray(block_tables, np.int64), np.asarray(context_lens, np.int64)
        if bt.ndim != 2 or bt.shape[0] != R or bt.shape[1] > MB or lens.shape != (R,):
            raise InvalidParameter(f"block_tables {bt.shape} and context_lens {lens.shape} of {R} requests")
        if (lens < 0).any() or (lens > bt.shape[1] * BS).any():
            raise InvalidParameter("a prompt is longer than its table")
        tables, ctx = np.zeros((R * W, MB), np.int32), np.zeros(R * W, np.int32)
        tables[::W, :bt.shape[1]], ctx[::W] = bt, lens
        refs = np.zeros(self.num_blocks, np.int32)
        for row, n in zip(bt, lens):
            used = row[:-(-int(n) // BS)]
            if ((used < 0) | (used >= self.num_blocks)).any():
                raise InvalidParameter(f"a block outside the pool of {self.num_blocks}")
            np.add.at(refs, used, 1)
        free = np.flatnonzero(refs == 0).astype(np.int32)
        scores = np.full((R, W), -np.inf, np.float32)
        scores[:, 0] = 0.0
        self._now, self._planned = 0, None
        self._tables[0].upload(tables)
        self._lens[0].upload(ctx)
        self.ref_counts.upload(refs)
        self.free_blocks.upload(np.pad(free, (0, self.num_blocks - len(free))))
        self.num_free.upload(np.array([len(free)], np.int32))
        self.scores.upload(scores)

    def select(self, logits: Ptr, logits_stride: Optional[int] = None,
               stream: Optional[Stream] = None) -> None:
        """The best continuations (beam_select) of logits [num_seqs, vocab], of the rows
        that brought a token in the plan() before; scores become those of the rows that
        go on."""
        step = self._its_step()
        beam_select(logits, self.scores, self.cand_scores, self.cand_rows, self.cand_tokens,
                    self.scores, self.next_rows, self.next_tokens, self._select_space,
                    self._select_space.nbytes, self.num_requests, self.beam_width, self.vocab,
                    self.num_candidates, dtype=self.dtype, logits_stride=logits_stride,
                    eos_id=self.eos_id, stream=stream,
                    query_offsets=None if step is None else step.query_offsets)

    def fork(self, key_caches: Sequence[Ptr], value_caches: Sequence[Ptr], num_kv_heads: int,
             head_dim: int, stream: Optional[Stream] = None) -> None:
        """The chosen rows' tables (fork_pages), and in every layer's caches the
        copies of the blocks that they are about to write."""
        self._check_caches(key_caches, value_caches, num_kv_heads, head_dim)
        now, planned = self._now, self._its_step()
        fork_pages(self._tables[1 - now], self._lens[1 - now], self._tables[now], self.context_lens,
                   self.next_rows, self.ref_counts, self.free_blocks, self.num_free,
                   self.copy_pairs, self.counts, self._pages_space, self._pages_space.nbytes,
                   self.num_seqs, self.max_num_blocks_per_seq, self.block_size, self.num_blocks,
                   taken=None if planned is None else planned.counts, new_lens=self.new_lens,
                   stream=stream)
        self._now, self._planned = 1 - now, None
        copy_blocks(key_caches, value_caches, self.copy_pairs, self.num_seqs, num_kv_heads,
                    head_dim, self.block_size, stream=stream)

    @staticmethod
    def _check_caches(key_caches: Sequence[Ptr], value_caches: Sequence[Ptr], num_kv_heads: int,
                      head_dim: int) -> None:
        """What copy_blocks would refuse, before tables change that its copies belong to."""
        if len(key_caches) != len(value_caches):
            raise InvalidParameter(f"{len(key_caches)} key caches but {len(value_caches)} value caches")
        if num_kv_heads <= 0 or head_dim <= 0:
            raise InvalidParameter(f"num_kv_heads {num_kv_heads} head_dim {head_dim}")
        if not all(_p(c) for c in (*key_caches, *value_caches)):
            raise InvalidParameter("null cache")

    def plan(self, step: AttentionStep, stream: Optional[Stream] = None) -> None:
        """step.plan() of the rows that go on, by requests where the step has groups."""
        if self._planned is not None:
            raise InvalidParameter("plan() twice without a fork() between")
        mine = (self.num_seqs, self.max_num_blocks_per_seq, self.block_size)
        its = (step.num_seqs, step.max_num_blocks_per_seq, step.block_size)
        if its != mine or step.num_groups not in (0, self.num_requests):
            raise InvalidParameter(f"a step of (sequences, blocks, block size) {its} and {step.num_groups} groups "
                                   f"for a search of {mine} and {self.num_requests} requests")
        step.plan(self.block_tables, self.context_lens, self.new_lens, self.free_blocks,
                  self.num_free, self.num_blocks, num_blocks=self.num_blocks, stream=stream,
                  group_offsets=self.group_offsets if step.num_groups else None)
        self._planned, self._plan_number = step, step.plans

    def compact(self, key_caches: Sequence[Ptr], value_caches: Sequence[Ptr], num_kv_heads: int,
                head_dim: int, new_ids: DeviceArray, max_moves: int,
                stream: Optional[Stream] = None) -> None:
        """After fork(): the blocks in use to the pool's front, at most max_moves of
        them (compact_pages), in the tables, the references and every layer's caches.
        new_ids int32 [num_blocks] is for whoever else holds blocks, compact_counts are
        (moves, blocks in use); counts stay those of the fork(). Waits for the
        device and allocates: not for a capture."""
        if self._planned is not None:
            raise InvalidParameter("compact() between plan() and fork()")
        if max_moves < 0:
            raise InvalidParameter(f"max_moves {max_moves}")
        self._check_caches(key_caches, value_caches, num_kv_heads, head_dim)
        pairs = DeviceArray((max(max_moves, 1), 2), np.int64)
        refs = DeviceArray((self.num_blocks,), np.int32)
        compact_pages(self.block_tables, refs, self.block_tables, self.context_lens,
                      self.ref_counts, self.free_blocks, self.num_free, pairs, new_ids, self.compact_counts,
                      self._pages_space, self._pages_space.nbytes, self.num_seqs,
                      self.max_num_blocks_per_seq, self.block_size, self.num_blocks, max_moves,
                      stream=stream)
        check(hip().hipMemcpyAsync(self.ref_counts.ptr, refs.ptr, refs.nbytes, HIP_MEMCPY_D2D, _s(stream)),
              "hipMemcpyAsync")
        copy_blocks(key_caches, value_caches, pairs, max_moves, num_kv_heads, head_dim,
                    self.block_size, stream=stream)
