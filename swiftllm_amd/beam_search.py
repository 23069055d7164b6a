"""Beam search over the paged cache, all of it on the device.

    beam_select    the best continuations of every request's beams

The reference has no beam search; its samplers are on the host
(crates/swiftllm-core/src/sampling/mod.rs, whose order of ties, the lower index
first, is kept). Device tensors are DeviceArrays or raw device pointers (ints).
Nothing here synchronises or allocates, so every call may be captured in a graph.
"""

from __future__ import annotations

from typing import Optional

from . import _lib
from ._hip import Stream
from .paged_attention import CudaError, NotSupported, Ptr, _p, _s, check_status

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
                eos_id: int = -1, stream: Optional[Stream] = None) -> None:
    """The num_candidates largest of beam_scores[row] + log softmax(logits[row])
    over the rows request * beam_width + beam of every request and their tokens,
    in descending order, and the first beam_width of them that do not end with
    eos_id (swiftllm_hip_beam_select): scores float32, rows and tokens int32,
    -inf, -1 and -1 where there is none. next_rows are the parents of
    pages.fork_pages; next_scores may be beam_scores."""
    if dtype not in LOGIT_DTYPES:
        raise NotSupported(f"dtype {dtype!r} (supported: {', '.join(LOGIT_DTYPES)})")
    check_status(_lib.lib().swiftllm_hip_beam_select(
        _p(logits), _p(beam_scores), _p(cand_scores), _p(cand_rows), _p(cand_tokens),
        _p(next_scores), _p(next_rows), _p(next_tokens), _p(workspace), workspace_bytes,
        LOGIT_DTYPES[dtype], num_requests, beam_width, vocab, num_candidates,
        vocab if logits_stride is None else logits_stride, eos_id, _s(stream)))
