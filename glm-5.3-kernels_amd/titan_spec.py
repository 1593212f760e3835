# SPDX-License-Identifier: Apache-2.0
"""The end of a speculative decode step on MI355X: drafted tokens against the
target's probabilities.

A speculative step runs each request's drafts and the token before them
through the model as one chunk - the indexer's rows with next_n > 1
(sparse_indexer), titan_mla.mla_chunk_attention_paged over the paged cache -
and verify_drafts says which of the drafts stand and what follows them.  The
kernels (csrc/verify_drafts.hip) run on the caller's current stream without
host synchronisation, so the call is graph-capturable.
"""
from __future__ import annotations

import functools

import torch

import _glm53_lib as _lib

_MAX_REQUESTS_PER_CALL = 65535


def verify_drafts(target_probs: torch.Tensor, draft_ids: torch.Tensor, draft_probs: torch.Tensor | None,
                  cu_rows: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor, max_drafts: int):
    """Accept, replace or follow up drafted tokens so that the tokens kept are
    distributed as the target's, from given random numbers.

    Request r has the target rows cu_rows[r] .. cu_rows[r + 1) (the chunk
    attention's cu_seqlens_q): one for each draft, in order, and a last one.
    Draft x is taken while accept_u * q(x) < p(x) (p the target's row, q the
    draft model's, 1 without draft_probs).  The first that is not taken is
    replaced by a token drawn from max(p - q, 0) (from p without x); where all
    are taken one more is drawn from the last row.  Token v weighs
    floor(min(max(p - q, 0), 1) * 2^40) in the draw, W is the weights' sum, and
    the token is the first whose running sum passes floor(sample_u * W): sums of
    whole numbers, the same however they are split.  Where every weight is 0
    the target's own row serves.

    Args:
        target_probs: fp32 [rows, vocab]
        draft_ids:    int32 / int64 [D], the requests' drafts one after another
                      (request r's begin at cu_rows[r] - r); an id outside the
                      vocabulary is not taken
        draft_probs:  fp32 [D, vocab] or None (drafts without probabilities)
        cu_rows:      int32 [R + 1], ascending
        accept_u:     fp32 [D], uniform in [0, 1)
        sample_u:     fp64 [R], uniform in [0, 1)
        max_drafts:   most drafts of a request; more than these are not looked at

    Returns (tokens int32 [R, max_drafts + 1], accepted int32 [R]): the accepted
    drafts, the drawn token, then -1.  A request with no target row (a padded
    batch), or whose rows lie outside target_probs or draft_ids, has only -1 and
    0; the drawn token is -1 where the target's row has no weight either.
    """
    # (sizes, strides and addresses are taken once: a small call's time is this function's)
    ps, id_type = target_probs.shape, draft_ids.dtype
    if len(ps) != 2 or target_probs.dtype is not torch.float32 or ps[1] < 1:
        raise ValueError(f"target_probs must be fp32 [rows, vocab], got {target_probs.dtype} {tuple(ps)}")
    rows, vocab = ps
    ids64 = id_type is torch.int64
    if not (ids64 or id_type is torch.int32) or draft_ids.dim() != 1:
        raise ValueError("draft_ids must be int32 or int64 [D]")
    D, R = draft_ids.numel(), cu_rows.numel() - 1
    if draft_probs is not None and (draft_probs.dtype is not torch.float32 or tuple(draft_probs.shape) != (D, vocab)):
        raise ValueError(f"draft_probs must be fp32 [{D}, {vocab}]")
    if cu_rows.dtype is not torch.int32 or cu_rows.dim() != 1 or R < 0:
        raise ValueError("cu_rows must be int32 [R + 1]")
    if accept_u.dtype is not torch.float32 or accept_u.dim() != 1 or accept_u.numel() != D:
        raise ValueError(f"accept_u must be fp32 [{D}]")
    if sample_u.dtype is not torch.float64 or sample_u.dim() != 1 or sample_u.numel() != R:
        raise ValueError(f"sample_u must be fp64 [{R}]")
    if max_drafts < 0:
        raise ValueError(f"max_drafts must be >= 0, got {max_drafts}")
    if R > _MAX_REQUESTS_PER_CALL:
        raise ValueError(f"at most {_MAX_REQUESTS_PER_CALL} requests per call, got {R}")
    index = target_probs.get_device()
    if index < 0 or draft_ids.get_device() != index or cu_rows.get_device() != index \
            or accept_u.get_device() != index or sample_u.get_device() != index \
            or (draft_probs is not None and draft_probs.get_device() != index):
        raise ValueError("verify_drafts requires CUDA (HIP) tensors on one device")
    dev = target_probs.device
    tokens = torch.empty((R, max_drafts + 1), dtype=torch.int32, device=dev)
    accepted = torch.empty(R, dtype=torch.int32, device=dev)
    if R == 0:
        return tokens, accepted
    if target_probs.stride(1) != 1:
        target_probs = target_probs.contiguous()
    draft_ptr, draft_step = None, 0
    if draft_probs is not None and D > 0:
        if draft_probs.stride(1) != 1:
            draft_probs = draft_probs.contiguous()
        draft_ptr, draft_step = draft_probs.data_ptr(), draft_probs.stride(0)
    draft_ids, cu_rows = draft_ids.contiguous(), cu_rows.contiguous()
    accept_u, sample_u = accept_u.contiguous(), sample_u.contiguous()
    L = _lib.load()
    with _lib.on_device(index):
        ws_bytes = _workspace_bytes(R, vocab)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        rc = L.glm53_verify_drafts(
            target_probs.data_ptr(), target_probs.stride(0), rows, draft_ptr, draft_step, draft_ids.data_ptr(), ids64, D,
            cu_rows.data_ptr(), accept_u.data_ptr(), sample_u.data_ptr(), R, vocab, max_drafts, workspace.data_ptr(),
            ws_bytes, tokens.data_ptr(), accepted.data_ptr(), _lib.raw_stream(index))
    if rc:
        _lib.check(rc, "glm53_verify_drafts")
    return tokens, accepted


@functools.lru_cache(maxsize=256)
def _workspace_bytes(requests, vocab):
    return int(_lib.load().glm53_verify_drafts_workspace_bytes(requests, vocab))
