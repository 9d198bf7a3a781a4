"""Attention over caches that a batch shares or that are about to be cut.

``shared_prefix_attention``: the sequences of a batch continue one prefix,
whose cache is held once and read once for all of them.  ``decode_accumulate``:
one query row per head, as decode_dense (reference
minference/backend_npu/attention.py:274-314), which also adds the attention
weights to a running score per key, the scores ``evict_kv_cache`` cuts a cache
by.  The reference has neither: it keeps one full cache per sequence.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _abi
from ..ops.common import (SUPPORTED_DTYPES, accepts_float32, check_written, dense_scale,
                          kernel_head_dim, kernel_view, make_out, pad_head_dim)
from ..ops.kv_eviction import check_scores

__all__ = ["shared_prefix_attention", "decode_accumulate"]


def _check_caches(q: torch.Tensor, pairs) -> None:
    """Shapes, types and devices of (name, k, v, batch) cache pairs against q."""
    qs = q.shape
    if len(qs) != 4:
        raise ValueError(f"q must be 4-D [B,H,S,D], got {len(qs)}-D")
    kv_heads = pairs[0][1].shape[1] if pairs[0][1].dim() > 1 else 0
    for name, k, v, batch in pairs:
        ks = k.shape
        if len(ks) != 4 or v.shape != ks:
            raise ValueError(f"k and v of the {name} must be 4-D [B,H_kv,S,D] of one shape, got "
                             f"{tuple(ks)} and {tuple(v.shape)}")
        if ks[0] != batch or ks[3] != qs[3]:
            raise ValueError(f"the {name} must be [{batch},H_kv,S,{qs[3]}] for q {tuple(qs)}, got "
                             f"{tuple(ks)}")
        if ks[1] < 1 or qs[1] % ks[1]:
            raise ValueError(f"q heads {qs[1]} not a multiple of {name} heads {ks[1]}")
        if ks[1] != kv_heads:
            raise ValueError("prefix and own caches must have the same kv heads")
    _abi.require_device(q, *(t for p in pairs for t in p[1:3]))
    dt = q.dtype
    if dt not in SUPPORTED_DTYPES:
        raise NotImplementedError(f"the MI355X kernels take bf16 or fp16 inputs, got {dt}")
    for _, k, v, _ in pairs:
        if k.dtype != dt or v.dtype != dt:
            raise ValueError("q, k and v must share one dtype")
    if qs[3] < 1:
        raise ValueError("head_dim must be positive")


def _finish(result, call, ts, q: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    """The output of valid arguments that the library did not take as they are
    (``result``: its status): rows that are not aligned are copied, head dims the
    kernels are not built for are zero-padded (no dot product changes) and cut
    again."""
    d = q.shape[3]
    dk = kernel_head_dim(d)
    if result.__class__ is int and result < 0 and dk != d:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        tmp = call([pad_head_dim(t, dk) for t in ts],
                   torch.empty((*q.shape[:3], dk), dtype=out.dtype, device=q.device))
        _abi.check_call(tmp)
        return out.copy_(tmp[..., :d])
    if result == _abi.MSA_E_ALIGN:
        result = call([kernel_view(t) for t in ts], out)
    _abi.check_call(result)
    return result


def _check_out(q: torch.Tensor, out: torch.Tensor, others=()) -> None:
    """``out`` may lie where q or a cache does: it is written after they are read."""
    make_out(q, out)
    check_written("out", out, others)


@accepts_float32(("q", "k_prefix", "v_prefix", "k_cache", "v_cache"))
def shared_prefix_attention(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    lens: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of a batch whose sequences continue one shared prefix.

    Args:
        q: ``[B, H, S_q, D]``, the last S_q tokens of each sequence (1 for
            decode; a short question or drafted tokens otherwise).
        k_prefix, v_prefix: ``[1, H_kv, S_p, D]``, seen by every row;
            ``H % H_kv == 0``; S_p may be 0.
        k_cache, v_cache: ``[B, H_kv, S_c, D]``, each sequence's own keys after
            the prefix, the queries' own among them; S_c may be 0.
        lens: int32 ``[B]`` on the device, keys of each own cache in use (None:
            S_c; values are clamped to [0, S_c]).  Row i sees own keys
            ``j <= lens[b] - S_q + i``.  Keys behind lens[b] are not used,
            whatever they hold.
        scale: 1/sqrt(D) by default.
        out: q's shape, q's dtype or fp32; may be q itself.

    The prefix is read once per 64 query rows (batch x heads of a kv head x
    S_q), not once per sequence.  Equal to dense attention over the
    concatenated caches.  A row that sees no key, or only scores of -inf, is 0.
    """
    if out is not None:
        _check_out(q, out)
    s = dense_scale(q.shape[-1]) if scale is None else float(scale)

    def call(ts, result):
        return _abi.calls().shared_prefix(*ts, result, lens, s)

    ts = (q, k_prefix, v_prefix, k_cache, v_cache)
    result = call(ts, out)
    if result is not None and result.__class__ is not int:
        return result
    _check_caches(q, [("prefix", k_prefix, v_prefix, 1), ("own cache", k_cache, v_cache, q.shape[0])])
    _abi.check_lens(lens, q.shape[0], q.device)
    if q.numel() == 0:
        return torch.empty_like(q) if out is None else out
    return _finish(result, call, ts, q, out)


@accepts_float32(("q", "k_cache", "v_cache"), once=True)
def decode_accumulate(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scores: torch.Tensor,
    *,
    lens: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    scores_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_dense over a ragged batch, with the attention weights added to a
    score per key: ``scores_out[b, g, j] = scores[b, g, j] + sum of the weights
    that the heads of kv head g give key j``, j < lens[b].

    Args:
        q: ``[B, H, 1, D]``; k_cache, v_cache: ``[B, H_kv, S, D]``.
        scores: float32 ``[B, H_kv, S]``, contiguous over the keys.
        lens: int32 ``[B]`` on the device, keys in use (None: S; values are
            clamped to [0, S]).  Keys behind are not used, whatever they hold,
            and their scores are left as they are.
        scale: 1/sqrt(D) by default.
        out: q's shape, q's dtype or fp32, apart from the scores; may be q itself.
        scores_out: where the sums go; ``scores`` itself by default.

    Returns (out, scores_out).  The same call gives the same bits.  With lens[b]
    = 0, or only scores of -inf, a row is 0 and adds nothing.
    """
    if k_cache.dim() != 4 or not q.is_cuda:
        _check_caches(q, [("cache", k_cache, v_cache, q.shape[0])])
    check_scores("scores", scores, k_cache, k_cache.shape[2])
    if scores_out is None or scores_out is scores:
        scores_out = scores
        check_written("scores", scores)
    else:
        check_scores("scores_out", scores_out, k_cache, k_cache.shape[2])
        same = (scores_out.data_ptr() == scores.data_ptr()
                and scores_out.stride() == scores.stride())
        check_written("scores_out", scores_out, () if same else (("scores", scores),))
    if out is not None:
        _check_out(q, out, (("scores", scores), ("scores_out", scores_out)))
    s = dense_scale(q.shape[-1]) if scale is None else float(scale)

    def call(ts, result):
        return _abi.calls().decode_accumulate(*ts, result, lens, scores, scores_out, s)

    ts = (q, k_cache, v_cache)
    result = call(ts, out)
    if result is not None and result.__class__ is not int:
        return result, scores_out
    _check_caches(q, [("cache", k_cache, v_cache, q.shape[0])])
    if q.shape[2] != 1:
        raise NotImplementedError("decode_accumulate takes one query row")
    _abi.check_lens(lens, q.shape[0], q.device)
    if q.numel() == 0:
        return torch.empty_like(q) if out is None else out, scores_out
    return _finish(result, call, ts, q, out), scores_out
