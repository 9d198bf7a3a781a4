"""Cutting a KV cache to the keys that were attended.

``attention_weight_sums`` gives a prompt's keys their starting scores,
``decode_accumulate`` adds to them with every token, ``evict_kv_cache`` keeps
the attention sinks, the recent keys and the best scored ones between them.
The reference keeps every key (its ``kv_type`` is "dense" only,
minference/minference_configuration.py).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _abi
from .common import (accepts_float32, check_supported, check_written, dense_scale,
                     kernel_head_dim, kernel_view, pad_head_dim)

__all__ = ["attention_weight_sums", "evict_kv_cache", "check_scores"]

CACHE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def check_scores(name: str, t: torch.Tensor, k: torch.Tensor, n: int) -> None:
    """Scores of n keys a kv head of the cache k: float32 [B, H_kv, n],
    contiguous over the keys."""
    sh, ks = t.shape, k.shape
    if (len(sh) != 3 or sh[0] != ks[0] or sh[1] != ks[1] or sh[2] != n
            or t.dtype is not torch.float32):
        raise ValueError(f"{name} must be float32 {(*ks[:2], n)}, got {t.dtype} {tuple(sh)}")
    if t.device != k.device:
        raise ValueError(f"{name} must be on the cache's device")
    if n > 1 and t.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous over the keys")


@accepts_float32(("q", "k"), has_out=False, once=True)
def attention_weight_sums(
    q: torch.Tensor,
    k: torch.Tensor,
    *,
    scale: Optional[float] = None,
    scores: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The attention weights of a prompt's rows, summed per key.

    Args:
        q: ``[B, H, S_q, D]``, the last S_q rows of the prompt (all of them, or
            a window: ``q[:, :, -64:]``), row i at position S_k - S_q + i.
        k: ``[B, H_kv, S_k, D]``, ``H % H_kv == 0``, S_q <= S_k.
        scale: 1/sqrt(D) by default.
        scores: float32 ``[B, H_kv, S_k]``, contiguous over the keys: added to
            and returned (a prompt in chunks); None: a new tensor.

    Returns float32 ``[B, H_kv, S_k]``: entry (b, g, j) is the sum over the heads
    of kv head g and the rows at or after j of their causal softmax weights of
    key j.  The same call gives the same bits.  Rows with only scores of -inf
    add nothing.
    """
    if scores is not None:
        if k.dim() == 4:
            check_scores("scores", scores, k, k.shape[2])
        check_written("scores", scores, (("q", q), ("k", k)))
    s = dense_scale(q.shape[-1]) if scale is None else float(scale)
    result = _abi.calls().weight_sums(q, k, scores, s)
    if result is not None and result.__class__ is not int:
        return result
    # not taken as they are: why, or copies that are
    if q.dim() != 4 or k.dim() != 4 or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q [B,H,S_q,D] and k [B,H_kv,S_k,D] expected, got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"q heads {q.shape[1]} not a multiple of k heads {k.shape[1]}")
    check_supported(q, k)
    if q.numel() == 0:
        return scores if scores is not None else torch.zeros(k.shape[:3], dtype=torch.float32,
                                                             device=k.device)
    dk = kernel_head_dim(q.shape[3])
    if result.__class__ is int and result < 0 and dk != q.shape[3]:
        result = _abi.calls().weight_sums(pad_head_dim(q, dk), pad_head_dim(k, dk), scores, s)
    elif result == _abi.MSA_E_ALIGN:
        result = _abi.calls().weight_sums(kernel_view(q), kernel_view(k), scores, s)
    _abi.check_call(result)
    return result


def evict_kv_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scores: torch.Tensor,
    keep: int,
    *,
    recent: int = 0,
    sinks: int = 0,
    lens: Optional[torch.Tensor] = None,
    out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The cache cut to ``keep`` keys per kv head, in their order.

    The first ``sinks`` and the last ``recent`` keys of each sequence stay, and
    of those between them the best scored; ties go to the lower position, a NaN
    score counts as the highest.  A sequence of at most ``keep`` keys keeps all.

    Args:
        k_cache, v_cache: ``[B, H_kv, S, D]`` bf16, fp16 or float32, any D.
        scores: float32 ``[B, H_kv, S]``, contiguous over the keys.
        keep: 1 <= keep <= S, sinks + recent <= keep.
        lens: int32 ``[B]`` on the device, keys in use (None: S; values are
            clamped to [0, S]).
        out: (k, v, scores) to write into, ``[B, H_kv, keep, D]`` twice and
            ``[B, H_kv, keep]`` (views of larger buffers are fine), apart from
            the inputs and from each other; None: new tensors.

    Returns (k, v, scores, positions, lens): the kept rows and their scores, the
    int32 ``[B, H_kv, keep]`` positions they had, and the int32 ``[B]`` lengths,
    min(lens, keep).  Rows behind a shorter sequence are 0, their positions -1.
    """
    outs = (None, None, None)
    if out is not None:
        outs = _check_outs(k_cache, v_cache, scores, keep, out)
    result = _abi.calls().evict(k_cache, v_cache, scores, lens, keep, recent, sinks, *outs)
    if result.__class__ is tuple:
        return result
    # not taken as they are: why, or copies that are
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache and v_cache must be [B,H_kv,S,D] of one shape, got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    B, H, S, D = k_cache.shape
    if not (1 <= keep <= S and sinks >= 0 and recent >= 0 and sinks + recent <= keep):
        raise ValueError(f"1 <= keep <= S and sinks + recent <= keep expected, got keep={keep}, "
                         f"S={S}, sinks={sinks}, recent={recent}")
    _abi.require_device(k_cache, v_cache)
    if k_cache.dtype not in CACHE_DTYPES or v_cache.dtype != k_cache.dtype:
        raise NotImplementedError(f"caches must both be one of {CACHE_DTYPES}, got "
                                  f"{k_cache.dtype} and {v_cache.dtype}")
    check_scores("scores", scores, k_cache, S)
    _abi.check_lens(lens, B, k_cache.device)
    if k_cache.numel() == 0:
        raise ValueError(f"the caches are empty: {tuple(k_cache.shape)}")
    if result == _abi.MSA_E_ALIGN:
        result = _abi.calls().evict(k_cache.contiguous(), v_cache.contiguous(), scores, lens, keep,
                                    recent, sinks, *outs)
    _abi.check_call(result)
    return result


def _check_outs(k_cache: torch.Tensor, v_cache: torch.Tensor, scores: torch.Tensor, keep: int, out):
    """evict_kv_cache's outputs: shapes, types, and apart from all else."""
    ko, vo, so = out
    want = (*k_cache.shape[:2], keep, *k_cache.shape[3:])
    for name, t in (("k", ko), ("v", vo)):
        if tuple(t.shape) != want or t.dtype != k_cache.dtype or t.device != k_cache.device:
            raise ValueError(f"out's {name} must be {k_cache.dtype} {want} on {k_cache.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"out's {name} must be contiguous over D")
    check_scores("out's scores", so, k_cache, keep)
    ins = [("k_cache", k_cache), ("v_cache", v_cache), ("scores", scores)]
    check_written("out's k", ko, ins)
    check_written("out's v", vo, ins + [("out's k", ko)])
    check_written("out's scores", so, ins + [("out's k", ko), ("out's v", vo)])
    return ko, vo, so
