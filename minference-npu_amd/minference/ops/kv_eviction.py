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
    if q.dim() != 4 or k.dim() != 4 or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q [B,H,S_q,D] and k [B,H_kv,S_k,D] expected, got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"q heads {q.shape[1]} not a multiple of k heads {k.shape[1]}")
    check_supported(q, k)
    add = scores is not None
    if add:
        check_scores("scores", scores, k, k.shape[2])
        check_written("scores", scores, (("q", q), ("k", k)))
    else:
        scores = torch.empty(k.shape[:3], dtype=torch.float32, device=k.device)
    if q.numel() == 0:
        return scores if add else scores.zero_()
    s = dense_scale(q.shape[-1]) if scale is None else float(scale)
    dk = kernel_head_dim(q.shape[3])
    if dk == q.shape[3]:
        q, k = kernel_view(q), kernel_view(k)
    else:
        q, k = pad_head_dim(q, dk), pad_head_dim(k, dk)
    _abi.attention_weight_sums(q, k, scores, add, s)
    return scores


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
    dev = k_cache.device
    check_scores("scores", scores, k_cache, S)
    if out is None:
        ko, vo = (torch.empty((B, H, keep, D), dtype=k_cache.dtype, device=dev) for _ in range(2))
        so = torch.empty((B, H, keep), dtype=torch.float32, device=dev)
    else:
        ko, vo, so = out
        for name, t in (("k", ko), ("v", vo)):
            if tuple(t.shape) != (B, H, keep, D) or t.dtype != k_cache.dtype or t.device != dev:
                raise ValueError(f"out's {name} must be {k_cache.dtype} {(B, H, keep, D)} on {dev}, "
                                 f"got {t.dtype} {tuple(t.shape)} on {t.device}")
            if D > 1 and t.stride(3) != 1:
                raise ValueError(f"out's {name} must be contiguous over D")
        check_scores("out's scores", so, k_cache, keep)
        ins = [("k_cache", k_cache), ("v_cache", v_cache), ("scores", scores)]
        check_written("out's k", ko, ins)
        check_written("out's v", vo, ins + [("out's k", ko)])
        check_written("out's scores", so, ins + [("out's k", ko), ("out's v", vo)])
    pos = torch.empty((B, H, keep), dtype=torch.int32, device=dev)
    new_lens = torch.empty((B,), dtype=torch.int32, device=dev)
    if k_cache.numel() == 0:
        raise ValueError(f"the caches are empty: {tuple(k_cache.shape)}")
    if D > 1 and k_cache.stride(3) != 1:
        k_cache = k_cache.contiguous()
    if D > 1 and v_cache.stride(3) != 1:
        v_cache = v_cache.contiguous()
    _abi.cache_evict(k_cache, v_cache, scores, lens, int(keep), int(recent), int(sinks), ko, vo, so,
                     pos, new_lens)
    return ko, vo, so, pos, new_lens
