"""64-bit oracles of the cache operators, and how far a kernel may be from them.

The bounds count roundings: a score is a sum of D products in fp32, off by at
most (D + 2) half steps of the sum of magnitudes, so exp of it (and of the row's
maximum) by twice that relatively; P is held in two 16-bit parts (the square of
the type's half step), in fp16 it may be one (a half step); the exponential, the sums over keys and the division add
a few fp32 half steps, taken as 2^-18 in all.  A weighted mean moves by at most
the weights' relative error times the largest |v|, and again for the divisor.
"""

from __future__ import annotations

import torch

INF = float("inf")


def score_error(q, k, scale):
    """Largest absolute error of a scaled score: q [..., S_q, D], k [..., S_k, D] (64-bit)."""
    mag = (q.abs() @ k.abs().transpose(-1, -2)).amax().item() if k.shape[-2] else 0.0
    return (q.shape[-1] + 2) * 2.0 ** -24 * mag * scale


def weight_error(q, k, scale, dtype):
    """Relative error of a softmax weight."""
    return 2 * score_error(q, k, scale) + 2.0 ** -18


def attention(q, k, v, see, scale):
    """softmax(q k^T scale, over see) v in 64 bits, and the weights; a row that
    sees nothing (or scores of -inf only) is 0."""
    s = (q @ k.transpose(-1, -2)) * scale
    s = torch.where(see, s, torch.tensor(-INF, dtype=s.dtype))
    m = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), -INF, dtype=s.dtype)
    p = torch.where(see, torch.exp(s - torch.where(m == -INF, 0.0, m)), 0.0)
    den = p.sum(-1, keepdim=True)
    p = torch.where(den > 0, p / den, torch.where(den == 0, 0.0, den))
    return p @ v, p


def repeat_kv(t, group):
    return t.repeat_interleave(group, 1)


def shared_prefix(q, kp, vp, k, v, lens, scale):
    """[B, H, S_q, D] in 64 bits from CPU tensors, one sequence at a time on
    its visible keys only."""
    B, H, Sq, D = q.shape
    group = H // k.shape[1]
    out = torch.zeros(B, H, Sq, D, dtype=torch.float64)
    for b in range(B):
        n = k.shape[2] if lens is None else max(0, min(int(lens[b]), k.shape[2]))
        kk = torch.cat([kp[0], k[b, :, :n]], 1).double().repeat_interleave(group, 0)
        vv = torch.cat([vp[0], v[b, :, :n]], 1).double().repeat_interleave(group, 0)
        for i in range(Sq):
            m = kp.shape[2] + max(0, min(n, n - Sq + i + 1))
            see = torch.ones(1, m, dtype=torch.bool)
            out[b, :, i:i + 1] = attention(q[b, :, i:i + 1].double(), kk[:, :m], vv[:, :m], see, scale)[0]
    return out


def decode_accumulate(q, k, v, scores, lens, scale):
    """(out, scores) in 64 bits."""
    B, H, _, D = q.shape
    Hkv, group = k.shape[1], H // k.shape[1]
    out = torch.zeros(B, H, 1, D, dtype=torch.float64)
    upd = scores.double().clone()
    for b in range(B):
        n = k.shape[2] if lens is None else max(0, min(int(lens[b]), k.shape[2]))
        kk = k[b, :, :n].double().repeat_interleave(group, 0)
        vv = v[b, :, :n].double().repeat_interleave(group, 0)
        o, p = attention(q[b].double(), kk, vv, torch.ones(1, n, dtype=torch.bool), scale)
        out[b] = o
        upd[b, :, :n] += p[:, 0].reshape(Hkv, group, n).sum(1)
    return out, upd


def weight_sums(q, k, scale):
    """[B, H_kv, S_k] in 64 bits: causal softmax weights summed over rows and heads."""
    B, H, Sq, _ = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    see = torch.arange(Sk) <= torch.arange(Sq)[:, None] + (Sk - Sq)
    kk = repeat_kv(k, H // Hkv).double()
    _, p = attention(q.double(), kk, kk, see, scale)
    p = torch.where(see, p, torch.zeros((), dtype=p.dtype))
    return p.sum(2).reshape(B, Hkv, H // Hkv, Sk).sum(2)


def kept_positions(scores, n, keep, recent, sinks):
    """Positions one kv head keeps, ascending: scores [S] (NaN highest, ties low)."""
    if n <= keep:
        return list(range(n))
    sure = set(range(sinks)) | set(range(n - recent, n))
    free = [j for j in range(n) if j not in sure]
    free.sort(key=lambda j: (0, 0.0, j) if scores[j] != scores[j] else (1, -scores[j], j))
    return sorted(sure | set(free[:keep - len(sure)]))
