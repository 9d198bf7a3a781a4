"""The cache operators of the package as measured calls: attention of a batch
over a shared prefix, decode that accumulates the attention weights, the
weights a prompt's rows give its keys, and eviction by those weights.

A case is a dict of plain values; ``op`` names the operator:

  prefix      shared_prefix_attention: B sequences, one prefix cache for all of
              them and a cache of its own for each
  accumulate  decode_accumulate: one query row per head against a cache, the
              weights of the row added to a running score per key
  sums        attention_weight_sums: what the last S_q rows of a prompt attend,
              summed per key
  evict       evict_kv_cache: the sinks, the recent keys and the best scored
              ones between them, moved together

Each has a plain form of elementary torch operations in 32 bits (``own`` false)
and the package's call (``own`` true).  Inputs are N(0, 1) with RoPE (theta
1e4) on q and k and the first four key rows times 8 (attention sinks).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _prefix(dtype, B, H, Hkv, D, Sp, Sc, Sq=1):
    return dict(op="prefix", dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, Sp=Sp, Sc=Sc, Sq=Sq)


def _accumulate(dtype, B, H, Hkv, D, S):
    return dict(op="accumulate", dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, S=S)


def _sums(dtype, B, H, Hkv, D, Sq, Sk):
    return dict(op="sums", dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, Sq=Sq, Sk=Sk)


def _evict(dtype, B, Hkv, D, S, keep, recent, sinks):
    return dict(op="evict", dtype=dtype, B=B, Hkv=Hkv, D=D, S=S, keep=keep, recent=recent,
                sinks=sinks)


def listed():
    return [
        # four answers sampled from one prompt of a few thousand tokens
        dict(name="prefix_b4_4k", **_prefix("bf16", 4, 32, 32, 96, 4096, 128)),
        # a batch of questions about one long document
        dict(name="prefix_b32_64k", **_prefix("bf16", 32, 32, 8, 128, 65536, 1024)),
        # many chats behind one long system prompt
        dict(name="prefix_b128_32k", **_prefix("fp16", 128, 32, 8, 128, 32768, 512)),
        # a few tokens of each sequence at once (drafted tokens, a short
        # question), odd lengths
        dict(name="prefix_rows16_20k", **_prefix("bf16", 8, 32, 32, 96, 20001, 700, 16)),
        # one token of a chat with a few thousand tokens of history
        dict(name="accumulate_4k", **_accumulate("bf16", 1, 32, 32, 96, 4113)),
        # small heads, odd lengths
        dict(name="accumulate_10k_d64", **_accumulate("fp16", 3, 16, 4, 64, 10007)),
        # a batch of long chats on a grouped-query model
        dict(name="accumulate_b8_64k", **_accumulate("bf16", 8, 32, 8, 128, 65536)),
        # what the last rows of a long prompt attend, before its cache is cut
        dict(name="sums_64_of_128k", **_sums("bf16", 1, 32, 32, 96, 64, 131072)),
        # one chunk of a prompt, odd lengths
        dict(name="sums_1000_of_5001", **_sums("fp16", 2, 32, 8, 96, 1000, 5001)),
        # every row of a prompt
        dict(name="sums_16k", **_sums("bf16", 1, 16, 4, 128, 16384, 16384)),
        # a chat's cache cut to a quarter
        dict(name="evict_4k", **_evict("bf16", 1, 32, 96, 4113, 1024, 256, 4)),
        # a batch of long caches cut to a quarter, ragged lengths
        dict(name="evict_b8_64k", **_evict("bf16", 8, 8, 128, 65536, 16384, 1024, 4)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges that the listed ones stand for."""
    op = rng.choice(["prefix", "prefix", "accumulate", "accumulate", "sums", "sums", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([64, 96, 96, 128, 128])
    group = rng.choice([1, 2, 4, 8])
    Hkv = rng.choice([2, 4, 8]) if group > 1 else rng.choice([8, 16, 32])
    H = Hkv * group
    if op == "prefix":
        Sq = rng.choice([1, 1, 1, _log(rng, 2, 40)])
        B = _log(rng, 1, 128 if Sq == 1 else 8)
        return _prefix(dtype, B, H, Hkv, D, _log(rng, 64, 32768), Sq + _log(rng, 1, 1000), Sq)
    if op == "accumulate":
        return _accumulate(dtype, rng.randint(1, 8), H, Hkv, D, _log(rng, 64, 40000))
    if op == "sums":
        Sq = _log(rng, 1, 4096)
        return _sums(dtype, rng.randint(1, 2), 16, 16 // group, D, Sq, max(Sq, _log(rng, 64, 16000)))
    S = _log(rng, 64, 60000)
    keep = max(16, S // rng.randint(2, 12))
    return _evict(dtype, rng.randint(1, 8), Hkv, D, S, keep, rng.randint(0, keep // 2),
                  rng.choice([0, 1, 4]))


def _lens(case):
    """Lengths of a ragged batch: from the longest down to a third of it."""
    hi = case["Sc"] if case["op"] == "prefix" else case["S"]
    B = case["B"]
    lo = case.get("Sq", 1)
    return [max(lo, hi - (i * (2 * hi // 3)) // max(1, B - 1)) for i in range(B)]


def _rope(x, offset=0):
    """Rotate-half RoPE of [B, H, S, D] fp32 at positions offset .. offset + S - 1."""
    D, S = x.shape[-1], x.shape[-2]
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    ang = torch.outer(torch.arange(S, dtype=torch.float64, device=x.device) + offset, inv)
    cos, sin = ang.cos().float(), ang.sin().float()
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, Hkv, D = case["B"], case["Hkv"], case["D"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    def keys(b, s, offset=0, sinks=True):
        k = _rope(randn(b, Hkv, s, D), offset)
        if sinks:
            k[:, :, :4] *= 8
        return k.to(dt)

    st = dict(case=case)
    if case["op"] == "prefix":
        H, Sp, Sc, Sq = case["H"], case["Sp"], case["Sc"], case["Sq"]
        st["q"] = _rope(randn(B, H, Sq, D), Sp + Sc - Sq).to(dt)
        st["kp"], st["vp"] = keys(1, Sp), randn(1, Hkv, Sp, D).to(dt)
        st["k"], st["v"] = keys(B, Sc, Sp, sinks=False), randn(B, Hkv, Sc, D).to(dt)
        st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEVICE)
    elif case["op"] == "accumulate":
        H, S = case["H"], case["S"]
        st["q"] = _rope(randn(B, H, 1, D), S - 1).to(dt)
        st["k"], st["v"] = keys(B, S), randn(B, Hkv, S, D).to(dt)
        st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEVICE)
        st["scores"] = torch.rand(B, Hkv, S, generator=g, device=DEVICE)
        st["updated"] = torch.zeros(B, Hkv, S, device=DEVICE)
    elif case["op"] == "sums":
        H, Sq, Sk = case["H"], case["Sq"], case["Sk"]
        st["q"] = _rope(randn(B, H, Sq, D), Sk - Sq).to(dt)
        st["k"] = keys(B, Sk)
    else:
        S = case["S"]
        st["k"], st["v"] = keys(B, S), randn(B, Hkv, S, D).to(dt)
        st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEVICE)
        # a few heavy keys, many small ones, and keys that nothing attended
        x = torch.exp(3 * randn(B, Hkv, S))
        st["scores"] = x * (torch.rand(B, Hkv, S, generator=g, device=DEVICE) > 0.2)
    return st


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "minference-npu_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import minference

    return minference


def run(state):
    case = state["case"]
    if own:
        m = _package()
        if case["op"] == "prefix":
            return m.shared_prefix_attention(state["q"], state["kp"], state["vp"], state["k"],
                                             state["v"], lens=state["lens"])
        if case["op"] == "accumulate":
            return m.decode_accumulate(state["q"], state["k"], state["v"], state["scores"],
                                       lens=state["lens"], scores_out=state["updated"])
        if case["op"] == "sums":
            return m.attention_weight_sums(state["q"], state["k"])
        return m.evict_kv_cache(state["k"], state["v"], state["scores"], case["keep"],
                                recent=case["recent"], sinks=case["sinks"], lens=state["lens"])
    return _PLAIN[case["op"]](state, case)


# ---- plain forms -----------------------------------------------------------


def _plain_prefix(st, c):
    B, H, Hkv, D, Sq, Sc = c["B"], c["H"], c["Hkv"], c["D"], c["Sq"], c["Sc"]
    G = H // Hkv
    q = st["q"].float().reshape(B, Hkv, G * Sq, D) / math.sqrt(D)
    # prefix: the rows of all sequences against one cache
    qp = q.transpose(0, 1).reshape(Hkv, B * G * Sq, D)
    sp = qp @ st["kp"][0].float().transpose(1, 2)
    sp = sp.reshape(Hkv, B, G * Sq, c["Sp"]).transpose(0, 1)
    so = q @ st["k"].float().transpose(2, 3)
    row = torch.arange(Sq, device=q.device).repeat(G)
    last = st["lens"].view(B, 1).long() - Sq + row  # last own key a row sees
    hidden = torch.arange(Sc, device=q.device) > last[:, None, :, None]
    so = so.masked_fill(hidden, -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    pp, po = torch.exp(sp - m), torch.exp(so - m)
    den = pp.sum(-1, keepdim=True) + po.sum(-1, keepdim=True)
    op = pp.transpose(0, 1).reshape(Hkv, B * G * Sq, c["Sp"]) @ st["vp"][0].float()
    o = op.reshape(Hkv, B, G * Sq, D).transpose(0, 1) + po @ st["v"].float()
    return (o / den).reshape(B, H, Sq, D).to(st["q"].dtype)


def _plain_accumulate(st, c):
    B, H, Hkv, D, S = c["B"], c["H"], c["Hkv"], c["D"], c["S"]
    q = st["q"].float().view(B, Hkv, H // Hkv, D) / math.sqrt(D)
    live = (torch.arange(S, device=q.device) < st["lens"].view(B, 1))[:, None]
    s = (q @ st["k"].float().transpose(2, 3)).masked_fill(~live[:, :, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p @ st["v"].float()).view(B, H, 1, D).to(st["q"].dtype)
    return o, torch.where(live, st["scores"] + p.sum(2), st["updated"])


def _plain_sums(st, c):
    B, H, Hkv, D, Sq, Sk = c["B"], c["H"], c["Hkv"], c["D"], c["Sq"], c["Sk"]
    q = st["q"].float().view(B, Hkv, (H // Hkv) * Sq, D) / math.sqrt(D)
    s = (q @ st["k"].float().transpose(2, 3)).view(B, H, Sq, Sk)
    row = torch.arange(Sq, device=q.device)[:, None] + (Sk - Sq)
    s = s.masked_fill_(torch.arange(Sk, device=q.device) > row, -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    s = s.div_(s.sum(-1, keepdim=True))
    return s.sum(2).view(B, Hkv, H // Hkv, Sk).sum(2)


def _plain_evict(st, c):
    S, keep, D = c["S"], c["keep"], c["D"]
    lens = st["lens"].view(-1, 1, 1).long()
    j = torch.arange(S, device=st["k"].device)
    score = st["scores"].masked_fill((j < c["sinks"]) | (j >= lens - c["recent"]), math.inf)
    score = score.masked_fill(j >= lens, -1.0)  # scores are sums of weights, not below 0
    pos = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    pos = torch.sort(pos, dim=-1).values
    gone = pos >= lens  # a sequence shorter than keep
    at = pos[..., None].expand(-1, -1, -1, D)
    k = torch.gather(st["k"], 2, at).masked_fill(gone[..., None], 0)
    v = torch.gather(st["v"], 2, at).masked_fill(gone[..., None], 0)
    scores = torch.gather(st["scores"], 2, pos).masked_fill(gone, 0)
    return (k, v, scores, pos.masked_fill(gone, -1).int(),
            st["lens"].clamp(max=keep))


_PLAIN = dict(prefix=_plain_prefix, accumulate=_plain_accumulate, sums=_plain_sums,
              evict=_plain_evict)


# ---- 64-bit results --------------------------------------------------------


def _root(c):
    return float(c["D"]) ** 0.5


def _exact_prefix(st, c):
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
    G, Sp, Sq = c["H"] // c["Hkv"], c["Sp"], c["Sq"]
    for b, n in enumerate(_lens(c)):
        see = torch.ones(Sq, Sp + n, device=DEVICE).tril(Sp + n - Sq).bool()
        for h in range(c["Hkv"]):
            k = torch.cat([st["kp"][0, h], st["k"][b, h, :n]]).double()
            v = torch.cat([st["vp"][0, h], st["v"][b, h, :n]]).double()
            x = torch.einsum("gid,jd->gij", st["q"][b, h * G:(h + 1) * G].double(), k)
            x = torch.where(see, x / _root(c), -math.inf)
            out[b, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v
    return out


def _exact_accumulate(st, c):
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
    scores = st["updated"].double().clone()
    G = c["H"] // c["Hkv"]
    for b, n in enumerate(_lens(c)):
        for h in range(c["Hkv"]):
            x = st["q"][b, h * G:(h + 1) * G, 0].double() @ st["k"][b, h, :n].double().t()
            w = torch.softmax(x / _root(c), -1)
            out[b, h * G:(h + 1) * G, 0] = w @ st["v"][b, h, :n].double()
            scores[b, h, :n] = st["scores"][b, h, :n].double() + w.sum(0)
    return out, scores


def _exact_sums(st, c):
    B, H, Hkv, Sq, Sk = c["B"], c["H"], c["Hkv"], c["Sq"], c["Sk"]
    out = torch.zeros(B, Hkv, Sk, dtype=torch.float64, device=DEVICE)
    for b in range(B):
        for h in range(H):
            for r in range(0, Sq, 4096):
                x = st["q"][b, h, r:r + 4096].double() @ st["k"][b, h * Hkv // H].double().t()
                past = torch.ones_like(x, dtype=torch.bool).triu(Sk - Sq + r + 1)
                x = (x / _root(c)).masked_fill(past, -math.inf)
                out[b, h * Hkv // H] += torch.softmax(x, -1).sum(0)
    return out


def _exact_evict(st, c):
    import numpy as np

    B, Hkv, D, keep = c["B"], c["Hkv"], c["D"], c["keep"]
    scores = st["scores"].cpu().numpy()
    pos = np.full((B, Hkv, keep), -1, np.int32)
    for b, n in enumerate(_lens(c)):
        sure = sorted(set(range(min(n, c["sinks"]))) | set(range(max(0, n - c["recent"]), n)))
        if n <= keep:
            pos[b, :, :n] = np.arange(n)
            continue
        free = np.setdiff1d(np.arange(n), sure)
        for h in range(Hkv):
            best = free[np.lexsort((free, -scores[b, h, free].astype(np.float64)))]
            pos[b, h] = np.sort(np.concatenate([best[:keep - len(sure)], np.array(sure, int)]))
    at = torch.from_numpy(pos).to(DEVICE).long()
    none = at < 0
    b, h = torch.arange(B, device=DEVICE)[:, None, None], torch.arange(Hkv, device=DEVICE)[:, None]
    kvs = [st[n][b, h, at.clamp(min=0)].double() for n in ("k", "v", "scores")]
    for t in kvs:
        t[none] = 0
    return (*kvs, at.int(), torch.tensor([min(n, keep) for n in _lens(c)], dtype=torch.int32))


_EXACT = dict(prefix=_exact_prefix, accumulate=_exact_accumulate, sums=_exact_sums,
              evict=_exact_evict)


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed), case)


# ---- work ------------------------------------------------------------------


def work(case):
    """Bytes of each input read once and each output written once, and the
    products of the visible (row, key) pairs."""
    c, B, Hkv, D = case, case["B"], case["Hkv"], case["D"]
    if c["op"] == "prefix":
        own_keys = sum(_lens(c))
        rows = c["H"] * c["Sq"]
        pairs = rows * (B * c["Sp"] + own_keys) - B * c["H"] * (c["Sq"] * (c["Sq"] - 1) // 2)
        return dict(bytes=4 * D * Hkv * (c["Sp"] + own_keys) + 4 * B * rows * D + 4 * B,
                    flops=4 * D * pairs)
    if c["op"] == "accumulate":
        keys = sum(_lens(c))
        return dict(bytes=Hkv * keys * (4 * D + 8) + 4 * B * c["H"] * D + 4 * B,
                    flops=4 * D * c["H"] * keys)
    if c["op"] == "sums":
        Sq, Sk = c["Sq"], c["Sk"]
        pairs = B * c["H"] * (Sq * Sk - Sq * (Sq - 1) // 2)
        return dict(bytes=2 * B * D * (c["H"] * Sq + Hkv * Sk) + 4 * B * Hkv * Sk,
                    flops=2 * D * pairs)
    lens = _lens(c)
    kept = sum(min(n, c["keep"]) for n in lens)
    return dict(bytes=Hkv * (4 * sum(lens) + kept * (4 * D + 4) + B * c["keep"] * (4 * D + 8)) + 8 * B,
                flops=Hkv * sum(lens))
