"""attention_weight_sums and evict_kv_cache on the GPU against 64-bit oracles,
and the cache operators run together as a serving loop uses them."""

from __future__ import annotations

import pytest
import torch

import cached_oracle as O
from test_gpu_cached import BF16, FP16, bshd, check_out, rand

pytestmark = pytest.mark.gpu


def sums_tol(ref, q, k, scale, base=None):
    """Bound of a column sum: each weight's error, and fp32 sums of 64 weights,
    of those, and of heads and waves."""
    G = q.shape[1] // k.shape[1]
    rel = O.weight_error(q.double(), O.repeat_kv(k.double(), G), scale, q.dtype)
    n = 64 + q.shape[2] * G / 256 + 32
    tol = (rel + n * 2.0 ** -24) * ref
    return tol if base is None else tol + 2.0 ** -23 * (base.double() + ref)


SUMS = [
    # B, H, Hkv, D, S_q, S_k, dtype
    (1, 1, 1, 64, 1, 1, BF16),
    (2, 4, 2, 96, 1, 300, BF16),
    (1, 8, 8, 96, 64, 5000, BF16),
    (2, 6, 2, 128, 77, 77, FP16),
    (1, 4, 1, 64, 200, 513, BF16),
    (1, 16, 2, 96, 17, 40, FP16),
    (3, 4, 4, 128, 130, 1001, BF16),
    (1, 2, 1, 256, 70, 200, BF16),
    (1, 2, 2, 512, 40, 90, FP16),
    (1, 2, 1, 80, 33, 100, BF16),
    (1, 20, 1, 64, 5, 70, BF16),
    (1, 32, 32, 96, 20, 9000, BF16),   # a key tile per wave
    (1, 4, 2, 96, 1500, 1500, BF16),   # row splits
    (1, 4, 4, 128, 16, 20000, FP16),   # key splits
    (2, 3, 3, 64, 64, 1000, FP16),     # a window, a kv head a head
    (1, 4, 4, 128, 1, 3001, BF16),
    (1, 5, 5, 256, 20, 700, BF16),
    (1, 3, 3, 512, 16, 500, FP16),
    (2, 2, 2, 96, 50, 50, BF16),
    (1, 32, 32, 64, 40, 86000, BF16),  # more keys than the caches hold
]


@pytest.mark.parametrize("case", SUMS, ids=lambda c: "x".join(map(str, c[:6])))
def test_weight_sums(gpu_device, case):
    from minference import attention_weight_sums

    B, H, Hkv, D, Sq, Sk, dt = case
    q, k = rand(1, B, H, Sq, D, dtype=dt), rand(2, B, Hkv, Sk, D, dtype=dt, sinks=True)
    scale = D ** -0.5
    ref = O.weight_sums(q, k, scale)
    dq, dk = q.to(gpu_device), k.to(gpu_device)
    got = attention_weight_sums(dq, dk)
    again = attention_weight_sums(dq, dk)
    torch.cuda.synchronize()
    assert torch.equal(got, again)
    err = (got.double().cpu() - ref).abs()
    tol = sums_tol(ref, q, k, scale)
    print(f"[sums] {case}: rel err {(err / ref.clamp(min=1e-300)).max():.2e}", flush=True)
    assert (err <= tol + 2.0 ** -126).all()
    # added to what a strided buffer holds, the rest of it untouched
    base = torch.rand(B, Hkv, Sk, generator=torch.Generator().manual_seed(3))
    buf = torch.full((B, Hkv, Sk + 3), -7.0, device=gpu_device)
    buf[:, :, 1:1 + Sk] = base.to(gpu_device)
    res = attention_weight_sums(bshd(dq), bshd(dk), scores=buf[:, :, 1:1 + Sk])
    torch.cuda.synchronize()
    assert res.data_ptr() == buf[:, :, 1:].data_ptr()
    assert (buf[:, :, 0] == -7).all() and (buf[:, :, 1 + Sk:] == -7).all()
    tol = sums_tol(ref, q, k, scale, base)
    assert ((res.double().cpu() - base.double() - ref).abs() <= tol).all()


def test_weight_sums_of_chunks(gpu_device):
    """A prompt in chunks adds up to the prompt."""
    from minference import attention_weight_sums

    q, k = rand(1, 1, 4, 700, 96), rand(2, 1, 2, 700, 96, sinks=True)
    ref = O.weight_sums(q, k, 96 ** -0.5)
    scores = torch.zeros(1, 2, 700, device=gpu_device)
    dq, dk = q.to(gpu_device), k.to(gpu_device)
    for a, b in ((0, 300), (300, 301), (301, 700)):
        attention_weight_sums(dq[:, :, a:b], dk[:, :, :b], scores=scores[:, :, :b])
    torch.cuda.synchronize()
    assert ((scores.double().cpu() - ref).abs() <= 3 * sums_tol(ref, q, k, 96 ** -0.5, scores.cpu())).all()


def test_weight_sums_nonfinite(gpu_device):
    """A NaN or +inf key makes the rows NaN that see it, so the keys they see; a
    -inf score weighs 0; rows of -inf only add nothing; keys behind are clean."""
    from minference import attention_weight_sums

    D, S = 64, 100
    q = torch.ones(1, 1, S, D, dtype=BF16)
    k = torch.zeros(1, 1, S, D, dtype=BF16)
    k[0, 0, 0] = float("-inf")  # row 0 sees nothing else
    got = attention_weight_sums(q.to(gpu_device), k.to(gpu_device)).cpu()[0, 0].double()
    see = torch.ones(S, S).tril().bool()
    see[:, 0] = False
    ref = (see.double() / see.sum(1, keepdim=True).clamp(min=1)).sum(0)
    assert (got - ref).abs().max() < 2.0 ** -18
    for bad in (float("nan"), float("inf")):
        k = torch.zeros(1, 1, S, D, dtype=BF16)
        k[0, 0, 40] = bad
        # rows 40.. see it; with only rows ..39 asked for, nothing is NaN
        full = attention_weight_sums(q.to(gpu_device), k.to(gpu_device)).cpu()
        assert torch.isnan(full[0, 0]).all()
        part = attention_weight_sums(q[:, :, :40].to(gpu_device), k[:, :, :40].to(gpu_device)).cpu()
        assert torch.isfinite(part).all()
    # a NaN query row reaches the keys it sees only
    k = torch.zeros(1, 1, S, D, dtype=BF16)
    q[0, 0, 50] = float("nan")
    got = attention_weight_sums(q.to(gpu_device), k.to(gpu_device)).cpu()
    assert torch.isnan(got[0, 0, :51]).all() and torch.isfinite(got[0, 0, 51:]).all()


EVICT = [
    # B, H, S, D, keep, recent, sinks, lens, dtype
    (1, 1, 1, 64, 1, 0, 0, None, BF16),
    (2, 3, 100, 96, 40, 10, 4, [100, 39], BF16),
    (2, 2, 5000, 128, 1000, 100, 4, [5000, 4097], FP16),
    (3, 2, 300, 80, 64, 64, 0, [300, 65, 0], BF16),     # recent only
    (1, 2, 300, 96, 64, 0, 64, None, BF16),             # sinks only
    (1, 2, 3000, 64, 500, 0, 0, None, torch.float32),   # scores only
    (2, 1, 70, 7, 30, 5, 5, [70, 31], BF16),            # rows of 14 bytes
    (1, 2, 300, 96, 300, 10, 4, None, BF16),            # nothing to drop
    (1, 2, 40000, 64, 9000, 1, 1, None, BF16),
    (2, 1, 70000, 64, 20000, 64, 4, [70000, 65537], BF16),
    (3, 1, 20000, 64, 5000, 4000, 1000, [20000, 5001, 4999], BF16),  # nothing by score
    (2, 33, 9001, 64, 4500, 100, 4, [9001, 8300], BF16),             # 66 rows, short stretches
    (1, 1, 300000, 64, 1000, 0, 0, None, BF16),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "x".join(map(str, c[:7])))
@pytest.mark.parametrize("kind", ["weights", "ties", "special"])
def test_evict(gpu_device, case, kind):
    from minference import evict_kv_cache

    B, H, S, D, keep, recent, sinks, lens, dt = case
    k, v = rand(1, B, H, S, D, dtype=dt), rand(2, B, H, S, D, dtype=dt)
    g = torch.Generator().manual_seed(5)
    scores = torch.exp(3 * torch.randn(B, H, S, generator=g))
    if kind == "ties":
        scores = torch.randint(0, 4, (B, H, S), generator=g).float()
    elif kind == "special":
        vals = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), -1.0, 1e-42, 3e38])
        scores = vals[torch.randint(0, 8, (B, H, S), generator=g)]
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu_device)
    buf = [torch.full((B, H, keep + 4, D), 9.0, dtype=dt, device=gpu_device) for _ in range(2)]
    sbuf = torch.full((B, H, keep + 4), 9.0, device=gpu_device)
    views = (buf[0][:, :, 2:2 + keep], buf[1][:, :, 2:2 + keep], sbuf[:, :, 2:2 + keep])
    dk, dv, ds = k.to(gpu_device), bshd(v.to(gpu_device)), scores.to(gpu_device)
    for out in (None, views):
        ko, vo, so, pos, nl = evict_kv_cache(dk, dv, ds, keep, recent=recent, sinks=sinks, lens=ln,
                                             out=out)
        torch.cuda.synchronize()
        assert pos.dtype == torch.int32 and nl.dtype == torch.int32
        ko, vo, so, pos = (t.cpu() for t in (ko, vo, so, pos))
        for b in range(B):
            n = S if lens is None else lens[b]
            assert int(nl[b]) == min(n, keep)
            for h in range(H):
                want = O.kept_positions(scores[b, h].tolist(), n, keep, recent, sinks)
                m = len(want)
                assert pos[b, h].tolist() == want + [-1] * (keep - m)
                at = torch.tensor(want, dtype=torch.long)
                assert torch.equal(ko[b, h, :m], k[b, h, at]) and (ko[b, h, m:] == 0).all()
                assert torch.equal(vo[b, h, :m], v[b, h, at]) and (vo[b, h, m:] == 0).all()
                assert torch.equal(torch.nan_to_num(so[b, h, :m]), torch.nan_to_num(scores[b, h, at]))
                assert (so[b, h, m:] == 0).all()
    for t in (*buf, sbuf):
        assert (t[:, :, :2] == 9).all() and (t[:, :, keep + 2:] == 9).all()


def test_serving_loop(gpu_device):
    """A prompt's keys scored, cut, decoded on with the scores kept up, cut
    again, then shared by a batch: every step against 64 bits."""
    from minference import (attention_weight_sums, decode_accumulate, dense_attention,
                            evict_kv_cache, shared_prefix_attention)

    H, Hkv, S, D, keep, steps = 8, 2, 600, 96, 200, 5
    dev, scale = gpu_device, D ** -0.5
    q, k, v = rand(1, 1, H, S, D), rand(2, 1, Hkv, S, D, sinks=True), rand(3, 1, Hkv, S, D)
    dq, dk, dv = q.to(dev), k.to(dev), v.to(dev)
    dense_attention(dq, dk.repeat_interleave(4, 1), dv.repeat_interleave(4, 1))
    sums = attention_weight_sums(dq, dk)
    # room for the tokens to come behind the kept keys
    cap = keep + steps
    kb, vb = (torch.zeros(1, Hkv, cap, D, dtype=BF16, device=dev) for _ in range(2))
    sb = torch.zeros(1, Hkv, cap, device=dev)
    *_, pos, lens = evict_kv_cache(dk, dv, sums, keep, recent=64, sinks=4,
                                   out=(kb[:, :, :keep], vb[:, :, :keep], sb[:, :, :keep]))
    for h in range(Hkv):
        want = O.kept_positions(sums[0, h].tolist(), S, keep, 64, 4)
        assert pos[0, h].tolist() == want
    assert torch.equal(kb[:, :, :keep], torch.gather(dk, 2, pos.long()[..., None].expand(-1, -1, -1, D)))
    for t in range(steps):
        kb[:, :, keep + t] = rand(10 + t, 1, Hkv, 1, D).to(dev)[:, :, 0]
        vb[:, :, keep + t] = rand(30 + t, 1, Hkv, 1, D).to(dev)[:, :, 0]
        lens = lens + 1
        x = rand(50 + t, 1, H, 1, D)
        before = sb.cpu()
        out, _ = decode_accumulate(x.to(dev), kb, vb, sb, lens=lens)
        torch.cuda.synchronize()
        ref, upd = O.decode_accumulate(x, kb.cpu(), vb.cpu(), before, [keep + t + 1], scale)
        check_out(out, ref, x, (kb.cpu(),), (vb.cpu(),), scale, f"step {t}")
        rel = O.weight_error(x.double(), O.repeat_kv(kb.cpu().double(), H // Hkv), scale, BF16)
        tol = rel * (upd - before.double()) + (H // Hkv + 2) * 2.0 ** -24 * upd
        assert ((sb.cpu().double() - upd).abs() <= tol).all()
    k2, v2, s2, pos, lens = evict_kv_cache(kb, vb, sb, 100, recent=16, sinks=4, lens=lens)
    B, Sc = 3, 7
    ko, vo, x = rand(70, B, Hkv, Sc, D), rand(71, B, Hkv, Sc, D), rand(72, B, H, 2, D)
    own = [7, 2, 5]
    got = shared_prefix_attention(x.to(dev), k2, v2, ko.to(dev), vo.to(dev),
                                  lens=torch.tensor(own, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    ref = O.shared_prefix(x, k2.cpu(), v2.cpu(), ko, vo, own, scale)
    check_out(got, ref, x, (k2.cpu(), ko), (v2.cpu(), vo), scale, "shared")


def test_eviction_graph_and_float32(gpu_device):
    """Captured and replayed with eager calls between; float32 inputs as their
    roundings, added once."""
    from minference import attention_weight_sums, evict_kv_cache

    q, k, v = (rand(i, 2, h, s, 96).to(gpu_device) for i, h, s in ((1, 8, 70), (2, 2, 900), (3, 2, 900)))
    lens = torch.tensor([900, 500], dtype=torch.int32, device=gpu_device)

    def step():
        s = attention_weight_sums(q, k)
        return (s, *evict_kv_cache(k, v, s, 128, recent=32, sinks=4, lens=lens))

    ref = [t.clone() for t in step()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for _ in range(3):
        for t in captured:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, ref))
        assert all(torch.equal(a, b) for a, b in zip(step(), ref))
    f = rand(4, 1, 2, 50, 96, dtype=torch.float32).to(gpu_device)
    one = torch.ones(1, 2, 50, device=gpu_device)
    assert torch.equal(attention_weight_sums(f, f, scores=one.clone()),
                       attention_weight_sums(f.half(), f.half(), scores=one.clone()))
    big = f.clone()
    big[0, 0, 0, 0] = 1e5
    assert torch.equal(attention_weight_sums(big, f, scores=one.clone()),
                       attention_weight_sums(big.bfloat16(), f.bfloat16(), scores=one.clone()))
