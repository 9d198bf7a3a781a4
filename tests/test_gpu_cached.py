"""shared_prefix_attention and decode_accumulate on the GPU against 64-bit
oracles (cached_oracle.py derives the bounds)."""

from __future__ import annotations

import pytest
import torch

import cached_oracle as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def rand(seed, *shape, dtype=BF16, sinks=False):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed))
    if sinks:
        x[:, :, :4] *= 8
    return x.to(dtype)


def bshd(t):
    """The same values with a token's heads adjacent in memory."""
    return t.transpose(1, 2).contiguous().transpose(1, 2)


def check_out(got, ref, q, ks, vs, scale, label):
    """got against ref: the weights' error times |v|, twice, and got's own rounding."""
    dt = q.dtype
    group = q.shape[1] // ks[0].shape[1]
    rel = 2.0 ** -18
    for k in ks:
        if k.shape[2]:
            rel = max(rel, O.weight_error(q.double(), O.repeat_kv(k.double(), group), scale, dt))
    vmax = max([v.double().abs().amax().item() for v in vs if v.numel()], default=0.0)
    p16 = (torch.finfo(dt).eps / 2) ** (2 if dt == BF16 else 1)
    tol = 2 * (rel + p16) * vmax + (torch.finfo(got.dtype).eps / 2) * ref.abs()
    err = (got.double().cpu() - ref).abs()
    print(f"[cached] {label}: err {err.max():.2e} tol {tol.min():.2e}", flush=True)
    assert (err <= tol).all(), (label, err.max().item())


PREFIX = [
    # B, H, Hkv, D, Sp, Sc, Sq, dtype, lens
    (1, 1, 1, 64, 1, 1, 1, BF16, None),
    (2, 4, 4, 96, 100, 17, 1, BF16, [17, 1]),
    (3, 8, 2, 128, 513, 40, 1, FP16, [40, 0, 13]),
    (5, 4, 1, 64, 33, 300, 1, BF16, [300, 129, 128, 31, 2]),
    (9, 8, 2, 128, 1000, 65, 1, BF16, None),            # 36 rows: two tiles, one short
    (20, 8, 1, 96, 2049, 9, 1, FP16, None),             # 160 rows: three row tiles
    (2, 40, 2, 128, 70, 70, 1, BF16, [70, 33]),         # 20 heads of a kv head
    (3, 4, 2, 96, 257, 50, 7, BF16, [50, 9, 7]),
    (2, 6, 3, 128, 31, 90, 33, FP16, [90, 64]),
    (3, 2, 1, 64, 128, 20, 8, BF16, [20, 3, 0]),        # fewer own keys than query rows
    (2, 4, 2, 256, 300, 33, 1, BF16, [33, 20]),
    (2, 4, 2, 256, 100, 33, 5, FP16, [33, 20]),
    (2, 2, 1, 512, 200, 40, 1, BF16, [40, 5]),
    (1, 2, 1, 512, 64, 40, 3, FP16, None),
    (2, 4, 4, 80, 77, 11, 1, BF16, [11, 4]),            # padded to 96
    (2, 4, 2, 96, 0, 40, 1, BF16, [40, 0]),             # no prefix, an empty sequence
    (2, 4, 2, 96, 50, 0, 1, BF16, None),                # no own cache
    (2, 4, 2, 64, 0, 30, 4, FP16, [30, 2]),             # rows that see nothing
    (3, 16, 1, 64, 700, 33, 1, BF16, [33, 32, 1]),      # 48 rows
    (7, 16, 1, 128, 300, 100, 1, FP16, None),           # 112 rows
    (2, 8, 1, 96, 65, 130, 20, FP16, [130, 97]),        # 160 rows of a sequence
    (1, 8, 8, 96, 20000, 600, 1, BF16, None),
    (130, 2, 1, 64, 40, 260, 1, BF16, [(7 * i) % 261 for i in range(130)]),
    (2, 2, 2, 128, 9000, 300, 40, BF16, [300, 150]),
    (3, 6, 2, 128, 200, 90, 6, FP16, [90, 5, 40]),      # 18 rows of a sequence, 54 in all
    (2, 32, 1, 96, 300, 150, 1, BF16, [150, 70]),       # 32 heads of a kv head
    (1, 20, 1, 64, 100, 300, 1, FP16, None),
    (9, 32, 1, 128, 500, 70, 1, BF16, [70 - 8 * i for i in range(9)]),
    (2, 8, 4, 96, 257, 60, 9, BF16, [60, 9]),
]


@pytest.mark.parametrize("case", PREFIX, ids=lambda c: "x".join(map(str, c[:7])))
@pytest.mark.parametrize("out32", [True, False])
def test_shared_prefix(gpu_device, case, out32):
    from minference import shared_prefix_attention

    B, H, Hkv, D, Sp, Sc, Sq, dt, lens = case
    q = rand(1, B, H, Sq, D, dtype=dt)
    kp, vp = rand(2, 1, Hkv, Sp, D, dtype=dt, sinks=True), rand(3, 1, Hkv, Sp, D, dtype=dt)
    k, v = rand(4, B, Hkv, Sc, D, dtype=dt), rand(5, B, Hkv, Sc, D, dtype=dt)
    scale = D ** -0.5
    ref = O.shared_prefix(q, kp, vp, k, v, lens, scale)
    if lens is not None:  # what lies behind a sequence is not used
        for b, n in enumerate(lens):
            k[b, :, n:], v[b, :, n:] = float("nan"), float("inf")
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu_device)
    out = torch.full(q.shape, float("nan"), dtype=torch.float32 if out32 else dt, device=gpu_device)
    got = shared_prefix_attention(*(t.to(gpu_device) for t in (q, kp, vp, k, v)), lens=ln, out=out)
    torch.cuda.synchronize()
    assert got is out
    if lens is not None:
        for b, n in enumerate(lens):
            k[b, :, n:], v[b, :, n:] = 0, 0
    check_out(got, ref, q, (kp, k), (vp, v), scale, case)


def test_shared_prefix_strided_views(gpu_device):
    """Heads adjacent per token, a part of a larger buffer, a strided output."""
    from minference import shared_prefix_attention

    B, H, Hkv, D, Sp, Sc, Sq = 2, 6, 2, 96, 150, 60, 3
    q, kp, vp = rand(1, B, H, Sq, D), rand(2, 1, Hkv, Sp, D), rand(3, 1, Hkv, Sp, D)
    k, v = rand(4, B, Hkv, Sc, D), rand(5, B, Hkv, Sc, D)
    lens = [60, 41]
    ref = O.shared_prefix(q, kp, vp, k, v, lens, 0.11)
    big = torch.full((B, Hkv, Sc + 40, D), float("nan"), dtype=BF16, device=gpu_device)
    bk, bv = big.clone()[:, :, 8:8 + Sc], big.clone()[:, :, 8:8 + Sc]
    bk.copy_(k)
    bv.copy_(v)
    out = bshd(torch.zeros(B, H, Sq, D, device=gpu_device))
    shared_prefix_attention(bshd(q).to(gpu_device), bshd(kp).to(gpu_device), bshd(vp).to(gpu_device),
                            bk, bv, lens=torch.tensor(lens, dtype=torch.int32, device=gpu_device),
                            scale=0.11, out=out)
    torch.cuda.synchronize()
    check_out(out, ref, q, (kp, k), (vp, v), 0.11, "strided")


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("Sq", [6, 40])
def test_shared_prefix_nonfinite_values(gpu_device, dt, Sq):
    """An Inf or NaN in V reaches the rows that see its key and no others;
    +-Inf and NaN keys behave as in softmax."""
    from minference import shared_prefix_attention

    B, H, Hkv, D, Sp, Sc = 2, 4, 2, 96, 40, 50
    q, kp, vp = rand(1, B, H, Sq, D, dtype=dt), rand(2, 1, Hkv, Sp, D, dtype=dt), rand(3, 1, Hkv, Sp, D, dtype=dt)
    k, v = rand(4, B, Hkv, Sc, D, dtype=dt), rand(5, B, Hkv, Sc, D, dtype=dt)
    lens = [50, 33]
    v[0, 0, 47, 5] = float("inf")   # the first rows of sequence 0 do not see it
    v[0, 0, 49, 17] = float("nan")  # only the last row sees it
    v[1, 1, 30, 3] = float("-inf")
    ref = O.shared_prefix(q, kp, vp, k, v, lens, D ** -0.5)
    got = shared_prefix_attention(*(t.to(gpu_device) for t in (q, kp, vp, k, v)),
                                  lens=torch.tensor(lens, dtype=torch.int32, device=gpu_device))
    torch.cuda.synchronize()
    got = got.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(torch.isinf(got), torch.isinf(ref))
    fin = torch.isfinite(ref)
    vf = torch.where(torch.isfinite(v), v, 0)
    check_out(torch.where(fin, got, 0), torch.where(fin, ref, 0.0), q, (kp, k), (vp, vf), D ** -0.5, "nonfinite")


def test_shared_prefix_infinite_scores(gpu_device):
    """A key of -inf scores gets weight 0; a row with only such keys is 0; +inf
    and NaN scores make the row NaN."""
    from minference import shared_prefix_attention

    D = 64
    q = torch.ones(1, 3, 1, D, dtype=BF16)
    kp = torch.zeros(1, 3, 40, D, dtype=BF16)
    vp = rand(3, 1, 3, 40, D)
    kp[0, 0] = float("-inf")       # head 0: every score -inf
    kp[0, 1, 7] = float("-inf")    # head 1: one of them
    kp[0, 2, 9] = float("inf")
    empty = torch.zeros(1, 3, 0, D, dtype=BF16)
    got = shared_prefix_attention(*(t.to(gpu_device) for t in (q, kp, vp, empty, empty)),
                                  out=torch.empty(1, 3, 1, D, device=gpu_device)).cpu()
    assert (got[0, 0] == 0).all()
    ref = (vp[0, 1].double().sum(0) - vp[0, 1, 7].double()) / 39
    assert (got[0, 1, 0].double() - ref).abs().max() < 2.0 ** -14 * vp.abs().max().double()
    assert torch.isnan(got[0, 2]).all()


ACCUMULATE = [
    # B, H, Hkv, D, S, dtype, lens
    (1, 1, 1, 64, 1, BF16, None),
    (1, 8, 8, 96, 1000, BF16, None),
    (3, 8, 2, 128, 777, FP16, [777, 0, 129]),
    (2, 16, 1, 64, 4097, BF16, [4097, 1]),
    (2, 40, 2, 96, 300, BF16, [300, 31]),   # 20 heads of a kv head
    (1, 4, 2, 256, 500, FP16, None),
    (2, 2, 2, 512, 130, BF16, [130, 64]),
    (1, 4, 4, 80, 65, BF16, None),
    (2, 4, 2, 64, 0, BF16, None),
    (1, 4, 2, 128, 30000, BF16, None),
    (70, 4, 2, 64, 400, BF16, [(37 * i) % 401 for i in range(70)]),  # more than 64 sequences
    (5, 2, 1, 96, 9000, FP16, [0, 9000, 0, 1, 0]),                    # one long among empty ones
]


@pytest.mark.parametrize("case", ACCUMULATE, ids=lambda c: "x".join(map(str, c[:5])))
@pytest.mark.parametrize("inplace", [True, False])
def test_decode_accumulate(gpu_device, case, inplace):
    from minference import decode_accumulate

    B, H, Hkv, D, S, dt, lens = case
    q = rand(1, B, H, 1, D, dtype=dt)
    k, v = rand(2, B, Hkv, S, D, dtype=dt, sinks=True), rand(3, B, Hkv, S, D, dtype=dt)
    scores = torch.rand(B, Hkv, S, generator=torch.Generator().manual_seed(4))
    scale = D ** -0.5
    ref, upd = O.decode_accumulate(q, k, v, scores, lens, scale)
    live = torch.ones(B, Hkv, S, dtype=torch.bool)
    for b, n in enumerate(lens or []):
        k[b, :, n:], v[b, :, n:] = float("nan"), float("nan")
        live[b, :, n:] = False
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu_device)
    dq, dk, dv = (t.to(gpu_device) for t in (q, k, v))
    runs = []
    for _ in range(2):  # the same call gives the same bits
        buf = torch.full((B, Hkv, S + 5), -7.0, device=gpu_device)
        ds = buf[:, :, 3:3 + S]
        if inplace:
            ds.copy_(scores)
        out, got = decode_accumulate(dq, dk, dv, ds if inplace else scores.to(gpu_device), lens=ln,
                                     out=torch.empty(q.shape, device=gpu_device),
                                     scores_out=None if inplace else ds)
        torch.cuda.synchronize()
        assert got is ds
        assert (buf[:, :, :3] == -7).all() and (buf[:, :, 3 + S:] == -7).all()
        runs.append((out.cpu(), got.cpu()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    out, got = runs[0]
    for b, n in enumerate(lens or []):
        k[b, :, n:], v[b, :, n:] = 0, 0
    check_out(out, ref, q, (k,), (v,), scale, case)
    behind = scores if inplace else torch.full_like(scores, -7.0)
    assert torch.equal(got[~live], behind[~live])
    rel = O.weight_error(q.double(), O.repeat_kv(k.double(), H // Hkv), scale, dt) if S else 0.0
    tol = rel * (upd - scores.double()) + (H // Hkv + 2) * 2.0 ** -24 * upd.abs()
    assert ((got.double() - upd).abs() <= tol)[live].all()


def test_decode_accumulate_infinite_scores(gpu_device):
    """Keys of -inf scores add nothing; only such keys: nothing and a row of 0."""
    from minference import decode_accumulate

    D, S = 64, 70
    q = torch.ones(1, 2, 1, D, dtype=BF16)
    k = torch.zeros(1, 2, S, D, dtype=BF16)
    k[0, 0] = float("-inf")
    k[0, 1, 3:] = float("-inf")
    v = rand(3, 1, 2, S, D)
    out, sc = decode_accumulate(*(t.to(gpu_device) for t in (q, k, v)),
                                torch.zeros(1, 2, S, device=gpu_device))
    torch.cuda.synchronize()
    assert (out[0, 0] == 0).all() and (sc[0, 0] == 0).all()
    assert (sc[0, 1, 3:] == 0).all()
    assert (sc[0, 1, :3] - 1 / 3).abs().max() < 2.0 ** -22


def test_float32_inputs_run_once(gpu_device):
    """float32 inputs: the call on their 16-bit roundings, the scores added
    once, also where a value lies beyond fp16's range."""
    from minference import decode_accumulate, shared_prefix_attention

    B, H, D, S = 2, 4, 96, 200
    for big in (1.0, 1e5):
        q, k, v = (rand(i, B, H, n, D, dtype=torch.float32) for i, n in ((1, 1), (2, S), (3, S)))
        v[0, 0, 0, 0] = big
        dt = FP16 if big == 1.0 else BF16
        dq, dk, dv = (t.to(gpu_device) for t in (q, k, v))
        zero = torch.zeros(B, H, S, device=gpu_device)
        out, sc = decode_accumulate(dq, dk, dv, zero.clone())
        ro, rs = decode_accumulate(dq.to(dt), dk.to(dt), dv.to(dt), zero.clone(),
                                   out=torch.empty_like(dq))
        assert out.dtype == torch.float32 and torch.equal(out, ro) and torch.equal(sc, rs)
        args = (dq, dk[:1, :, :150], dv[:1, :, :150], dk, dv)
        out = shared_prefix_attention(*args)
        ref = shared_prefix_attention(*(t.to(dt) for t in args), out=torch.empty_like(dq))
        assert torch.equal(out, ref)


def test_cached_graph_and_streams(gpu_device):
    """Captured and replayed, with eager calls between the replays, and on a
    side stream: the eager bits every time."""
    from minference import decode_accumulate, shared_prefix_attention

    B, H, Hkv, D, Sp, Sc = 3, 8, 2, 128, 700, 90
    q = rand(1, B, H, 1, D).to(gpu_device)
    kp, vp = (rand(i, 1, Hkv, Sp, D).to(gpu_device) for i in (2, 3))
    k, v = (rand(i, B, Hkv, Sc, D).to(gpu_device) for i in (4, 5))
    lens = torch.tensor([90, 1, 40], dtype=torch.int32, device=gpu_device)
    start = torch.rand(B, Hkv, Sc, device=gpu_device)

    def step(sc):
        a = shared_prefix_attention(q, kp, vp, k, v, lens=lens)
        return a, *decode_accumulate(q, k, v, start, lens=lens, scores_out=sc)

    zero = torch.zeros_like(start)
    ref = [t.clone() for t in step(zero.clone())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(zero.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    buf = zero.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step(buf)
    for _ in range(3):
        buf.zero_()
        captured[0].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, ref))
        eager = step(zero.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, ref))
