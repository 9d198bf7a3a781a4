"""The cache operators as callers may use them beside the usual: long offsets,
broadcast and unaligned views, outputs over inputs, lengths out of range, empty
batches, calls on two streams at once, two captured graphs."""

from __future__ import annotations

import pytest
import torch

from test_gpu_cached import BF16, bshd, rand

pytestmark = pytest.mark.gpu


def call_all(q, kp, vp, k, v, lens=None):
    """Every operator once on prefix and own caches of one sequence or more."""
    from minference import (attention_weight_sums, decode_accumulate, evict_kv_cache,
                            shared_prefix_attention)

    sc = torch.linspace(0, 1, k.shape[2], device=k.device).expand(*k.shape[:2], -1).contiguous()
    return (shared_prefix_attention(q, kp, vp, k, v, lens=lens),
            *decode_accumulate(q[:, :, -1:], k, v, sc.clone(), lens=lens),
            attention_weight_sums(q, k),
            *evict_kv_cache(k, v, sc.sin(), k.shape[2] // 3, recent=3, sinks=2, lens=lens))


def same(a, b):
    torch.cuda.synchronize()
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("Sq", [1, 40])
def test_offsets_past_32_bits(gpu_device, Sq):
    """2^20 keys 16 KiB apart: as the same keys side by side."""
    S, D = 1 << 20, 64
    buf = torch.empty(S, 8192, dtype=BF16, device=gpu_device)
    buf[:, :4 * D] = torch.randn(S, 4 * D, device=gpu_device, generator=torch.Generator(gpu_device).manual_seed(1))
    k = buf[:, None, :2 * D].view(S, 1, 2, D).permute(1, 2, 0, 3)
    v = buf[:, None, 2 * D:4 * D].view(S, 1, 2, D).permute(1, 2, 0, 3)
    q = rand(2, 1, 4, Sq, D).to(gpu_device)
    got = call_all(q, k, v, k, v)
    assert same(got, call_all(q, *(t.contiguous() for t in (k, v, k, v))))


@pytest.mark.parametrize("Sq", [1, 5])
def test_broadcast_and_unaligned_views(gpu_device, Sq):
    B, H, D, Sp, Sc = 3, 4, 96, 200, 70
    q, kp, vp = (rand(i, b, h, s, D).to(gpu_device) for i, b, h, s in ((1, B, H, Sq), (2, 1, 1, Sp), (3, 1, 1, Sp)))
    k, v = (rand(i, 1, 1, Sc, D).to(gpu_device) for i in (4, 5))
    ks, vs = k.expand(B, 2, Sc, D), v.expand(B, 2, Sc, D)
    kps, vps = kp.expand(1, 2, Sp, D), vp.expand(1, 2, Sp, D)
    lens = torch.tensor([Sc, 3, 40], dtype=torch.int32, device=gpu_device)
    ref = call_all(q, *(t.contiguous() for t in (kps, vps, ks, vs)), lens)
    assert same(call_all(q, kps, vps, ks, vs, lens), ref)

    def off(t):  # rows 97 elements apart, from an odd element on
        b = torch.empty(*t.shape[:3], 97, dtype=t.dtype, device=t.device)[..., 1:]
        return b.copy_(t)

    assert same(call_all(*map(off, (q, kps, vps, ks, vs)), lens), ref)


def test_output_over_the_query(gpu_device):
    from minference import decode_accumulate, shared_prefix_attention

    B, H, Hkv, D, Sp, Sc = 5, 8, 2, 128, 900, 300
    kp, vp = (rand(i, 1, Hkv, Sp, D).to(gpu_device) for i in (2, 3))
    k, v = (rand(i, B, Hkv, Sc, D).to(gpu_device) for i in (4, 5))
    for Sq in (1, 20):
        q = bshd(rand(1, B, H, Sq, D)).to(gpu_device)
        ref = shared_prefix_attention(q, kp, vp, k, v)
        x = q.clone()
        assert shared_prefix_attention(x, kp, vp, k, v, out=x) is not None
        assert same([x], [ref])
    q = rand(1, B, H, 1, D).to(gpu_device)
    sc = torch.rand(B, Hkv, Sc, device=gpu_device)
    ref = decode_accumulate(q, k, v, sc.clone())
    assert same(decode_accumulate(q, k, v, sc, out=q), ref)


def test_output_apart_from_the_scores(gpu_device):
    from minference import decode_accumulate

    q, k = (rand(i, 1, 1, s, 64, dtype=torch.float16).to(gpu_device) for i, s in ((1, 1), (2, 64)))
    buf = torch.zeros(128, device=gpu_device)
    out, other = buf[48:112].view(1, 1, 1, 64), torch.zeros(1, 1, 64, device=gpu_device)
    for sc, so in ((buf[:64].view(1, 1, 64), None), (other, buf[:64].view(1, 1, 64)),
                   (buf[:64].view(1, 1, 64), other)):
        with pytest.raises(ValueError, match="out shares memory"):
            decode_accumulate(q, k, k, sc, out=out, scores_out=so)


def test_lengths_out_of_range_are_clamped(gpu_device):
    B, H, Hkv, D, S = 4, 4, 2, 64, 150
    q, k, v = (rand(i, B, h, s, D).to(gpu_device) for i, h, s in ((1, H, 2), (2, Hkv, S), (3, Hkv, S)))
    kp, vp = (rand(i, 1, Hkv, 33, D).to(gpu_device) for i in (4, 5))

    def lens(*x):
        return torch.tensor(x, dtype=torch.int32, device=gpu_device)

    far = call_all(q, kp, vp, k, v, lens(-5, S + 1, 2 ** 31 - 1, -2 ** 31))
    assert same(far, call_all(q, kp, vp, k, v, lens(0, S, S, 0)))


def test_empty_batches(gpu_device):
    from minference import attention_weight_sums, decode_accumulate, shared_prefix_attention

    def z(*s, dtype=BF16):
        return torch.zeros(*s, dtype=dtype, device=gpu_device)

    kp, none = z(1, 2, 9, 96), torch.zeros(0, dtype=torch.int32, device=gpu_device)
    assert shared_prefix_attention(z(0, 4, 1, 96), kp, kp, z(0, 2, 5, 96), z(0, 2, 5, 96),
                                   lens=none).shape == (0, 4, 1, 96)
    assert shared_prefix_attention(z(2, 4, 0, 96), kp, kp, z(2, 2, 5, 96), z(2, 2, 5, 96)).shape == (2, 4, 0, 96)
    out, sc = decode_accumulate(z(0, 4, 1, 96), z(0, 2, 5, 96), z(0, 2, 5, 96),
                                z(0, 2, 5, dtype=torch.float32), lens=none)
    assert out.shape == (0, 4, 1, 96) and sc.shape == (0, 2, 5)
    assert (attention_weight_sums(z(1, 4, 0, 96), z(1, 2, 5, 96)) == 0).all()
    # nothing to see, from a buffer whose rows lie far apart
    far = torch.empty(1, dtype=BF16, device=gpu_device).as_strided((2, 2, 0, 96), (96, 96, 1 << 23, 1))
    q = rand(1, 2, 4, 1, 96).to(gpu_device)
    v = rand(2, 1, 2, 9, 96).to(gpu_device)
    got = shared_prefix_attention(q, kp, v, far, far)
    torch.cuda.synchronize()
    mean = v.double().mean(2)[:, :, None].repeat_interleave(2, 1)
    # 9 weights of 1/9, in two bf16 parts, and the output's rounding
    assert ((got.double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -14 * v.abs().max().double()).all()
    out, _ = decode_accumulate(q, far, far, torch.zeros(2, 2, 0, device=gpu_device))
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_two_streams_at_once_and_two_graphs(gpu_device):
    sets, refs = [], []
    for seed, (B, Sp, Sc, Sq) in enumerate(((3, 3000, 9000, 1), (2, 500, 700, 20))):
        q = rand(10 * seed, B, 8, Sq, 128).to(gpu_device)
        kp, vp = (rand(10 * seed + i, 1, 2, Sp, 128).to(gpu_device) for i in (1, 2))
        k, v = (rand(10 * seed + i, B, 2, Sc, 128).to(gpu_device) for i in (3, 4))
        lens = torch.tensor([Sc, Sc - 7, 5][:B], dtype=torch.int32, device=gpu_device)
        sets.append((q, kp, vp, k, v, lens))
        refs.append([t.clone() for t in call_all(*sets[-1])])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call_all(*sets[i]))
    torch.cuda.synchronize()
    assert all(same(g, refs[i]) for i in (0, 1) for g in got[i])
    graphs = []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured = call_all(*a)
        graphs.append((g, captured))
    for _ in range(3):
        for _, captured in graphs:
            for t in captured:
                t.zero_()
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):  # both at once
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(same(c, r) for (_, c), r in zip(graphs, refs))
        assert all(same(call_all(*a), r) for a, r in zip(sets, refs))
