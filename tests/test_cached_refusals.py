"""Arguments the cache operators refuse, before anything is launched (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from minference import (_abi, attention_weight_sums, decode_accumulate, evict_kv_cache,
                        shared_prefix_attention)
from minference.ops.common import check_written
from test_abi import FAKE, t4

F32 = _abi.MSA_DTYPE_FP32
REF = ctypes.byref


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_shared_prefix_refusals():
    q, kp, k = z(2, 4, 1, 96), z(1, 2, 8, 96), z(2, 2, 5, 96)
    with pytest.raises(RuntimeError, match="GPU only"):
        shared_prefix_attention(q, kp, kp, k, k)
    with pytest.raises(ValueError, match="4-D"):
        shared_prefix_attention(q[0], kp, kp, k, k)
    with pytest.raises(ValueError, match="prefix must be"):
        shared_prefix_attention(q, k, k, k, k)  # a prefix per sequence
    with pytest.raises(ValueError, match="of one shape"):
        shared_prefix_attention(q, kp, z(1, 2, 7, 96), k, k)
    with pytest.raises(ValueError, match="own cache must be"):
        shared_prefix_attention(q, kp, kp, z(3, 2, 5, 96), z(3, 2, 5, 96))
    with pytest.raises(ValueError, match="own cache must be"):
        shared_prefix_attention(q, kp, kp, z(2, 2, 5, 64), z(2, 2, 5, 64))
    with pytest.raises(ValueError, match="not a multiple"):
        shared_prefix_attention(q, z(1, 3, 8, 96), z(1, 3, 8, 96), k, k)
    with pytest.raises(ValueError, match="same kv heads"):
        shared_prefix_attention(q, z(1, 4, 8, 96), z(1, 4, 8, 96), k, k)


def test_decode_accumulate_refusals():
    q, k, s = z(2, 4, 1, 96), z(2, 2, 5, 96), z(2, 2, 5, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="GPU only"):
        decode_accumulate(q, k, k, s)
    with pytest.raises(ValueError, match="not a multiple"):
        decode_accumulate(z(2, 3, 1, 96), k, k, s)
    with pytest.raises(ValueError, match="of one shape"):
        decode_accumulate(q, k, z(2, 2, 6, 96), s)


def test_weight_sums_refusals():
    q, k = z(1, 4, 6, 96), z(1, 2, 6, 96)
    with pytest.raises(RuntimeError, match="GPU only"):
        attention_weight_sums(q, k)
    with pytest.raises(ValueError, match="not a multiple"):
        attention_weight_sums(q, z(1, 3, 6, 96))
    with pytest.raises(ValueError, match="expected"):
        attention_weight_sums(q, z(2, 2, 6, 96))
    with pytest.raises(ValueError, match="expected"):
        attention_weight_sums(q, z(1, 2, 6, 64))


@pytest.mark.parametrize("keep,kw", [(0, {}), (7, {}), (3, dict(recent=4)), (3, dict(sinks=4)),
                                     (3, dict(recent=2, sinks=2)), (3, dict(recent=-1)),
                                     (3, dict(sinks=-1))])
def test_evict_counts_refused(keep, kw):
    k = z(1, 2, 6, 96)
    with pytest.raises(ValueError, match="keep"):
        evict_kv_cache(k, k, z(1, 2, 6, dtype=torch.float32), keep, **kw)


def test_evict_refusals():
    k, s = z(1, 2, 6, 96), z(1, 2, 6, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="GPU only"):
        evict_kv_cache(k, k, s, 3)
    with pytest.raises(ValueError, match="of one shape"):
        evict_kv_cache(k, z(1, 2, 5, 96), s, 3)
    with pytest.raises(ValueError):
        evict_kv_cache(z(1, 2, 0, 96), z(1, 2, 0, 96), z(1, 2, 0, dtype=torch.float32), 1)


def test_check_written():
    """Outputs whose elements share memory, with each other or with an input."""
    buf = torch.zeros(2, 4, 10, 16)
    check_written("out", buf[:, :, 2:5], [("in", buf[:, :, 5:9])])
    check_written("out", buf[..., :8], [("in", buf[..., 8:])])       # side by side
    check_written("out", buf[:, :2], [("in", buf[:, 2:])])
    check_written("out", buf.transpose(1, 2))
    check_written("out", torch.zeros(0, 4))
    for bad in (buf[:, :, 4:8], buf[:, 1:3, 3:6], buf[..., 4:12]):
        with pytest.raises(ValueError, match="shares memory with in"):
            check_written("out", buf[:, :, 2:5], [("in", bad)])
    with pytest.raises(ValueError, match="share memory"):
        check_written("out", torch.zeros(1, 4).expand(3, 4))
    with pytest.raises(ValueError, match="share memory"):
        check_written("out", torch.zeros(100).as_strided((5, 10), (4, 1)))


# ---- the C ABI: fake pointers, nothing is read or launched ----

Q, KP, KV = [2, 4, 1, 96], [1, 2, 100, 96], [2, 2, 50, 96]


def prefix(q=None, kp=None, vp=None, k=None, v=None, o=None, scale=0.1, ws=FAKE, wsb=1 << 40):
    lib = _abi.load_library()
    ts = [t if t is not None else t4(s) for t, s in ((q, Q), (kp, KP), (vp, KP), (k, KV), (v, KV), (o, Q))]
    return lib.msa_shared_prefix_attention(*map(REF, ts), None, scale, ws, wsb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(q=t4(Q, data=0)), _abi.MSA_E_NULL),
    (dict(kp=t4(KP, data=0)), _abi.MSA_E_NULL),
    (dict(kp=t4([2, 2, 100, 96]), vp=t4([2, 2, 100, 96])), _abi.MSA_E_RANK),
    (dict(vp=t4([1, 2, 99, 96])), _abi.MSA_E_RANK),
    (dict(kp=t4([1, 4, 100, 96]), vp=t4([1, 4, 100, 96])), _abi.MSA_E_RANK),
    (dict(k=t4([2, 2, 50, 64]), v=t4([2, 2, 50, 64])), _abi.MSA_E_RANK),
    (dict(o=t4([2, 4, 2, 96])), _abi.MSA_E_RANK),
    (dict(v=t4(KV, _abi.MSA_DTYPE_FP16)), _abi.MSA_E_DTYPE),
    (dict(o=t4(Q, _abi.MSA_DTYPE_FP16)), _abi.MSA_E_DTYPE),
    (dict(k=t4(KV, strides=[9600, 4800, 96, 2])), _abi.MSA_E_ALIGN),
    (dict(k=t4(KV, data=FAKE + 8)), _abi.MSA_E_ALIGN),
    (dict(k=t4(KV, strides=[1 << 30, 1 << 30, (1 << 23) + 64, 1])), _abi.MSA_E_SEQ),
    (dict(kp=t4([1, 2, (1 << 20) + 1, 96]), vp=t4([1, 2, (1 << 20) + 1, 96])), _abi.MSA_E_SEQ),
    (dict(scale=0.0), _abi.MSA_E_HEADS),
    (dict(scale=float("nan")), _abi.MSA_E_HEADS),
    (dict(ws=None), _abi.MSA_E_WORKSPACE),
    (dict(ws=FAKE + 4), _abi.MSA_E_ALIGN),
    (dict(wsb=64), _abi.MSA_E_WORKSPACE),
])
def test_prefix_abi_refusals(kw, want):
    assert prefix(**kw) == want


def test_prefix_abi_other_head_dim_and_workspace():
    bad = [t4([s[0], s[1], s[2], 80]) for s in (Q, KP, KP, KV, KV, Q)]
    assert prefix(*bad) == _abi.MSA_E_HEAD_DIM
    lib = _abi.load_library()
    ts = [t4(s) for s in (Q, KP, KP, KV, KV)]
    need = lib.msa_shared_prefix_workspace_bytes(*map(REF, ts))
    assert need > 0 and prefix(wsb=need - 1) == _abi.MSA_E_WORKSPACE
    # a long prefix with rows of 16 MiB: ranges below 2 GiB each, or refused
    big = t4([1, 2, 1 << 20, 96], strides=[1 << 40, 96, (1 << 22), 1])
    assert lib.msa_shared_prefix_workspace_bytes(REF(ts[0]), REF(big), REF(big), REF(ts[3]), REF(ts[4])) == 0


@pytest.mark.parametrize("stride", [1 << 23, 1 << 40, 1 << 62])
def test_empty_caches_of_any_stride(stride):
    # rows of an empty cache may lie any distance apart; a division by the
    # keys of 2 GiB once ended the process here
    lib = _abi.load_library()
    ts = [t4(s) for s in (Q, KP, KP)]
    empty = t4([2, 2, 0, 96], strides=[0, 0, stride, 1])
    assert lib.msa_shared_prefix_workspace_bytes(*map(REF, ts), REF(empty), REF(empty)) > 0
    assert lib.msa_decode_accumulate_workspace_bytes(REF(ts[0]), REF(empty), REF(empty)) > 0
    one = t4([2, 2, 1, 96], strides=[0, 0, stride, 1])
    assert lib.msa_decode_accumulate_workspace_bytes(REF(ts[0]), REF(one), REF(one)) == 0


@pytest.mark.parametrize("kw,want", [
    (dict(q=t4([2, 4, 2, 96]), o=t4([2, 4, 2, 96])), _abi.MSA_E_SEQ),
    (dict(s=t4([2, 2, 49, 1], F32)), _abi.MSA_E_RANK),
    (dict(s=t4([2, 2, 50, 1])), _abi.MSA_E_DTYPE),
    (dict(r=t4([2, 2, 50, 1], F32, strides=[200, 100, 2, 1])), _abi.MSA_E_ALIGN),
    (dict(r=t4([2, 2, 50, 1], F32, data=0)), _abi.MSA_E_NULL),
    (dict(q=t4([2, 258, 1, 96]), o=t4([2, 258, 1, 96])), _abi.MSA_E_HEADS),
    (dict(wsb=64), _abi.MSA_E_WORKSPACE),
])
def test_accumulate_abi_refusals(kw, want):
    lib = _abi.load_library()
    a = dict(q=t4(Q), k=t4(KV), v=t4(KV), o=t4(Q), s=t4([2, 2, 50, 1], F32), r=t4([2, 2, 50, 1], F32),
             wsb=1 << 40)
    a.update(kw)
    st = lib.msa_decode_accumulate(REF(a["q"]), REF(a["k"]), REF(a["v"]), REF(a["o"]), None, REF(a["s"]),
                                   REF(a["r"]), 0.1, FAKE, a["wsb"], None)
    assert st == want


@pytest.mark.parametrize("kw,want", [
    (dict(q=t4([2, 4, 51, 96])), _abi.MSA_E_SEQ),
    (dict(q=t4([2, 3, 5, 96])), _abi.MSA_E_RANK),
    (dict(s=t4([2, 2, 51, 1], F32)), _abi.MSA_E_RANK),
    (dict(s=t4([2, 2, 50, 1])), _abi.MSA_E_DTYPE),
    (dict(add=2), _abi.MSA_E_FLAGS),
    (dict(scale=-1.0), _abi.MSA_E_HEADS),
    (dict(wsb=16), _abi.MSA_E_WORKSPACE),
])
def test_sums_abi_refusals(kw, want):
    lib = _abi.load_library()
    a = dict(q=t4([2, 4, 5, 96]), k=t4(KV), s=t4([2, 2, 50, 1], F32), add=0, scale=0.1, wsb=1 << 40)
    a.update(kw)
    st = lib.msa_attention_weight_sums(REF(a["q"]), REF(a["k"]), REF(a["s"]), a["add"], a["scale"], FAKE,
                                       a["wsb"], None)
    assert st == want


@pytest.mark.parametrize("kw,want", [
    (dict(keep=0), _abi.MSA_E_RANK),
    (dict(keep=51, ko=t4([2, 2, 51, 96]), vo=t4([2, 2, 51, 96])), _abi.MSA_E_TOPK),
    (dict(recent=9, sinks=2), _abi.MSA_E_TOPK),
    (dict(recent=-1), _abi.MSA_E_TOPK),
    (dict(ko=t4([2, 2, 11, 96])), _abi.MSA_E_RANK),
    (dict(vo=t4([2, 2, 10, 96], F32)), _abi.MSA_E_DTYPE),
    (dict(so=t4([2, 2, 11, 1], F32)), _abi.MSA_E_RANK),
    (dict(k=t4(KV, strides=[9600, 4800, 96, 2])), _abi.MSA_E_ALIGN),
    (dict(pos=None), _abi.MSA_E_NULL),
    (dict(k=t4([2, 2, 9000, 96]), v=t4([2, 2, 9000, 96]), s=t4([2, 2, 9000, 1], F32), wsb=16),
     _abi.MSA_E_WORKSPACE),
])
def test_evict_abi_refusals(kw, want):
    lib = _abi.load_library()
    a = dict(k=t4(KV), v=t4(KV), s=t4([2, 2, 50, 1], F32), keep=10, recent=2, sinks=2, ko=t4([2, 2, 10, 96]),
             vo=t4([2, 2, 10, 96]), so=t4([2, 2, 10, 1], F32), pos=FAKE, wsb=1 << 30)
    a.update(kw)
    st = lib.msa_cache_evict(REF(a["k"]), REF(a["v"]), REF(a["s"]), None, a["keep"], a["recent"], a["sinks"],
                             REF(a["ko"]), REF(a["vo"]), REF(a["so"]), a["pos"], FAKE, FAKE, a["wsb"], None)
    assert st == want
