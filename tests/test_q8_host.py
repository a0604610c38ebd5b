"""The 8-bit cache's entry points without a GPU: shapes that are refused,
arguments that are refused before any device call, the views of its records
and the frequency helpers."""
import ctypes
import math

import numpy as np
import pytest
import torch

from rvllm_amd import _lib
from rvllm_amd._lib import RvkvError
from rvllm_amd.q8_storage import HipQ8Storage
from rvllm_amd.rope import rope_cos_sin, rope_inv_freq, rope_yarn


def host_pool(n_layers=2, nb=4, bs=16, kv=2, hd=64):
    """A pool over host memory: every call that would launch is refused or
    fails before it."""
    L = _lib.load()
    n = L.rvkv_q8_pool_bytes(n_layers, nb, bs, kv, hd)
    mem = torch.zeros(n + 256, dtype=torch.uint8)
    at = -mem.data_ptr() % 256
    return HipQ8Storage(n_layers, nb, bs, kv, hd, memory=mem[at:at + n])


@pytest.mark.parametrize("shape,code", [
    ((0, 1, 16, 1, 64), _lib.RVKV_EINVAL),
    ((1, 1, 16, 1, 0), _lib.RVKV_EINVAL),
    ((1, 1, 16, 1, 72), _lib.RVKV_EUNSUPPORTED),
    ((1, 1, 16, 1, 272), _lib.RVKV_EUNSUPPORTED),
    ((1, 1, 8, 1, 64), _lib.RVKV_EUNSUPPORTED),
    ((1, 1, 24, 1, 64), _lib.RVKV_EUNSUPPORTED),
    ((1, 1, 16, 5000, 64), _lib.RVKV_EUNSUPPORTED),
    ((1, 1, 4096, 4096, 256), _lib.RVKV_EUNSUPPORTED),
    ((65535, 0xFFFFFFFF, 4096, 16, 256), _lib.RVKV_EINVAL),
])
def test_pool_shapes_that_are_refused(shape, code):
    assert _lib.load().rvkv_q8_pool_bytes(*shape) == 0
    with pytest.raises(RvkvError, match="^q8_pool_") as e:
        HipQ8Storage(*shape)
    assert e.value.code == code


def test_pool_memory_is_checked():
    L, h = _lib.load(), ctypes.c_void_p()
    n = L.rvkv_q8_pool_bytes(1, 2, 16, 1, 64)
    assert n == 2 * 2 * 1280  # 16 * 68 = 1088, in records of 256 bytes
    args = (1, 2, 16, 1, 64)
    assert L.rvkv_q8_pool_create(*args, 256, n - 1, None,
                                 ctypes.byref(h)) == _lib.RVKV_EINVAL
    assert L.rvkv_q8_pool_create(*args, 128, n, None,
                                 ctypes.byref(h)) == _lib.RVKV_EINVAL
    assert L.rvkv_q8_pool_create(*args, None, 0, None, None) == \
        _lib.RVKV_EINVAL
    L.rvkv_q8_pool_destroy(None)
    assert L.rvkv_q8_pool_set_stream(None, None) == _lib.RVKV_EINVAL


def test_views_are_the_records():
    st = host_pool()
    st.codes(1, 1)[2, 1, 5, 7] = -3
    st.scales(1, 0)[3, 1, 15] = 2.5
    rec = 16 * 2 * 68 + (-(16 * 2 * 68)) % 256
    raw = st.memory.numpy().reshape(2, 2, 4, rec)
    assert raw[1, 1, 2].view(np.int8)[64 * 16 + 7 * 16 + 5] == -3
    assert raw[1, 0, 3][2048:2048 + 128].view(np.float32)[31] == 2.5
    for bad in ((2, 0), (-1, 0), (0, 2)):
        with pytest.raises(RvkvError):
            st.codes(*bad)


def test_append_refuses():
    st = host_pool()
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    i = torch.zeros(3, dtype=torch.int32)
    inv = torch.ones(32)

    def bad(match, layer=0, q=q, k=k, v=k, pos=i, inv=inv, blk=i, off=i, **kw):
        with pytest.raises(RvkvError, match=match):
            st.rope_append(layer, q, k, v, pos, inv, blk, off, **kw)

    bad("layer out of range", layer=2)
    bad("rows, heads, head_dim", q=q[:2])
    bad("rows, heads, head_dim", k=k[:, :, :32])
    bad("n_kv_heads", k=torch.zeros(3, 1, 64))
    bad("float32 or float16", q=q.half())
    bad("float32 or float16", q=q.double(), k=k.double(), v=k.double())
    bad("one behind the other", k=torch.zeros(3, 64, 2).transpose(1, 2))
    bad("contiguous int32", pos=i.long())
    bad("contiguous int32", blk=i[:2])
    bad("rot_dim", inv=torch.ones(33))
    bad("inv_freq", inv=torch.ones(32).double())
    bad("norm weights", q_norm=torch.ones(32))
    bad("match q", q_out=torch.zeros(3, 4, 64).half())
    bad("multiple of n_kv_heads", q=torch.zeros(3, 3, 64))
    with pytest.raises(RvkvError, match="k/v len is 0"):
        st.write_tokens(0, i[:0], i[:0], k[:0], k[:0])
    # no rows: nothing to do
    st.rope_append(0, q[:0], k[:0], k[:0], i[:0], inv, i[:0], i[:0])
    L = _lib.load()
    assert L.rvkv_rope_append(*[None if t is ctypes.c_void_p else 1 for t in
                                _lib.SIGNATURES["rvkv_rope_append"][1]]) == \
        _lib.RVKV_EINVAL
    p, f = k.data_ptr(), 1.0
    n = i.data_ptr()

    def raw(qs=256, ks=128, dtype=_lib.RVKV_F32, rows=3, inter=0, rot=64,
            pos=n, kp=p, heads=4):
        return L.rvkv_q8_rope_append(st._pool, 0, q.data_ptr(), qs, kp, ks, p,
                                     128, dtype, rows, heads, None, None, f,
                                     pos, inv.data_ptr(), rot, inter, f, n, n,
                                     q.data_ptr())

    assert raw(rows=1) == _lib.RVKV_EINVAL  # (q_out is q)
    assert b"overlaps" in L.rvkv_last_error()
    assert raw(qs=255) == _lib.RVKV_EINVAL
    assert raw(ks=127) == _lib.RVKV_EINVAL
    assert raw(dtype=5) == _lib.RVKV_EINVAL
    assert raw(inter=2) == _lib.RVKV_EINVAL
    assert raw(rot=63) == _lib.RVKV_EINVAL
    assert raw(pos=None) == _lib.RVKV_EINVAL
    assert raw(kp=None) == _lib.RVKV_EINVAL
    assert raw(kp=p + 1) == _lib.RVKV_EINVAL
    assert raw(rows=1 << 24) == _lib.RVKV_EUNSUPPORTED


def test_decode_refuses():
    st = host_pool()
    q = torch.zeros(2, 4, 64)
    t = torch.zeros(2, 4, dtype=torch.int32)
    c = torch.ones(2, dtype=torch.int32)

    def bad(match, layer=0, q=q, t=t, c=c, top=64, **kw):
        with pytest.raises(RvkvError, match=match):
            st.paged_decode(layer, q, t, c, top, **kw)

    bad("layer out of range", layer=5)
    bad("contiguous", q=q.transpose(0, 1))
    bad("head_dim", q=torch.zeros(2, 4, 32))
    bad("block_tables must be", t=t[:1])
    bad("int32", t=t.long())
    bad("ctx_lens length", c=c[:1])
    bad("out must match", out=torch.zeros(2, 4, 64).half())
    bad("multiple of n_kv_heads", q=torch.zeros(2, 3, 64))
    bad("max_blocks", t=torch.zeros(2, 0, dtype=torch.int32))
    assert st.decode_workspace_bytes(2, 4, 100) == 0
    need = st.decode_workspace_bytes(2, 4, 5000)
    assert need > 0 and need % 256 == 0
    bad("smaller than", top=5000,
        ws=torch.zeros(need - 1, dtype=torch.uint8))
    # a window bounds the partitions
    assert st.decode_workspace_bytes(2, 4, 5000, window=100) == 0
    assert _lib.load().rvkv_q8_decode_workspace_bytes(None, 1, 1, 1, 0) == 0
    assert st.paged_decode(0, q[:0], t[:0], c[:0], 64).shape == (0, 4, 64)


def test_prefill_refuses():
    st = host_pool()
    q = torch.zeros(5, 4, 64)
    t = torch.zeros(2, 4, dtype=torch.int32)
    s = torch.tensor([0, 2, 5], dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)

    def bad(match, layer=0, q=q, s=s, t=t, o=n, r=n, **kw):
        with pytest.raises(RvkvError, match=match):
            st.packed_prefill(layer, q, s, t, o, r, **kw)

    bad("layer out of range", layer=5)
    bad("head_dim", q=torch.zeros(5, 4, 32))
    bad("batch \\+ 1", s=s[:2])
    bad("must be \\[batch", t=t[0])
    bad("length must equal batch", o=n[:1])
    bad("int32", r=n.long())
    bad("multiple of n_kv_heads", q=torch.zeros(5, 3, 64))
    bad("max_blocks", t=torch.zeros(2, 0, dtype=torch.int32))
    need = st.prefill_workspace_bytes(5, 2, 4, 400)
    assert need > 0
    bad("smaller than", t=torch.zeros(2, 400, dtype=torch.int32),
        ws=torch.zeros(need - 256, dtype=torch.uint8))
    empty = st.packed_prefill(0, q[:0], s * 0, t, n, n)
    assert empty.shape == (0, 4, 64)


def test_gather_and_copy_refuse():
    from rvllm_amd.kv_storage import HipGatherPlan
    st = host_pool()
    plan = HipGatherPlan([([0, 1], 20)], device="cpu")
    out = torch.zeros(1, 2, 20, 64)
    for match, k, v in [("output length", out[:, :, :19], out),
                        ("output length", out.transpose(1, 2), out),
                        ("float32 or float16", out, out.half()),
                        ("float32 or float16", out.double(), out.double())]:
        with pytest.raises(RvkvError, match=match):
            st.gather(0, plan, k, v)
    with pytest.raises(RvkvError, match="layer"):
        st.gather(9, plan, out, out)
    with pytest.raises(RvkvError, match="max_blocks \\* block_size"):
        st.gather(0, HipGatherPlan([([0], 20)], device="cpu"), out, out)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RvkvError, match="different lengths"):
        st.copy_blocks(i, i[:2])
    with pytest.raises(RvkvError, match="contiguous int32"):
        st.copy_blocks(i.long(), i.long())
    st.copy_blocks(i[:0], i[:0])  # nothing to do


def test_a_call_without_a_device_fails_and_says_so():
    if torch.cuda.is_available():
        pytest.skip("needs a host without a GPU")
    st = host_pool()
    with pytest.raises(RvkvError) as e:
        st.paged_decode(0, torch.zeros(1, 2, 64),
                        torch.zeros(1, 1, dtype=torch.int32),
                        torch.ones(1, dtype=torch.int32), 16)
    assert e.value.code == _lib.RVKV_EHIP


def test_inv_freq():
    inv = rope_inv_freq(1e4, 64)
    cos, _ = rope_cos_sin(1e4, 64, [1])
    assert np.allclose(np.cos(inv.astype(np.float64)), cos[0], atol=1e-7)
    assert np.array_equal(rope_inv_freq(1e4, 64, 8.0),
                          (1e4 ** (-np.arange(0, 64, 2) / 64) / 8
                           ).astype(np.float32))


def test_yarn():
    """Frequencies that turn often stay, those that turn less than once are
    divided, and the scale is monotone between."""
    inv, factor = rope_yarn(1e4, 128, 4.0, 4096)
    base = rope_inv_freq(1e4, 128).astype(np.float64)
    ratio = base / inv
    turns = 4096 * base / (2 * math.pi)
    assert np.allclose(ratio[turns > 40], 1, atol=1e-6)
    assert np.allclose(ratio[turns < 0.8], 4, atol=1e-5)
    assert (np.diff(ratio) > -1e-5).all()
    assert factor == pytest.approx(1.138629, abs=1e-6)
