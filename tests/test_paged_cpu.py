"""Refusals of the paged-cache entry points: every check answers before a device is touched."""
import ctypes

import pytest
import torch

from cutile_rs_b200 import _lib, api, launch, paged
from cutile_rs_b200.tensor import KernelLaunchError, TensorError

I2, I3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
P = 4096   # an aligned address that no refused call reads


def _cache(**kw):
    d = dict(k=P, v=P, k_scales=P, v_scales=P, k_strides=I3(8192, 2048, 128), v_strides=I3(8192, 2048, 128),
             k_scale_strides=I3(512, 128, 8), v_scale_strides=I3(512, 128, 8), k_global=1.0, v_global=1.0, format=0,
             num_pages=4, kv_heads=4, page_size=16, head_dim=128)
    d.update(kw)
    return ctypes.pointer(_lib.PagedCacheC(**d))


def _batch(**kw):
    d = dict(block_table=P, block_table_pitch=8, cu_q=P, kv_lens=P, batch=2, max_pages=8, max_q_len=4)
    d.update(kw)
    return ctypes.pointer(_lib.PagedBatchC(**d))


def _attend(c, b, dtype=b"bf16", q=P, out=P, tokens=4, heads=8, qs=I2(1024, 128), os=I2(1024, 128), scale=0.1, causal=1,
            window=0, cap=0.0, ws=P, ws_bytes=1 << 40):
    lib = _lib.load()
    rc = lib.b200tile_paged_attention(dtype, c, b, q, out, tokens, heads, qs, os, scale, causal, window, cap, ws, ws_bytes,
                                      None)
    return rc, lib.b200tile_last_error().decode()


def _append(c, b, q=P, q_out=P, rot=128, f=P, tokens=4, heads=8, k=P, v=P, ks=I2(512, 128), dtype=b"bf16"):
    lib = _lib.load()
    rc = lib.b200tile_paged_kv_append(dtype, c, b, q, k, v, q_out, f, tokens, heads, rot, I2(1024, 128), ks, ks,
                                      I2(1024, 128), None)
    return rc, lib.b200tile_last_error().decode()


CACHE_FAULTS = [
    (dict(format=2), _lib.ERR_UNSUPPORTED, "format"), (dict(head_dim=96), _lib.ERR_UNSUPPORTED, "head_dim"),
    (dict(num_pages=0), _lib.ERR_INVALID, "positive"), (dict(page_size=24), _lib.ERR_UNSUPPORTED, "page_size"),
    (dict(page_size=8), _lib.ERR_UNSUPPORTED, "page_size"), (dict(k=None), _lib.ERR_INVALID, "K pool is null"),
    (dict(v=P + 8), _lib.ERR_ALIGN, "V pool"), (dict(k_strides=I3(8192, 2044, 128)), _lib.ERR_ALIGN, "K pool"),
    (dict(v_strides=I3(0, 2048, 128)), _lib.ERR_INVALID, "positive"),
    (dict(format=1, k_scales=None), _lib.ERR_INVALID, "K scale"),
    (dict(format=1, v_scales=P + 4), _lib.ERR_ALIGN, "V scale"),
    (dict(format=1, k_global=0.0), _lib.ERR_INVALID, "k_global"),
    (dict(format=1, v_global=float("nan")), _lib.ERR_INVALID, "v_global"),
    (dict(format=1, k_strides=I3(8192, 2048, 72)), _lib.ERR_ALIGN, "K pool"),
    (dict(format=1, v_strides=I3(1 << 31, 2048, 128)), _lib.ERR_UNSUPPORTED, "2^31"),
]


@pytest.mark.parametrize("change,code,text", CACHE_FAULTS)
def test_cache_faults(change, code, text):
    for rc, msg in (_attend(_cache(**change), _batch()), _append(_cache(**change), _batch())):
        assert rc == code and text in msg
    lib = _lib.load()
    rc = lib.b200tile_paged_kv_gather(b"f16", _cache(**change), _batch(), P, P, 4, I2(512, 128), I2(512, 128), None)
    assert rc == code


@pytest.mark.parametrize("change,code,text", [
    (dict(batch=-1), _lib.ERR_INVALID, "negative"), (dict(cu_q=None), _lib.ERR_INVALID, "required"),
    (dict(kv_lens=P + 2), _lib.ERR_ALIGN, "4-byte"), (dict(max_q_len=0), _lib.ERR_INVALID, "max_q_len"),
    (dict(max_pages=0), _lib.ERR_INVALID, "max_pages"), (dict(block_table_pitch=7), _lib.ERR_INVALID, "pitch"),
    (dict(max_pages=1 << 27, block_table_pitch=1 << 27), _lib.ERR_UNSUPPORTED, "positions"),
])
def test_batch_faults(change, code, text):
    for rc, msg in (_attend(_cache(), _batch(**change)), _append(_cache(), _batch(**change))):
        assert rc == code and text in msg


def test_attention_arguments():
    c, b = _cache(), _batch()
    for kw, code, text in ((dict(dtype=b"f32"), _lib.ERR_UNSUPPORTED, "element type"), (dict(dtype=None), _lib.ERR_INVALID, "dtype"),
                           (dict(q=None), _lib.ERR_INVALID, "q and"), (dict(out=P + 2), _lib.ERR_ALIGN, "out"),
                           (dict(qs=I2(1023, 128)), _lib.ERR_ALIGN, "q must"), (dict(heads=6), _lib.ERR_INVALID, "multiple"),
                           (dict(scale=0.0), _lib.ERR_INVALID, "qk_scale"), (dict(scale=float("inf")), _lib.ERR_INVALID, "qk_scale"),
                           (dict(cap=-1.0), _lib.ERR_INVALID, "softcap"), (dict(cap=float("nan")), _lib.ERR_INVALID, "softcap"),
                           (dict(window=-1), _lib.ERR_INVALID, "window"), (dict(window=5, causal=0), _lib.ERR_INVALID, "causal"),
                           (dict(ws=None), _lib.ERR_INVALID, "workspace"), (dict(ws_bytes=64), _lib.ERR_INVALID, "workspace"),
                           (dict(ws=P + 8), _lib.ERR_ALIGN, "workspace"), (dict(tokens=-1), _lib.ERR_INVALID, "negative")):
        rc, msg = _attend(c, b, **kw)
        assert rc == code and text in msg, (kw, rc, msg)
    assert _attend(None, b)[0] == _lib.ERR_INVALID and _attend(c, None)[0] == _lib.ERR_INVALID
    assert _attend(c, b, tokens=0)[0] == _lib.OK and _attend(c, _batch(batch=0))[0] == _lib.OK


def test_append_arguments():
    c, b = _cache(), _batch()
    for kw, code, text in ((dict(rot=20), _lib.ERR_UNSUPPORTED, "rotary_dim"), (dict(rot=144), _lib.ERR_UNSUPPORTED, "rotary_dim"),
                           (dict(f=None), _lib.ERR_INVALID, "inv_freq"), (dict(f=P + 1), _lib.ERR_ALIGN, "inv_freq"),
                           (dict(q_out=None), _lib.ERR_INVALID, "together"), (dict(heads=0), _lib.ERR_INVALID, "q_heads"),
                           (dict(k=None), _lib.ERR_INVALID, "k and"), (dict(v=P + 8), _lib.ERR_ALIGN, "v must"),
                           (dict(ks=I2(512, 130)), _lib.ERR_ALIGN, "k must")):
        rc, msg = _append(c, b, **kw)
        assert rc == code and text in msg, (kw, rc, msg)
    rc, msg = _append(_cache(format=1), b, rot=48)
    assert rc == _lib.ERR_UNSUPPORTED and "multiple of 32" in msg
    assert _append(c, b, tokens=0)[0] == _lib.OK


def test_rows_that_are_written_share_no_memory():
    lib = _lib.load()
    for st in (I2(0, 128), I2(1024, 0)):
        assert _attend(_cache(), _batch(), os=st)[0] == _lib.ERR_INVALID
        rc = lib.b200tile_paged_kv_append(b"bf16", _cache(), _batch(), P, P, P, P, None, 4, 8, 0, I2(1024, 128), I2(512, 128),
                                          I2(512, 128), st, None)
        assert rc == _lib.ERR_INVALID and b"q_out" in lib.b200tile_last_error()
        for ks, vs, name in ((st, I2(512, 128), b"k_out"), (I2(512, 128), st, b"v_out")):
            assert lib.b200tile_paged_kv_gather(b"bf16", _cache(), _batch(), P, P, 4, ks, vs, None) == _lib.ERR_INVALID
            assert name in lib.b200tile_last_error()


def test_workspace_grows_with_what_it_holds():
    lib = _lib.load()
    size = lambda **kw: lib.b200tile_paged_attention_workspace_bytes(_cache(), _batch(**kw), 8)  # noqa: E731
    assert 0 < size(max_pages=8) < size(max_pages=4096, block_table_pitch=4096) < 1 << 26
    assert size(batch=0) == 0


def test_containers_and_python_refusals():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 2, 16, 32, dtype=torch.uint8), torch.zeros(4, 2, 16, 4, dtype=torch.uint8)
    c = paged.PagedKvCache(k.permute(0, 1, 2, 3), k.clone())
    assert (c.head_dim, c.kv_heads, c.page_size, c.num_pages) == (64, 2, 16, 4)
    assert paged.PagedKvCache(codes, codes, scales, scales).head_dim == 64
    for bad in (lambda: paged.PagedKvCache(k, k[:3]), lambda: paged.PagedKvCache(k.float(), k.float()),
                lambda: paged.PagedKvCache(codes, codes, scales), lambda: paged.PagedKvCache(codes, codes, scales[:2], scales),
                lambda: paged.PagedKvCache(k.transpose(2, 3), k.transpose(2, 3)),
                lambda: paged.PagedKvCache(k, k, scales, scales)):
        with pytest.raises(TensorError):
            bad()
    i32 = dict(dtype=torch.int32)
    table, cu, lens = torch.zeros(2, 4, **i32), torch.zeros(3, **i32), torch.zeros(2, **i32)
    b = paged.PagedBatch(table, cu, lens, 1)
    for bad in ((table, cu[:2], lens), (table.long(), cu, lens), (table.t()[:2], cu, lens), (table[0], cu, lens)):
        with pytest.raises(TensorError):
            paged.PagedBatch(*bad, 1)
    q = api.from_torch(torch.zeros(2, 4, 64, dtype=torch.bfloat16))
    kv = api.from_torch(torch.zeros(2, 2, 64, dtype=torch.bfloat16))
    half = api.from_torch(torch.zeros(2, 4, 64, dtype=torch.float16))
    with pytest.raises(KernelLaunchError, match="expected"):
        launch.paged_attention(q, api.from_torch(torch.zeros(2, 4, 32, dtype=torch.bfloat16)), c, b, 0.1)
    with pytest.raises(KernelLaunchError, match="different element types"):
        launch.paged_attention(q, half, c, b, 0.1)
    with pytest.raises(KernelLaunchError, match="the cache holds bf16"):
        launch.paged_attention(half, half, c, b, 0.1)
    with pytest.raises(KernelLaunchError, match="together"):
        launch.paged_kv_append(c, b, kv, kv, q=q)
    with pytest.raises(KernelLaunchError, match="inv_freq"):
        launch.paged_kv_append(c, b, kv, kv, inv_freq=kv)
    with pytest.raises(KernelLaunchError, match="expected"):
        launch.paged_kv_gather(q, kv, c, b)
    with pytest.raises(KernelLaunchError, match="current device"):
        launch.paged_attention(q, q, c, b, 0.1)
