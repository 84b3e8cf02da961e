"""Host checks of the C entries of the key / value cache, and of the Python surface over them (no GPU needed:
everything here is refused before a launch)."""
import ctypes
import os

import pytest
import torch

from minimaxh3_amd import _native as N
from minimaxh3_amd.kernels.kv_cache import FP8KVCache, append_kv, cached_attention, read_kv

D = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.lib_path()):
        pytest.fail("libmxf8.so is not built (run __graft_entry__.build())")
    return N.load()


def refused(lib, rc, text):
    assert rc == 1 and text in lib.mxf8_last_error().decode(), (rc, lib.mxf8_last_error())


POOL = ({"kc": None}, {"vs": None}, {"kc": ODD}, {"vc": ODD}, {"page": 24}, {"page": 8}, {"page": 256}, {"d": 96},
        {"pages": -1}, {"pages": 1 << 31}, {"width": -1}, {"width": 1 << 28}, {"b": -1}, {"b": 1 << 16}, {"h": -1},
        {"h": 1 << 16}, {"table": None}, {"b": 2, "ts": 3})
TEXT = ("null", "null", "aligned", "aligned", "page holds", "page holds", "page holds", "D must be", "shape", "shape", "shape",
        "shape", "shape", "shape", "shape", "shape", "null page table", "overlap")


def test_kv_append(lib):
    st = N._I64x4(64, 16, 8, 1)

    def call(k=D, v=D, dtype=0, b=1, h=2, s=3, d=64, turns=D, tb=0, p=8, eps=1e-6, table=D, ts=4, width=4, starts=D, kc=D,
             vc=D, ks=D, vs=D, pages=9, page=16, kst=st, vst=st):
        return lib.mxf8_kv_append(k, kst, v, vst, dtype, b, h, s, d, turns, tb, p, None, eps, 1, table, ts, width, starts,
                                  None, kc, vc, ks, vs, pages, page, None)

    for bad, text in zip(POOL, TEXT):
        refused(lib, call(**bad), text)
    refused(lib, call(s=-1), "shape")
    refused(lib, call(s=(1 << 30) + 1), "shape")
    refused(lib, call(s=1 << 30), "too large")
    refused(lib, call(p=33), "pairs")
    refused(lib, call(p=-1), "pairs")
    refused(lib, call(dtype=3), "dtype")
    refused(lib, call(eps=-1.0), "eps")
    refused(lib, call(eps=float("nan")), "eps")
    for null in ("k", "v", "starts", "turns"):
        refused(lib, call(**{null: None}), "null")
    refused(lib, call(turns=ctypes.c_void_p(260)), "aligned")
    refused(lib, call(tb=3), "aligned")
    for bad in ("kst", "vst"):
        refused(lib, call(**{bad: N._I64x4(64, 16, 8, 2)}), "contiguous")
    for none in ({"b": 0}, {"h": 0}, {"s": 0}, {"width": 0}, {"pages": 0}):
        assert call(**none) == 0


def test_kv_read(lib):
    def call(kc=D, vc=D, ks=D, vs=D, pages=9, h=2, page=16, d=64, table=D, ts=4, width=4, b=1, starts=D, t=5, k=D, v=D, dtype=0):
        return lib.mxf8_kv_read(kc, vc, ks, vs, pages, h, page, d, table, ts, width, b, starts, t, None, k, v, dtype, None)

    for bad, text in zip(POOL, TEXT):
        refused(lib, call(**bad), text)
    refused(lib, call(t=-1), "shape")
    refused(lib, call(t=(1 << 30) + 1), "shape")
    refused(lib, call(t=1 << 30, page=128, d=128), "too large")
    refused(lib, call(dtype=4), "dtype")
    for null in ("starts", "k", "v"):
        refused(lib, call(**{null: None}), "null")
    for none in ({"b": 0}, {"h": 0}, {"t": 0}):
        assert call(**none) == 0


def test_kv_attend(lib):
    st = N._I64x4(64, 16, 8, 1)

    def call(q=D, dtype=0, b=1, hq=4, s=3, d=64, kc=D, vc=D, ks=D, vs=D, pages=9, h=2, page=16, table=D, ts=4, width=4,
             lengths=D, scale=0.1, out=D, qst=st, ost=st, ws=D):
        return lib.mxf8_kv_attend(q, qst, dtype, b, hq, s, d, kc, vc, ks, vs, pages, h, page, table, ts, width, lengths, None,
                                  0, scale, out, ost, ws, None)

    for bad, text in zip(POOL, TEXT):
        refused(lib, call(**bad), text)
    refused(lib, call(s=-1), "shape")
    refused(lib, call(hq=-1), "shape")
    refused(lib, call(hq=5), "key heads")
    refused(lib, call(h=0), "key heads")
    refused(lib, call(dtype=2), "dtype")
    refused(lib, call(scale=float("inf")), "scale")
    refused(lib, call(scale=float("nan")), "scale")
    for null in ("q", "out", "lengths"):
        refused(lib, call(**{null: None}), "null")
    for bad in ("qst", "ost"):
        refused(lib, call(**{bad: N._I64x4(64, 16, 8, 2)}), "contiguous")
    for none in ({"b": 0}, {"hq": 0, "h": 0}, {"s": 0}):
        assert call(**none) == 0


def test_attend_workspace(lib):
    need = lib.mxf8_kv_attend_workspace_bytes
    for none in ((0, 4, 2, 3, 64, 4, 16), (1, 0, 0, 3, 64, 4, 16), (1, 4, 2, 0, 64, 4, 16), (1, 4, 2, 3, 64, 0, 16),
                 (-1, 4, 2, 3, 64, 4, 16), (1, 4, 3, 3, 64, 4, 16)):
        assert need(*none) == 0


def test_cache_refusals():
    t = lambda *s, dt=torch.uint8: torch.zeros(s, dtype=dt)  # noqa: E731
    codes, scale = t(5, 2, 16, 64), t(5, 2)
    ok = FP8KVCache.from_tensors(codes, codes.clone(), scale, scale.clone())
    assert (ok.pages, ok.heads, ok.page_size, ok.head_dim) == (5, 2, 16, 64) and ok.k.dtype == torch.float8_e4m3fn
    assert ok.k.data_ptr() == codes.data_ptr()
    assert FP8KVCache(3, 2, 128, device="cpu").k.shape == (3, 2, 64, 128)
    for bad in ((codes.float(), codes, scale, scale), (codes, codes[:4], scale, scale), (codes[0], codes[0], scale, scale),
                (codes, codes, scale[:, :1], scale), (codes, codes, scale, scale.int()), (codes.transpose(0, 1),) * 2 + (scale.t(),) * 2,
                (t(5, 2, 24, 64), t(5, 2, 24, 64), scale, scale), (t(5, 2, 16, 96), t(5, 2, 16, 96), scale, scale),
                (codes, codes.to("meta"), scale, scale)):
        with pytest.raises(ValueError):
            FP8KVCache.from_tensors(*bad)
    for bad in ((3, 2, 128, 48), (3, 2, 80, 64)):
        with pytest.raises(ValueError):
            FP8KVCache(*bad, device="cpu")


def test_cpu_tensors_are_refused():
    cache, n = FP8KVCache(3, 2, 64, device="cpu"), torch.zeros(1, dtype=torch.int32)
    table, x = torch.zeros((1, 2), dtype=torch.int32), torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        append_kv(cache, table, n, x, x)
    with pytest.raises(ValueError):
        cached_attention(x, cache, table, n)
    with pytest.raises(ValueError):
        read_kv(cache, table, n, 4)


def test_fake_kernels_give_the_shapes_of_the_real_ones():
    from minimaxh3_amd import ops

    cache, n = FP8KVCache(3, 2, 64, device="meta"), torch.empty(2, dtype=torch.int32, device="meta")
    table = torch.empty((2, 5), dtype=torch.int32, device="meta")
    q = torch.empty((2, 9, 4, 64), dtype=torch.float16, device="meta").transpose(1, 2)
    o = ops.kv_attend(q, *cache.tensors(), table, n, None, True, 0.1)
    assert o.shape == q.shape and o.dtype == q.dtype and o.transpose(1, 2).is_contiguous()
    k, v = ops.kv_read(*cache.tensors(), table, n, 7, None, torch.float32)
    assert k.shape == v.shape == (2, 2, 7, 64) and k.dtype == torch.float32
    assert ops.kv_append(*cache.tensors(), table, n, k, v, None, None, None, 1e-6, True) is None


def test_the_extension_is_aliased():
    import sys

    import minimaxh3_amd

    saved = {k: v for k, v in sys.modules.items() if k == "kernels" or k.startswith("kernels.")}
    try:
        minimaxh3_amd.install_as_kernels()
        from kernels.kv_cache import FP8KVCache as aliased
        assert aliased is FP8KVCache
    finally:
        for k in [k for k in sys.modules if k == "kernels" or k.startswith("kernels.")]:
            del sys.modules[k]
        sys.modules.update(saved)


def test_import_registers_the_native_kernels():
    import minimaxh3_amd.ops  # noqa: F401

    for op in ("kv_append", "kv_read", "kv_attend"):
        for key in ("CUDA", "AutogradCUDA"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key("mxf8::" + op, key), (op, key)
