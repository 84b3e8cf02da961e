"""Host checks of the C entries for rotary positions, gated residual norms and 4-bit blocks, and of the Python
surface over them (no GPU needed: everything here is refused before a launch)."""
import ctypes
import os

import pytest
import torch

from minimaxh3_amd import _native as N
from minimaxh3_amd.kernels.block_norms import gated_residual_norm
from minimaxh3_amd.kernels.mxfp4_linear import MXFP4Linear, dequantize_mxfp4, quantize_mxfp4
from minimaxh3_amd.kernels.rotary import rotary_table, rotate_qk

D = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.lib_path()):
        pytest.fail("libmxf8.so is not built (run __graft_entry__.build())")
    return N.load()


def refused(lib, rc, text):
    assert rc == 1 and text in lib.mxf8_last_error().decode(), (rc, lib.mxf8_last_error())


def dims(*d):
    return (ctypes.c_int64 * len(d))(*d)


def test_rotary_table(lib):
    call = lambda pos=D, typ=0, n=4, axes=2, d=dims(4, 6), theta=1e4, table=D: lib.mxf8_rotary_table(  # noqa: E731
        pos, typ, n, axes, d, theta, table, None)
    refused(lib, call(n=-1), "negative")
    refused(lib, call(axes=0), "axes")
    refused(lib, call(axes=5, d=dims(2, 2, 2, 2, 2)), "axes")
    refused(lib, call(d=None), "axes")
    refused(lib, call(d=dims(4, 5)), "even")
    refused(lib, call(d=dims(4, 0)), "even")
    refused(lib, call(d=dims(4, -2)), "even")
    refused(lib, call(d=dims(512, 2)), "pairs")
    refused(lib, call(d=dims(4, 2 ** 40)), "even")
    refused(lib, call(theta=0.0), "theta")
    refused(lib, call(theta=float("nan")), "theta")
    refused(lib, call(theta=float("inf")), "theta")
    refused(lib, call(pos=None), "null")
    refused(lib, call(table=None), "null")
    refused(lib, call(table=ctypes.c_void_p(260)), "aligned")
    refused(lib, call(typ=4), "type")
    assert call(n=0, pos=None, table=None) == 0


def test_rotate_qk(lib):
    st = N._I64x4(64, 16, 8, 1)

    def call(q=D, hq=2, k=D, hk=1, dtype=0, b=1, s=3, d=8, table=D, tb=0, p=4, eps=1e-6, qst=st, qo=D, ko=D):
        return lib.mxf8_rotate_qk(q, qst, hq, k, st, hk, dtype, b, s, d, table, tb, p, None, None, eps, 1, qo, st, ko, st,
                                  None)

    for bad in ({"b": -1}, {"s": -1}, {"hq": -1}, {"hk": -1}, {"d": 0}, {"d": 5000}):
        refused(lib, call(**bad), "shape")
    refused(lib, call(p=5), "pairs")
    refused(lib, call(p=-1), "pairs")
    refused(lib, call(dtype=3), "dtype")
    refused(lib, call(eps=-1.0), "eps")
    refused(lib, call(eps=float("nan")), "eps")
    refused(lib, call(hq=1 << 15), "too large")
    refused(lib, call(b=1 << 20, s=1 << 20), "too large")
    for null in ("q", "k", "table", "qo", "ko"):
        refused(lib, call(**{null: None}), "null")
    refused(lib, call(table=ctypes.c_void_p(260)), "aligned")
    refused(lib, call(tb=3), "aligned")
    refused(lib, call(qst=N._I64x4(64, 16, 8, 2)), "contiguous")
    assert call(s=0) == 0 and call(hq=0, hk=0) == 0


def test_gated_residual_norm(lib):
    def call(x=D, branch=D, dtype=0, b=1, s=4, c=32, gate=D, spans=1, bw=None, eps=1e-6, quant=0, r=D, y=D, codes=D,
             scales=D):
        return lib.mxf8_gated_residual_norm(x, 128, 32, branch, 128, 32, dtype, b, s, c, gate, 32, 0, None, 0, 0, None, 0,
                                            0, spans, bw, None, 1, eps, 1.0, quant, r, y, codes, scales, None)

    for bad in ({"b": -1}, {"s": -1}, {"c": 0}):
        refused(lib, call(**bad), "shape")
    refused(lib, call(c=16385), "16384")
    refused(lib, call(dtype=7), "dtype")
    refused(lib, call(quant=3), "quantization")
    refused(lib, call(quant=-1), "quantization")
    refused(lib, call(quant=2, c=40), "multiple of 32")
    refused(lib, call(eps=-1e-6), "eps")
    refused(lib, call(spans=0), "spans")
    refused(lib, call(spans=3), "spans")
    refused(lib, call(b=1 << 12, s=1 << 20), "too large")
    refused(lib, call(x=None), "null")
    refused(lib, call(r=None), "null")
    refused(lib, call(y=None), "null")
    refused(lib, call(quant=1, codes=None), "null")
    refused(lib, call(quant=2, scales=None), "null")
    refused(lib, call(branch=None), "need a branch")
    refused(lib, call(branch=None, gate=None, bw=D), "need a branch")
    refused(lib, call(quant=2, codes=ctypes.c_void_p(258)), "aligned")
    assert call(s=0) == 0


def test_mxfp4(lib):
    assert lib.mxf8_mxfp4_scale_bytes(5, 288) == 2 * 5 * 8 and lib.mxf8_mxfp4_scale_bytes(0, 32) == 0
    quant = lambda x=D, dtype=0, m=4, k=64, ld=64, c=D, s=D: lib.mxf8_mxfp4_quant(x, dtype, m, k, ld, c, s, None)  # noqa: E731
    refused(lib, quant(m=-1), "shape")
    refused(lib, quant(k=0), "shape")
    refused(lib, quant(k=48), "multiple of 32")
    refused(lib, quant(k=(1 << 22) + 32, ld=1 << 23), "too large")
    refused(lib, quant(ld=32), "ldx")
    refused(lib, quant(dtype=5), "dtype")
    for null in ("x", "c", "s"):
        refused(lib, quant(**{null: None}), "null")
    refused(lib, quant(c=ctypes.c_void_p(258)), "aligned")
    assert quant(m=0) == 0
    refused(lib, lib.mxf8_mxfp4_dequant(D, D, 4, 40, D, 0, None), "multiple of 32")
    refused(lib, lib.mxf8_mxfp4_dequant(D, None, 4, 64, D, 0, None), "null")
    refused(lib, lib.mxf8_mxfp4_dequant(D, D, 4, 64, D, 3, None), "dtype")
    refused(lib, lib.mxf8_mxfp4_dequant(ctypes.c_void_p(257), D, 4, 64, D, 0, None), "aligned")

    def gemm(a=D, w=D, sa=D, sw=D, act=0, out=D, m=4, n=8, k=64, ld=8):
        return lib.mxf8_gemm_mxfp4(a, w, sa, sw, None, act, out, m, n, k, ld, None)

    for bad in ({"m": -1}, {"n": -1}, {"k": -32}):
        refused(lib, gemm(**bad), "negative")
    refused(lib, gemm(k=0), "multiple of 32")
    refused(lib, gemm(k=48), "multiple of 32")
    for null in ("a", "w", "sa", "sw", "out"):
        refused(lib, gemm(**{null: None}), "null")
    refused(lib, gemm(ld=7), "ld_out")
    refused(lib, gemm(act=2), "act")
    refused(lib, gemm(m=(1 << 27) + 1), "too large")
    refused(lib, gemm(k=(1 << 22) + 32), "too large")
    refused(lib, gemm(a=ctypes.c_void_p(264)), "aligned")
    refused(lib, gemm(sw=ctypes.c_void_p(260)), "aligned")
    assert gemm(m=0, a=None) == 0 and gemm(n=0, w=None) == 0

    def linear(x=D, dtype=0, ldx=64, w=D, sw=D, act=0, out=D, m=40, n=8, k=64, ld=8, ws=D):
        return lib.mxf8_mxfp4_linear(x, dtype, ldx, w, sw, None, act, out, m, n, k, ld, ws, None)

    need = lib.mxf8_mxfp4_linear_workspace_bytes
    assert need(16, 96, 288, 0) == 0 and need(0, 96, 288, 0) == 0
    assert need(17, 96, 288, 0) == 17 * 144 + 2 * 17 * 8 and need(1, 96, 288, 2) == 144 + 16
    assert need(1, 9216, 3072, 0) == 0 and need(12, 9216, 3072, 0) == 12 * (1536 + 12 * 8)
    assert need(1, 3072, 12288, 0) == 0 and need(6, 3072, 12288, 0) == 6 * (6144 + 48 * 8)
    refused(lib, linear(m=-1), "negative")
    refused(lib, linear(k=0), "multiple of 32")
    for null in ("x", "w", "sw", "out"):
        refused(lib, linear(**{null: None}), "null")
    refused(lib, linear(ldx=63), "ldx")
    refused(lib, linear(ld=7), "ld_out")
    refused(lib, linear(dtype=3), "dtype")
    refused(lib, linear(act=9), "act")
    refused(lib, linear(ws=None), "workspace")
    refused(lib, linear(ws=ctypes.c_void_p(264)), "workspace")
    refused(lib, linear(w=ctypes.c_void_p(264)), "aligned")
    assert linear(m=0, x=None) == 0 and linear(n=0, w=None) == 0


def test_sizes_that_no_launch_takes(lib):
    """2^32 threads or more: refused with their own words, not at the launch."""
    refused(lib, lib.mxf8_rotary_table(D, 0, 1 << 35, 1, dims(2), 1e4, D, None), "too many")
    st = N._I64x4(64, 16, 8, 1)
    for s, d in ((1 << 27, 8), (1 << 26, 128), (1 << 25, 1024)):
        for dtype in (0, 1, 2):
            for inter in (0, 1):
                rc = lib.mxf8_rotate_qk(D, st, 2, D, st, 1, dtype, 1, s, d, D, 0, 4, None, None, 1e-6, inter, D, st, D, st,
                                        None)
                refused(lib, rc, "too large")
    # (tokens, channels): a row takes 8 threads, 64 and 256 of 256, 512
    for s, c in ((1 << 29, 32), (1 << 26, 1024), (1 << 24, 4096), (1 << 23, 16384)):
        for dtype in (0, 2):
            for quant in (0, 1, 2):
                rc = lib.mxf8_gated_residual_norm(D, 0, c, D, 0, c, dtype, 1, s, c, None, 0, 0, None, 0, 0, None, 0, 0, 1,
                                                  None, None, 1, 1e-6, 1.0, quant, D, D, D, D, None)
                refused(lib, rc, "too large")
    for m, k in ((1 << 28, 32), (1 << 24, 1 << 13)):
        refused(lib, lib.mxf8_mxfp4_quant(D, 0, m, k, k, D, D, None), "too large")
        refused(lib, lib.mxf8_mxfp4_dequant(D, D, m, k, D, 0, None), "too large")


def test_cpu_tensors_are_refused():
    x = torch.zeros((4, 64))
    with pytest.raises(ValueError):
        quantize_mxfp4(x)
    with pytest.raises(ValueError):
        dequantize_mxfp4(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 4, 8), dtype=torch.uint8))
    with pytest.raises(ValueError):
        rotary_table(x[:, :1], (4,))
    with pytest.raises(ValueError):
        rotate_qk(x.view(1, 1, 4, 64), None, torch.zeros((4, 8, 2)))
    with pytest.raises(ValueError):
        gated_residual_norm(x[None], x[None])
    with pytest.raises(ValueError):
        gated_residual_norm(x[None], x[None], norm="group")
    with pytest.raises(ValueError):
        MXFP4Linear.from_quantized(torch.zeros((4, 24), dtype=torch.uint8), torch.zeros((1, 4, 8), dtype=torch.uint8))


def test_fake_kernels_give_the_shapes_of_the_real_ones():
    from minimaxh3_amd import ops

    t = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="meta")  # noqa: E731
    q = t(2, 9, 3 * 4 * 64)[..., :256].unflatten(-1, (4, 64)).transpose(1, 2)
    qo, ko = ops.rotate_qk(q, None, t(9, 16, 2, dt=torch.float32), None, None, 1e-6, True)
    assert qo.shape == q.shape and qo.transpose(1, 2).is_contiguous() and ko.shape == (0,)
    assert ops.rotary_table(t(2, 9, 3), [4, 6, 2], 1e4).shape == (2, 9, 6, 2)
    x = t(2, 9, 288)
    r, y, codes, scales = ops.gated_residual_norm(x, x, None, None, None, None, None, True, 1e-6, 1.0, 2, False)
    assert r.shape == x.shape and y.shape == (0,) and codes.shape == (18, 144) and scales.shape == (2, 18, 8)
    codes, scales = ops.mxfp4_quant(t(5, 288))
    assert codes.shape == (5, 144) and scales.shape == (2, 5, 8)
    assert ops.gemm_mxfp4(codes, codes, scales, scales, None, 0).shape == (5, 5)
    assert ops.mxfp4_dequant(codes, scales, torch.float16).dtype == torch.float16


def test_import_registers_the_native_kernels():
    """Before any call: a kernel registered later would change a table that the dispatcher reads without a lock."""
    import minimaxh3_amd.ops  # noqa: F401

    for op in ("rotary_table", "rotate_qk", "gated_residual_norm", "mxfp4_quant", "mxfp4_dequant", "gemm_mxfp4",
               "mxfp4_linear"):
        for key in ("CUDA", "AutogradCUDA"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key("mxf8::" + op, key), (op, key)
