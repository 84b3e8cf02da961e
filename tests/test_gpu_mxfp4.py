"""4-bit blocks: the quantizer and its inverse against the oracle bit for bit, the product and the module against
64-bit sums of the same values."""
import numpy as np
import pytest
import torch
import torch.nn as nn

from minimaxh3_amd import ops
from minimaxh3_amd.kernels.mxfp4_linear import (MXFP4Linear, convert_transformer_to_mxfp4, dequantize_mxfp4,
                                                quantize_mxfp4)
from oracle import dit_block as ob

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def randn(seed, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def check_quant(x):
    codes, scales = quantize_mxfp4(x)
    rc, rs = ob.mxfp4_quantize(f64(x))
    assert np.array_equal(scales.cpu().numpy(), rs)
    nan = np.repeat(rs.transpose(1, 0, 2).reshape(x.shape[0], -1)[:, : x.shape[1] // 32] == 255, 16, 1)
    assert np.array_equal(np.where(nan, 0, codes.cpu().numpy()), np.where(nan, 0, rc))
    ref = ob.mxfp4_values(rc, rs)
    # exact in bf16 and fp32 (but 4 x 2^126, which a block's largest value from 7 / 4 x 2^127 on rounds to, is past
    # them and becomes infinite); rounded in fp16
    for dt in (torch.bfloat16, torch.float32, torch.float16):
        want = torch.from_numpy(ref).to(dt)
        if dt != torch.float16:
            assert np.array_equal(f64(want), np.where(np.abs(ref) >= 2.0 ** 128, np.inf * ref, ref), equal_nan=True)
        assert np.array_equal(f64(dequantize_mxfp4(codes, scales, dt)), f64(want), equal_nan=True), dt


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 3072), (5, 96), (17, 288), (33, 4640), (130, 1056), (3, 12288),
                                 (6000, 3072)])
def test_quantizer(m, k, dtype):
    check_quant(randn(m + k, m, k, dtype=DT[dtype]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_quantizer_on_every_16_bit_value(dtype):
    """All 16-bit patterns, in blocks of neighbours and in blocks scattered over the range: every exponent and
    rounding, subnormals, infinities and NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    v = bits.view(torch.float16 if dtype == "fp16" else torch.bfloat16)
    v = v.float() if dtype == "fp32" else v
    check_quant(v.reshape(-1, 64).cuda())
    perm = torch.randperm(65536, generator=torch.Generator().manual_seed(0))
    check_quant(v[perm].reshape(-1, 1024).cuda())
    # (with few non-finite blocks: finite values only)
    v = v[torch.isfinite(v.float())]
    check_quant(v[: v.numel() // 32 * 32].reshape(-1, 32).cuda())


def test_quantizer_on_scaled_grids():
    """Values on and next to every code and midpoint, under scales from the smallest to the largest."""
    grid = torch.tensor(sorted(set(ob.GRID) | {(a + b) / 2 for a, b in zip(ob.GRID, ob.GRID[1:])}))
    near = torch.cat([grid, torch.nextafter(grid.float(), torch.tensor(9.0)).double(),
                      torch.nextafter(grid.float(), torch.tensor(-9.0)).double(), torch.tensor([6.5, 6.99])])
    row = torch.zeros(64, dtype=torch.float64)
    row[: near.numel()] = near
    row[32:] = row[32:].flip(0) * -1
    rows = torch.stack([row * 2.0 ** e for e in range(-150, 126)])
    check_quant(rows.float().cuda())


def test_quantizer_layouts():
    x = randn(3, 40, 300)
    view = x[1:34:2, 5:293]
    want = quantize_mxfp4(view.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(quantize_mxfp4(view), want))
    t = view.t().contiguous().t()
    assert all(torch.equal(a, b) for a, b in zip(quantize_mxfp4(t), want))
    row = x[:1, :32].expand(7, 32)
    assert torch.equal(quantize_mxfp4(row)[0], quantize_mxfp4(row.contiguous())[0])
    codes, scales = quantize_mxfp4(x[:0, :32])
    assert codes.shape == (0, 16) and scales.shape == (1, 0, 8) and dequantize_mxfp4(codes, scales).shape == (0, 32)


def product(m, n, k, seed=0, bias=True, act=0, spread=0):
    a, w = randn(seed, m, k), randn(seed + 1, n, k, std=0.05)
    if spread:  # block magnitudes over 2^+-spread
        g = torch.Generator().manual_seed(seed + 2)
        for t in (a, w):
            e = torch.randint(-spread, spread + 1, (t.shape[0], k // 32), generator=g).cuda()
            t.copy_((t.float().view(t.shape[0], -1, 32) * torch.exp2(e.float()).unsqueeze(-1)).view(t.shape))
    b = randn(seed + 3, n, std=0.5) if bias else None
    a4, sa = quantize_mxfp4(a)
    w4, sw = quantize_mxfp4(w)
    out = ops.gemm_mxfp4(a4, w4, sa, sw, b, act)
    va, vw = ob.mxfp4_values(a4.cpu().numpy(), sa.cpu().numpy()), ob.mxfp4_values(w4.cpu().numpy(), sw.cpu().numpy())
    ref, bound = ob.mxfp4_linear(va, vw, None if b is None else f64(b), bool(act))
    err = np.abs(f64(out) - ref)
    ok = err <= bound + ob.half_step(np.abs(ref) + bound, "bf16")
    assert out.shape == (m, n) and out.dtype == torch.bfloat16
    assert ok.all(), ((err - bound).max(), np.argwhere(~ok)[:4], (~ok).sum())
    return out


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 32), (1, 64, 3072), (1, 9216, 3072), (2, 33, 64), (7, 1001, 288), (16, 64, 256), (17, 130, 512),
    (32, 3072, 1024), (33, 96, 1056), (64, 64, 12288), (100, 200, 96), (128, 128, 256), (129, 257, 544),
    (256, 256, 4640), (300, 1000, 224), (513, 768, 3072), (1000, 520, 480), (2048, 384, 320),
])
def test_product(m, n, k):
    product(m, n, k, seed=m + n)


@pytest.mark.parametrize("m,n,k", [(4096, 8192, 96), (4097, 4224, 800)])
def test_product_of_many_tiles(m, n, k):
    product(m, n, k, seed=m)


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("m,n,k", [(1, 9216, 3072), (7, 1001, 288), (3, 64, 8224), (17, 130, 512), (33, 2100, 96),
                                   (200, 2100, 800), (70, 1999, 2080), (130, 4100, 800), (300, 4100, 320),
                                   (256, 9216, 2080), (513, 12288, 800), (2100, 1001, 768), (4100, 4104, 256),
                                   (6000, 4100, 288)])
def test_every_kernel(m, n, k, act):
    """Each of the product's kernels (tests/test_mxfp4_tiles.py), with whole and cut stages and tiles, rows of
    outputs at any alignment."""
    product(m, n, k, seed=m + k, act=act)


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("m,n,k", [(200, 2100, 768), (130, 4100, 768), (300, 4100, 768), (256, 9216, 2048),
                                   (513, 12288, 768), (8200, 4100, 768), (4097, 8200, 1024), (2100, 4100, 1536)])
def test_every_tile_kernel_with_whole_stages(m, n, k, act):
    """K in whole stages of 256, three and more of them (tests/test_mxfp4_tiles.py: the ring and the persistent kernels,
    256 x 256 tiles in one round of workgroups and in several)."""
    product(m, n, k, seed=m + k, act=act)


@pytest.mark.parametrize("k", [768, 800, 1280])
def test_a_token_does_not_depend_on_the_others(k):
    """Bit for bit, among the sizes that go to the ring and the persistent kernels, which add in one order; and among
    those of up to 16 tokens."""
    n = 4100
    (a4, sa), (w4, sw) = quantize_mxfp4(randn(1, 8200, k)), quantize_mxfp4(randn(2, n, k))
    b = randn(3, n)
    whole = ops.gemm_mxfp4(a4, w4, sa, sw, b, 1)
    part = lambda i, m: ops.gemm_mxfp4(a4[i: i + m], w4, sa[:, i: i + m].contiguous(), sw, b, 1)  # noqa: E731
    for m in (60, 130, 300, 700, 1100, 2100, 4200):
        for i in (0, 8200 - m):
            assert torch.equal(part(i, m), whole[i: i + m]), (m, i)
    few = part(3, 16)
    for m in (1, 2, 7, 15):
        assert torch.equal(part(3, m), few[:m])


@pytest.mark.parametrize("m,n,k", [(1, 48, 3072), (20, 70, 96), (130, 300, 320), (700, 256, 768), (4500, 4100, 64)])
@pytest.mark.parametrize("bias", [True, False])
def test_product_with_activation(m, n, k, bias):
    product(m, n, k, seed=n, bias=bias, act=1)


@pytest.mark.parametrize("m,n,k", [(3, 40, 512), (70, 130, 1056), (513, 300, 288)])
def test_product_of_widely_scaled_blocks(m, n, k):
    product(m, n, k, seed=k, spread=6)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1, 9216, 3072), (1, 3, 32), (5, 1001, 288), (16, 64, 8224), (16, 5200, 3072),
                                   (11, 5200, 4640), (2, 96, 288), (4, 5201, 288), (3, 6145, 6176), (17, 96, 544),
                                   (600, 300, 96), (16, 64, 4000), (12, 4001, 5280), (7, 5200, 4640), (1, 48, 65536),
                                   (8, 100, 8192), (1, 33, 65568)])
def test_linear_in_one_call_is_the_quantizer_and_the_product(m, n, k, dtype):
    x, w, b = randn(m, m, k, dtype=DT[dtype]), randn(n, n, k, std=0.05), randn(3, n)
    x[0, :32] = 0
    x[m // 2, 5] = 1e-7
    w4, sw = quantize_mxfp4(w)
    for act in (0, 1):
        want = ops.gemm_mxfp4(*[(q, w4, s, sw) for q, s in [quantize_mxfp4(x)]][0], b, act)
        assert torch.equal(ops.mxfp4_linear(x, w4, sw, b, act), want)
    wide = torch.zeros((m, k + 7), dtype=x.dtype, device="cuda")
    wide[:, 3: k + 3] = x
    assert torch.equal(ops.mxfp4_linear(wide[:, 3: k + 3], w4, sw, b, 1), want)
    assert torch.equal(ops.mxfp4_linear(x.t().contiguous().t(), w4, sw, b, 1), want)
    x[m - 1, k - 1] = float("nan")
    x[0, 2] = -float("inf")
    out = ops.mxfp4_linear(x, w4, sw, b, 0)
    assert out[m - 1].isnan().all() and out[0].isnan().all() and torch.isfinite(out[1: m - 1]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_linear_quantizes_every_16_bit_value_as_the_quantizer(dtype):
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16 if dtype == "fp16" else torch.bfloat16)
    v = v[torch.randperm(65536, generator=torch.Generator().manual_seed(1))].float()
    v = v.nan_to_num(0.5, 1.0, -1.0).to(DT[dtype]).reshape(-1, 1024).cuda()
    w4, sw = quantize_mxfp4(torch.eye(1024, device="cuda"))  # (each output is one value of the row)
    for rows in v.split(16):
        (a4, sa), got = quantize_mxfp4(rows), ops.mxfp4_linear(rows, w4, sw, None, 0)
        assert torch.equal(got, ops.gemm_mxfp4(a4, w4, sa, sw, None, 0))
        assert torch.equal(got, dequantize_mxfp4(a4, sa))


def test_scale_bytes_past_k_are_ignored():
    """K = 288 fills one block of the second slab; the others' bytes may hold anything, NaN among it."""
    for m in (3, 40, 140, 4100):
        a, w = randn(1, m, 288), randn(2, 4200 if m > 4096 else 96, 288)
        (a4, sa), (w4, sw) = quantize_mxfp4(a), quantize_mxfp4(w)
        want = ops.gemm_mxfp4(a4, w4, sa, sw, None, 0)
        assert (sa[1, :, 1:] == 127).all()
        sa, sw = sa.clone(), sw.clone()
        sa[1, :, 1:] = 255
        sw[1, :, 1:] = 254
        assert torch.equal(ops.gemm_mxfp4(a4, w4, sa, sw, None, 0), want)
        assert torch.equal(dequantize_mxfp4(a4, sa), dequantize_mxfp4(*quantize_mxfp4(a)))


@pytest.mark.parametrize("m", [1, 20, 140, 4200])
def test_nan_blocks_reach_their_row_and_column_alone(m):
    n = 4200 if m > 4096 else 80
    a, w = randn(1, m, 544), randn(2, n, 544)
    clean = ops.gemm_mxfp4(*_args(a, w))
    a[m // 2, 100] = float("inf")
    w[3, 543] = float("nan")
    out = ops.gemm_mxfp4(*_args(a, w))
    bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    bad[m // 2], bad[:, 3] = True, True
    assert out[bad].isnan().all() and torch.equal(out[~bad], clean[~bad])


def _args(a, w):
    (a4, sa), (w4, sw) = quantize_mxfp4(a), quantize_mxfp4(w)
    return a4, w4, sa, sw, None, 0


def test_smallest_and_largest_scales():
    """Blocks at the ends of the scales' range: 2^-127 times codes, and products that meet in the middle."""
    a = torch.full((33, 64), 2.0 ** -126, device="cuda")
    a[:, 32:] = 0.0
    w = torch.full((40, 64), 2.0 ** 120, device="cuda")
    out = ops.gemm_mxfp4(*_args(a, w))
    va = ob.mxfp4_values(*(t.cpu().numpy() for t in quantize_mxfp4(a)))
    vw = ob.mxfp4_values(*(t.cpu().numpy() for t in quantize_mxfp4(w)))
    assert np.array_equal(f64(out), va @ vw.T)


def test_every_pair_of_codes():
    """All 256 products of two codes, one per output, exactly."""
    vals = torch.tensor(np.concatenate([ob.GRID, -ob.GRID]), dtype=torch.float32, device="cuda")
    a = torch.zeros((16, 32), device="cuda")
    a[:, 0], a[:, 1] = vals, 6.0
    w = torch.zeros((16, 32), device="cuda")
    w[:, 0], w[:, 2] = vals, 6.0
    out = ops.gemm_mxfp4(*_args(a, w))
    assert torch.equal(out.float(), vals[:, None] * vals[None])


def test_empty_products():
    a4, w4, sa, sw, _, _ = _args(randn(1, 4, 64), randn(2, 5, 64))
    assert ops.gemm_mxfp4(a4[:0], w4, sa[:, :0], sw, None, 0).shape == (0, 5)
    assert ops.gemm_mxfp4(a4, w4[:0], sa, sw[:, :0], None, 0).shape == (4, 0)


def test_product_is_the_same_every_time_and_on_another_stream():
    args = _args(randn(1, 700, 1056), randn(2, 900, 1056))
    one = _args(randn(1, 1, 3072), randn(2, 512, 3072))
    want, want1 = ops.gemm_mxfp4(*args), ops.gemm_mxfp4(*one)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.gemm_mxfp4(*args) for _ in range(3)]
        got1 = [ops.gemm_mxfp4(*one) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got) and all(torch.equal(g, want1) for g in got1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_module(dtype):
    lin = nn.Linear(288, 176).to("cuda", torch.bfloat16)
    w, b = lin.weight.detach().clone(), lin.bias.detach().clone()
    x = randn(5, 2, 9, 288, dtype=DT[dtype])
    mod = MXFP4Linear.from_linear(lin)
    assert lin.weight is None and (mod.in_features, mod.out_features) == (288, 176)
    y = mod(x)
    assert y.shape == (2, 9, 176) and y.dtype == DT[dtype]
    xv, wv = (f64(dequantize_mxfp4(*quantize_mxfp4(t.reshape(-1, 288)), torch.float32)) for t in (x, w))
    ref, bound = ob.mxfp4_linear(xv, wv, f64(b))
    err = np.abs(f64(y).reshape(18, 176) - ref)
    assert (err <= bound + 1.01 * ob.half_step(np.abs(ref) + bound, "bf16")).all()
    again = MXFP4Linear.from_quantized(mod.w4, mod.w_scale, mod.bias)
    assert torch.equal(again(x), y) and set(dict(mod.named_buffers())) == {"w4", "w_scale", "bias"}
    assert torch.equal(mod.forward_quantized(*quantize_mxfp4(x.reshape(-1, 288))).to(y.dtype), y.reshape(18, 176))
    # LoRA and the activation
    A, B = randn(6, 8, 288, std=0.1), randn(7, 176, 8, std=0.1)
    mod.adapters.append((A, B, 0.5))
    got = mod(x.to(torch.bfloat16)).reshape(18, 176)
    plain = again(x.to(torch.bfloat16)).reshape(18, 176)
    x2 = x.to(torch.bfloat16).reshape(18, 288)
    assert torch.equal(got, plain + ((x2 @ A.t()) @ B.t() * 0.5))
    mod.act = 1
    assert torch.equal(mod(x.to(torch.bfloat16)).reshape(18, 176), torch.nn.functional.gelu(got, approximate="tanh"))
    with pytest.raises(ValueError):
        mod.forward_quantized(*quantize_mxfp4(x2))


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_adapters_add_in_the_input_s_dtype(dtype, act):
    """The product, then each branch and the activation, in x's dtype, as FP8Linear does it."""
    mod = MXFP4Linear.from_linear(nn.Linear(288, 176, device="cuda", dtype=torch.bfloat16))
    x = randn(5, 2, 9, 288, dtype=DT[dtype])
    want = mod(x)
    mod.act = act
    for i, (rank, scale) in enumerate(((8, 0.5), (3, 1.7))):
        A, B = randn(6 + i, rank, 288, std=0.1), randn(8 + i, 176, rank, std=0.1)
        mod.adapters.append((A, B, scale))
        want = want + (((x.to(A.dtype) @ A.t()) @ B.t()) * scale).to(x.dtype)
    if act:
        want = torch.nn.functional.gelu(want, approximate="tanh")
    assert want.dtype == DT[dtype] and torch.equal(mod(x), want)


def test_conversion_of_a_transformer():
    class Proj(nn.Module):
        def __init__(self):
            super().__init__()
            self.proj = nn.Linear(64, 128)
            self.approximate = "tanh"

        def forward(self, x):
            return torch.nn.functional.gelu(self.proj(x), approximate="tanh")

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.up, self.down, self.norm_lin = Proj(), nn.Linear(128, 64), nn.Linear(64, 64)
            self.odd = nn.Linear(64, 72)

        def forward(self, x):
            return x + self.down(self.up(x)) + self.norm_lin(x)

    net = nn.Module()
    net.blocks = nn.ModuleList(Block() for _ in range(4))
    net = net.to("cuda", torch.bfloat16)
    x = randn(1, 3, 64)
    before = net.blocks[1](x)
    assert convert_transformer_to_mxfp4(net, "norm", 1, fuse_gelu=True) == 4
    assert isinstance(net.blocks[1].up.proj, MXFP4Linear) and net.blocks[1].up.proj.act == 1
    assert isinstance(net.blocks[2].down, MXFP4Linear) and isinstance(net.blocks[0].down, nn.Linear)
    assert isinstance(net.blocks[1].norm_lin, nn.Linear) and isinstance(net.blocks[1].odd, nn.Linear)
    after = net.blocks[1](x)
    # two 4-bit linears: each value within a quarter of itself at most, errors that mostly cancel
    assert (after - before).float().norm() < 0.2 * before.float().norm()


def test_refusals():
    x = randn(1, 4, 64)
    a4, w4, sa, sw, _, _ = _args(x, x)
    for bad in (x[0], x.cpu(), x[:, :48], x.to(torch.float64), x[:, :0]):
        with pytest.raises(ValueError):
            quantize_mxfp4(bad)
    for args in ((a4.cpu(), sa), (a4, sa.cpu()), (a4[:3], sa), (a4.to(torch.int32), sa), (a4, sa.to(torch.int32)),
                 (a4[:, :24].contiguous(), sa), (a4[:, :16], sa), (a4, sa[..., :4])):
        with pytest.raises(ValueError):
            dequantize_mxfp4(*args)
    with pytest.raises(ValueError):
        dequantize_mxfp4(a4, sa, torch.float64)
    b = torch.zeros(4, dtype=torch.bfloat16, device="cuda")
    for args in ((a4, w4[:, :16].contiguous(), sa, sw, None, 0), (a4, w4, sa, sw[:, :2], None, 0),
                 (a4, w4, sa, sw, b[:3], 0), (a4, w4, sa, sw, b.float(), 0), (a4, w4, sa, sw, b.cpu(), 0),
                 (a4, w4.cpu(), sa, sw.cpu(), None, 0)):
        with pytest.raises(ValueError):
            ops.gemm_mxfp4(*args)
    with pytest.raises(RuntimeError, match="act"):
        ops.gemm_mxfp4(a4, w4, sa, sw, b, 5)
    for args in ((x[:, :32], w4, sw, b, 0), (x[0], w4, sw, b, 0), (x.cpu(), w4, sw, b, 0), (x, w4, sw[:, :3], b, 0),
                 (x, w4, sw, b[:2], 0), (x.double(), w4, sw, b, 0), (x, w4.cpu(), sw.cpu(), None, 0)):
        with pytest.raises(ValueError):
            ops.mxfp4_linear(*args)
    with pytest.raises(RuntimeError, match="act"):
        ops.mxfp4_linear(x, w4, sw, b, 2)
    with pytest.raises(ValueError):
        MXFP4Linear.from_quantized(w4, sw[:, :3])
    with pytest.raises(ValueError):
        MXFP4Linear.from_quantized(w4.to(torch.int8), sw)
