"""The gated residual with its norms against the 64-bit oracle, and its quantized outputs against the quantizers of
the stored result, bit for bit."""
import numpy as np
import pytest
import torch

from minimaxh3_amd.kernels.block_norms import gated_residual_norm
from minimaxh3_amd.kernels.fp8_linear import quantize_rows
from minimaxh3_amd.kernels.mxfp4_linear import quantize_mxfp4
from oracle import dit_block as ob

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t):
    return None if t is None else t.detach().to("cpu", torch.float64).numpy()


def make(seed, b, s, c, dtype, groups=1, sandwich=False, weighted=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *sh: torch.randn(sh, generator=g)  # noqa: E731
    x, branch = (rn(b, s, c) * 2 + 0.5).to(DT[dtype]).cuda(), rn(b, s, c).to(DT[dtype]).cuda()
    mod = (rn(b, groups, 3 * c) * 0.4).to(DT[dtype]).cuda()
    parts = [mod[..., i * c: (i + 1) * c] for i in range(3)]
    gate, shift, scale = parts if groups > 1 else [p[:, 0] for p in parts]
    w = [(1 + 0.2 * rn(c)).to(DT[dtype]).cuda() for _ in range(2)]
    return {"x": x, "branch": branch, "gate": gate, "shift": shift, "scale": scale,
            "branch_weight": w[0] if sandwich else None, "weight": w[1] if weighted else None}


def check(a, dtype, norm, rs=1.0, eps=1e-6):
    r, y = gated_residual_norm(**a, norm=norm, residual_scale=rs, eps=eps)
    rr, yy, br, by = ob.gated_residual_norm(**{k: f64(v) for k, v in a.items()}, norm=norm, residual_scale=rs, eps=eps)
    for what, got, ref, bound in (("r", r, rr, br), ("y", y, yy, by)):
        assert got.dtype == DT[dtype] and tuple(got.shape) == ref.shape
        err = np.abs(f64(got) - ref)
        ok = err <= bound + ob.half_step(np.abs(ref) + bound, dtype)
        assert ok.all(), (what, (err - bound).max(), np.argwhere(~ok)[:4])


SHAPES = [(1, 1, 3072), (2, 3, 3072), (1, 2, 1), (2, 5, 7), (1, 3, 8), (3, 4, 33), (1, 6, 512), (1, 3, 2730),
          (1, 2, 4096), (1, 2, 4104), (2, 2, 8192), (1, 1, 12288), (1, 1, 16384), (1, 1, 16383), (1, 4099, 72),
          (1, 4097, 96), (1, 4200, 1000), (1, 9000, 9), (1, 8200, 515),
          (3, 43, 64), (2, 35, 120), (1, 37, 128), (1, 21, 250), (5, 17, 256), (1, 9, 257)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("b,s,c", SHAPES)
def test_against_the_oracle(b, s, c, norm, dtype):
    odd = (s + c) % 2 == 1
    # (one channel: a LayerNorm of one value is its shift; of few, the deviations may be tiny: a larger eps keeps the
    # bound meaningful)
    check(make(c + s, b, s, c, dtype, sandwich=odd, weighted=norm == "rms"), dtype, norm, rs=0.75 if odd else 1.0,
          eps=1e-2 if c < 64 else 1e-6)


@pytest.mark.parametrize("absent", ["gate", "shift", "scale", "branch", "all"])
def test_operands_left_out(absent):
    a = make(1, 2, 6, 264, "bf16")
    for k in {"branch": ("branch", "gate"), "all": ("gate", "shift", "scale")}.get(absent, (absent,)):
        a[k] = None
    if absent == "branch":
        r, y = gated_residual_norm(**a)
        assert r is a["x"]
        ref = gated_residual_norm(a["x"], torch.zeros_like(a["x"]), None, a["shift"], a["scale"])
        assert torch.equal(y, ref[1]) and torch.equal(a["x"], ref[0])
    else:
        check(a, "bf16", "layer")


@pytest.mark.parametrize("groups", [2, 3, 12])
@pytest.mark.parametrize("s", [12, 4104])
def test_modulation_per_span(groups, s):
    check(make(groups, 2, s, 40, "bf16", groups=groups, sandwich=True), "bf16", "rms")
    a = make(groups, 1, s, 40, "fp32", groups=groups)
    a["gate"] = a["gate"][:, :1].expand(1, groups, 40)  # one row for all spans, stride 0
    check(a, "fp32", "layer")


def test_layouts():
    a = make(4, 2, 9, 96, "bf16", groups=3)
    want = gated_residual_norm(**a)
    odd = torch.zeros((2, 9, 205), dtype=torch.bfloat16, device="cuda")
    odd[..., 3:99], odd[..., 101:197] = a["x"], a["branch"]
    got = gated_residual_norm(**{**a, "x": odd[..., 3:99], "branch": odd[..., 101:197]})
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    swapped = {**a, "x": a["x"].transpose(0, 1).contiguous().transpose(0, 1),
               "branch": a["branch"].transpose(1, 2).contiguous().transpose(1, 2)}
    assert all(torch.equal(p, q) for p, q in zip(gated_residual_norm(**swapped), want))
    chan = {**a, "shift": a["shift"].transpose(1, 2).contiguous().transpose(1, 2)}
    assert all(torch.equal(p, q) for p, q in zip(gated_residual_norm(**chan), want))
    one = a["x"][:1].expand(2, 9, 96)
    assert torch.equal(gated_residual_norm(**{**a, "x": one})[1], gated_residual_norm(**{**a, "x": one.contiguous()})[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("b,s,c", [(1, 1, 3072), (2, 7, 96), (1, 4098, 288), (1, 3, 4640), (1, 2, 8192), (1, 2, 16384),
                                   (2, 3, 32), (1, 4100, 4096), (3, 37, 160), (1, 45, 256), (1, 19, 64)])
def test_quantized_outputs_are_the_quantizers_of_y(b, s, c, dtype):
    a = make(c, b, s, c, dtype, sandwich=c == 96, weighted=c == 288)
    a["x"][0, 0, :32] = 0
    r, y = gated_residual_norm(**a)
    y2 = y.reshape(-1, c)
    for fmt, quant in (("e4m3", quantize_rows), ("mxfp4", quantize_mxfp4)):
        want = quant(y2)
        r1, codes, scales, y1 = gated_residual_norm(**a, quantize=fmt, return_modulated=True)
        assert torch.equal(r1, r) and torch.equal(y1, y)
        assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)), fmt
        assert codes.shape == want[0].shape and torch.equal(scales, want[1]), fmt
        r1, codes, scales = gated_residual_norm(**a, quantize=fmt)
        assert torch.equal(r1, r) and torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(scales, want[1])


@pytest.mark.parametrize("c", [1, 5, 7, 9, 15, 33, 1001, 2730, 4099, 16383])
def test_e4m3_codes_of_odd_widths(c):
    a = make(c, 2, 5, c, "bf16")
    _, y = gated_residual_norm(**a)
    want = quantize_rows(y.reshape(-1, c))
    _, codes, scales = gated_residual_norm(**a, quantize="e4m3")
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


LARGE = [("bf16", 8200, 3072), ("fp16", 8197, 2730), ("bf16", 8192, 1032), ("bf16", 8200, 2000), ("fp16", 8192, 2560),
         ("fp32", 8200, 1536), ("fp32", 8195, 1029)]


@pytest.mark.parametrize("norm,sandwich", [("layer", False), ("rms", True)])
@pytest.mark.parametrize("dtype,s,c", LARGE)
def test_one_wave_a_row_against_the_oracle(dtype, s, c, norm, sandwich):
    """1025 channels and more, from 8192 rows on."""
    check(make(c + s, 1, s, c, dtype, sandwich=sandwich, weighted=sandwich), dtype, norm, rs=0.75 if sandwich else 1.0)


@pytest.mark.parametrize("sandwich", [False, True])
@pytest.mark.parametrize("dtype,s,c", [*LARGE, ("bf16", 8200, 1056), ("fp16", 8200, 2336), ("fp32", 8192, 1312)])
def test_codes_of_one_wave_a_row_are_the_quantizers_of_y(dtype, s, c, sandwich):
    a = make(c, 1, s, c, dtype, sandwich=sandwich, weighted=sandwich)
    a["x"][0, 0, :32] = 0
    r, y = gated_residual_norm(**a)
    for fmt, quant in (("e4m3", quantize_rows), ("mxfp4", quantize_mxfp4)):
        if fmt == "e4m3" or c % 32 == 0:
            want = quant(y[0])
            r1, codes, scales = gated_residual_norm(**a, quantize=fmt)
            assert torch.equal(r1, r) and torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)), fmt
            assert torch.equal(scales, want[1]), fmt


@pytest.mark.parametrize("norm,sandwich,weighted", [("layer", False, False), ("rms", True, True), ("layer", True, False)])
@pytest.mark.parametrize("dtype,c", [("bf16", 3072), ("bf16", 1032), ("fp16", 2730), ("bf16", 2048), ("fp16", 1600),
                                     ("fp32", 1536), ("fp32", 1030), ("fp32", 3072), ("bf16", 1024), ("bf16", 33),
                                     ("bf16", 4104)])
def test_a_token_does_not_depend_on_the_others(c, dtype, norm, sandwich, weighted):
    """Bit for bit: from 8192 tokens on one wave holds a row that four share below."""
    s = 8300
    a = make(c, 1, s, c, dtype, sandwich=sandwich, weighted=weighted)
    per_call = {"norm": norm}
    formats = [None, "e4m3"] + ["mxfp4"] * (c % 32 == 0)
    whole = {q: gated_residual_norm(**a, **per_call, quantize=q) for q in formats}
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    for n in (1, 5, 700, 8191):
        for i in (0, s - n):
            cut = {**a, "x": a["x"][:, i: i + n], "branch": a["branch"][:, i: i + n]}
            for q in formats:
                got, want = gated_residual_norm(**cut, **per_call, quantize=q), whole[q]
                assert torch.equal(got[0], want[0][:, i: i + n])
                if q is None:
                    assert torch.equal(got[1], want[1][:, i: i + n])
                else:
                    scale = want[2][:, i: i + n] if q == "mxfp4" else want[2][i: i + n]
                    assert torch.equal(as_bytes(got[1]), as_bytes(want[1][i: i + n])) and torch.equal(got[2], scale)


@pytest.mark.parametrize("s", [3, 4100])
def test_non_finite_values_stay_in_their_token(s):
    a = make(8, 1, s, 96, "bf16", sandwich=True)
    clean = gated_residual_norm(**a, quantize="mxfp4", return_modulated=True)
    a["x"][0, 1, 4] = float("nan")
    a["branch"][0, 2, 50] = float("inf")
    got = gated_residual_norm(**a, quantize="mxfp4", return_modulated=True)
    keep = torch.ones(s, dtype=torch.bool, device="cuda")
    keep[1] = keep[2] = False
    assert torch.equal(got[0][:, keep], clean[0][:, keep]) and torch.equal(got[3][:, keep], clean[3][:, keep])
    assert torch.equal(got[1][keep], clean[1][keep]) and torch.equal(got[2][:, keep], clean[2][:, keep])
    assert got[3][0, 1].isnan().all() and got[3][0, 2].isnan().all() and (got[2][0, 1, :3] == 255).all()
    assert got[0][0, 1].isnan().sum() == 1
    # constant rows: LayerNorm of equal values is the shift
    a = make(8, 1, 2, 96, "fp32")
    a["x"].fill_(3.0)
    a["branch"].fill_(0.0)
    assert torch.equal(gated_residual_norm(**a)[1], a["shift"][:, None].expand(1, 2, 96))


def test_empty():
    a = make(8, 2, 0, 96, "bf16")
    r, y = gated_residual_norm(**a)
    assert r.shape == y.shape == (2, 0, 96)
    r, codes, scales = gated_residual_norm(**a, quantize="mxfp4")
    assert codes.shape == (0, 48) and scales.shape == (1, 0, 8)


def test_refusals():
    a = make(1, 2, 6, 96, "bf16", groups=3, sandwich=True, weighted=True)
    x = a["x"]
    bad = [
        {"x": x[0]}, {"x": x.cpu()}, {"x": x.to(torch.float64)}, {"branch": a["branch"][:, :5]},
        {"branch": a["branch"].float()}, {"branch": a["branch"].cpu()}, {"branch": None},
        {"gate": a["gate"][..., :95]}, {"gate": a["gate"].float()}, {"gate": a["gate"][:1]}, {"gate": a["gate"][:, 0]},
        {"gate": a["gate"].cpu()}, {"shift": a["shift"][:, :2]}, {"weight": a["weight"][:5]},
        {"weight": a["weight"].float()}, {"branch_weight": a["branch_weight"].repeat(2)[::2]},
        {"norm": "batch"}, {"quantize": "int8"}, {"gate": None, "shift": None, "scale": x[:, :4]},
    ]
    for change in bad:
        with pytest.raises(ValueError):
            gated_residual_norm(**{**a, **change})
    with pytest.raises(ValueError):
        gated_residual_norm(x, None, residual_scale=0.5)
    with pytest.raises(ValueError):
        gated_residual_norm(x[..., :40].contiguous(), x[..., :40].contiguous(), quantize="mxfp4")
    wide = torch.zeros((1, 1, 16392), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="16384"):
        gated_residual_norm(wide, wide)
    with pytest.raises(RuntimeError, match="eps"):
        gated_residual_norm(x, x, eps=-1.0)
