"""Rotary tables and the rotation of q and k against the 64-bit oracle.  Bounds come with the oracle's results
(fp32 arithmetic) plus half a step of the output type."""
import numpy as np
import pytest
import torch

from minimaxh3_amd.kernels.rotary import rotary_table, rotate_qk
from oracle import dit_block as ob

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


@pytest.mark.parametrize("dims", [(64,), (44, 42, 42), (2, 2, 2, 2), (256, 256), (8, 20, 20, 16)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("shape", [(1,), (2, 77), (1031,)])
def test_table(dims, dtype, shape):
    g = torch.Generator().manual_seed(len(dims) + sum(shape))
    pos = (torch.rand((*shape, len(dims)), generator=g, dtype=torch.float64) - 0.2) * 5000
    pos = pos.to(dtype)
    t = rotary_table(pos.cuda(), dims, theta=500.0)
    assert t.shape == (*shape, sum(dims) // 2, 2) and t.dtype == torch.float32
    # the reduced angle, at most pi / 4, is rounded once (2^-25), the series end at 2^-26 and are evaluated with
    # at most three roundings of values up to 1; the angle itself is off by a few 2^-53 of at most 5000
    assert np.abs(f64(t) - ob.rotary_table(f64(pos), dims, 500.0)).max() <= 2.0 ** -22


def test_table_of_far_and_special_positions():
    far = torch.tensor([[0.0], [-0.0], [1.0], [2.0 ** 24], [-3.0e6], [1.0e9], [2.0 ** 40]], dtype=torch.float64)
    t = f64(rotary_table(far.cuda(), (16,), theta=10000.0))
    ref = ob.rotary_table(f64(far), (16,), 10000.0)
    # fp64 angles: the frequency and the product are each off by up to 4 steps of 2^-53
    assert (np.abs(t - ref) <= 2.0 ** -22 + 8 * 2.0 ** -53 * np.abs(f64(far))[..., None]).all()
    assert (t[0] == [1.0, 0.0]).all() and (np.abs(t[1]) == [1.0, 0.0]).all()
    bad = torch.tensor([[float("inf")], [float("nan")], [2.0]])
    t = f64(rotary_table(bad.cuda(), (4,)))
    assert np.isnan(t[:2]).all() and np.isfinite(t[2]).all()


def test_table_of_strided_and_empty_positions():
    pos = torch.arange(60, device="cuda", dtype=torch.float32).reshape(10, 6)
    assert torch.equal(rotary_table(pos[::2, 1::2], (4, 6, 2)), rotary_table(pos[::2, 1::2].contiguous(), (4, 6, 2)))
    assert rotary_table(pos[:0, :3], (4, 6, 2)).shape == (0, 6, 2)


def make(seed, b, s, hq, hk, d, p, dtype, weights, per_batch):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((b, s, (hq + 2 * hk) * d), generator=g).to(DT[dtype]).cuda()
    q = qkv[..., : hq * d].unflatten(-1, (hq, d)).transpose(1, 2)
    k = qkv[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d)).transpose(1, 2) if hk else None
    a = torch.rand((b, s, p) if per_batch else (s, p), generator=g) * 7
    table = torch.stack([a.cos(), a.sin()], -1).cuda()
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(DT[dtype]).cuda() if weights else None for _ in range(2))
    return q, k, table, qw, kw if hk else None


def check(out, x, table, w, dtype, interleaved, eps=1e-6):
    ref, bound = ob.rotate(f64(x), f64(table), None if w is None else f64(w), eps, interleaved)
    err = np.abs(f64(out) - ref)
    assert (err <= bound + ob.half_step(np.abs(ref) + bound, dtype)).all(), (err - bound).max()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("b,s,hq,hk,d,p", [
    (1, 1, 1, 1, 8, 4),        # one token, one head
    (1, 1, 24, 24, 128, 64),   # one token of the 480p block
    (2, 37, 24, 24, 128, 64),
    (1, 700, 5, 3, 64, 24),    # channels that pass through; heads that do not fill a wave
    (3, 9, 4, 2, 96, 48),      # 12 chunks in 16 lanes
    (1, 5, 3, 1, 72, 36),      # 36 pairs: a half-split pair spans two lanes' chunks
    (2, 6, 7, 2, 50, 25),      # a head of 50 channels
    (1, 3, 2, 2, 256, 128),
    (1, 3, 2, 1, 512, 256),
    (1, 2, 2, 1, 520, 200),    # wider than a wave
    (2, 4, 3, 0, 80, 33),      # q alone
    (1, 4, 2, 2, 64, 0),       # nothing turns
    (1, 2, 2, 2, 1, 0),
])
def test_rotate(b, s, hq, hk, d, p, dtype, weights, interleaved):
    q, k, table, qw, kw = make(d + s, b, s, hq, hk, d, p, dtype, weights, per_batch=b > 1)
    qo, ko = rotate_qk(q, k, table, qw, kw, interleaved=interleaved)
    assert qo.shape == q.shape and qo.dtype == q.dtype
    check(qo, q, table, qw, dtype, interleaved)
    if k is None:
        assert ko is None
    else:
        check(ko, k, table, kw, dtype, interleaved)


def test_layouts():
    """Any strides and alignment, the results in the inputs' order of dimensions."""
    q, k, table, qw, kw = make(3, 2, 33, 4, 4, 64, 32, "bf16", True, False)
    want = rotate_qk(q.contiguous(), k.contiguous(), table, qw, kw)
    got = rotate_qk(q, k, table, qw, kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0].transpose(1, 2).is_contiguous() and want[0].is_contiguous()
    # a view that starts one element into its storage, with odd row strides
    store = torch.zeros((2, 4, 33, 67), dtype=torch.bfloat16, device="cuda")
    view = store[..., 1:65]
    view.copy_(q)
    assert torch.equal(rotate_qk(view, None, table, qw)[0], want[0])
    # channels that are not neighbours, and one head for all (stride 0)
    chan = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert chan.stride(3) != 1 and torch.equal(rotate_qk(chan, None, table, qw)[0], want[0])
    one = q[:, :1].expand(2, 4, 33, 64)
    assert torch.equal(rotate_qk(one, None, table, qw)[0], want[0][:, :1].expand(2, 4, 33, 64))


def test_non_finite_values_stay_in_their_head():
    q, _, table, qw, _ = make(5, 1, 4, 3, 0, 64, 32, "bf16", True, False)
    q = q.contiguous()
    q[0, 1, 2, 5] = float("nan")
    q[0, 2, 0, 7] = float("inf")
    o = rotate_qk(q, None, table, qw)[0]
    bad = torch.zeros((1, 3, 4), dtype=torch.bool, device="cuda")
    bad[0, 1, 2] = bad[0, 2, 0] = True
    assert torch.isfinite(o[~bad]).all() and o[0, 1, 2].isnan().all() and not torch.isfinite(o[0, 2, 0, 6:8]).any()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,p", [(64, 24), (64, 20), (96, 40), (96, 37), (50, 20), (128, 0), (520, 200)])
def test_channels_that_pass_through_are_untouched(d, p, dtype, interleaved):
    """Bit for bit, infinities and negative zeros too, and nothing of them in the channels that turn."""
    q, k, table, _, _ = make(d, 1, 9, 3, 2, d, p, dtype, False, False)
    q, k = q.contiguous(), k.contiguous()
    for x in (q, k):
        x[..., 2 * p:: 3] = -0.0
        x[..., 2 * p + 1:: 5] = float("inf")
        x[..., 2 * p + 2:: 7] = float("nan")
    for x, o in zip((q, k), rotate_qk(q, k, table, interleaved=interleaved)):
        bits = torch.int32 if dtype == "fp32" else torch.int16
        nan = x.isnan()
        same = (o.view(bits) == x.view(bits)) | (o.isnan() & nan)
        assert same[..., 2 * p:].all() and torch.isfinite(o[..., : 2 * p]).all()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("d,p", [(128, 64), (96, 37)])
def test_a_token_does_not_depend_on_the_others(d, p, weights, interleaved):
    """Bit for bit: few tokens split their heads over waves, many do not."""
    q, k, table, qw, kw = make(4, 1, 3000, 24, 5, d, p, "bf16", weights, False)
    qo, ko = rotate_qk(q, k, table, qw, kw, interleaved=interleaved)
    for n in (1, 5, 80, 700):
        for i in (0, 1500, 3000 - n):
            part = rotate_qk(q[:, :, i: i + n], k[:, :, i: i + n], table[i: i + n].contiguous(), qw, kw,
                             interleaved=interleaved)
            assert torch.equal(part[0], qo[:, :, i: i + n]) and torch.equal(part[1], ko[:, :, i: i + n])


def _apart(x, stride):
    """x [B, H, S, D] as a view whose heads lie `stride` elements apart."""
    b, h, s, d = x.shape
    store = torch.empty((h - 1) * stride + b * s * d, dtype=x.dtype, device="cuda")
    return store.as_strided((b, h, s, d), (s * d, stride, d, 1)).copy_(x)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("b,s,hq,hk,d,p", [(2, 9, 5, 3, 128, 64), (1, 37, 9, 1, 64, 24), (1, 5, 3, 2, 96, 37),
                                           (2, 4, 3, 1, 50, 25), (1, 3, 2, 2, 256, 128), (1, 3, 2, 1, 72, 36)])
def test_heads_far_apart(b, s, hq, hk, d, p, dtype, weights, interleaved):
    """The values, bit for bit, that heads which are neighbours get."""
    q, k, table, qw, kw = make(d + s, b, s, hq, hk, d, p, dtype, weights, False)
    want = rotate_qk(q, k, table, qw, kw, interleaved=interleaved)
    got = rotate_qk(_apart(q, 2 ** 24 + 24), _apart(k, 2 ** 24 + 56), table, qw, kw, interleaved=interleaved)
    for x, w, g, n in ((q, qw, got[0], want[0]), (k, kw, got[1], want[1])):
        check(g, x, table, w, dtype, interleaved)
        assert torch.equal(g, n)


@pytest.mark.parametrize("stride", [306_783_300, 306_783_400, 320_000_000])
@pytest.mark.parametrize("weights,interleaved", [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize("d,p", [(64, 32), (50, 25)])
def test_heads_at_and_past_32_bit_offsets(d, p, weights, interleaved, stride):
    """Eight heads: the last one's offset is on either side of 2^32 bytes."""
    q, _, table, qw, _ = make(d, 1, 3, 8, 0, d, p, "bf16", weights, False)
    want = rotate_qk(q, None, table, qw, interleaved=interleaved)[0]
    assert torch.equal(rotate_qk(_apart(q, stride), None, table, qw, interleaved=interleaved)[0], want)


@pytest.mark.parametrize("h,s,d,p", [(5, 140_001, 128, 64), (8, 5_000_001, 64, 4)])
def test_long_head_major_sequences(h, s, d, p):
    """[B, H, S, D] as it lies in memory, results too; a token as it is in a short sequence, bit for bit."""
    q = torch.zeros((1, h, s, d), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(s)
    spots = [0, 1, s // 2, s - 2, s - 1]
    q[:, :, spots] = torch.randn((1, h, 5, d), generator=g).bfloat16().cuda()
    table, w = torch.rand((s, p, 2), device="cuda"), (1 + 0.2 * torch.randn(d, generator=g)).bfloat16().cuda()
    for interleaved in (True, False):
        got = rotate_qk(q, None, table, w, interleaved=interleaved)[0]
        assert got.is_contiguous()
        few = rotate_qk(q[:, :, spots], None, table[spots], w, interleaved=interleaved)[0]
        assert torch.equal(got[:, :, spots], few)
        check(few, q[:, :, spots], table[spots], w, "bf16", interleaved)


def test_zero_heads_and_zero_tokens():
    q, k, table, qw, kw = make(5, 1, 0, 3, 1, 64, 32, "bf16", True, False)
    qo, ko = rotate_qk(q, k, table, qw, kw)
    assert qo.shape == (1, 3, 0, 64) and ko.shape == (1, 1, 0, 64)
    z = torch.zeros((1, 2, 3, 64), device="cuda")
    assert (rotate_qk(z, None, torch.rand((3, 32, 2), device="cuda"), torch.ones(64, device="cuda"))[0] == 0).all()


def test_refusals():
    q, k, table, qw, kw = make(1, 2, 5, 2, 2, 64, 32, "bf16", True, False)
    bad = [
        (q[0], k, table, qw, kw), (q, k[..., :32], table, qw, kw), (q, k[:1], table, qw, kw),
        (q, k.float(), table, qw, kw), (q, k, table[:4], qw, kw), (q, k, table.double(), qw, kw),
        (q, k, table[..., 0], qw, kw), (q, k, table.expand(3, 5, 32, 2).contiguous(), qw, kw),
        (q, k, torch.cat([table, table], 1), qw, kw), (q, k, table, qw[:32], kw), (q, k, table, qw.float(), kw),
        (q, k, table.cpu(), qw, kw), (q, k, table, qw.cpu(), kw), (q, None, table, qw, kw), (q.cpu(), k, table, qw, kw),
        (q.to(torch.float64), None, table, None, None), (q, k, table.transpose(0, 1), qw, kw),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            rotate_qk(*args)
    pos = torch.zeros((3, 2), device="cuda")
    for p, dims in ((pos, (4,)), (pos, (4, 3)), (pos, (4, 0)), (pos[0], (4, 4)), (pos.to(torch.int8), (4, 4)), (pos.cpu(), (4, 4))):
        with pytest.raises(ValueError):
            rotary_table(p, dims)
    for dims, theta in (((2, 512), 1e4), ((4, 4), 0.0), ((4, 4), float("nan"))):
        with pytest.raises((ValueError, RuntimeError)):
            rotary_table(pos, dims, theta=theta)
