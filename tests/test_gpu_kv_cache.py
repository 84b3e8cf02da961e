"""The paged e4m3 cache of keys and values, and the attention over it, against the 64-bit oracle.

Codes are exact but where the unrounded key lies within its 32-bit evaluation's bound of a border between two.
The attention's outputs: half a step of the output type, and 2^-10 of sum p |v| / sum p.  Of that half are the
probabilities' own half steps in fp16 (2^-11 each); the scores' fp32 sums over D products (D 2^-24 of
sum |q k| scale, under 2^-13 for scores of size 10), exp2 and the row sum share the other half.  Probabilities below fp16's
normal range add 2^-32 of the row's largest p 2^e each, times their code (`oracle.kv_cache.attend_small`): with the values
and scores of most tests here too little to count."""
import math

import numpy as np
import pytest
import torch

from minimaxh3_amd import ops
from minimaxh3_amd.kernels.kv_cache import FP8KVCache, append_kv, cached_attention, read_kv
from minimaxh3_amd.kernels.rotary import rotary_table, rotate_qk
from oracle import dit_block as ob
from oracle import kv_cache as ok
from oracle.numerics import e4m3_decode

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def raw(cache):
    return ([t.view(torch.uint8).cpu().numpy() for t in (cache.k, cache.v)],
            [t.cpu().numpy() for t in (cache.k_scale, cache.v_scale)])


def random_cache(seed, pages, heads, page, d, spread=3):
    """Any codes but NaN, under exponents of -spread - 6 ... spread - 6."""
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 127, (pages, heads, page, d), generator=g, dtype=torch.uint8)
             + 128 * torch.randint(0, 2, (pages, heads, page, d), generator=g, dtype=torch.uint8) for _ in range(2)]
    # (sizes up to 448 would let one product decide a row: most codes of 1 and below)
    codes = [torch.where(c % 128 > 56, c - 56 // 8 * 8, c) for c in codes]
    scales = [torch.randint(121 - spread, 122 + spread, (pages, heads), generator=g, dtype=torch.uint8) for _ in range(2)]
    return FP8KVCache.from_tensors(*[t.cuda() for t in codes + scales])


def normal_cache(seed, pages, heads, page, d, table, lengths, k_std=1.0, v_std=1.0):
    """A cache that holds normal keys and values, appended."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = FP8KVCache(pages, heads, d, page)
    S, B = table.shape[1] * page, table.shape[0]
    k, v = (torch.randn((B, heads, S, d), generator=g, device="cuda") * s for s in (k_std, v_std))
    append_kv(cache, table, torch.zeros(B, dtype=torch.int32, device="cuda"), k, v, counts=lengths)
    return cache


def pages_for(seed, b, width, extra=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(b * width + extra, generator=g)[: b * width].to(torch.int32).view(b, width).cuda()


# ---------------------------------------------------------------------------------------
# append, read
# ---------------------------------------------------------------------------------------

def check_append(cache, table, starts, k, v, counts=None, turns=None, weight=None, interleaved=True):
    pool = ok.Pool(*raw(cache))
    before = pool.copy()
    append_kv(cache, table, starts, k, v, counts=counts, table=turns, k_weight=weight, interleaved=interleaved)
    tb, st = table.cpu().numpy(), starts.cpu().numpy()
    cn = None if counts is None else counts.cpu().numpy()
    key, _, bound = ok.append(pool, tb, st, f64(k), f64(v), cn, None if turns is None else f64(turns),
                              None if weight is None else f64(weight), 1e-6, interleaved)
    codes, scales = raw(cache)
    assert np.array_equal(scales[0], pool.scales[0]) and np.array_equal(scales[1], pool.scales[1])
    assert np.array_equal(codes[1], pool.codes[1])
    wrong = codes[0] != pool.codes[0]
    if turns is None and weight is None:
        assert not wrong.any()
    elif wrong.any():
        # each as near to the unrounded key as the oracle's, within what 32 bits may add
        for b in range(len(st)):
            for s in range(k.shape[2] if cn is None else min(max(cn[b], 0), k.shape[2])):
                at = pool.at(tb, b, int(st[b]) + s)
                if at is None or not wrong[at[0], :, at[1]].any():
                    continue
                e = pool.scales[0][at[0]].astype(int)[:, None] - 127
                got, ref = (np.ldexp(e4m3_decode(c[0][at[0], :, at[1]]).astype(np.float64), e) for c in (codes, pool.codes))
                x, near = key[b, :, s], bound[b, :, s]
                assert (np.abs(got - x) <= np.abs(ref - x) + 2 * near).all()
                wrong[at[0], :, at[1]] = False
        assert not wrong.any()  # and nothing else differs
    return before, pool


@pytest.mark.parametrize("d,page", [(128, 16), (128, 32), (128, 64), (128, 128), (64, 16), (64, 32), (64, 64), (64, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_append_plain(d, page, dtype):
    g = torch.Generator().manual_seed(page + d)
    b, h, s = 3, 3, 2 * page + 5
    cache = random_cache(1, 40, h, page, d)
    table = pages_for(2, b, 6)
    qkv = (torch.randn((b, s, 3, h, d), generator=g) * torch.exp2(torch.randint(-9, 9, (b, s, 1, 1, 1), generator=g))).to(DT[dtype]).cuda()
    k, v = (qkv[:, :, i].transpose(1, 2) for i in (1, 2))
    check_append(cache, table, i32(0, page - 1, 2 * page + 3), k, v)
    check_append(cache, table, i32(5, page, 3 * page - 7), k, v, counts=i32(s, 1, s + 9))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("d,p", [(128, 64), (128, 48), (128, 21), (64, 32), (64, 8), (64, 1), (64, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_append_turned(interleaved, weighted, d, p, dtype):
    g = torch.Generator().manual_seed(p)
    b, h, s, page = 2, 2, 83, 32
    cache, table = random_cache(3, 16, h, page, d), pages_for(4, b, 5)
    k, v = (torch.randn((b, h, s, d), generator=g).to(DT[dtype]).cuda() for _ in range(2))
    angle = torch.rand((b, s, p) if p == 48 else (s, p), generator=g) * 7
    turns = torch.stack([angle.cos(), angle.sin()], -1).cuda()
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(DT[dtype]).cuda() if weighted else None
    check_append(cache, table, i32(0, 40), k, v, turns=turns, weight=w, interleaved=interleaved)


@pytest.mark.parametrize("turned,interleaved", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("d,page,dtype", [(128, 64, "bf16"), (64, 128, "fp32"), (128, 64, "fp16")])
def test_append_many_workgroups(d, page, dtype, turned, interleaved):
    """More than a thousand pages and heads in a call."""
    g = torch.Generator().manual_seed(7)
    b, h, s = 8, 9, 15 * page - 3
    cache, table = random_cache(8, b * 17 + 3, h, page, d), pages_for(9, b, 17)
    k, v = (torch.randn((b, h, s, d), generator=g).to(DT[dtype]).cuda() for _ in range(2))
    angle = torch.rand((s, d // 2 - (3 if interleaved else 8)), generator=g) * 7
    turns = torch.stack([angle.cos(), angle.sin()], -1).cuda() if turned else None
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(DT[dtype]).cuda() if turned else None
    starts = i32(*[i * page // 5 for i in range(b)])
    check_append(cache, table, starts, k, v, counts=i32(*[s - 11 * i for i in range(b)]), turns=turns, weight=w,
                 interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_any_sizes(interleaved, weighted, dtype):
    """Tokens and weights of any size in one page, exact zeros, ties between codes, turns by whole quarters."""
    g = torch.Generator().manual_seed(11)
    s, d, page = 150, 128, 32
    cache, table = FP8KVCache(8, 2, d, page), pages_for(1, 1, 6)
    x = torch.randn((1, 2, s, d), generator=g)
    top = 38 if dtype == "bf16" else 4
    x[0, 0] *= 10.0 ** (torch.rand((s, 1), generator=g) * 2 * top - top)
    x[0, 1, ::3, ::5], x[0, 1, 7] = 0.0, 0.0
    x[0, 1, 64:] = (torch.randint(-31, 32, (s - 64, d), generator=g) * 2.0 ** -3)  # codes and the ties between them
    angle = torch.rand((s, 64), generator=g) * 7
    angle[70:90] = torch.pi / 2 * torch.arange(20)[:, None]
    turns = torch.stack([angle.cos(), angle.sin()], -1)
    turns[70:90] = turns[70:90].round()
    w = None
    if weighted:
        w = torch.randn(d, generator=g) * 10.0 ** (torch.rand(d, generator=g) * top - top / 2)
        w = w.to(DT[dtype]).cuda()
    for n in (64, 24):
        check_append(cache, table, i32(0), x.to(DT[dtype]).cuda(), x.to(DT[dtype]).cuda(), weight=w,
                     turns=turns[:, :n].contiguous().cuda(), interleaved=interleaved)


@pytest.mark.parametrize("d,page", [(128, 64), (64, 16), (128, 128)])
def test_append_one_token_at_a_time(d, page):
    """Sizes that grow and fall: pages whose exponent rises under what they hold."""
    g = torch.Generator().manual_seed(5)
    cache, table = FP8KVCache(12, 2, d, page), pages_for(6, 2, 3)
    for t in range(0, 2 * page + 3, 3 if page > 16 else 1):
        k, v = (torch.randn((2, 2, 1, d), generator=g) * 2.0 ** float(torch.randint(-6, 7, (1,), generator=g)) for _ in range(2))
        check_append(cache, table, i32(t, max(0, t - 5)), k.bfloat16().cuda(), v.bfloat16().cuda())


def test_append_small_halves():
    """fp16's own subnormals, under exponents that keep them."""
    cache, table = FP8KVCache(8, 2, 64, 16), pages_for(1, 1, 4)
    x = torch.randint(-1500, 1500, (1, 2, 40, 64), generator=torch.Generator().manual_seed(1)) * 2.0 ** -24
    check_append(cache, table, i32(0), x.half().cuda(), (x * 2.0 ** -1).half().cuda())


def test_append_far_from_one():
    """A page's values at both ends of the exponents' range, and past them."""
    cache, table = FP8KVCache(12, 1, 128, 16), pages_for(1, 1, 8)
    x = torch.randn((1, 1, 128, 128), generator=torch.Generator().manual_seed(1))
    size = torch.tensor([2.0 ** -36, 2.0 ** -44, 1e-38, 2.0 ** 60, 2.0 ** 71, 2.0 ** 72, 1e30, 1.0]).repeat_interleave(16)
    check_append(cache, table, i32(0), (x * size[:, None]).cuda(), (x * size.flip(0)[:, None]).cuda())
    check_append(cache, table, i32(0), (x * size[:, None]).bfloat16().cuda(), (x * size.flip(0)[:, None]).bfloat16().cuda())


def test_append_special_values():
    cache, table = FP8KVCache(8, 1, 64, 16), pages_for(1, 1, 4)
    x = torch.randn((1, 1, 48, 64), generator=torch.Generator().manual_seed(1))
    x[0, 0, 3, 7], x[0, 0, 20] = float("inf"), 0.0
    x[0, 0, 33, 5], x[0, 0, 34, 5], x[0, 0, 35] = 3e38, -1e-38, 1e25
    v = x.clone()
    v[0, 0, 9, 63], x[0, 0, 11, 1] = float("nan"), float("nan")
    x[0, 0, 16:32], v[0, 0, 16:32] = 0.0, -0.0
    check_append(cache, table, i32(0), x.cuda(), v.cuda())
    k, w = read_kv(cache, table, i32(0), 48, dtype=torch.float32)
    assert torch.isnan(k[0, 0, 9, 0]) and torch.isnan(k[0, 0, 11, 0]) and torch.isfinite(w).all()
    assert torch.isnan(k).sum() == 2 and (k[0, 0, 16:32] == 0).all()
    # a value of the page is the largest, an infinity as large as the scale allows; the other tokens keep theirs
    assert k[0, 0, 3, 7] == k[0, 0, 3, 7].abs() > 2 and (w[0, 0, 0] - v[0, 0, 0].cuda()).abs().max() < 0.2


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_append_special_values_turned(interleaved, dtype):
    """A NaN, an infinity or an overflow on the way makes its token's keys what they are, and leaves the others alone."""
    cache, table = FP8KVCache(8, 2, 64, 32), pages_for(1, 1, 3)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((1, 2, 70, 64), generator=g).to(DT[dtype])
    angle = torch.rand((70, 32), generator=g) * 7
    turns = torch.stack([angle.cos(), angle.sin()], -1).cuda()
    clean = FP8KVCache(8, 2, 64, 32)
    append_kv(clean, table, i32(0), x.cuda(), x.cuda(), table=turns, interleaved=interleaved)
    bad = x.clone()
    bad[0, 0, 3, 7], bad[0, 0, 40, 5], bad[0, 0, 66, 9] = float("nan"), float("inf"), torch.finfo(DT[dtype]).max
    append_kv(cache, table, i32(0), bad.cuda(), x.cuda(), table=turns, interleaved=interleaved)
    k, v = read_kv(cache, table, i32(0), 70, dtype=torch.float32)
    kc, vc = read_kv(clean, table, i32(0), 70, dtype=torch.float32)
    assert torch.equal(v, vc) and torch.equal(k[:, 1], kc[:, 1])
    assert torch.isnan(k[0, 0, 3, 0]) and (torch.isnan(k[0, 0]).any(-1).nonzero()[:, 0].tolist() == [3])
    same = torch.ones(64, dtype=torch.bool)
    same[[3, 40]] = False
    assert torch.equal(k[0, 0, :64][same], kc[0, 0, :64][same]) and k[0, 0, 66].abs().max() > 1e4


def test_append_where_there_is_no_page():
    page, d = 16, 64
    cache, g = random_cache(8, 6, 2, page, d), torch.Generator().manual_seed(2)
    k, v = (torch.randn((4, 2, 40, d), generator=g).bfloat16().cuda() for _ in range(2))
    table = torch.tensor([[0, -1, 1], [6, 2, 2 ** 31 - 1], [-(2 ** 31), 3, 4], [5, -1, -1]], dtype=torch.int32, device="cuda")
    # behind the table's end, before its beginning, and all of a sequence
    check_append(cache, table, i32(3, 30, -20, 2 ** 30), k, v)
    before = raw(cache)
    for kwargs in ({"counts": i32(0, -3, 0, 0)}, {}):
        append_kv(cache, table[:, :0] if not kwargs else table, i32(0, 0, 0, 0), k, v, **kwargs)
    append_kv(cache, table[:0], i32(), k[:0], v[:0])
    append_kv(cache, table, i32(0, 0, 0, 0), k[:, :, :0], v[:, :, :0])
    assert all(np.array_equal(a, b) for x, y in zip(before, raw(cache)) for a, b in zip(x, y))


def test_append_any_strides():
    g = torch.Generator().manual_seed(3)
    base = torch.randn((2, 3, 41, 2 * 64 + 1), generator=g).bfloat16().cuda()
    for view in (base[..., 1:65], base[..., ::2][..., :64], base[..., :64].transpose(0, 1)[:2], base[:1, :, :, :64].expand(2, -1, -1, -1)):
        h = view.shape[1]
        a, b = FP8KVCache(12, h, 64, 16), FP8KVCache(12, h, 64, 16)
        table = pages_for(3, 2, 4, extra=4)
        for cache, x in ((a, view), (b, view.contiguous())):
            append_kv(cache, table, i32(7, 16), x, x)
        assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a.tensors(), b.tensors()))
    wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = table
    c = FP8KVCache(12, h, 64, 16)
    append_kv(c, wide[:, 2:6], i32(7, 16), view, view)  # a view of a table
    assert torch.equal(c.k.view(torch.uint8), b.k.view(torch.uint8))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16)])
def test_read(dtype, d, page):
    cache, table = random_cache(4, 9, 3, page, d), pages_for(5, 2, 4, extra=0)
    table[1, 1] = -1
    pool = ok.Pool(*raw(cache))
    for starts, t, lengths in ((i32(0, 3), 4 * page + 3, None), (i32(page - 1, -2), 11, i32(page + 4, 5)), (i32(1, 1), 0, None)):
        got = read_kv(cache, table, starts, t, lengths=lengths, dtype=DT[dtype])
        ref = ok.read(pool, table.cpu().numpy(), starts.cpu().numpy(), t, None if lengths is None else lengths.cpu().numpy())
        for a, b in zip(got, ref):
            assert a.dtype == DT[dtype] and torch.equal(a.cpu(), torch.from_numpy(b).to(DT[dtype]))


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------

def check_attend(q, cache, table, lengths, causal=False, q_lengths=None, scale=None):
    got = cached_attention(q, cache, table, lengths, causal=causal, q_lengths=q_lengths, scale=scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    pool = ok.Pool(*raw(cache))
    tb, T = table.cpu().numpy(), table.shape[1] * cache.page_size
    k, v = ok.read(pool, tb, np.zeros(len(tb), int), T)
    there = np.repeat((tb >= 0) & (tb < cache.pages), cache.page_size, 1)
    c = q.shape[-1] ** -0.5 if scale is None else scale
    o, a = ok.attend(f64(q), k, v, there, lengths.cpu().numpy(), c, causal,
                     None if q_lengths is None else q_lengths.cpu().numpy())
    name = "bf16" if q.dtype == torch.bfloat16 else "fp16"
    tol = 2.0 ** -10 * a
    err = np.abs(f64(got) - o)
    assert (err <= tol + ob.half_step(np.abs(o) + tol, name)).all(), ((err - tol).max(), np.argwhere(err > tol + ob.half_step(np.abs(o) + tol, name))[:5])
    assert (f64(got)[a.sum(-1) == 0] == 0).all()  # rows that see nothing
    return got


SHAPES = [  # B, H, Hk, S, D, page
    (1, 1, 1, 1, 64, 16), (2, 4, 4, 1, 128, 64), (3, 8, 2, 1, 128, 16), (2, 7, 1, 1, 64, 32), (1, 16, 1, 1, 128, 128),
    (2, 5, 5, 3, 64, 64), (1, 40, 8, 5, 64, 32), (2, 8, 1, 2, 128, 64), (1, 4, 2, 13, 128, 16), (2, 3, 1, 17, 128, 32),
    (1, 2, 2, 64, 64, 16), (1, 2, 2, 65, 128, 64), (1, 6, 2, 100, 128, 16), (2, 1, 1, 129, 64, 128), (1, 2, 1, 150, 64, 32),
    (1, 2, 2, 257, 128, 64),
]


@pytest.mark.parametrize("B,H,Hk,S,D,page", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend(B, H, Hk, S, D, page, causal, dtype):
    g = torch.Generator().manual_seed(S + H)
    width = -(-(S + 70) // page) + 1
    table = pages_for(S, B, width)
    T = width * page
    lengths = torch.tensor([T, S + 33, 1][:B], dtype=torch.int32, device="cuda")
    cache = normal_cache(D + page, B * width + 3, Hk, page, D, table, lengths)
    q = torch.randn((B, S, H, D), generator=g).to(DT[dtype]).cuda().transpose(1, 2)
    got = check_attend(q, cache, table, lengths, causal)
    assert got.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 4), (1, 8, 2), (5, 4, 1), (70, 2, 2), (140, 2, 1)])
@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 300])
def test_attend_lengths(S, H, Hk, length):
    table = pages_for(length, 1, 20)
    cache = normal_cache(length, 23, Hk, 16, 64, table, i32(length))
    q = torch.randn((1, H, S, 64), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    check_attend(q, cache, table, i32(length))
    check_attend(q, cache, table, i32(length), causal=True)


@pytest.mark.parametrize("S,H,Hk,D", [(1, 4, 4, 128), (3, 8, 2, 64), (90, 2, 2, 128), (200, 4, 2, 64)])
def test_attend_ragged(S, H, Hk, D):
    """Queries that are not there, sequences longer than their tables, shorter than nothing, or fewer than the queries."""
    B, page, width = 6, 32, 7
    table = pages_for(9, B, width)
    lengths = i32(100, 224, 3, 0, 10 ** 6, -5)
    cache = normal_cache(2, B * width + 3, Hk, page, D, table, lengths)
    q = torch.randn((B, H, S, D), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    q[1, :, 1:] = float("nan")  # not there
    q_lengths = i32(S, 1, S, S, S + 5, S)
    for causal in (False, True):
        check_attend(torch.nan_to_num(q), cache, table, lengths, causal, q_lengths)
        got = cached_attention(q, cache, table, lengths, causal=causal, q_lengths=q_lengths)
        assert torch.equal(got, cached_attention(torch.nan_to_num(q), cache, table, lengths, causal=causal, q_lengths=q_lengths))
        assert (got[1, :, 1:] == 0).all()
    check_attend(torch.nan_to_num(q), cache, table, lengths, True, i32(0, -1, S, 1, S, S))


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (2, 4, 1), (80, 2, 2)])
def test_attend_missing_pages(S, H, Hk):
    table = pages_for(3, 2, 12)
    cache = normal_cache(3, 27, Hk, 16, 128, table, i32(192, 192))
    table[0, 2:5], table[0, 11], table[1, :] = -1, 27, 2 ** 31 - 1
    q = torch.randn((2, H, S, 128), generator=torch.Generator().manual_seed(3)).half().cuda()
    got = check_attend(q, cache, table, i32(190, 192))
    assert (got[1] == 0).all()
    check_attend(q, cache, table, i32(190, 192), causal=True)


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (6, 4, 1), (130, 2, 2)])
@pytest.mark.parametrize("byte", [0, 255])
def test_attend_missing_pages_beside_a_page_of_nothing(S, H, Hk, byte):
    """Pages that nobody names hold NaN codes under any scale, page 0 among them."""
    table = pages_for(4, 1, 12, extra=0) + 1
    lengths = i32(16 * 11 + 5)
    cache = normal_cache(4, 14, Hk, 16, 64, table, lengths)
    holes = table.clone()
    holes[0, 3:6], holes[0, 9] = -1, 14
    q = torch.randn((1, H, S, 64), generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    want = [check_attend(q, cache, holes, lengths, c) for c in (False, True)]
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[0], t.view(torch.uint8)[13] = 0xFF, 0x7F
    for t in (cache.k_scale, cache.v_scale):
        t[0], t[13] = byte, byte
    for c, w in zip((False, True), want):
        assert torch.equal(cached_attention(q, cache, holes, lengths, causal=c), w)


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (6, 4, 1), (130, 2, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_what_is_not_there_changes_nothing(S, H, Hk, D):
    """NaN codes and any scales behind a sequence's end and in pages that it does not name."""
    table = pages_for(4, 1, 12)
    lengths = i32(16 * 9 + 5)
    cache = normal_cache(4, 15, Hk, 16, D, table, lengths)
    q = torch.randn((1, H, S, D), generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    want = [cached_attention(q, cache, table, lengths, causal=c) for c in (False, True)]
    used = set(table[0, :10].tolist())
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[int(table[0, 9]), :, 5:] = 0x7F
        for p in set(range(15)) - used:
            t.view(torch.uint8)[p] = 0xFF
            cache.k_scale[p], cache.v_scale[p] = 255, 0
    for c, w in zip((False, True), want):
        assert torch.equal(cached_attention(q, cache, table, lengths, causal=c), w)


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (20, 2, 1), (150, 2, 2)])
def test_attend_nan_reaches_those_that_see_it(S, H, Hk):
    """A NaN in one token's value: rows that see the token are NaN, causal rows before it are not."""
    table, n = pages_for(5, 1, 12), 180
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn((1, Hk, n, 64), generator=g).bfloat16().cuda() for _ in range(2))
    at = n - S // 2 - 1
    v[0, 0, at, 3] = float("nan")
    cache = FP8KVCache(15, Hk, 64, 16)
    append_kv(cache, table, i32(0), k, v)
    q = torch.randn((1, H, S, 64), generator=g).bfloat16().cuda()
    bad = torch.isnan(cached_attention(q, cache, table, i32(n), causal=True)).all(-1)
    part = torch.isnan(cached_attention(q, cache, table, i32(n), causal=True)).any(-1)
    sees = (torch.arange(S) + n - S >= at).cuda()
    heads = (torch.arange(H) // (H // Hk) == 0).cuda()
    assert torch.equal(bad[0], sees & heads[:, None]) and torch.equal(bad, part)


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (3, 8, 1), (100, 2, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_any_scales(S, H, Hk, D):
    """Pages, values, queries and scores of very different sizes."""
    table = pages_for(6, 1, 12)
    q = torch.randn((1, H, S, D), generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    cache = random_cache(6, 15, Hk, 16, D, spread=5)
    check_attend(q, cache, table, i32(185), scale=0.3)
    cache.v_scale.copy_(torch.randint(95, 191, cache.v_scale.shape, generator=torch.Generator().manual_seed(7)))
    check_attend(q, cache, table, i32(185), scale=0.01)
    # one page of the largest values, one of the smallest, the others zeros of the lowest exponent
    cache = FP8KVCache.from_tensors(cache.k.view(torch.uint8), torch.zeros_like(cache.v.view(torch.uint8)), cache.k_scale,
                                    torch.full_like(cache.v_scale, 95))
    cache.v_scale[int(table[0, 1])], cache.v_scale[int(table[0, 8])] = 190, 95
    cache.v[int(table[0, 1])], cache.v[int(table[0, 8])] = 448.0, 0.5
    check_attend(q, cache, table, i32(185), scale=0.05)
    cache.v_scale[int(table[0, 1])] = 127
    for size in (2.0 ** -40, 2.0 ** 30):  # queries beyond fp16's range under a scale that brings the scores back
        check_attend((q.float() * size).bfloat16(), cache, table, i32(185), scale=0.1 / size)
    check_attend(torch.zeros_like(q), cache, table, i32(185))
    for scale in (0.0, -0.1, 1e-30):
        check_attend(q, cache, table, i32(185), scale=scale)


@pytest.mark.parametrize("S,H,Hk", [(1, 2, 2), (4, 8, 2), (70, 2, 1)])
def test_attend_scores_that_grow(S, H, Hk):
    """Each page's scores larger than the last's, and the other way round: the running maximum moves at every step."""
    table = pages_for(7, 1, 16)
    k = torch.randn((1, Hk, 256, 64), generator=torch.Generator().manual_seed(8))
    v = torch.randn((1, Hk, 256, 64), generator=torch.Generator().manual_seed(9))
    q = torch.randn((1, H, S, 64), generator=torch.Generator().manual_seed(10)).bfloat16()
    q[..., 0] = 8.0
    for ramp in (torch.linspace(0, 60, 256), torch.linspace(60, 0, 256), 30 * torch.sin(torch.arange(256.0))):
        k[..., 0] = ramp
        cache = FP8KVCache(19, Hk, 64, 16)
        append_kv(cache, table, i32(0), k.cuda(), v.cuda())
        check_attend(q.cuda(), cache, table, i32(256), scale=0.125)


def test_attend_strides():
    table = pages_for(8, 2, 10)
    cache = normal_cache(8, 23, 2, 16, 64, table, i32(150, 160))
    base = torch.randn((2, 4, 90, 2 * 64 + 1), generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    for n in (1, 3, 90):
        for view in (base[:, :, :n, 1:65], base[:, :, :n, ::2][..., :64], base[:1, :, :n, 3:67].expand(2, -1, -1, -1),
                     base[:, :2, :n, :64].repeat_interleave(2, 1)):
            want = cached_attention(view.contiguous(), cache, table, i32(150, 160), causal=True)
            assert torch.equal(cached_attention(view, cache, table, i32(150, 160), causal=True), want)
    wide = torch.full((2, 15), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:12] = table
    assert torch.equal(cached_attention(view, cache, wide[:, 2:12], i32(150, 160), causal=True), want)


def test_attend_empty():
    cache = FP8KVCache(2, 2, 64)
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    q = torch.randn((1, 2, 3, 64), device="cuda").bfloat16()
    assert (cached_attention(q, cache, table[:, :0], i32(5)) == 0).all()
    assert cached_attention(q[:, :, :0], cache, table, i32(5)).shape == (1, 2, 0, 64)
    assert cached_attention(q[:0], cache, table[:0], i32()).shape == (0, 2, 3, 64)
    assert (cached_attention(q, FP8KVCache(0, 2, 64), table, i32(5)) == 0).all()


def reference(q, cache, table, lengths, causal, q_lengths=None):
    """Larger calls in 64 bits on the GPU: (o, sum p |v| / sum p)."""
    B, H, S, D = q.shape
    T = table.shape[1] * cache.page_size
    k, v = (t.double() for t in read_kv(cache, table, torch.zeros_like(lengths), T, dtype=torch.float32))
    o, a = torch.zeros((2, B, H, S, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        n, length = S if q_lengths is None else int(q_lengths[b]), int(lengths[b])
        for h in range(H):
            kk, vv = (t[b, h * cache.heads // H, :length] for t in (k, v))
            x = q[b, h, :n].double() @ kk.t() / math.sqrt(D)
            if causal:
                x = x.masked_fill(torch.arange(length, device="cuda") > length - n + torch.arange(n, device="cuda")[:, None], -math.inf)
            p = torch.softmax(x, -1)
            o[b, h, :n], a[b, h, :n] = p @ vv, p @ vv.abs()
    return o, a


@pytest.mark.parametrize("B,H,Hk,S,D,page,length,causal,dtype", [
    (1, 24, 24, 1, 128, 64, 20281, False, "bf16"),    # one query of a whole clip
    (1, 32, 8, 1, 128, 64, 131072, False, "bf16"),    # a very long cache, split
    (5, 16, 2, 3, 64, 16, 5001, True, "fp16"),
    (9, 8, 8, 1, 128, 128, 1999, True, "bf16"),
    (1, 24, 24, 1560, 128, 64, 4680, False, "bf16"),  # a frame over three
    (2, 8, 2, 777, 64, 32, 2049, True, "fp16"),
    (1, 4, 4, 5000, 128, 64, 513, False, "bf16"),     # a clip over its text
    (1, 2, 1, 3001, 128, 16, 3001, True, "bf16"),     # a prompt
    (1, 1, 1, 300, 128, 64, 50001, False, "bf16"),    # few rows over many keys
])
def test_attend_large(B, H, Hk, S, D, page, length, causal, dtype):
    width = -(-length // page)
    lengths = torch.tensor([length - i * (length // (B + 1)) for i in range(B)], dtype=torch.int32, device="cuda")
    q_lengths = None if B == 1 else torch.tensor([max(1, S - i * 40) for i in range(B)], dtype=torch.int32, device="cuda")
    table = pages_for(length, B, width)
    cache = normal_cache(length, B * width + 3, Hk, page, D, table, lengths, k_std=1.5)
    q = torch.randn((B, S, H, D), generator=torch.Generator().manual_seed(S)).to(DT[dtype]).cuda().transpose(1, 2)
    got = cached_attention(q, cache, table, lengths, causal=causal, q_lengths=q_lengths)
    o, a = reference(q, cache, table, lengths, causal, q_lengths)
    tol = 2.0 ** -10 * a
    tol = tol + (o.abs() + tol) * torch.finfo(q.dtype).eps / 2 + 2.0 ** -25
    assert ((got.double() - o).abs() <= tol).all(), ((got.double() - o).abs() / tol).max()
    assert torch.equal(got, cached_attention(q, cache, table, lengths, causal=causal, q_lengths=q_lengths))


def test_pages_beyond_four_gigabytes():
    """Pages and tensors whose offsets need more than 32 bits."""
    pages, page, h, d = 700_000, 16, 4, 128  # 5.7e9 codes each
    cache = FP8KVCache(pages, h, d, page)
    table = torch.tensor([[pages - 1, 5, pages - 2, pages // 2]], dtype=torch.int32, device="cuda")
    small, low = FP8KVCache(4, h, d, page), torch.arange(4, dtype=torch.int32, device="cuda")[None]
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((1, h, 60, d), generator=g).bfloat16().cuda() for _ in range(2))
    for c, t in ((cache, table), (small, low)):
        append_kv(c, t, i32(2), k, v)
    for a, b in zip(read_kv(cache, table, i32(0), 62), read_kv(small, low, i32(0), 62)):
        assert torch.equal(a, b)
    for s in (1, 90):
        q = torch.randn((1, 8, s, d), generator=g).bfloat16().cuda()
        assert torch.equal(cached_attention(q, cache, table, i32(62)), cached_attention(q, small, low, i32(62)))


# ---------------------------------------------------------------------------------------
# a run of them
# ---------------------------------------------------------------------------------------

H, D, FRAME = 3, 128, 60


class Clip:
    """Frames generated one after another: each is appended at every denoising step at the same place, and attends to
    the clip and itself."""

    def __init__(self, frames=5, page=32):
        self.cache = FP8KVCache(frames * FRAME // page + 3, H, D, page)
        self.table = pages_for(11, 1, frames * FRAME // page + 1, extra=0)
        g = torch.Generator().manual_seed(11)
        self.qw, self.kw = ((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().cuda() for _ in range(2))

    def step(self, x, frame, start, length):
        """x [1, S, 3, H, D]; start, length: device tensors."""
        pos = torch.stack([torch.full((FRAME,), frame), torch.arange(FRAME) // 10, torch.arange(FRAME) % 10], -1)
        table = self.turns[frame] if hasattr(self, "turns") else rotary_table(pos.cuda(), (44, 42, 42))
        q, k, v = (t.transpose(1, 2) for t in x.unbind(2))
        q, _ = rotate_qk(q, None, table, self.qw)
        append_kv(self.cache, self.table, start, k, v, table=table, k_weight=self.kw)
        return cached_attention(q, self.cache, self.table, length), q, table


@torch.no_grad()
def test_a_clip_frame_by_frame():
    clip, g = Clip(), torch.Generator().manual_seed(12)
    pool = ok.Pool(*raw(clip.cache))
    tb = clip.table.cpu().numpy()
    for frame in range(5):
        start, length = i32(frame * FRAME), i32((frame + 1) * FRAME)
        for step in range(2):
            x = torch.randn((1, FRAME, 3, H, D), generator=g).bfloat16().cuda()
            got, q, table = clip.step(x, frame, start, length)
            k, v = (x[:, :, i].transpose(1, 2) for i in (1, 2))
            ok.append(pool, tb, [frame * FRAME], f64(k), f64(v), None, f64(table), f64(clip.kw))
            codes, scales = raw(clip.cache)
            assert (codes[0] != pool.codes[0]).mean() < 1e-4 and np.array_equal(codes[1], pool.codes[1])
            assert all(np.array_equal(s, t) for s, t in zip(scales, pool.scales))
            pool.codes[0] = codes[0]  # (a border's other side, as above)
            kk, vv = ok.read(pool, tb, [0], (frame + 1) * FRAME)
            o, a = ok.attend(f64(q), kk, vv, np.ones((1, kk.shape[2]), bool), [kk.shape[2]], D ** -0.5)
            tol = 2.0 ** -10 * a
            assert (np.abs(f64(got) - o) <= tol + ob.half_step(np.abs(o) + tol, "bf16")).all()


@torch.no_grad()
@pytest.mark.parametrize("S,Hq,Hk", [(FRAME, 3, 3), (1, 12, 3)])
def test_a_captured_step_replays(S, Hq, Hk):
    """One graph for every token or frame: starts and lengths are read on the device.  Eager work in between."""
    cache, eager = FP8KVCache(40, Hk, D, 16), FP8KVCache(40, Hk, D, 16)
    table = pages_for(13, 1, 30)
    g = torch.Generator().manual_seed(13)
    q, k, v = (torch.zeros((1, h, S, D), dtype=torch.bfloat16, device="cuda") for h in (Hq, Hk, Hk))
    start, length = i32(0), i32(S)

    def step():
        append_kv(cache, table, start, k, v)
        o = cached_attention(q, cache, table, length, causal=True)
        start.add_(S)
        length.add_(S)
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    start.zero_(), length.fill_(S)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(6):
        new = [torch.randn(t.shape, generator=g).bfloat16().cuda() for t in (q, k, v)]
        for t, n in zip((q, k, v), new):
            t.copy_(n)
        graph.replay()
        append_kv(eager, table, i32(i * S), new[1], new[2])
        want = cached_attention(new[0], eager, table, i32(i * S + S), causal=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


@torch.no_grad()
def test_two_streams_and_graphs_at_once():
    table = pages_for(14, 1, 200)
    caches = [normal_cache(s, 203, 4, 16, D, table, i32(3100)) for s in (1, 2)]
    qs = [torch.randn((1, 8, s, D), generator=torch.Generator().manual_seed(s)).bfloat16().cuda() for s in (1, 130)]
    lengths = i32(3100)
    want = [[cached_attention(q, c, table, lengths) for q in qs] for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    for _ in range(5):
        got = []
        for c, st in zip(caches, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append([cached_attention(q, c, table, lengths) for q in qs])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs, outs = [], []
    for c in caches:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([cached_attention(q, c, table, lengths) for q in qs])
    for _ in range(4):
        for gr, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        eager = cached_attention(qs[0], caches[0], table, lengths)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0][0])
        assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))


@torch.no_grad()
def test_compiled_step():
    clip, ref = Clip(), Clip()
    x = torch.randn((1, FRAME, 3, H, D), generator=torch.Generator().manual_seed(15)).bfloat16().cuda()
    pos = torch.stack([torch.zeros(FRAME), torch.arange(FRAME) // 10, torch.arange(FRAME) % 10], -1)
    clip.turns = ref.turns = [rotary_table(pos.cuda(), (44, 42, 42))]
    start, length = i32(0), i32(FRAME)
    want = ref.step(x, 0, start, length)[0]

    def f(x, start, length):
        return clip.step(x, 0, start, length)[0]

    compiled = torch.compile(f, backend="eager", fullgraph=True)
    assert torch.equal(compiled(x, start, length), want)
    assert torch.equal(clip.cache.k.view(torch.uint8), ref.cache.k.view(torch.uint8))


def test_dispatcher_checks_and_derivatives():
    cache, table = random_cache(1, 6, 2, 16, 64), pages_for(1, 1, 3)
    k, v = (torch.randn((1, 2, 5, 64), device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((1, 4, 3, 64), device="cuda").bfloat16()
    tests = ("test_faketensor",)  # (test_schema compares inputs by a product, which torch has none of in e4m3)
    torch.library.opcheck(ops.kv_append, (*cache.tensors(), table, i32(3), k, v, None, None, None, 1e-6, True), test_utils=tests)
    torch.library.opcheck(ops.kv_read, (*cache.tensors(), table, i32(3), 7, None, torch.float16), test_utils=tests)
    torch.library.opcheck(ops.kv_attend, (q, *cache.tensors(), table, i32(30), None, False, 0.1), test_utils=tests)
    version = cache.k._version
    append_kv(cache, table, i32(3), k.requires_grad_(), v)
    assert cache.k._version > version  # a write in place, for whoever saved the codes
    out = cached_attention(q.requires_grad_(), cache, table, i32(30))
    with pytest.raises(RuntimeError, match="kv_attend"):
        out.float().sum().backward()


def test_refusals():
    cache, table = FP8KVCache(6, 2, 64, 16), pages_for(1, 1, 3)
    k = torch.zeros((1, 2, 5, 64), device="cuda", dtype=torch.bfloat16)
    q, n = torch.zeros((1, 4, 3, 64), device="cuda", dtype=torch.bfloat16), i32(3)
    turns = torch.zeros((5, 32, 2), device="cuda")

    def append(cache=cache, table=table, starts=n, k=k, v=k, **kw):
        append_kv(cache, table, starts, k, v, **kw)

    for bad in ({"k": k[0]}, {"v": k[:, :, :4]}, {"v": k.float()}, {"k": k.double(), "v": k.double()}, {"k": k[:, :1], "v": k[:, :1]},
                {"k": k[..., :32], "v": k[..., :32]}, {"table": table.long()}, {"table": table[0]}, {"table": table.repeat(2, 1)},
                {"starts": n.long()}, {"starts": i32(1, 2)}, {"starts": n.cpu()}, {"counts": i32(1, 2)}, {"counts": n.float()},
                {"table": table.cpu()}, {"v": k.cpu()}):
        with pytest.raises(ValueError):
            append(**bad)
    for bad in ({"table": turns.double()}, {"table": turns[:4]}, {"table": turns.repeat(1, 2, 1)}, {"table": turns.transpose(0, 1)},
                {"table": turns.cpu()}, {"k_weight": k[0, 0, 0].float()}, {"k_weight": k[0, 0, 0, :32]}):
        with pytest.raises(ValueError):
            append_kv(cache, table, n, k, k, **bad)
    with pytest.raises(RuntimeError, match="eps"):
        append(eps=-1.0)

    def attend(q=q, cache=cache, table=table, lengths=n, **kw):
        return cached_attention(q, cache, table, lengths, **kw)

    for bad in ({"q": q[0]}, {"q": q.float()}, {"q": q[:, :3]}, {"q": q[..., :32]}, {"table": table.long()}, {"table": table.cpu()},
                {"table": table.repeat(2, 1)}, {"lengths": n.long()}, {"lengths": i32(1, 2)}, {"q_lengths": i32(1, 2)},
                {"q_lengths": n.cpu()}):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(RuntimeError, match="scale"):
        attend(scale=float("nan"))
    with pytest.raises(ValueError):
        read_kv(cache, table, n, -1)
    with pytest.raises(ValueError):
        read_kv(cache, table, n, 3, dtype=torch.float64)
    with pytest.raises(ValueError):
        read_kv(cache, table, i32(1, 2), 3)
    bad = FP8KVCache(6, 2, 64, 16)
    bad.k_scale = bad.k_scale[:, :1]
    with pytest.raises(ValueError):
        attend(cache=bad)


# ---------------------------------------------------------------------------------------
# scores of any size, probabilities far below the largest, lengths past the table
# ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (4, 8, 1), (40, 1, 1), (70, 2, 2), (130, 1, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_scores_of_any_size(S, H, Hk, D):
    """Scores up to the largest fp32 number, of either sign.  Keys are one row times 1, 2 or 4: a row's weight is spread
    evenly over those of the largest score."""
    page, n = 16, 300
    table = pages_for(D, 1, 20)
    g = torch.Generator().manual_seed(D)
    factor = 2.0 ** torch.randint(0, 3, (n,), generator=g)
    v = torch.randn((1, Hk, n, D), generator=g).clamp(-4, 4)
    v[..., 0] = 4.0  # (one exponent for all pages: it is added to scores whose last bits are larger)
    for key, query, size in ((3.0, 5.0, 2.0 ** 15), (3.0, 5.0, 2.0 ** 20), (1.0, 7.0, 2.0 ** 25), (3.0, 5.0, 2.0 ** 40), (3.0, 3.0, 2.0 ** 70),
                             (1.0, 1.0, 2.0 ** 110)):
        k = (key * 2.0 ** 20 * factor)[None, None, :, None].expand(1, Hk, n, D)
        cache = FP8KVCache(23, Hk, D, page)
        append_kv(cache, table, i32(0), k.cuda(), v.cuda())
        _, w = read_kv(cache, table, i32(0), n, dtype=torch.float32)
        for sign in (1, -1):
            q = torch.full((1, H, S, D), sign * query * size / 2 ** 20).bfloat16().cuda()
            best = (factor == (4 if sign > 0 else 1)).cuda()
            want = w[:, :, best].double().mean(2).repeat_interleave(H // Hk, 1)[:, :, None]
            tol = 2.0 ** -10 * w[:, :, best].double().abs().mean(2).repeat_interleave(H // Hk, 1)[:, :, None]
            got = cached_attention(q, cache, table, i32(n), scale=0.11).double()
            tol = tol + (want.abs() + tol) * 2.0 ** -8
            assert ((got - want).abs() <= tol).all(), (size, sign, ((got - want).abs() / tol).max())


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (40, 1, 1), (70, 2, 2)])
def test_attend_no_scores(S, H, Hk):
    """A scale of 0, and rows that are large only where all keys are 0: every key weighs the same."""
    table = pages_for(1, 1, 20)
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.float16, torch.bfloat16):
        k, v = (torch.randn((1, Hk, 300, 128), generator=g) for _ in range(2))
        k[:, :, :, :8] = 0.0
        cache = FP8KVCache(23, Hk, 128, 16)
        append_kv(cache, table, i32(0), k.cuda() * 2.0 ** 70, v.cuda())
        _, w = read_kv(cache, table, i32(0), 300, dtype=torch.float32)
        want, a = (t.double().mean(2, keepdim=True).repeat_interleave(H // Hk, 1) for t in (w, w.abs()))
        full = torch.full((1, H, S, 128), torch.finfo(dtype).max, dtype=dtype, device="cuda")
        part = torch.zeros_like(full)
        part[..., :8] = full[..., :8]
        for q, scale in ((full, 0.0), (part, 1.0), (part, -3.0)):
            got = cached_attention(q, cache, table, i32(300), scale=scale).double()
            tol = 2.0 ** -10 * a
            tol = tol + (want.abs() + tol) * torch.finfo(dtype).eps / 2
            assert ((got - want).abs() <= tol).all(), (dtype, scale, ((got - want).abs() / tol).max())


def check_attend_small(q, cache, table, lengths, causal=False, scale=None):
    """As check_attend, with what the oracle says that probabilities below fp16's normal numbers may add."""
    got = cached_attention(q, cache, table, lengths, causal=causal, scale=scale)
    pool = ok.Pool(*raw(cache))
    tb = table.cpu().numpy()
    T, c = tb.shape[1] * cache.page_size, q.shape[-1] ** -0.5 if scale is None else scale
    k, v = ok.read(pool, tb, np.zeros(len(tb), int), T)
    e = np.repeat(pool.scales[1][tb].astype(int) - 127, cache.page_size, 1).transpose(0, 2, 1)  # [B, Hk, T]
    o, a, small = ok.attend_small(f64(q), k, v, e, lengths.cpu().numpy(), c, causal)
    tol = 2.0 ** -10 * a + small
    err = np.abs(f64(got) - o)
    tol = tol + ob.half_step(np.abs(o) + tol, "bf16" if q.dtype == torch.bfloat16 else "fp16")
    assert (err <= tol).all(), ((err / tol).max(), (err / np.abs(o).mean()).max())


@pytest.mark.parametrize("below", [18, 22, 26])
@pytest.mark.parametrize("S,H,Hk,D,n", [(1, 4, 2, 64, 20280), (3, 8, 1, 128, 3001), (33, 1, 1, 64, 9001), (70, 1, 1, 64, 20280),
                                        (66, 2, 2, 128, 4099)])
def test_attend_many_keys_far_below_the_largest(S, H, Hk, D, n, below):
    """Keys with all the weight and values of 0 among thousands that are 2^18 to 2^26 times less likely: the output is
    the sum of these."""
    g = torch.Generator().manual_seed(below)
    table = pages_for(below, 1, -(-n // 64))
    k = torch.randn((1, Hk, n, D), generator=g)
    v = 1 + 0.25 * torch.randn((1, Hk, n, D), generator=g)
    k[..., 0], k[..., ::32, 0], v[..., ::32, :] = 0.0, float(below), 0.0
    q = torch.randn((1, H, S, D), generator=g) * 8 / math.sqrt(D)  # scores of the other channels: 1 in powers of two
    q[..., 0] = 8.0
    cache = FP8KVCache(table.numel() + 3, Hk, D, 64)
    append_kv(cache, table, i32(0), k.cuda(), v.cuda())
    check_attend_small(q.bfloat16().cuda(), cache, table, i32(n), scale=math.log(2) / 8)


@pytest.mark.parametrize("spread", [16, 24])
@pytest.mark.parametrize("S,H,Hk,D", [(1, 4, 2, 64), (5, 8, 1, 128), (40, 1, 1, 64), (70, 2, 2, 64), (130, 1, 1, 128)])
def test_attend_pages_large_in_one_channel(S, H, Hk, D, spread):
    """Every other page has values 2^16 or 2^24 times the rest, in one channel, and zeros in the others."""
    g = torch.Generator().manual_seed(spread)
    n, table = 16 * 40 - 3, pages_for(spread, 1, 40)
    k, v = (torch.randn((1, Hk, n, D), generator=g) for _ in range(2))
    big = torch.arange(n) // 16 % 2 == 1
    v[:, :, big] = 0.0
    v[:, :, big, 5] = 1.5 * 2.0 ** spread
    q = torch.randn((1, H, S, D), generator=g).bfloat16().cuda()
    cache = FP8KVCache(table.numel() + 3, Hk, D, 16)
    append_kv(cache, table, i32(0), k.cuda(), v.cuda())
    check_attend_small(q, cache, table, i32(n))
    check_attend_small(q, cache, table, i32(n), causal=True)


@pytest.mark.parametrize("S,H,Hk", [(1, 4, 2), (12, 2, 1), (80, 2, 2), (150, 1, 1)])
@pytest.mark.parametrize("past", [1, 7, 100])
def test_attend_causal_past_the_table(S, H, Hk, past):
    """Tokens behind the table's last page are dropped, and the other tokens' queries see what they would with more
    entries that name no page."""
    page, width = 16, 12
    length = page * width + past
    table = pages_for(past, 1, width)
    g = torch.Generator().manual_seed(past)
    k, v = (torch.randn((1, Hk, length, 64), generator=g).bfloat16().cuda() for _ in range(2))
    cache = FP8KVCache(width + 3, Hk, 64, page)
    append_kv(cache, table, i32(0), k, v)
    q = torch.randn((1, H, S, 64), generator=g).bfloat16().cuda()
    wide = torch.cat([table, torch.full((1, 8), -1, dtype=torch.int32, device="cuda")], 1)
    check_attend(q, cache, wide, i32(length), causal=True)
    got = check_attend(q, cache, table, i32(length), causal=True)
    # the last query sees all that is there
    want = cached_attention(q[:, :, -1:], cache, table, i32(length))
    assert (got[:, :, -1:] - want).abs().max() <= 2.0 ** -7 * want.abs().max()


# ---------------------------------------------------------------------------------------
# key codes of the keys in 64 bits
# ---------------------------------------------------------------------------------------

def fp32_keys(k, turns, weight, eps, interleaved):
    """The keys [1, H, S, D] in 32 bits."""
    x = k.float().cpu()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float().cpu()
    p, t = turns.shape[-2], turns.cpu()
    a, b = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if interleaved else (slice(0, p), slice(p, 2 * p))
    u, v, y = x[..., a], x[..., b], x.clone()
    y[..., a], y[..., b] = u * t[..., 0] - v * t[..., 1], u * t[..., 1] + v * t[..., 0]
    return f64(y)


def check_codes_of_64_bits(k, turns, weight, interleaved, page, eps, undecided):
    """Codes and scales of k [1, H, S, D] in an empty cache: those of the key in 64 bits, exactly where all of its
    arithmetic is that of the oracle, else but where `undecided` of its size changes the oracle's code.  The key in 32
    bits has another code somewhere, or the inputs would not test this."""
    _, H, S, D = k.shape
    table = pages_for(S, 1, -(-S // page))
    cache = FP8KVCache(table.numel() + 3, H, D, page)
    append_kv(cache, table, i32(0), k, k, table=turns, k_weight=weight, eps=eps, interleaved=interleaved)
    codes, scales = raw(cache)
    key, _ = ob.rotate(f64(k), f64(turns), None if weight is None else f64(weight), eps, interleaved)
    single = fp32_keys(k, turns, weight, eps, interleaved)
    others = 0
    for i, p in enumerate(table[0].tolist()):
        for h in range(H):
            x = key[0, h, i * page: (i + 1) * page]
            e = ok.exponent(np.abs(x).max())
            assert int(scales[0][p, h]) - 127 == e, (i, h)
            got = codes[0][p, h, : len(x)]
            near = [ok.round_codes(x * (1 + d), e) for d in (-undecided, undecided)]
            assert ((got == near[0]) | (got == near[1])).all(), (i, h, np.argwhere((got != near[0]) & (got != near[1]))[:5])
            y = single[0, h, i * page: (i + 1) * page]
            others += int((ok.round_codes(y, ok.exponent(np.abs(y).max())) != got).sum())
    assert others


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("d,p", [(128, 64), (128, 56), (128, 21), (64, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_append_keys_beside_borders(interleaved, weighted, d, p, dtype):
    """Keys 2^-26 of their size above or below a border of two codes, normal and subnormal, or of two scales."""
    g = torch.Generator().manual_seed(d + p)
    h, page, s = 2, 32, 32 * 6 - 5
    rnd = lambda n, *shape: torch.randint(0, n, shape, generator=g)  # noqa: E731
    mids = torch.from_numpy((e4m3_decode(np.arange(126, dtype=np.uint8)).astype(np.float64)
                             + e4m3_decode(np.arange(1, 127, dtype=np.uint8))) / 2)
    c = mids[rnd(126, s, p)]
    c[:: page, 0] = 448.0  # each page's largest, on a scale's border or beside it
    c = c * torch.exp2(torch.tensor([-8.0, 0.0, 5.0])[torch.arange(s) // page % 3])[:, None]
    side = rnd(2, s, p) * 2 - 1
    side[:: page, 0] = rnd(3, len(range(0, s, page))) - 1
    turns = torch.stack([c * (rnd(2, s, p) * 2 - 1), c * side * 2.0 ** -16], -1).float().cuda()
    # one of a pair's two is 1 and the other 2^-10, times cos and 2^-16 of it
    small = rnd(2, p).bool()
    size = torch.ones(d)
    size[slice(0, 2 * p, 2) if interleaved else slice(0, p)] = torch.where(small, 2.0 ** -10, 1.0)
    size[slice(1, 2 * p, 2) if interleaved else slice(p, 2 * p)] = torch.where(small, 1.0, 2.0 ** -10)
    x = (rnd(2, 1, h, s, d) * 2 - 1) * (1.0 if weighted else size)
    weight = size.to(DT[dtype]).cuda() if weighted else None
    check_codes_of_64_bits(x.to(DT[dtype]).cuda(), turns, weight, interleaved, page, 0.0, 0.0)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,weighted", [("bf16", True), ("fp16", True), ("bf16", False), ("fp16", False)])
def test_append_codes_of_many_keys(interleaved, dtype, weighted):
    """Two or three keys of a million are in 32 bits on the other side of a border."""
    g = torch.Generator().manual_seed(21)
    s, h, d = 8192, 4, 128
    k = torch.randn((1, h, s, d), generator=g).to(DT[dtype]).cuda()
    angle = torch.rand((s, d // 2), generator=g) * 7
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(DT[dtype]).cuda() if weighted else None
    check_codes_of_64_bits(k, torch.stack([angle.cos(), angle.sin()], -1).cuda(), w, interleaved, 64, 1e-6, 2.0 ** -45 if weighted else 0.0)


@torch.no_grad()
def test_compiled_step_keeps_its_writes():
    """Through the shape kernels, with the writes in place taken out of the graph and put back after it: later
    steps see them, in the tensors that the cache was made of too."""
    torch._dynamo.reset()
    try:
        clip, ref = Clip(), Clip()
        g = torch.Generator().manual_seed(16)
        pos = torch.stack([torch.zeros(FRAME), torch.arange(FRAME) // 10, torch.arange(FRAME) % 10], -1)
        clip.turns = ref.turns = [rotary_table(pos.cuda(), (44, 42, 42))]
        codes = [t.view(torch.uint8) for t in (clip.cache.k, clip.cache.v)]
        run = torch.compile(lambda x, start, length: clip.step(x, 0, start, length)[0], backend="aot_eager", fullgraph=True)
        for i in range(3):
            x = torch.randn((1, FRAME, 3, H, D), generator=g).bfloat16().cuda()
            start, length = i32(i * FRAME), i32((i + 1) * FRAME)
            assert torch.equal(run(x, start, length), ref.step(x, 0, start, length)[0]), i
            for a, b, c in zip(clip.cache.tensors(), ref.cache.tensors(), codes + [None] * 2):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                assert c is None or c.data_ptr() == a.data_ptr()
    finally:
        torch._dynamo.reset()
