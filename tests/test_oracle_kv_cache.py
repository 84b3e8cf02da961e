"""The 64-bit restatement of the key / value cache against closed forms (no GPU)."""
import numpy as np
import pytest
import torch

from oracle import kv_cache as ok
from oracle.numerics import e4m3_decode


def empty(pages, heads, page, d):
    return ok.Pool([np.zeros((pages, heads, page, d), np.uint8)] * 2, [np.full((pages, heads), 127, np.uint8)] * 2)


@pytest.mark.parametrize("amax,e", [(0.0, -32), (448.0, 0), (448.0001, 1), (224.0, -1), (225.0, 0), (1e-30, -32),
                                    (448 * 2.0 ** -32, -32), (449 * 2.0 ** -32, -31), (1e30, 63)])
def test_exponent(amax, e):
    assert ok.exponent(amax) == e


def test_codes_are_the_nearest_numbers():
    x = np.concatenate([np.linspace(-500, 500, 4001), [2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, np.inf, -np.inf]])
    got = ok.round_codes(x, 0)
    ref = torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(got, ref)
    assert np.array_equal(ok.round_codes(x * 8, 3), got)


def test_a_page_grows_and_shrinks():
    pool, table = empty(3, 1, 16, 64), np.array([[2, 0]])
    ones = np.ones((1, 1, 3, 64))
    ok.append(pool, table, [0], ones, 2 * ones)
    assert pool.scales[0][2, 0] == 127 - 8 and pool.scales[1][2, 0] == 127 - 7
    assert (e4m3_decode(pool.codes[0][2, 0, :3]) == 256).all()
    ok.append(pool, table, [3], 1000 * ones, 0 * ones)  # raises the keys' exponent, and leaves the values'
    assert pool.scales[0][2, 0] == 129 and pool.scales[1][2, 0] == 127 - 7
    assert (e4m3_decode(pool.codes[0][2, 0, :3]) == 0.25).all()
    k, v = ok.read(pool, table, [0], 8, [6])
    assert (k[0, 0, :3] == 1).all() and (k[0, 0, 3:6] == 4 * 256).all() and (k[0, 0, 6:] == 0).all()
    assert (v[0, 0, :3] == 2).all() and (v[0, 0, 3:] == 0).all()
    ok.append(pool, table, [0], ones[:, :, :1], ones[:, :, :1])  # from the first token again
    assert pool.scales[0][2, 0] == 127 - 8
    ok.append(pool, table, [15], ones, ones, counts=[2])  # over the page's end
    assert (ok.read(pool, table, [15], 3)[0][0, 0] == [[1.0], [1.0], [0.0]]).all()


def test_tokens_without_a_page_are_dropped():
    pool = empty(2, 1, 16, 64)
    before = pool.copy()
    x = np.ones((1, 1, 5, 64))
    ok.append(pool, np.array([[-1, 7]]), [14], x, x)
    ok.append(pool, np.array([[0]]), [16], x, x)
    assert all(np.array_equal(a, b) for a, b in zip(pool.codes + pool.scales, before.codes + before.scales))


def test_nan_stays_in_the_key():
    pool, x = empty(1, 1, 16, 64), np.ones((1, 1, 2, 64))
    v = x.copy()
    v[0, 0, 1, 5] = np.nan
    ok.append(pool, np.array([[0]]), [0], x, v)
    k, v = ok.read(pool, np.array([[0]]), [0], 2)
    assert np.isnan(k[0, 0, 1, 0]) and np.isfinite(k[0, 0, 0]).all() and (v[0, 0, :, 5] == [1, 0]).all()


def test_attention_is_the_softmax_of_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((2, h, s, 64), generator=g, dtype=torch.float64) for h, s in ((4, 3), (2, 9), (2, 9)))
    for causal in (False, True):
        mask = torch.ones(3, 9, dtype=torch.bool).tril(6) if causal else None
        ref = torch.nn.functional.scaled_dot_product_attention(
            q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1), attn_mask=mask, scale=0.2)
        o, a = ok.attend(q.numpy(), k.numpy(), v.numpy(), np.ones((2, 9), bool), [9, 9], 0.2, causal)
        assert np.allclose(o, ref.numpy(), atol=1e-12) and (a >= np.abs(o) - 1e-12).all()
    o, _ = ok.attend(q.numpy(), k.numpy(), v.numpy(), np.ones((2, 9), bool), [1, 0], 0.2, True, [3, 2])
    assert (o[0, :, :2] == 0).all() and (o[1] == 0).all() and np.allclose(o[0, :, 2], v[0, :, 0].repeat_interleave(2, 0))
