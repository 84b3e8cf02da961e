"""The 64-bit restatements of the DiT block's operators against closed forms (no GPU)."""
import numpy as np
import pytest

from oracle import dit_block as ob


def test_rotary_table_of_one_axis_is_the_textbook_one():
    t = ob.rotary_table(np.arange(5)[:, None], (8,), 10000.0)
    for s in range(5):
        for i in range(4):
            a = s / 10000.0 ** (i / 4)
            assert np.allclose(t[s, i], [np.cos(a), np.sin(a)], atol=1e-15)


def test_rotation_depends_on_relative_positions_only():
    rng = np.random.default_rng(0)
    q, k = rng.standard_normal((2, 1, 1, 1, 24))
    dims = (8, 6, 10)

    def score(pq, pk, interleaved):
        tq, tk = (ob.rotary_table(np.asarray(p, float)[None], dims, 100.0) for p in (pq, pk))
        return (ob.rotate(q, tq, interleaved=interleaved)[0] * ob.rotate(k, tk, interleaved=interleaved)[0]).sum()

    for interleaved in (True, False):
        s0 = score((3, 1, 4), (1, 5, 9), interleaved)
        assert np.isclose(s0, score((13, 21, 4.5), (11, 25, 9.5), interleaved), rtol=1e-12)
        assert not np.isclose(s0, score((3, 1, 4), (2, 5, 9), interleaved), rtol=1e-3)


@pytest.mark.parametrize("value", ob.GRID)
def test_grid_values_are_their_own_codes(value):
    x = np.full((1, 32), 6.0)
    x[0, 1], x[0, 2] = value, -value
    codes, scales = ob.mxfp4_quantize(x)
    assert scales[0, 0, 0] == 127 and (scales[0, 0, 1:] == 127).all()
    assert np.array_equal(ob.mxfp4_values(codes, scales), x)


def test_ties_go_to_the_even_code_and_the_scale_to_the_next_power_at_seven_quarters():
    x = np.zeros((1, 32))
    x[0, :9] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25]
    v = ob.mxfp4_values(*ob.mxfp4_quantize(x))
    assert v[0, :9].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0]
    for top, scale, got in ((6.99, 127, 6.0), (7.0, 128, 8.0), (3.5, 127, 4.0), (3.49, 126, 3.0), (5.01, 127, 6.0)):
        x = np.full((1, 32), 0.0)
        x[0, 31] = top
        codes, scales = ob.mxfp4_quantize(x)
        assert scales[0, 0, 0] == scale and ob.mxfp4_values(codes, scales)[0, 31] == got, top


def test_blocks_with_an_infinity_or_nan_read_as_nan_and_zeros_as_zeros():
    x = np.ones((2, 96))
    x[0, 3], x[0, 40], x[1, 64:] = np.inf, np.nan, 0.0
    codes, scales = ob.mxfp4_quantize(x)
    v = ob.mxfp4_values(codes, scales)
    assert np.isnan(v[0, :64]).all() and (v[0, 64:] == 1).all() and (v[1, 64:] == 0).all()
    assert scales[0, 1, 2] == 0 and scales.shape == (1, 2, 8)


def test_residual_norm_of_a_plain_layer_norm():
    rng = np.random.default_rng(1)
    x, br = rng.standard_normal((2, 2, 6, 40))
    r, y, b_r, b_y = ob.gated_residual_norm(x, br, eps=0.0)
    assert np.allclose(r, x + br) and np.allclose(y.mean(-1), 0) and np.allclose(y.var(-1), 1)
    assert (b_r > 0).all() and (b_y < 1e-3).all()
