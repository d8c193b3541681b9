"""What the checks of Connected4 and WindowAttention tell apart: operands of 11 bits do not pass where operands of 22 do."""
import numpy as np
import pytest

from tests import sequence_oracle as oracle
from tests.helpers import normal, rng


def half(a):
    """As one fp16 number, the largest of all at 2^13."""
    scale = 2.0 ** (13 - np.floor(np.log2(np.abs(a).max())))
    return (np.asarray(a, np.float64) * scale).astype(np.float16).astype(np.float64) / scale


def halves(a):
    """As two of them."""
    hi = half(a)
    return hi + half(a - hi)


@pytest.mark.parametrize("rows,n_in,group", [(13, 5000, 32), (16, 4096, 64), (128, 4096, 128), (1, 16384, 128)])
def test_connected4_of_half_the_bits_does_not_pass(rows, n_in, group):
    groups = -(-n_in // group)
    codes = rng(1).integers(0, 2 ** 32, (60, n_in // 8), dtype=np.uint32)
    steps = (0.02 * np.exp(0.3 * normal(2, (60, groups)))).astype(np.float32)
    x = normal(3, (rows, n_in))
    want, _ = oracle.connected4(x, codes, steps, None, None, group)
    allowed = oracle.whole_connected4(n_in)
    oracle.assert_close_on_the_whole(oracle.connected4(halves(x), codes, steps, None, None, group)[0], want, allowed)
    with pytest.raises(AssertionError):
        oracle.assert_close_on_the_whole(oracle.connected4(half(x), codes, steps, None, None, group)[0], want, allowed)


@pytest.mark.parametrize("dim,keys", [(64, 4000), (128, 300), (128, 4000), (256, 1000)])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_attention_of_half_the_bits_does_not_pass(dim, keys, which):
    a = {"q": normal(4, (40, dim)), "k": normal(5, (keys, dim)), "v": normal(6, (keys, dim))}
    args = (keys - 40, keys, 0, 0, 1, dim ** -0.5)
    want, _ = oracle.attention_of_head(a["q"], a["k"], a["v"], *args)
    allowed = oracle.whole_attention(dim, keys)
    for cut, passes in ((halves, True), (half, False)):
        b = dict(a, **{which: cut(a[which])})
        got, _ = oracle.attention_of_head(b["q"], b["k"], b["v"], *args)
        if passes:
            oracle.assert_close_on_the_whole(got, want, allowed)
        else:
            with pytest.raises(AssertionError):
                oracle.assert_close_on_the_whole(got, want, allowed)


def test_bounds_by_columns_do_not_grow_with_other_columns():
    """The bound of a column, a row and a key that nothing far off touches is what it is without."""
    q, k, v = normal(7, (5, 32)), normal(8, (50, 32)), normal(9, (50, 32))
    args = (45, 50, 0, 0, 1, 0.2)
    y, bound = oracle.attention_of_head(q, k, v, *args)
    v2 = v.copy()
    v2[:, 3] *= 1e9
    y2, bound2 = oracle.attention_of_head(q, k, v2, *args)
    keep = np.arange(32) != 3
    assert (y[:, keep] == y2[:, keep]).all() and np.allclose(bound[:, keep], bound2[:, keep], rtol=1e-12)
    whole, wide = oracle.window_attention(q[None, :, None], k[None, None], v[None, None], [45], [5], 0, 0, 1, 0.2)
    assert np.allclose(whole[0, :, 0], y, atol=1e-12) and (bound <= wide[0, :, 0] * (1 + 1e-9)).all()
