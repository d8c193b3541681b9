"""Connected4, RotaryNorm and WindowAttention on finite inputs far from size 1: largest values that meet weights of zero,
columns and keys of very different sizes, sums that would leave fp32's range on their way."""
import numpy as np
import pytest

from tests import sequence_oracle as oracle
from tests.helpers import normal, rng
from tests.test_gpu_attention_layer import check_rotary_norm, inputs, run_attention, run_connected4, run_rotary_norm, weights

pytestmark = pytest.mark.gpu
F = np.float32


def away(seed, shape):
    """Numbers of either sign, from 0.5 to 1.5 in size."""
    g = rng(seed)
    return ((0.5 + g.random(shape)) * np.where(g.random(shape) < 0.5, -1, 1)).astype(F)


# rows, in, out, group: one row, two to eight, by sixteen, and in tiles (more than 4096 rows)
FORMS = [(1, 4096, 40, 128), (7, 4096, 40, 64), (20, 2048, 48, 32), (4100, 1024, 40, 128), (4100, 1096, 33, 64), (4100, 1096, 33, 32)]


@pytest.mark.parametrize("rows,n_in,n_out,group", FORMS)
@pytest.mark.parametrize("lows", [False, True])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e12, 1e20])
def test_connected4_largest_value_meets_weights_of_zero(gpu, rows, n_in, n_out, group, lows, size):
    """One value of each row is `size` times the others, in a group whose steps and lows are 0: the result does not depend on it."""
    codes, steps, low = weights(81, n_in, n_out, group, lows)
    of = 3
    steps[:, of] = 0
    if lows:
        low[:, of] = 0
    x = normal(82, (rows, n_in))
    x[np.arange(rows), of * group + np.arange(rows) % group] = size
    y = run_connected4(x, codes, steps, low, None, group)
    oracle.assert_within(y, *oracle.connected4(x, codes, steps, low, None, group), "connected4")


@pytest.mark.parametrize("rows,n_in,n_out,group", FORMS)
@pytest.mark.parametrize("lows", [False, True])
def test_connected4_groups_of_very_different_sizes(gpu, rows, n_in, n_out, group, lows):
    """Groups of x from 1e-9 to 1e9 with steps the other way round: every group counts as much as the next."""
    codes, steps, low = weights(83, n_in, n_out, group, lows)
    groups = steps.shape[1]
    sizes = np.exp(np.linspace(-20, 20, groups))[rng(84).permutation(groups)].astype(F)
    steps /= sizes
    if lows:
        low /= sizes
    x = normal(85, (rows, n_in)) * np.repeat(sizes, group)[:n_in]
    bias = normal(86, n_out)
    y = run_connected4(x, codes, steps, low, bias, group)
    oracle.assert_within(y, *oracle.connected4(x, codes, steps, low, bias, group), "connected4")


@pytest.mark.parametrize("rows,n_in,n_out,group", FORMS)
@pytest.mark.parametrize("lows", [False, True])
@pytest.mark.parametrize("size", [3e38, 2e35, 1e-37, 1e-40, 1e-43])
def test_connected4_of_values_at_the_ends_of_the_range(gpu, rows, n_in, n_out, group, lows, size):
    """Sums of code * x and of x may leave fp32's range where x and the result are within it."""
    codes, steps, low = weights(87, n_in, n_out, group, lows)
    scale = F(1e-6) if size > 1 else F(50 * 1e-37 / size)
    steps *= scale
    if lows:
        low *= scale
    x = (np.abs(normal(88, (rows, n_in))).clip(0, 1) * F(size)).astype(F)
    y = run_connected4(x, codes, steps, low, None, group)
    want, bound = oracle.connected4(x, codes, steps, low, None, group)
    assert np.isfinite(y).all()
    # results of 1e-37 are near the least normal number: what is subnormal on the way has steps of 2^-149
    oracle.assert_within(y, want, bound - 1e-37 + n_in * 2.0 ** -148, "connected4")


# batch, length, q_heads, kv_heads: a token, a few rows, tiles
SPANS = [(2, 1, 4, 2), (1, 3, 4, 2), (1, 70, 4, 2), (1, 200, 2, 2)]


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
@pytest.mark.parametrize("dim", [64, 100, 128, 160])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e15])
def test_attention_of_a_column_far_larger_than_the_others(gpu, batch, length, q_heads, kv_heads, dim, size):
    """One column of v is `size` times the others: they do not depend on it."""
    capacity = 300
    q, k, _ = inputs(91, batch, length, q_heads, kv_heads, dim, capacity)
    v = away(92, (batch, kv_heads, capacity, dim))
    v[..., 17] *= F(size)
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, dim ** -0.5)
    oracle.attention_by_heads(run_attention(q, k, v, *args), q, k, v, *args)


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
@pytest.mark.parametrize("dim,size", [(64, 20), (128, 40), (160, 300)])
def test_attention_of_scores_of_thousands(gpu, batch, length, q_heads, kv_heads, dim, size):
    """Rows and keys of 20 to 300 standard deviations: a key takes all the weight, or two share it."""
    capacity = 300
    q, k, _ = inputs(106, batch, length, q_heads, kv_heads, dim, capacity)
    v = away(107, (batch, kv_heads, capacity, dim))
    q, k = q * F(size), k * F(size)
    k[:, :, 1::2] = k[:, :, ::2] + normal(108, k[:, :, ::2].shape, 0.1 / size)
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, dim ** -0.5)
    oracle.attention_by_heads(run_attention(q, k, v, *args), q, k, v, *args)


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
@pytest.mark.parametrize("dim", [64, 128, 160])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e8, 1e9, 1e12])
def test_attention_of_scores_beyond_units(gpu, batch, length, q_heads, kv_heads, dim, size):
    """Scores whose steps are units and more: weights are those of rounded scores, results finite and between the seen values."""
    capacity = 300
    q, k, _ = inputs(109, batch, length, q_heads, kv_heads, dim, capacity)
    v = away(110, (batch, kv_heads, capacity, dim))
    k *= np.exp(np.linspace(0, np.log(size), capacity))[rng(111).permutation(capacity)].astype(F)[:, None]
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, 1.0)
    y = run_attention(q, k, v, *args)
    assert np.isfinite(y).all()
    wide = np.abs(v).max() * (1 + 2.0 ** -18)
    assert (np.abs(y) <= wide).all()
    oracle.attention_by_heads(y, q, k, v, *args)


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
@pytest.mark.parametrize("size", [30, 1e4, 1e7, 1e9, 1e12])
@pytest.mark.parametrize("period", [1, 32, 90])
def test_attention_of_large_values_with_small_weights(gpu, batch, length, q_heads, kv_heads, size, period):
    """Every other `period` keys have values `size` times the others' and weights smaller by as much or more."""
    capacity, dim = 400, 64
    q, k, _ = inputs(95, batch, length, q_heads, kv_heads, dim, capacity)
    v = away(96, (batch, kv_heads, capacity, dim))
    large = np.arange(capacity) // period % 2 == 1
    v[:, :, large] *= F(size)
    q[..., 0], k[..., 0] = 4, 0
    k[:, :, large, 0] = F(-np.log(size) / (4 * 0.125))
    for extra in (0, 4):
        k[:, :, large, 0] -= F(extra)
        args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, 0.125)
        oracle.attention_by_heads(run_attention(q, k, v, *args), q, k, v, *args)


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
@pytest.mark.parametrize("size", [1e2, 1e5, 1e9, 1e18])
@pytest.mark.parametrize("where", ["q", "k", "both"])
def test_attention_of_columns_that_do_not_meet(gpu, batch, length, q_heads, kv_heads, size, where):
    """Columns of q and of k that are `size` times the others meet zeros: scores do not depend on them."""
    capacity, dim = 300, 64
    q, k, _ = inputs(93, batch, length, q_heads, kv_heads, dim, capacity)
    v = away(94, (batch, kv_heads, capacity, dim))
    if where != "k":
        q[..., 5], k[..., 5] = F(size), 0
    if where != "q":
        k[..., 40], q[..., 40] = F(size), 0
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, 0.3)
    oracle.attention_by_heads(run_attention(q, k, v, *args), q, k, v, *args)


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
@pytest.mark.parametrize("size", [1e30, 1e33, 1e35, 1e36])
def test_attention_of_large_finite_values_and_keys(gpu, batch, length, q_heads, kv_heads, size):
    """Some seen values, then some seen keys, near the end of fp32's range; scores and results are within it."""
    capacity, dim = 250, 64
    q, k, _ = inputs(97, batch, length, q_heads, kv_heads, dim, capacity)
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, 0.125)
    v = away(98, (batch, kv_heads, capacity, dim))
    v[:, :, 3::40] *= F(size)
    v[:, :, 100:110] *= F(1e-9)
    y = run_attention(q, k, v, *args)
    assert np.isfinite(y).all()
    oracle.attention_by_heads(y, q, k, v, *args, what="large values")
    v = away(99, (batch, kv_heads, capacity, dim))
    k[:, :, 5::50] *= F(size)
    q *= F(1e-4)
    for scale, what in ((1e-33, "one key or none"), (1e-2, "one key")):
        args = args[:5] + (scale,)
        y = run_attention(q, k, v, *args)
        assert np.isfinite(y).all()
        oracle.attention_by_heads(y, q, k, v, *args, what="large keys, " + what)


@pytest.mark.parametrize("length,capacity", [(1, 64), (3, 64), (1, 700), (3, 3000), (70, 300), (200, 2000)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_attention_of_values_that_are_not_finite_and_weigh_nothing(gpu, length, capacity, bad):
    """A seen value that is not finite shows in its column, however small its weight: also where a wave, or a part of the keys,
    has weights of e^-480 and nothing else."""
    q, k, v = inputs(101, 1, length, 4, 2, 64, capacity)
    q[..., 0], k[..., 0] = 8, 0
    k[:, :, :capacity // 4, 0] = -60
    v[:, :, 5, 3] = bad
    y = run_attention(q, k, v, [capacity - length], [length], 0, 0, 1, 1.0)
    assert not np.isfinite(y[..., 3]).any()


@pytest.mark.parametrize("batch,length,q_heads,kv_heads", SPANS)
def test_attention_of_keys_that_are_not_finite(gpu, batch, length, q_heads, kv_heads):
    """A key that makes a score +inf or NaN leaves its row not finite, one that makes it -inf has weight 0."""
    capacity, dim = 300, 64
    q, k, v = inputs(102, batch, length, q_heads, kv_heads, dim, capacity)
    q[..., 7] = np.where(np.arange(q_heads) % 2, 1, -1) * np.abs(q[..., 7])
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, 0.125)
    gone = ([capacity - length - 1] * batch,) + args[1:]
    for bad, hurt in ((np.inf, 1), (-np.inf, 0)):
        k[:, :, 9, 7] = bad
        y = run_attention(q, k, v, *args)
        for h in range(q_heads):
            if h % 2 == hurt:
                assert not np.isfinite(y[:, :, h]).any()
            else:  # as if the key were not there
                oracle.attention_by_heads(y, q, np.delete(k, 9, 2), np.delete(v, 9, 2), *gone, pairs=[(b, h) for b in range(batch)])
    k[:, :, 9, 7] = np.nan
    assert not np.isfinite(run_attention(q, k, v, *args)).any()


@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, 0), (128, 64, 1), (256, 0, 0), (80, 36, 0), (65, 30, 1)])
@pytest.mark.parametrize("size", [3e38, 1e25, 1e19, 1e-12, 1e-19, 1e-25, 1e-37])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_rotary_norm_of_heads_at_the_ends_of_the_range(gpu, dim, rotary, interleaved, size, eps):
    """Squares may leave fp32's range where the heads and their norms are within it."""
    x = (away(103, (2, 5, 8, dim)) / F(1.5) * F(size)).astype(F)
    x[0, 1], x[1, 2, 3] = normal(104, (8, dim)), 0 if eps else 1
    scale = (1 + normal(105, dim, 0.1)).astype(F)
    frequency = np.linspace(1, 0.01, rotary // 2).astype(F)
    args = (4, 2, rotary, interleaved, 1, eps, scale, scale, frequency, [4, 9], None, 20)
    check_rotary_norm(run_rotary_norm(x, *args), x, *args)
