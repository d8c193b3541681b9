"""Connected4, RotaryNorm and WindowAttention on finite inputs far from size 1: largest values that meet weights of zero,
columns and keys of very different sizes, sums that would leave fp32's range on their way."""
import numpy as np
import pytest

from tests import sequence_oracle as oracle
from tests.helpers import normal, rng
from tests.test_gpu_attention_layer import run_connected4, weights

pytestmark = pytest.mark.gpu
F = np.float32


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
@pytest.mark.parametrize("size", [3e38, 2e35, 1e-37])
def test_connected4_of_values_at_the_ends_of_the_range(gpu, rows, n_in, n_out, group, lows, size):
    """Sums of code * x and of x may leave fp32's range where x and the result are within it."""
    codes, steps, low = weights(87, n_in, n_out, group, lows)
    scale = F(1e-6) if size > 1 else F(50)
    steps *= scale
    if lows:
        low *= scale
    x = (np.abs(normal(88, (rows, n_in))).clip(0, 1) * F(size)).astype(F)
    y = run_connected4(x, codes, steps, low, None, group)
    want, bound = oracle.connected4(x, codes, steps, low, None, group)
    assert np.isfinite(y).all()
    # results of 1e-37 are near the least normal number: what is subnormal on the way has steps of 2^-149
    oracle.assert_within(y, want, bound - 1e-37 + n_in * 2.0 ** -148, "connected4")
