"""Kernels of Connected4 and WindowAttention that only some sizes take, each at sizes that take it; rules that pick them are
restated here, so that a change of theirs shows."""
import numpy as np
import pytest

from tests import sequence_oracle as oracle
from tests.helpers import rng
from tests.test_gpu_attention_layer import inputs, run_attention

pytestmark = pytest.mark.gpu
F = np.float32


# ---- eight waves that share a tile: heads of 97 to 128 values, and 512 workgroups of 256 rows at least ----
EIGHT = [
    # batch, length, q_heads, kv_heads, dim, capacity, window, sinks, causal
    (64, 70, 8, 8, 128, 420, 0, 0, 1),
    (64, 67, 8, 8, 100, 300, 90, 5, 1),
    (64, 65, 8, 8, 97, 200, 40, 3, 0),
    (32, 300, 8, 8, 128, 300, 0, 0, 1),
    (16, 257, 32, 8, 128, 500, 64, 40, 1),
    (128, 66, 4, 4, 125, 66, 0, 0, 0),
]


def eight_waves(batch, length, q_heads, kv_heads, dim):
    rows = length * (q_heads // kv_heads)
    return rows > 64 and 96 < dim <= 128 and -(-rows // 256) * batch * kv_heads >= 512


@pytest.mark.parametrize("batch,length,q_heads,kv_heads,dim,capacity,window,sinks,causal", EIGHT)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("kind", ["plain", "ragged", "outliers"])
def test_attention_of_eight_waves(gpu, batch, length, q_heads, kv_heads, dim, capacity, window, sinks, causal, offset, kind):
    """Every eighth pair of a sequence and a head, against the definition; tiles that need fp32 among the others."""
    assert eight_waves(batch, length, q_heads, kv_heads, dim)
    q, k, v = inputs(201, batch, length, q_heads, kv_heads, dim, capacity)
    starts, lengths = np.full(batch, capacity - length), np.full(batch, length)
    if kind == "ragged":
        lengths = 1 + rng(202).integers(0, length, batch)
        starts = (rng(203).integers(0, capacity - length + 1, batch)).astype(int)
        lengths[::7], starts[3::11] = 0, -20
    pairs = [(b, (b * 5 + h) % q_heads) for b in range(batch) for h in range(0, q_heads, 8)][::2]
    if kind == "outliers":
        v[::3, :, capacity // 2, :] *= F(1e7)                    # a row of values, a column of values, a column of keys
        v[1::3, :, : capacity // 2, 9] *= F(1e9)
        k[2::3, :, capacity // 3 : capacity // 3 + 40, 7] = F(1e9)
        q[2::3, :, :, 7] = 0
    args = (list(starts), list(lengths), window, sinks, causal, dim ** -0.5)
    y = run_attention(q, k, v, *args, offset=offset)
    oracle.attention_by_heads(y, q, k, v, *args, pairs=pairs)
    for b in range(batch):
        assert (y[b, max(0, lengths[b]):] == -7).all(), "rows that do not count"


def test_attention_of_eight_waves_keeps_what_is_not_finite_in_its_rows(gpu):
    batch, length, heads, dim, capacity = 64, 80, 8, 128, 260
    q, k, v = inputs(204, batch, length, heads, heads, dim, capacity)
    args = ([capacity - length] * batch, [length] * batch, 0, 0, 1, dim ** -0.5)
    clean = run_attention(q, k, v, *args)
    hurt = capacity - 30  # seen by the last 30 queries
    v[5, 2, hurt, 3], v[6, 2, hurt, 4], k[7, 2, hurt, 5] = np.nan, np.inf, np.nan
    y = run_attention(q, k, v, *args)
    assert not np.isfinite(y[5, 50:, 2, 3]).any() and not np.isfinite(y[6, 50:, 2, 4]).any() and not np.isfinite(y[7, 50:, 2]).any()
    keep = np.ones(y.shape, bool)
    keep[5:8, 50:, 2] = False
    near = np.zeros(y.shape, bool)
    near[5:8, :50, 2] = True  # share tiles with what is hurt
    assert (y[keep & ~near] == clean[keep & ~near]).all()
    for b in (5, 6, 7):
        want, bound = oracle.attention_of_head(q[b, :50, 2], k[b, 2], v[b, 2], capacity - length, capacity - 30, 0, 0, 1, dim ** -0.5)
        oracle.assert_within(y[b, :50, 2], want, bound, "rows in front of it")


def test_attention_of_eight_waves_is_the_same_on_every_call(gpu):
    q, k, v = inputs(205, 64, 70, 8, 8, 128, 700)
    args = ([630] * 64, None, 0, 0, 1, 0.09)
    first = run_attention(q, k, v, *args)
    for _ in range(4):
        assert (run_attention(q, k, v, *args) == first).all()
