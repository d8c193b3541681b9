"""Kernels of Connected4 and WindowAttention that only some sizes take, each at sizes that take it; rules that pick them are
restated here, so that a change of theirs shows."""
import numpy as np
import pytest

import shadow_amd
from shadow_amd import Buffer, check
from tests import sequence_oracle as oracle
from tests.helpers import normal, rng
from tests.test_gpu_attention_graphs import Chain, Graph, streams  # noqa: F401 (a fixture)
from tests.test_gpu_attention_layer import inputs, run_attention, run_connected4, weights

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


# ---- Connected4: two tiles of outputs a workgroup (8192 outputs and more, up to eight rows) ----
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8])
@pytest.mark.parametrize("n_in,n_out,group", [(264, 8192, 32), (1000, 8200, 64), (520, 16384, 128)])
@pytest.mark.parametrize("lows", [False, True])
def test_connected4_of_many_outputs(gpu, rows, n_in, n_out, group, lows):
    assert rows <= 8 and n_out >= 16 * 512
    codes, steps, low = weights(211, n_in, n_out, group, lows)
    x, bias = normal(212, (rows, n_in)), normal(213, n_out)
    y = run_connected4(x, codes, steps, low, bias, group)
    oracle.assert_within(y, *oracle.connected4(x, codes, steps, low, bias, group), "connected4")


# ---- Connected4: tiles ----
def in_tiles(rows, n_in, n_out):
    sets, tiles = -(-rows // 16), -(-rows // 128)
    return rows > 64 and (rows > 4096 or n_in * n_out * (165 * sets - 800 * tiles) > 11000 << 20)


def tile_bytes(rows, n_in):
    """What the two parts of x take of the workspace in tiles of 128 rows, stages of 64 codes, an even number."""
    return -(-rows // 128) * 128 * (-(-n_in // 128) * 128) * 4


@pytest.mark.parametrize("rows,n_in,n_out,group", [(96, 4096, 16400, 64), (97, 8200, 8190, 32), (700, 2048, 2500, 128), (200, 5000, 9000, 32)])
@pytest.mark.parametrize("lows", [False, True])
def test_connected4_in_tiles(gpu, rows, n_in, n_out, group, lows):
    """Fewer than 4096 rows on weights from which on tiles are faster; against the definition at some of the outputs."""
    assert in_tiles(rows, n_in, n_out)
    assert shadow_amd.hip().shdw_hip_connected4_workspace_bytes(rows, n_in, n_out, group) >= tile_bytes(rows, n_in)
    codes, steps, low = weights(221, n_in, n_out, group, lows)
    x = normal(222, (rows, n_in))
    x[3::9] *= np.repeat(np.exp(np.linspace(-25, 25, -(-n_in // group))), group)[:n_in].astype(F)  # groups with powers of their own
    y = run_connected4(x, codes, steps, low, None, group)
    some = np.r_[0:70, n_out // 2:n_out // 2 + 40, n_out - 70:n_out]
    want = oracle.connected4(x, codes[some], steps[some], None if low is None else low[some], None, group)
    oracle.assert_within(y[:, some], *want, "connected4")


class Long(Chain):
    """A pass of more than 4096 tokens: projections in tiles, the second in parts that are joined."""

    def __init__(self, workspace=None):
        super().__init__(2100, hidden=256, q_heads=16, kv_heads=2, dim=64, window=40, workspace=workspace)
        size = self.lib.shdw_hip_connected4_workspace_bytes
        for n_in, n_out, parts in ((256, self.width, 1), (self.inner, 256, 2)):
            assert in_tiles(self.rows, n_in, n_out)
            sums = size(self.rows, n_in, n_out, 64) - tile_bytes(self.rows, n_in)
            assert (sums > parts * self.rows * n_out * 4) == (parts > 1)


def test_replays_of_a_graph_of_tiles(streams):  # noqa: F811
    recorded, eager = Long(), Long()
    graph = Graph(recorded.run, streams[0])
    for turn in range(4):
        for chain in (recorded, eager):
            chain.feed(230 + turn, [0, 30 * turn])
            if turn == 2:  # groups far below their rows' largest values
                x = normal(239, (chain.rows, chain.hidden))
                x[::50, :64] *= F(1e9)
                chain.x.upload(x)
        eager.run(None)
        check(eager.lib.shdw_hip_stream_sync(None))
        graph.replay()
        for got, want in zip(recorded.result(), eager.result()):
            assert (got == want).all(), "replay %d" % turn
    graph.close()


def test_a_graph_of_tiles_and_one_of_a_token_share_a_workspace(streams):  # noqa: F811
    alone = [Long(), Chain(1)]
    shared = Buffer(max(c.need for c in alone))
    chains = [Long(workspace=shared), Chain(1, workspace=shared)]
    graphs = [Graph(c.run, streams[0]) for c in chains]
    for turn in range(3):
        for chain, single, graph in zip(chains, alone, graphs):
            for c in (chain, single):
                c.feed(240 + turn, [100 + turn, 5])
            single.run(None)
            graph.replay()
            for got, want in zip(chain.result(), single.result()):
                assert (got == want).all(), "replay %d" % turn
    for g in graphs:
        g.close()


def test_tiles_on_streams_side_by_side(streams):  # noqa: F811
    pair, single = [Long(), Long()], Long()
    single.feed(250, [7, 50])
    single.run(None)
    want = single.result()
    for c in pair:
        c.feed(250, [7, 50])
    for _ in range(2):
        for c, s in zip(pair, streams):
            c.run(s)
    for c, s in zip(pair, streams):
        check(c.lib.shdw_hip_stream_sync(s))
        for got, w in zip(c.result(), want):
            assert (got == w).all()
