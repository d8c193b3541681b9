"""Connected4 and WindowAttention on the whole: the 2-norm of the error over the result's, for every kernel.  The bounds of single
elements add up every rounding at its worst, so that at thousands of products they would let fp16 operands pass
(tests/test_attention_accuracy_cpu.py); these do not."""
import numpy as np
import pytest

from tests import sequence_oracle as oracle
from tests.helpers import normal
from tests.test_gpu_attention_layer import inputs, run_attention, run_connected4, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n_in,n_out,group", [
    (1, 4096, 500, 128), (1, 16384, 8200, 64), (3, 4096, 300, 32), (4, 4096, 8200, 64), (8, 5000, 400, 128), (7, 4096, 8192, 32),
    (13, 5000, 4099, 32), (16, 4096, 300, 64), (48, 4096, 4200, 128), (64, 4096, 16384, 64), (700, 4096, 2048, 128), (200, 8192, 5000, 32),
    (4100, 4096, 64, 64)])
@pytest.mark.parametrize("lows", [False, True])
def test_connected4_on_the_whole(gpu, rows, n_in, n_out, group, lows):
    codes, steps, low = weights(301, n_in, n_out, group, lows)
    x = normal(302, (rows, n_in))
    y = run_connected4(x, codes, steps, low, None, group)
    some = np.r_[0:min(n_out, 200), max(0, n_out - 60):n_out]
    want, _ = oracle.connected4(x, codes[some], steps[some], None if low is None else low[some], None, group)
    oracle.assert_close_on_the_whole(y[:, some], want, oracle.whole_connected4(n_in), "connected4")


@pytest.mark.parametrize("batch,length,q_heads,kv_heads,dim,capacity,window,causal", [
    (1, 1, 8, 2, 64, 4000, 0, 1), (2, 1, 8, 2, 128, 3000, 0, 1), (40, 1, 16, 8, 128, 500, 0, 1), (1, 5, 8, 4, 192, 700, 100, 1),
    (1, 3, 4, 1, 256, 900, 0, 1), (2, 60, 2, 2, 100, 600, 0, 1),
    (1, 300, 2, 1, 32, 900, 0, 1), (2, 300, 2, 1, 64, 300, 0, 0), (1, 400, 3, 1, 80, 2000, 512, 1), (1, 500, 4, 1, 128, 1500, 0, 1),
    (64, 70, 8, 8, 128, 300, 0, 1), (1, 200, 2, 1, 160, 800, 0, 1), (1, 200, 2, 1, 192, 800, 64, 1), (1, 300, 2, 1, 256, 1500, 0, 1)])
def test_attention_on_the_whole(gpu, batch, length, q_heads, kv_heads, dim, capacity, window, causal):
    q, k, v = inputs(303, batch, length, q_heads, kv_heads, dim, capacity)
    start, args = capacity - length, (window, 0, causal, dim ** -0.5)
    y = run_attention(q, k, v, [start] * batch, None, *args)
    for b, h in [(b, h) for b in range(0, batch, 9) for h in range(q_heads)]:
        g = h // (q_heads // kv_heads)
        want, _ = oracle.attention_of_head(q[b, :, h], k[b, g], v[b, g], start, capacity, *args)
        keys = window if window and causal else capacity
        oracle.assert_close_on_the_whole(y[b, :, h], want, oracle.whole_attention(dim, keys), "head %d of %d" % (h, b))
