"""The attention layer's operators by their definitions, in fp64 numpy, with the bound that
each result may be off by: every rounding of an fp32 evaluation counted with half a step of
its operand (2^-24), nothing measured."""
import numpy as np

HALF = 2.0 ** -24  # half a step of fp32, relative


def unpack(codes, n_in):
    """[out][in / 8] words -> [out][in] codes 0..15."""
    words = np.ascontiguousarray(codes).view(np.uint32)
    return ((words[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(words.shape[0], -1)[:, :n_in]


def connected4(x, codes, steps, lows, bias, group):
    """(y, bound): y[r][o] = sum_k x[r][k] (low + step * code) + bias.

    The bound, relative to the sum of |x| (|low| + 15 |step|): two parts of an operand with 11 bits each leave
    2^-22 of it; sums of 32 products, in / 32 of them one after another, and six steps of scaling and joining."""
    x = np.asarray(x, np.float64)
    n_in = x.shape[1]
    of = np.arange(n_in) // group
    step = np.asarray(steps, np.float64)[:, of]
    low = -8.0 * step if lows is None else np.asarray(lows, np.float64)[:, of]
    w = low + step * unpack(codes, n_in)
    y = x @ w.T
    size = np.abs(x) @ (np.abs(low) + 15.0 * np.abs(step)).T
    if bias is not None:
        y = y + np.asarray(bias, np.float64)
        size = size + np.abs(np.asarray(bias, np.float64))
    return y, size * (2.0 ** -22 + (32 + n_in / 32 + 6) * HALF) + 1e-37


def rotary_norm(x, q_heads, kv_heads, rotary, interleaved, normalize, eps, q_scale, k_scale, frequency, starts, lengths):
    """(heads, bound) of all tokens: heads [batch][length][q_heads + 2 kv_heads][dim].

    The bound, relative to |a| + |b| of a pair: the mean of `dim` squares and what is made of it (dim / 2 + 8 half
    steps), an angle whose rest of up to half a turn is an fp32 number (pi * 2^-24), cos and sin to two steps, two
    products and a sum."""
    x = np.asarray(x, np.float64)
    batch, length, heads, dim = x.shape
    turned = q_heads + kv_heads
    y = x.copy()
    bound = np.zeros_like(x)
    body = y[:, :, :turned]
    if normalize:
        body = body / np.sqrt((body ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if q_scale is not None:
            body[:, :, :q_heads] *= np.asarray(q_scale, np.float64)
        if k_scale is not None:
            body[:, :, q_heads:] *= np.asarray(k_scale, np.float64)
    size = np.abs(body)
    half = rotary // 2
    if half:
        pair = np.arange(half)
        a, b = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + half)
        position = np.asarray(starts, np.float64)[:, None] + np.arange(length)
        t = position[:, :, None, None] * np.asarray(frequency, np.float64)
        out, both = body.copy(), size.copy()
        out[..., a] = body[..., a] * np.cos(t) - body[..., b] * np.sin(t)
        out[..., b] = body[..., b] * np.cos(t) + body[..., a] * np.sin(t)
        both[..., a] = both[..., b] = size[..., a] + size[..., b]
        body, size = out, both
    y[:, :, :turned] = body
    bound[:, :, :turned] = size * ((dim / 2 + 8 + np.pi + 8) * HALF) if normalize or half else 0.0
    return y, bound


def reach(p, keys, window, sinks, causal):
    """Boolean [keys]: which keys the query at position p sees."""
    j = np.arange(keys)
    near = np.ones(keys, bool) if window == 0 else (j > p - window if causal else np.abs(p - j) < window)
    seen = near | (j < sinks)
    return seen & (j <= p) if causal else seen


def window_attention(q, k, v, starts, lengths, window, sinks, causal, scale, y0=None):
    """(y, bound); rows of queries that do not count are y0's (0 without), with bound 0.

    A score is off by d = scale * |q| |k| (2^-21 + dim half steps) and three roundings of its own size, which shows in
    the weights as e^(2 d): first order 2 d of the largest visible |v|; the weights themselves are off by an exponential
    (four half steps) and a split into 22 bits, the sum over the keys by 32 + keys / 16 roundings."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    batch, length, q_heads, dim = q.shape
    kv_heads, capacity = k.shape[1], k.shape[2]
    y = np.zeros_like(q) if y0 is None else np.asarray(y0, np.float64).copy()
    bound = np.zeros_like(q)
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), length)
        keys = min(max(int(starts[b]) + n, 0), capacity)
        for t in range(n):
            seen = np.flatnonzero(reach(int(starts[b]) + t, keys, window, sinks, causal))
            for h in range(q_heads):
                g = h // (q_heads // kv_heads)
                if seen.size == 0:
                    y[b, t, h] = 0.0
                    continue
                kk, vv = k[b, g, seen], v[b, g, seen]
                s = scale * (kk @ q[b, t, h])
                w = np.exp(s - s.max())
                w /= w.sum()
                y[b, t, h] = w @ vv
                d = (abs(scale) * (np.abs(kk) @ np.abs(q[b, t, h])) * (2.0 ** -21 + dim * HALF) + np.abs(s) * 3 * HALF).max()
                bound[b, t, h] = np.abs(vv).max() * (2 * d + 2.0 ** -20 + (32 + seen.size / 16) * HALF) + 1e-37
    return y, bound


def assert_within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, "%s: shape %s vs %s" % (what, got.shape, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / np.maximum(bound, 1e-300), 0)), off.shape)
        raise AssertionError("%s: %d of %d outside; worst at %s: got %r want %r, off %.3g, allowed %.3g" % (
            what, bad.sum(), off.size, at, got[at], want[at], off[at], bound[at]))


def attention_of_head(q, k, v, start, keys, window, sinks, causal, scale):
    """(y, bound) of one head of one sequence: q [n][dim] from position `start` on, k and v [at least keys][dim].

    The bound of a value is relative to its own column, and to what the weights leave of it: sum_j w_j |v_j| times the
    same roundings as in window_attention.  So it does not grow with columns, keys or values that the result does not depend on."""
    q, k, v = np.asarray(q, np.float64), np.asarray(k, np.float64)[:keys], np.asarray(v, np.float64)[:keys]
    n, dim = q.shape
    seen = np.zeros((n, keys), bool)
    for t in range(n):
        seen[t] = reach(start + t, keys, window, sinks, causal)
    if not seen.any():
        return np.zeros_like(q), np.zeros_like(q)
    s = scale * (q @ k.T)
    off = abs(scale) * (np.abs(q) @ np.abs(k).T) * (2.0 ** -21 + dim * HALF) + np.abs(s) * 3 * HALF
    d = np.where(seen, off, 0.0).max(1, keepdims=True)
    top = np.where(seen, s, -np.inf).max(1, keepdims=True)
    w = np.where(seen, np.exp(np.minimum(s - np.where(np.isfinite(top), top, 0.0), 0.0)), 0.0)
    w /= np.maximum(w.sum(1, keepdims=True), 1e-300)
    count = seen.sum(1, keepdims=True)
    return w @ v, (w @ np.abs(v)) * (2 * d + 2.0 ** -20 + (32 + count / 16) * HALF) + 1e-37


def attention_by_heads(y, q, k, v, starts, lengths, window, sinks, causal, scale, pairs=None, what="attention"):
    """Holds y against attention_of_head, for all (sequence, query head) or the `pairs` given."""
    batch, length, q_heads, _ = q.shape
    group, capacity = q_heads // k.shape[1], k.shape[2]
    for b, h in pairs or [(b, h) for b in range(batch) for h in range(q_heads)]:
        n = min(max(int(lengths[b]), 0), length)
        keys = min(max(int(starts[b]) + n, 0), capacity)
        want, bound = attention_of_head(q[b, :n, h], k[b, h // group], v[b, h // group], int(starts[b]), keys, window, sinks, causal, scale)
        assert_within(y[b, :n, h], want, bound, "%s, head %d of sequence %d" % (what, h, b))


def whole_connected4(n_in):
    """What the result of `n_in` products of random signs may be off by on the whole, 2-norm over 2-norm: operands of 22 bits,
    and the sums' roundings, which do not line up: twice the square root of their number, the numbers summed being
    up to twice the result's size."""
    return 2.0 ** -22 + 2 * HALF * np.sqrt(32 + n_in / 32 + 6)


def whole_attention(dim, keys):
    """The same for attention on numbers of size 1 and scores of size 1: a score's products and sum, an exponential of four
    half steps, two operands of 22 bits, the sum over the keys."""
    return 2 * 2.0 ** -22 + 4 * HALF + HALF * (np.sqrt(dim) + 2 * np.sqrt(32 + keys / 16))


def assert_close_on_the_whole(got, want, allowed, what=""):
    """2-norm of the error over the result's, for all of it and for every row (the last axis and what is in front of it
    apart), where a row may be off by four times that."""
    got, want = np.asarray(got, np.float64).reshape(-1, np.shape(want)[-1]), np.asarray(want, np.float64).reshape(-1, np.shape(want)[-1])
    off, size = np.linalg.norm(got - want, axis=1), np.linalg.norm(want, axis=1)
    assert np.linalg.norm(off) <= allowed * np.linalg.norm(size), "%s: %.3g on the whole, allowed %.3g" % (
        what, np.linalg.norm(off) / np.linalg.norm(size), allowed)
    worst = np.argmax(off / np.maximum(size, 1e-300))
    assert (off <= 4 * allowed * size).all(), "%s: row %d off by %.3g, allowed %.3g" % (what, worst, off[worst] / size[worst], 4 * allowed)
