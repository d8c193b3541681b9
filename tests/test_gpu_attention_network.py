"""Connected4, RotaryNorm and WindowAttention as operators of a workspace and of a text
model: an attention layer over caches, a prompt first and then token by token."""
import ctypes

import numpy as np
import pytest

import shadow_amd
from oracle import net as onet
from shadow_amd import ShadowError, Workspace
from tests import sequence_oracle as oracle
from tests.helpers import normal, rng

pytestmark = pytest.mark.gpu
F = np.float32


def op(typ, name, bottom, top, *args):
    return {"type": typ, "name": name, "bottom": list(bottom), "top": list(top), "arg": list(args)}


def arg_i(name, v):
    return (name, "s_i", int(v))


class Layer:
    """x -> 4-bit projection -> norms, rotation, caches -> windowed attention -> 4-bit projection -> + x."""

    def __init__(self, hidden=96, q_heads=6, kv_heads=2, dim=32, capacity=48, window=12, sinks=2, group=32, batch=3, length=16):
        self.q_heads, self.kv_heads, self.dim, self.capacity = q_heads, kv_heads, dim, capacity
        self.window, self.sinks, self.group, self.hidden = window, sinks, group, hidden
        width = (q_heads + 2 * kv_heads) * dim
        self.w_in, self.w_out = self.weights(1, hidden, width), self.weights(2, q_heads * dim, hidden)
        self.bias = normal(3, width, 0.1)
        self.scales = [(1 + normal(s, dim, 0.1)).astype(F) for s in (4, 5)]
        self.frequency = (100.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(F)
        blobs = [("in_codes", "int32", self.w_in[0]), ("in_steps", "float", self.w_in[1]), ("in_bias", "float", self.bias),
                 ("frequency", "float", self.frequency), ("q_scale", "float", self.scales[0]), ("k_scale", "float", self.scales[1]),
                 ("out_codes", "int32", self.w_out[0]), ("out_steps", "float", self.w_out[1]), ("out_lows", "float", self.w_out[2])]
        both = [arg_i("has_starts", 1), arg_i("has_lengths", 1)]
        self.net = {
            "name": "attention", "arg": [("out_blob", "v_s", ["y"])],
            "blob": [(name, kind, list(a.shape)) for name, kind, a in blobs],
            "op": [
                op("Input", "in", [], ["x", "starts", "lengths"], ("x", "v_i", [batch, length, hidden]), ("starts", "v_i", [batch]),
                   ("lengths", "v_i", [batch]), ("starts_type", "s_s", "int32"), ("lengths_type", "s_s", "int32")),
                op("Connected4", "project", ["x", "in_codes", "in_steps", "in_bias"], ["qkv"], arg_i("group", group),
                   arg_i("has_bias", 1)),
                op("RotaryNorm", "heads", ["qkv", "frequency", "q_scale", "k_scale", "starts", "lengths"], ["q", "k", "v"],
                   arg_i("q_heads", q_heads), arg_i("kv_heads", kv_heads), arg_i("head_dim", dim), arg_i("has_scale", 1),
                   arg_i("capacity", capacity), *both),
                op("WindowAttention", "attend", ["q", "k", "v", "starts", "lengths"], ["a"], arg_i("window", window),
                   arg_i("sinks", sinks), *both),
                op("Connected4", "join", ["a", "out_codes", "out_steps", "out_lows"], ["o"], arg_i("group", group),
                   arg_i("axis", 2), arg_i("has_lows", 1)),
                op("Eltwise", "add", ["x", "o"], ["y"], arg_i("operation", 1)),
            ]}
        self.packed = [a.view(F) for _, _, a in blobs]  # the bits of an int32 blob travel as they are

    def weights(self, seed, n_in, n_out):
        groups = -(-n_in // self.group)
        codes = rng(seed).integers(0, 2 ** 32, (n_out, n_in // 8), dtype=np.uint32).view(np.int32)
        steps = (0.02 * np.exp(normal(seed, (n_out, groups), 0.3))).astype(F)
        return codes, steps, (steps * (-7.5 + normal(seed + 9, (n_out, groups)))).astype(F)

    def step(self, nw, x, starts, lengths, caches):
        """One run of the model, every operator held against its definition on what the operator in front of it gave."""
        starts, lengths = np.asarray(starts, np.int32), np.asarray(lengths, np.int32)
        nw.forward({"x": x, "starts": starts.view(F), "lengths": lengths.view(F)}, reshape=True)
        batch, length = x.shape[:2]
        qkv = nw.blob("qkv")
        want, bound = oracle.connected4(x.reshape(-1, self.hidden), *self.w_in[:2], None, self.bias, self.group)
        oracle.assert_within(qkv.reshape(batch * length, -1), want, bound, "projection")
        heads, bound = oracle.rotary_norm(qkv.reshape(batch, length, -1, self.dim), self.q_heads, self.kv_heads, self.dim, 0, 1, 1e-6,
                                          *self.scales, self.frequency, starts, lengths)
        q, k, v, a, o, y = (nw.blob(n) for n in ("q", "k", "v", "a", "o", "y"))
        for b in range(batch):
            n, rows = lengths[b], slice(starts[b], starts[b] + lengths[b])
            oracle.assert_within(q[b, :n], heads[b, :n, :self.q_heads], bound[b, :n, :self.q_heads], "q")
            for got, first, old in ((k, self.q_heads, caches[0]), (v, self.q_heads + self.kv_heads, caches[1])):
                part = slice(first, first + self.kv_heads)
                oracle.assert_within(got[b, :, rows].transpose(1, 0, 2), heads[b, :n, part], bound[b, :n, part] + 1e-37, "cache")
                old[b, :, rows] = got[b, :, rows]
                assert (got[b, :, :starts[b] + n] == old[b, :, :starts[b] + n]).all(), "rows of earlier runs changed"
        want, bound = oracle.window_attention(q, k, v, starts, lengths, self.window, self.sinks, 1, self.dim ** -0.5)
        for b in range(batch):
            n = lengths[b]
            oracle.assert_within(a[b, :n], want[b, :n], bound[b, :n], "attention")
            want_o, bound_o = oracle.connected4(a[b, :n].reshape(n, -1), *self.w_out, None, self.group)
            oracle.assert_within(o[b, :n], want_o, bound_o, "join")
            assert (y[b, :n] == (F(0) + x[b, :n]) + o[b, :n]).all()
        return y


def test_layer_over_caches_prompt_then_tokens(gpu):
    layer = Layer()
    text = onet.write_text(layer.net)
    batch, length = 3, 16
    caches = [np.zeros((batch, layer.kv_heads, layer.capacity, layer.dim), F) for _ in range(2)]
    with shadow_amd.Network(text, layer.packed) as nw:
        lengths = np.array([16, 5, 11], np.int32)
        layer.step(nw, normal(20, (batch, length, layer.hidden)), np.zeros(batch, np.int32), lengths, caches)
        starts = lengths.copy()
        for t in range(6):  # token by token: past the window, to the sinks and what is near
            layer.step(nw, normal(30 + t, (batch, 1, layer.hidden)), starts, np.ones(batch, np.int32), caches)
            starts += 1
        # a sequence that pauses, and a piece of several tokens
        layer.step(nw, normal(50, (batch, 4, layer.hidden)), starts, np.array([4, 1, 2], np.int32), caches)


def test_a_run_gives_the_same_again(gpu):
    layer = Layer()
    with shadow_amd.Network(onet.write_text(layer.net), layer.packed) as nw:
        x = normal(60, (3, 16, layer.hidden))
        zero, full = np.zeros(3, np.int32), np.full(3, 16, np.int32)
        first = layer.step(nw, x, zero, full, [np.zeros((3, 2, 48, 32), F) for _ in range(2)])
        nw.run()
        assert (nw.blob("y") == first).all()


def test_extension_registry(gpu):
    lib = shadow_amd.host()
    buf = ctypes.create_string_buffer(256)
    lib.shdw_host_extension_keys(buf, 256)
    assert buf.value.decode().split("\n") == ["Connected4", "RotaryNorm", "WindowAttention"]


def test_operator_refusals(gpu):
    """The operators' own checks, which come before any launch."""
    codes = np.zeros((8, 4), np.int32)
    with Workspace() as ws:
        ws.set_blob("x", normal(1, (2, 3, 32)))
        ws.set_blob("codes", codes, "int32")
        ws.set_blob("steps", np.ones((8, 1), F))
        ws.set_blob("wrong", np.ones((8, 2), F))
        ws.set_blob("one", np.ones(1, F))
        ws.set_blob("starts", np.zeros(2, np.int32), "int32")
        ws.set_blob("q", normal(2, (2, 3, 4, 8)))
        ws.set_blob("k", normal(3, (2, 2, 5, 8)))
        ws.set_blob("k3", normal(3, (2, 3, 5, 8)))

        def refused(typ, bottoms, tops, args, text):
            with pytest.raises(ShadowError) as e:
                ws.create_op(typ, bottoms, tops, args).run()
            assert text in str(e.value), str(e.value)

        refused("Connected4", ["x", "codes", "steps"], ["y"], {"group": 16}, "group must be")
        refused("Connected4", ["x", "steps", "steps"], ["y"], {"group": 32}, "codes must be an int32 blob")
        refused("Connected4", ["x", "codes", "wrong"], ["y"], {"group": 32}, "steps")
        refused("Connected4", ["x", "codes", "steps"], ["y"], {"group": 32, "has_bias": 1}, "no input for bias")
        refused("Connected4", ["x", "codes", "steps", "one"], ["y"], {"group": 32}, "left over")
        refused("Connected4", ["x", "codes", "steps"], ["x"], {"group": 32}, "")
        refused("RotaryNorm", ["x", "one"], ["a", "b"], {"q_heads": 2, "kv_heads": 1, "head_dim": 8}, "q, k and v")
        refused("RotaryNorm", ["x", "one"], ["a", "b", "c"], {"q_heads": 2, "kv_heads": 1, "head_dim": 8}, "frequency")
        refused("RotaryNorm", ["x", "one"], ["a", "b", "c"], {"q_heads": 3, "kv_heads": 1, "head_dim": 8}, "")
        refused("RotaryNorm", ["x"], ["a", "b", "c"], {"q_heads": 2, "kv_heads": 1, "head_dim": 8, "rotary_dim": 3}, "frequency")
        refused("RotaryNorm", ["x", "steps"], ["a", "b", "c"], {"q_heads": 2, "kv_heads": 1, "head_dim": 8, "rotary_dim": 16}, "")
        refused("RotaryNorm", ["x", "one"], ["a", "b", "c"],
                {"q_heads": 2, "kv_heads": 1, "head_dim": 8, "rotary_dim": 2, "has_lengths": 1}, "no input for lengths")
        refused("WindowAttention", ["q", "k3", "k3"], ["y"], {}, "")
        refused("WindowAttention", ["q", "k", "k3"], ["y"], {}, "")
        refused("WindowAttention", ["q", "k", "k"], ["q"], {}, "")
        refused("WindowAttention", ["q", "k", "k"], ["y"], {"window": -1}, "")
        refused("WindowAttention", ["q", "k", "k", "one"], ["y"], {"has_starts": 1}, "starts must be an int32 blob")
        # and the same calls put right run
        for typ, bottoms, tops, args in (
                ("Connected4", ["x", "codes", "steps"], ["y1"], {"group": 32}),
                ("RotaryNorm", ["x", "one"], ["y2", "y3", "y4"], {"q_heads": 2, "kv_heads": 1, "head_dim": 8, "rotary_dim": 2}),
                ("WindowAttention", ["q", "k", "k", "starts"], ["y5"], {"has_starts": 1})):
            ws.create_op(typ, bottoms, tops, args).run()
        ws.sync()
        assert ws.blob_shape("y1") == [2, 3, 8] and ws.blob_shape("y3") == [2, 1, 3, 8] and ws.blob_shape("y5") == [2, 3, 4, 8]
        want, bound = oracle.window_attention(ws.get_blob("q"), ws.get_blob("k"), ws.get_blob("k"), [0, 0], [3, 3], 0, 0, 1, 8 ** -0.5)
        oracle.assert_within(ws.get_blob("y5"), want, bound, "attention")


def test_operators_refuse_an_output_that_is_an_input(gpu):
    """Every input, not the first alone: what an output's new shape frees would still be read."""
    with Workspace() as ws:
        ws.set_blob("x", normal(1, (2, 3, 32)))
        ws.set_blob("codes", np.zeros((8, 4), np.int32), "int32")
        for name, size in (("steps", 8), ("lows", 8), ("bias", 8), ("frequency", 4), ("q_scale", 8), ("k_scale", 8)):
            ws.set_blob(name, np.ones((8, 1) if size == 8 and name in ("steps", "lows") else size, F))
        for name in ("starts", "lengths"):
            ws.set_blob(name, np.ones(2, np.int32), "int32")
        for name, heads in (("q", 4), ("k", 2), ("v", 2)):
            ws.set_blob(name, normal(2, (2, 3, 4, 8) if name == "q" else (2, heads, 5, 8)))
        both = {"has_starts": 1, "has_lengths": 1}
        connected = ["x", "codes", "steps", "lows", "bias"]
        rotary = ["x", "frequency", "q_scale", "k_scale", "starts", "lengths"]
        attention = ["q", "k", "v", "starts", "lengths"]
        heads = {"q_heads": 2, "kv_heads": 1, "head_dim": 8, "has_scale": 1}
        cases = [("Connected4", connected, [n], {"group": 32, "has_lows": 1, "has_bias": 1}) for n in connected]
        cases += [("RotaryNorm", rotary, [n if i == at else "o%d" % i for i in range(3)], dict(heads, **both))
                  for n in rotary for at in range(3)]
        cases += [("WindowAttention", attention, [n], both) for n in attention]
        for typ, bottoms, tops, args in cases:
            with pytest.raises(ShadowError) as e:
                ws.create_op(typ, bottoms, tops, args).run()
            assert "output" in str(e.value), (typ, tops, str(e.value))
        with pytest.raises(ShadowError) as e:  # 2^32 + 4 heads are not 4
            ws.create_op("RotaryNorm", ["x", "frequency"], ["a", "b", "c"],
                         {"q_heads": 2 ** 31 - 2, "kv_heads": 2 ** 30 + 3, "head_dim": 8, "rotary_dim": 8}).run()
        assert "values of a token" in str(e.value)
