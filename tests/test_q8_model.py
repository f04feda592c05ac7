"""OpModel over 8-bit weights against a forward pass written down apart from it:
which weight, which norm and which residual stands where. The checkpoint's norm
weights are all different, so none passes in another's place.

On the CPU OpModel runs on a device of numpy arrays whose operations are the
restatements of test_q8.py and the oracle's, the same ones that the forward pass
calls, so the two are equal bit for bit unless they compute different things.

On the GPU sums are taken in another order, and a value next to the middle of two
integers may become the other one: one more draw of the roundings to 8 bits, at
worst of all of them. So the distance from the model without 8 bits (in f32 and
f64) may be as large as the restatement's own, D, and is held to twice that."""

import numpy as np
import pytest

import titania_b200 as tb
from oracle import oracle as orc
from titania_b200 import synth
from titania_b200.model import Config, rope_table, tensor_names
from test_q8 import F32, bf16, ref_matmul, ref_norm, ref_rows, same

MODEL = dict(synth.TINY, num_hidden_layers=3)


def checkpoint(tied):
    """(config, {name: (bf16 bits, f32 values)}), of magnitudes at which every part counts."""
    spec = dict(MODEL, tie_word_embeddings=tied)
    rng, w = np.random.default_rng(11), {}
    for name, shape, init in synth.tensor_list(spec):
        v = 1 + 0.3 * rng.standard_normal(shape) if init == "ones" else rng.standard_normal(shape)
        if len(shape) == 2 and not name.startswith("model.embed"):
            v = v * shape[1] ** -0.5
        bits, f = bf16(v.reshape(-1))
        w[name] = bits.reshape(shape), f.reshape(shape)
    c = Config(**spec)
    assert set(w) == {n for n, _ in tensor_names(c)}
    return c, w


def rms(x, weight, eps):
    """Oracle's rmsnorm over rows of weight.size."""
    out = np.ascontiguousarray(x, dtype=F32).reshape(-1).copy()
    orc.rmsnorm(out, weight, eps)
    return out.reshape(x.shape)


# ---- the forward pass, apart ---------------------------------------------------------

def forward(c, w, tokens, eight):
    """Logits of every position, [n, vocab]."""
    n, hd, heads, kv = len(tokens), c.head_dim(), c.num_attention_heads, c.num_key_value_heads
    eps, table = c.rms_norm_eps, rope_table(n, hd, c.rope_theta)

    def rows(values):  # activations as the next product reads them
        return ref_rows(values) if eight else values

    def product(name, a):
        if eight:
            return ref_matmul(*ref_rows(w[name][1]), *a)
        return (np.asarray(a, dtype=np.float64) @ w[name][1].astype(np.float64).T).astype(F32)

    def normed(x, name):
        return rows(ref_norm(x, None, w[name][1], eps)[1])

    def roped(x, n_heads):
        x = np.ascontiguousarray(x).reshape(-1).copy()
        orc.rope(x, table, 0, n_heads, hd)
        return x

    x = w["model.embed_tokens.weight"][1][tokens]
    for i in range(c.num_hidden_layers):
        at = f"model.layers.{i}."
        a = normed(x, at + "input_layernorm.weight")
        q, k, v = (product(f"{at}self_attn.{p}_proj.weight", a) for p in "qkv")
        q = roped(rms(q, w[at + "self_attn.q_norm.weight"][0], eps), heads)
        k = roped(rms(k, w[at + "self_attn.k_norm.weight"][0], eps), kv)
        mixed = np.zeros(n * heads * hd, dtype=F32)
        orc.attention(mixed, q, k, np.ascontiguousarray(v).reshape(-1), 0, heads, hd, kv)
        x = (x + product(at + "self_attn.o_proj.weight", rows(mixed.reshape(n, -1)))).astype(F32)
        a = normed(x, at + "post_attention_layernorm.weight")
        gate = np.ascontiguousarray(product(at + "mlp.gate_proj.weight", a)).reshape(-1).copy()
        orc.silu_mul(gate, np.ascontiguousarray(product(at + "mlp.up_proj.weight", a)).reshape(-1))
        x = (x + product(at + "mlp.down_proj.weight", rows(gate.reshape(n, -1)))).astype(F32)
    head = "model.embed_tokens.weight" if c.tie_word_embeddings else "lm_head.weight"
    return product(head, normed(x, "model.norm.weight"))


def log_softmax(logits):
    z = logits.astype(np.float64)
    z -= z.max(axis=1, keepdims=True)
    return z - np.log(np.exp(z).sum(axis=1, keepdims=True))


# ---- a device of numpy arrays -----------------------------------------------------------

class Array:
    def __init__(self, n):
        self.all, self.n = np.zeros(n, dtype=F32), n

    @property
    def v(self):
        return self.all[:self.n]


class Rows8:
    def __init__(self, q, s):
        self.q, self.s, self.n = q, s, len(s)

    @property
    def v(self):
        return self.q[:self.n], self.s[:self.n]


class NumpyDevice:
    """The operations that OpModel(q8=True) calls."""

    def alloc(self, n):
        return Array(n)

    def resize(self, b, n):
        assert n <= b.all.size
        b.n = n

    def read(self, b):
        return b.v.copy()

    def write(self, b, data):
        b.v[:] = data

    def copy(self, dst, to, src, at, n):
        assert to + n <= dst.n and at + n <= src.n
        dst.v[to:to + n] = src.v[at:at + n]

    def embed(self, out, table, tokens):
        out.v[:] = table[1][list(tokens)].reshape(-1)

    def rmsnorm(self, x, weight, eps):
        x.v[:] = rms(x.v, weight[0], eps)

    def rope(self, x, table, pos, n_heads, head_dim):
        orc.rope(x.v, table.v, pos, n_heads, head_dim)

    def attention(self, out, q, k, v, pos, n_heads, head_dim, n_kv_heads):
        orc.attention(out.v, q.v, k.v, v.v, pos, n_heads, head_dim, n_kv_heads)

    def silu_mul(self, gate, up):
        orc.silu_mul(gate.v, up.v)

    def q8(self, rows, cols):
        return Rows8(np.zeros((rows, cols), np.int8), np.zeros(rows, F32))

    def resize_q8(self, q, rows):
        assert rows <= len(q.s)
        q.n = rows

    def quantize_weight(self, w):
        return Rows8(*ref_rows(w[1]))

    def _set(self, out, n):
        out.v[0][:], out.v[1][:] = ref_rows(n)

    def quantize(self, out, x):
        self._set(out, x.v.reshape(out.n, -1))

    def add_rmsnorm_q8(self, out, x, y, weight, eps):
        h, n = ref_norm(x.v.reshape(out.n, -1), None if y is None else y.v.reshape(out.n, -1), weight[1], eps)
        x.v[:] = h.reshape(-1)
        self._set(out, n)

    def matmul_q8(self, out, w, x):
        out.v[:] = ref_matmul(*w.v, *x.v).reshape(-1)


@pytest.mark.parametrize("tied", [True, False])
def test_each_weight_stands_in_its_place(tied):
    """A prompt of more than one batch and two tokens after it: equal bits."""
    c, w = checkpoint(tied)
    tokens = synth.prompt_tokens(72, c.vocab_size, seed=5)
    m = tb.OpModel(c, NumpyDevice(), w, q8=True)
    st, exp = m.state(80), forward(c, w, tokens, True)
    same(m.forward(st, tokens[:70], 0), exp[69])
    same(m.forward(st, tokens[70:71], 70), exp[70])
    same(m.forward(st, tokens[71:], 71), exp[71])


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
def test_distance_from_the_model_without_8_bits(b200, tied):
    c, w = checkpoint(tied)
    tokens = synth.prompt_tokens(72, c.vocab_size, seed=5)
    exact, eight = forward(c, w, tokens, False), forward(c, w, tokens, True)
    d = np.linalg.norm(eight - exact)
    assert d < 0.1 * np.linalg.norm(exact)  # small enough that another model would show
    m = tb.OpModel(c, b200, {k: b200.upload(tb.Tensor(v[0].shape, v[0])) for k, v in w.items()}, q8=True)
    st = m.state(80)
    got = np.stack([m.forward(st, tokens[i:i + 1], i) for i in range(72)])
    assert np.linalg.norm(got - exact) <= 2 * d
    st = m.state(80)
    whole = [m.forward(st, tokens[:70], 0), m.forward(st, tokens[70:], 70)]
    for i, logits in zip((69, 71), whole):
        assert np.linalg.norm(logits - exact[i]) <= 4 * d / 72 ** 0.5  # one row: twice the mean of 72
    given = np.arange(71), tokens[1:]
    lp_exact, lp_eight = log_softmax(exact)[given], log_softmax(eight)[given]
    lp = m.score(m.state(80), tokens, 0)[0]
    assert np.linalg.norm(lp - lp_exact) <= 2 * np.linalg.norm(lp_eight - lp_exact)
