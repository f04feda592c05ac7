"""8-bit rows (tb200_q8: quantize, add_rmsnorm_q8, dequantize, matmul_q8)
against restatements in 64 bits, and OpModel over them.

Every comparison is for equal bits. The integers of a row are defined by
64-bit arithmetic (of which h * w and h^2 are exact), so another order of the
sum of squares moves a value by about 1e-16 of itself: it would have to lie that
near to the middle of two integers, or the scale that near to the middle of two
f32 values, to come out different. A product's integer sum is exact, and what
follows it is two f32 roundings in a fixed order."""

import ctypes

import numpy as np
import pytest

import titania_b200 as tb
from titania_b200 import _lib, synth

F32 = np.float32


# ---- restatements --------------------------------------------------------------------

def bf16(a):
    """f32 values rounded to bf16, as bits and as f32."""
    bits = synth.f32_to_bf16_bits(np.asarray(a, dtype=F32))
    return bits, (bits.astype(np.uint32) << 16).view(F32)


def ref_rows(n):
    """(integers, scales) of rows of f64 values."""
    n = np.asarray(n, dtype=np.float64)
    with np.errstate(all="ignore"):
        scale = (np.abs(n).max(axis=1) / 127.0).astype(F32)  # NaN where a row has one
        scale = np.where(np.isfinite(scale), scale, F32(np.nan))
        step = scale.astype(np.float64)[:, None]
        q = np.clip(np.rint(n / step), -127, 127)
    return np.where(step > 0, q, 0).astype(np.int8), scale


def ref_norm(x, y, w, eps):
    """(x + y in f32, its normalised rows in f64)."""
    h = x if y is None else (x + y).astype(F32)
    with np.errstate(all="ignore"):
        d = h.astype(np.float64)
        r = 1.0 / np.sqrt((d * d).mean(axis=1, keepdims=True) + np.float64(F32(eps)))
        return h, d * w.astype(np.float64) * r


def ref_matmul(wq, ws, xq, xs):
    acc = xq.astype(np.int64) @ wq.astype(np.int64).T
    return acc.astype(F32) * (ws[None, :] * xs[:, None])


def buf(dev, values):
    b = dev.alloc(values.size)
    dev.write(b, values.reshape(-1))
    return b


def rows_of(dev, values, scales):
    q = dev.q8(*values.shape)
    dev.write_q8(q, values, scales)
    return q


def same(a, b):
    """Equal bits, every NaN alike."""
    a, b = np.asarray(a), np.asarray(b)
    assert a.shape == b.shape and a.dtype == b.dtype
    if a.dtype.kind == "f":
        assert np.array_equal(np.isnan(a), np.isnan(b))
        a, b = np.where(np.isnan(a), 0, a), np.where(np.isnan(b), 0, b)
    bad = np.flatnonzero(a.reshape(-1) != b.reshape(-1))
    assert bad.size == 0, (f"{bad.size} of {a.size} differ, first at {np.unravel_index(bad[0], a.shape)}: "
                           f"{a.reshape(-1)[bad[0]]!r} for {b.reshape(-1)[bad[0]]!r}")


# ---- no GPU ----------------------------------------------------------------------------

def test_restatement_of_a_row():
    q, s = ref_rows(np.array([[1.5, -3.0, 381.0, 4.5, 10.5], [0, 0, 0, 0, 0], [1, np.nan, 2, 3, 4],
                              [np.inf, 1, 2, 3, 4]]))
    assert s[0] == 3 and q[0].tolist() == [0, -1, 127, 2, 4]  # 0.5 -> 0, 1.5 -> 2, 3.5 -> 4
    assert s[1] == 0 and not q[1].any()
    assert np.isnan(s[2:]).all() and not q[2:].any()


NULLS = [("tb200_q8_new", (None, 1, 1, None)), ("tb200_q8_resize", (None, None, 1)),
         ("tb200_q8_shape", (None, None, None)), ("tb200_q8_read", (None, None, None, None)),
         ("tb200_q8_write", (None, None, None, None)), ("tb200_q8_data", (None, None, None, None)),
         ("tb200_quantize", (None, None, None)), ("tb200_quantize_weight", (None, None, None)),
         ("tb200_dequantize", (None, None, None)), ("tb200_add_rmsnorm_q8", (None, None, None, None, None, 0.0)),
         ("tb200_matmul_q8", (None, None, None, None))]


@pytest.mark.parametrize("name,args", NULLS, ids=[n for n, _ in NULLS])
def test_null_handles_are_errors(name, args):
    with pytest.raises(tb.DeviceError, match="null") as e:
        _lib.call(name, *args)
    assert e.value.code == _lib.TB200_ERR_ARG
    assert _lib.lib().tb200_q8_free(None, None) == 0
    assert not _lib.lib().tb200_buffer_data(None)


# ---- rows in 8 bits ----------------------------------------------------------------------

SHAPES = [(1, 1), (3, 5), (1, 64), (2, 127), (1, 1024), (61, 1001), (5, 2048), (300, 1024), (700, 96), (64, 2560),
          (1200, 40), (9, 9728), (2, 10240), (3, 16388), (2, 33001), (1, 140000)]


def sample_rows(rows, cols, seed):
    """Rows of different size with a few large channels, one of zeros, and
    one whose values lie in the middle of two integers."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)).astype(F32)
    x *= np.exp(rng.standard_normal((rows, 1)) * 3).astype(F32)
    x[:, rng.integers(0, cols, 1 + cols // 100)] *= F32(20)
    if rows > 1:
        x[rows // 2] = 0
    if rows > 2:
        x[-1] = rng.integers(-127, 128, cols).astype(F32) * F32(3) - F32(1.5)
        x[-1, 0] = 381  # scale 3: everything else is a tie
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(b200, rows, cols):
    x = sample_rows(rows, cols, rows * 7 + cols)
    q = b200.q8(rows, cols)
    b200.quantize(q, buf(b200, x))
    got, exp = b200.read_q8(q), ref_rows(x)
    same(got[1], exp[1])
    same(got[0], exp[0])
    out = b200.alloc(x.size)
    b200.dequantize(out, q)
    same(b200.read(out).reshape(rows, cols), exp[0].astype(F32) * exp[1][:, None])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_weight(b200, rows, cols):
    bits, w = bf16(sample_rows(rows, cols, rows * 11 + cols))
    got, exp = b200.read_q8(b200.quantize_weight(b200.upload(tb.Tensor([rows, cols], bits)))), ref_rows(w)
    same(got[1], exp[1])
    same(got[0], exp[0])


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_add_rmsnorm_q8(b200, rows, cols, residual):
    x = sample_rows(rows, cols, rows * 13 + cols)
    rng = np.random.default_rng(cols)
    y = rng.standard_normal((rows, cols)).astype(F32) if residual else None
    bits, w = bf16(1 + 0.3 * rng.standard_normal(cols))
    xb, q = buf(b200, x), b200.q8(rows, cols)
    yb = buf(b200, y) if residual else None
    b200.add_rmsnorm_q8(q, xb, yb, b200.upload(tb.Tensor([cols], bits)), 1e-6)
    h, n = ref_norm(x, y, w, 1e-6)
    same(b200.read(xb).reshape(rows, cols), h)
    got, exp = b200.read_q8(q), ref_rows(n)
    same(got[1], exp[1])
    same(got[0], exp[0])
    if residual:
        same(b200.read(yb).reshape(rows, cols), y)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [7, 64, 1024, 2560, 20000])
def test_rows_that_are_not_ordinary(b200, cols):
    """NaN, infinities, the largest and the smallest numbers, a zero norm
    weight; eps of zero on a row of zeros is 0 / 0."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((12, cols)).astype(F32)
    x[0, 3], x[1, cols - 1], x[2, 0], x[2, 1] = np.nan, np.inf, np.inf, -np.inf
    x[3] *= F32(1e38)
    x[4] *= F32(1e-38)
    x[5] = F32(1e-45)
    x[6] = 0
    x[7], x[7, 2] = 0, F32(3.4e38)
    x[8], x[8, 5] = 0, F32(-1e-45)
    x[9] = F32(-0.0)
    q = b200.q8(*x.shape)
    b200.quantize(q, buf(b200, x))
    for got, exp in zip(b200.read_q8(q), ref_rows(x)):
        same(got, exp)
    bits, w = bf16(rng.standard_normal(cols))
    bits[1], w[1] = 0, 0
    for eps in (1e-6, 0.0):
        for add in (None, np.zeros_like(x)):
            b200.add_rmsnorm_q8(q, buf(b200, x), None if add is None else buf(b200, add),
                                b200.upload(tb.Tensor([cols], bits)), eps)
            for got, exp in zip(b200.read_q8(q), ref_rows(ref_norm(x, add, w, eps)[1])):
                same(got, exp)


@pytest.mark.gpu
def test_resized_rows(b200):
    """Fewer rows than a handle was made for: the rows behind them stay."""
    x = sample_rows(6, 200, 3)
    q = b200.q8(6, 200)
    b200.quantize(q, buf(b200, x))
    before = b200.read_q8(q)
    b200.resize_q8(q, 2)
    assert q.shape == (2, 200)
    y = sample_rows(2, 200, 4)
    b200.quantize(q, buf(b200, y))
    b200.resize_q8(q, 6)
    got = b200.read_q8(q)
    for g, b, e in zip(got, before, ref_rows(y)):
        same(g[:2], e)
        same(g[2:], b[2:])
    with pytest.raises(tb.DeviceError, match="can't hold"):
        b200.resize_q8(q, 7)


# ---- products ---------------------------------------------------------------------------

PRODUCTS = [
    # tokens, channels, columns
    (3, 17000, 2600), (4, 40001, 1100), (1, 1, 1), (1, 5, 16), (1, 4096, 1024), (1, 33, 1001), (1, 1000, 10240),
    (2, 128, 128), (3, 257, 96), (4, 9, 2560),
    (5, 300, 130), (7, 131, 777), (8, 1024, 512), (9, 640, 2560), (15, 40, 3000), (16, 128, 64), (17, 129, 1001),
    (31, 1000, 31), (33, 77, 4100), (48, 4096, 1024), (63, 2560, 96), (64, 640, 2560), (65, 130, 200), (100, 1, 100),
    (128, 1024, 1024), (129, 513, 640), (200, 2560, 257), (256, 256, 9728), (300, 1200, 1100), (511, 1023, 511),
    (513, 3001, 160), (1025, 260, 384), (2050, 130, 48),
    # few tokens on both sides of the change to tensor cores
    (5, 9001, 300), (6, 2000, 1001), (6, 9000, 64), (7, 8999, 33), (8, 9002, 272), (5, 27001, 1000), (6, 1500, 15000),
    (7, 10001, 1930), (8, 17009, 1001), (8, 1000, 20000), (1, 1001, 3001), (4, 600, 129),
    # a long K over few channels, cut over the CTAs of a cluster
    (64, 2560, 9728), (20, 1001, 5000), (130, 300, 4000), (8, 100, 20000), (5, 16, 1025), (128, 2000, 2048),
    # pairs of CTAs: a second CTA with no tokens, with some, odd channels
    (1100, 515, 2100), (1025, 260, 2048), (1290, 64, 2500), (1999, 1000, 2176),
]


def product_inputs(tokens, channels, cols, seed):
    rng = np.random.default_rng(seed)
    v = [rng.integers(-127, 128, (n, cols)).astype(np.int8) for n in (channels, tokens)]
    s = [np.exp(rng.standard_normal(n)).astype(F32) for n in (channels, tokens)]
    return v[0], s[0], v[1], s[1]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,channels,cols", PRODUCTS)
def test_matmul_q8(b200, tokens, channels, cols):
    wq, ws, xq, xs = product_inputs(tokens, channels, cols, tokens + 3 * channels + 5 * cols)
    out = buf(b200, np.full(tokens * channels + 64, 7, dtype=F32))  # 64 values behind the output
    b200.resize(out, tokens * channels)
    b200.matmul_q8(out, rows_of(b200, wq, ws), rows_of(b200, xq, xs))
    exp = ref_matmul(wq, ws, xq, xs)
    same(b200.read(out).reshape(tokens, channels), exp)
    b200.resize(out, tokens * channels + 64)
    assert np.all(b200.read(out)[tokens * channels:] == 7)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3, 20, 70])
def test_matmul_q8_largest_sums(b200, tokens):
    """131071 columns of -128 sum to 2^31 - 16384; alternating signs to 0."""
    cols = 131071
    xq = np.full((tokens, cols), -128, dtype=np.int8)
    wq = np.full((3, cols), -128, dtype=np.int8)
    wq[1], wq[2, ::2] = 127, 127
    s = np.array([1.0, 0.5, 3.0], dtype=F32)
    out = b200.alloc(3 * tokens)
    b200.matmul_q8(out, rows_of(b200, wq, s), rows_of(b200, xq, np.ones(tokens, dtype=F32)))
    same(b200.read(out).reshape(tokens, 3), ref_matmul(wq, s, xq, np.ones(tokens, dtype=F32)))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 6, 40, 300])
def test_matmul_q8_scales(b200, tokens):
    """Scales of zero, NaN and infinity, and a product of scales below f32's
    smallest number; tokens of which fewer are used than the handle holds."""
    wq, ws, xq, xs = product_inputs(tokens + 5, 200, 320, tokens)
    ws[:4] = [0, np.nan, np.inf, 1e-30]
    xs[:1] = F32(1e-30)
    xs[tokens - 1] = np.nan if tokens > 1 else xs[tokens - 1]
    x = rows_of(b200, xq, xs)
    b200.resize_q8(x, tokens)
    out = b200.alloc(200 * tokens)
    b200.matmul_q8(out, rows_of(b200, wq, ws), x)
    with np.errstate(all="ignore"):
        same(b200.read(out).reshape(tokens, 200), ref_matmul(wq, ws, xq[:tokens], xs[:tokens]))


@pytest.mark.gpu
def test_product_of_rows_with_themselves(b200):
    wq, ws, _, _ = product_inputs(1, 150, 260, 1)
    q, out = rows_of(b200, wq, ws), b200.alloc(150 * 150)
    b200.matmul_q8(out, q, q)
    same(b200.read(out).reshape(150, 150), ref_matmul(wq, ws, wq, ws))


@pytest.mark.gpu
def test_products_past_32_bit_offsets(b200):
    """Output offsets past 2^31 elements: 18000 tokens by 120001 channels."""
    tokens, channels, cols = 18000, 120001, 32
    wq, ws, xq, xs = product_inputs(tokens, channels, cols, 9)
    out = b200.alloc(tokens * channels)
    b200.matmul_q8(out, rows_of(b200, wq, ws), rows_of(b200, xq, xs))
    part = b200.alloc(channels)
    for t in (0, 9000, 17895, 17999):
        b200.copy(part, 0, out, t * channels, channels)
        same(b200.read(part)[None], ref_matmul(wq, ws, xq[t:t + 1], xs[t:t + 1]))


# ---- refusals and empty calls -------------------------------------------------------------

@pytest.mark.gpu
def test_refusals(b200):
    q, x, w = b200.q8(4, 64), b200.alloc(4 * 64), b200.upload(tb.Tensor([64], np.zeros(64, np.uint16)))
    with pytest.raises(tb.DeviceError, match="columns"):
        b200.q8(1, 0)
    with pytest.raises(tb.DeviceError, match="columns"):
        b200.q8(0, 2 ** 30 + 1)
    with pytest.raises(tb.DeviceError, match="rows"):
        b200.q8(2 ** 30 + 1, 1)
    with pytest.raises(tb.DeviceError, match="expected 256"):
        b200.quantize(q, b200.alloc(255))
    with pytest.raises(tb.DeviceError, match="expected 256"):
        b200.dequantize(b200.alloc(257), q)
    with pytest.raises(tb.DeviceError, match="x holds"):
        b200.add_rmsnorm_q8(q, b200.alloc(3 * 64), None, w, 1e-6)
    with pytest.raises(tb.DeviceError, match="y holds"):
        b200.add_rmsnorm_q8(q, x, b200.alloc(3 * 64), w, 1e-6)
    with pytest.raises(tb.DeviceError, match="same buffer"):
        b200.add_rmsnorm_q8(q, x, x, w, 1e-6)
    with pytest.raises(tb.DeviceError, match="weight holds"):
        b200.add_rmsnorm_q8(q, x, None, b200.upload(tb.Tensor([63], np.zeros(63, np.uint16))), 1e-6)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(tb.DeviceError, match="eps"):
            b200.add_rmsnorm_q8(q, x, None, w, eps)
    with pytest.raises(tb.DeviceError, match="not a matrix"):
        b200.quantize_weight(w)
    with pytest.raises(tb.DeviceError, match="weight has 65 columns, input 64"):
        b200.matmul_q8(b200.alloc(8), b200.q8(2, 65), q)
    with pytest.raises(tb.DeviceError, match="output holds"):
        b200.matmul_q8(b200.alloc(9), b200.q8(2, 64), q)
    with pytest.raises(tb.DeviceError, match="131071"):
        b200.matmul_q8(b200.alloc(1), b200.q8(1, 131072), b200.q8(1, 131072))
    with pytest.raises(ValueError, match="int32"):
        b200.write_q8(q, np.zeros((4, 64), np.int32), np.zeros(4, F32))
    with pytest.raises(ValueError, match="shape"):
        b200.write_q8(q, np.zeros((4, 63), np.int8), np.zeros(4, F32))
    b200.sync()


@pytest.mark.gpu
def test_calls_with_no_rows(b200):
    q, e, w = b200.q8(0, 64), b200.alloc(0), b200.upload(tb.Tensor([64], np.zeros(64, np.uint16)))
    b200.quantize(q, e)
    b200.dequantize(e, q)
    b200.add_rmsnorm_q8(q, e, b200.alloc(0), w, 1e-6)
    b200.matmul_q8(e, b200.q8(5, 64), q)
    b200.matmul_q8(e, q, b200.q8(5, 64))
    assert [a.shape for a in b200.read_q8(q)] == [(0, 64), (0,)]
    b200.write_q8(q, np.zeros((0, 64), np.int8), np.zeros(0, F32))
    assert b200.quantize_weight(b200.upload(tb.Tensor([0, 64], np.zeros(0, np.uint16)))).shape == (0, 64)


@pytest.mark.gpu
def test_operands_of_another_device(b200):
    """Refused before anything is launched; here another device is another handle of the same GPU."""
    other = tb.B200(0)
    bits = np.full((4, 64), 0x3F80, np.uint16)
    q, x, w = b200.q8(4, 64), b200.alloc(256), b200.upload(tb.Tensor([64], bits[0]))
    m = b200.upload(tb.Tensor([4, 64], bits))
    q2, x2, w2, out = other.q8(4, 64), other.alloc(256), other.upload(tb.Tensor([64], bits[0])), b200.alloc(16)
    for call in (lambda: b200.quantize(q2, x), lambda: b200.quantize(q, x2), lambda: b200.dequantize(x2, q),
                 lambda: b200.dequantize(x, q2), lambda: b200.add_rmsnorm_q8(q2, x, None, w, 1e-6),
                 lambda: b200.add_rmsnorm_q8(q, x2, None, w, 1e-6), lambda: b200.add_rmsnorm_q8(q, x, x2, w, 1e-6),
                 lambda: b200.add_rmsnorm_q8(q, x, None, w2, 1e-6), lambda: b200.matmul_q8(out, q2, q),
                 lambda: b200.matmul_q8(out, q, q2), lambda: b200.matmul_q8(x2, q, q), lambda: other.quantize_weight(m),
                 lambda: b200.read_q8(q2), lambda: b200.resize_q8(q2, 2),
                 lambda: b200.write_q8(q2, np.zeros((4, 64), np.int8), np.zeros(4, F32)),
                 lambda: tb.LogProbs(b200, 4, 64).score(x2, [0])):
        with pytest.raises(tb.DeviceError, match="another device"):
            call()
    other.sync()
    b200.sync()


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(b200):
    """2.2 M rows of 2048: 4.5 G values and 8-bit integers, products of up to 2.3 G values."""
    torch = pytest.importorskip("torch")
    rows, cols = 2200003, 2048
    at = [0, 1048577, 2097153, rows - 1]
    v = sample_rows(4, cols, 91)
    x, q = b200.alloc(rows * cols), b200.q8(rows, cols)
    for i, r in enumerate(at):
        b200.copy(x, r * cols, buf(b200, v[i]), 0, cols)

    def rows_at(q):
        b200.sync()
        return (torch.as_tensor(q.values, device="cuda")[at].cpu().numpy(),
                torch.as_tensor(q.scales, device="cuda")[at].cpu().numpy())

    b200.quantize(q, x)
    for got, exp in zip(rows_at(q), ref_rows(v)):
        same(got, exp)
    wq, ws = rows_at(q)
    b200.dequantize(x, q)
    b200.sync()
    same(torch.as_tensor(x, device="cuda").view(rows, cols)[at].cpu().numpy(), wq.astype(F32) * ws[:, None])
    for i, r in enumerate(at):
        b200.copy(x, r * cols, buf(b200, v[i]), 0, cols)
    bits, w = bf16(np.random.default_rng(5).standard_normal(cols).astype(F32))
    b200.add_rmsnorm_q8(q, x, None, b200.upload(tb.Tensor([cols], bits)), 1e-6)
    for got, exp in zip(rows_at(q), ref_rows(ref_norm(v, None, w, 1e-6)[1])):
        same(got, exp)
    del x

    wq, ws = rows_at(q)
    out = b200.alloc(1030 * rows)
    for tokens in (3, 20, 1000, 1030):
        _, _, xq, xs = product_inputs(tokens, 1, cols, tokens)
        b200.resize(out, tokens * rows)
        b200.matmul_q8(out, q, rows_of(b200, xq, xs))
        b200.sync()
        got = torch.as_tensor(out, device="cuda").view(tokens, rows)[:, at].cpu().numpy()
        same(got, ref_matmul(wq, ws, xq, xs))


# ---- with torch, and captured --------------------------------------------------------------

@pytest.mark.gpu
def test_device_arrays_share_memory_with_torch(b200):
    torch = pytest.importorskip("torch")
    wq, ws, xq, xs = product_inputs(5, 70, 33, 2)
    w, x = b200.q8(70, 33), b200.q8(5, 33)
    b200.sync()
    for q, v, s in ((w, wq, ws), (x, xq, xs)):
        torch.as_tensor(q.values, device="cuda").copy_(torch.from_numpy(v))
        torch.as_tensor(q.scales, device="cuda").copy_(torch.from_numpy(s))
    out = b200.alloc(5 * 70)
    torch.cuda.synchronize()
    b200.matmul_q8(out, w, x)
    b200.sync()
    same(torch.as_tensor(out, device="cuda").cpu().numpy().reshape(5, 70), ref_matmul(wq, ws, xq, xs))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 40, 300])
def test_captured_chain(b200, tokens):
    """Norm, product and quantisation captured into a CUDA graph on the
    device's stream, replayed on other inputs, and interleaved with plain calls."""
    torch = pytest.importorskip("torch")
    cols, channels = 320, 200
    rng = np.random.default_rng(tokens)
    wq, ws, _, _ = product_inputs(1, channels, cols, tokens)
    bits, nw = bf16(1 + 0.1 * rng.standard_normal(cols))
    norm, w = b200.upload(tb.Tensor([cols], bits)), rows_of(b200, wq, ws)
    x, y = b200.alloc(tokens * cols), b200.alloc(tokens * cols)
    q, out, oq = b200.q8(tokens, cols), b200.alloc(tokens * channels), b200.q8(tokens, channels)

    def chain():
        b200.add_rmsnorm_q8(q, x, y, norm, 1e-6)
        b200.matmul_q8(out, w, q)
        b200.quantize(oq, out)

    def check(call):
        a, b = sample_rows(tokens, cols, 5), rng.standard_normal((tokens, cols)).astype(F32)
        b200.write(x, a.reshape(-1))
        b200.write(y, b.reshape(-1))
        call()
        h, n = ref_norm(a, b, nw, 1e-6)
        product = ref_matmul(wq, ws, *ref_rows(n))
        b200.sync()
        same(b200.read(x).reshape(h.shape), h)
        same(b200.read(out).reshape(product.shape), product)
        for g, e in zip(b200.read_q8(oq), ref_rows(product)):
            same(g, e)

    check(chain)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.ExternalStream(b200.stream)
    with torch.cuda.graph(graph, stream=stream):
        chain()

    def replay():
        with torch.cuda.stream(stream):
            graph.replay()

    for call in (replay, chain, replay):
        check(call)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 8, 40])
def test_operands_written_by_the_kernel_before(b200, tokens):
    """Each kernel starts while the one that writes its input still runs: two inputs in turns through the same
    buffers, nothing waited for, and every result as when it is computed alone."""
    torch = pytest.importorskip("torch")
    cols, channels = 1024, 1500
    wq, ws, _, _ = product_inputs(1, channels, cols, tokens)
    w, ids = rows_of(b200, wq, ws), torch.arange(tokens, dtype=torch.int32, device="cuda")
    x = [buf(b200, np.random.default_rng(i).standard_normal((tokens, cols)).astype(F32)) for i in range(2)]
    q, out, back = b200.q8(tokens, cols), b200.alloc(tokens * channels), b200.alloc(tokens * cols)
    lp = tb.LogProbs(b200, tokens, channels, 5)
    torch.cuda.synchronize()

    def chain(i):
        b200.quantize(q, x[i])
        b200.dequantize(back, q)
        b200.quantize(q, back)
        b200.matmul_q8(out, w, q)
        lp.enqueue(out, ids)
        with torch.cuda.stream(torch.cuda.ExternalStream(b200.stream)):
            return [torch.as_tensor(a, device="cuda").clone() for a in (out, lp.logprob, lp.top_ids)]

    alone = []
    for i in range(2):
        alone.append(chain(i))
        b200.sync()
    assert not torch.equal(alone[0][0], alone[1][0])
    for i, got in [(n % 2, chain(n % 2)) for n in range(60)]:
        b200.sync()
        assert all(torch.equal(g, a) for g, a in zip(got, alone[i]))


@pytest.mark.gpu
def test_two_devices_at_once(b200):
    """Products of every kind and scores on two handles' streams, nothing waited for between them."""
    torch = pytest.importorskip("torch")
    other = tb.B200(0)
    shapes = [(1, 4096, 1024), (5, 1000, 4000), (40, 2000, 1024), (64, 512, 9728), (300, 1200, 1100), (1100, 640, 2176)]
    work = []
    for k, dev in enumerate((b200, other)):
        for tokens, channels, cols in shapes:
            wq, ws, xq, xs = product_inputs(tokens, channels, cols, tokens + k)
            lp = tb.LogProbs(dev, tokens, channels, 3)
            work.append((dev, rows_of(dev, wq, ws), rows_of(dev, xq, xs), dev.alloc(tokens * channels), lp,
                         torch.arange(tokens, dtype=torch.int32, device="cuda") % channels, ref_matmul(wq, ws, xq, xs)))
    torch.cuda.synchronize()
    for _ in range(20):
        for dev, w, x, out, lp, ids, _ in work:
            dev.matmul_q8(out, w, x)
            lp.enqueue(out, ids)
    b200.sync()
    other.sync()
    for dev, _, _, out, lp, ids, exp in work:
        same(dev.read(out).reshape(exp.shape), exp)
        now = [torch.as_tensor(a, device="cuda").clone() for a in (lp.logprob, lp.entropy, lp.top_ids)]
        torch.cuda.synchronize()
        lp.enqueue(out, ids)
        dev.sync()
        assert all(torch.equal(torch.as_tensor(a, device="cuda"), b)
                   for a, b in zip((lp.logprob, lp.entropy, lp.top_ids), now))


# ---- a whole model --------------------------------------------------------------------------

class Checked:
    """A device that checks each 8-bit call against its restatement on the
    inputs that the call was given."""

    def __init__(self, dev):
        self._dev, self.seen = dev, []

    def __getattr__(self, name):
        return getattr(self._dev, name)

    def _q8(self, q, n):
        for g, e in zip(self._dev.read_q8(q), ref_rows(n)):
            same(g, e)

    def add_rmsnorm_q8(self, out, x, y, weight, eps):
        d = self._dev
        a, b = d.read(x).reshape(out.shape), None if y is None else d.read(y).reshape(out.shape)
        d.add_rmsnorm_q8(out, x, y, weight, eps)
        h, n = ref_norm(a, b, np.ones(out.cols, F32), eps)  # the synthetic checkpoint's norm weights are 1
        same(d.read(x).reshape(out.shape), h)
        self._q8(out, n)
        self.seen.append("norm")

    def quantize(self, out, x):
        self._dev.quantize(out, x)
        self._q8(out, self._dev.read(x).reshape(out.shape))
        self.seen.append("quantize")

    def matmul_q8(self, out, w, x):
        d = self._dev
        d.matmul_q8(out, w, x)
        same(d.read(out).reshape(x.shape[0], w.shape[0]), ref_matmul(*d.read_q8(w), *d.read_q8(x)))
        self.seen.append("matmul")


@pytest.mark.gpu
def test_model_over_8_bit_weights(b200, tiny_model_dir):
    """A prompt and three single tokens through OpModel(q8=True): every 8-bit
    call equals its restatement, and scoring a prompt (all positions of a
    batch at once) gives what forward's logits, one position at a time, say."""
    checked = Checked(b200)
    m = tb.OpModel.load(tiny_model_dir, checked, q8=True)
    c = m.config
    prompt = synth.prompt_tokens(70, c.vocab_size, seed=3)  # more than one batch of 64
    st = m.state(80)
    first = m.forward(st, prompt, 0)
    m.forward(st, [int(np.argmax(first))], 70)
    layers = c.num_hidden_layers
    per_pass = ["norm"] + ["matmul"] * 3 + ["quantize", "matmul", "norm", "matmul", "matmul", "quantize", "matmul"]
    assert checked.seen == (per_pass * layers + ["norm", "matmul"]) * 3

    plain = tb.OpModel.load(tiny_model_dir, b200, q8=True)
    lp, ent, ids, top = plain.score(plain.state(80), prompt, 0, top=3)
    assert lp.shape == ent.shape == (69,) and ids.shape == top.shape == (69, 3)
    st = plain.state(80)
    for i in range(69):
        logits = plain.forward(st, prompt[i:i + 1], i).astype(np.float64)
        logp = logits - logits.max()
        logp -= np.log(np.exp(logp).sum())
        # f32 sums of 1024 terms, rounded logits of magnitude below 16
        tol = 1100 * 2.0 ** -24 + 2.0 ** -19
        assert abs(lp[i] - logp[prompt[i + 1]]) <= tol
        assert abs(ent[i] + (np.exp(logp) * logp).sum()) <= 8 * tol
        order = np.lexsort((np.arange(logp.size), -logits))[:3]
        assert ids[i].tolist() == order.tolist()
        assert np.all(np.abs(top[i] - logp[order]) <= tol)
    same(plain.forward(plain.state(80), prompt, 0), first)


@pytest.mark.gpu
def test_score_over_bf16_weights(b200, tiny_model_dir):
    m = tb.OpModel.load(tiny_model_dir, b200)
    prompt = synth.prompt_tokens(9, m.config.vocab_size, seed=4)
    lp, ent, ids, _ = m.score(m.state(16), prompt, 0)
    assert ids.shape == (8, 0)
    for i in range(8):
        logits = m.forward(m.state(16), prompt[:i + 1], 0).astype(np.float64)
        logp = logits - logits.max()
        logp -= np.log(np.exp(logp).sum())
        assert abs(lp[i] - logp[prompt[i + 1]]) <= 1e-3  # the batched product sums in another order
    with pytest.raises(ValueError, match="no tokens"):
        m.score(m.state(16), [], 0)
    assert m.score(m.state(16), prompt[:1], 0)[0].shape == (0,)
