"""Log probabilities of given tokens, entropies and alternatives (LogProbs,
tb200_score) against log-softmax in 64 bits.

Tolerances. A row's sum of exponentials is positive terms added in f32, so its
relative error is at most (longest chain of additions + the exponentials' own
few units) * 2^-24; CHAIN bounds both. That is the absolute error of log Z. The
difference l - m rounds once, and once more against log Z: 2^-24 each, relative
to numbers of at most |l - m| + |log Z|. The entropy's second term adds the same
again, times its terms' magnitudes."""

import numpy as np
import pytest

import titania_b200 as tb
from titania_b200 import _lib

F32 = np.float32
CHAIN = 1100
EPS = 2.0 ** -24


def reference(logits, tokens, top):
    """(logprob, entropy, ids, top logprobs) in f64."""
    l = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        z = l - l.max(axis=1, keepdims=True)
        logz = np.log(np.exp(z).sum(axis=1, keepdims=True))
        logp = z - logz
        p = np.exp(logp)
        ent = -np.where(p > 0, p * logp, 0).sum(axis=1)
        ent = np.where(np.isnan(logz[:, 0]), np.nan, ent)
    lp = np.array([logp[i, t] if t < l.shape[1] else np.nan for i, t in enumerate(tokens)])
    b = logits.view(np.int32).astype(np.int64)
    key = np.where(b < 0, b ^ 0x7FFFFFFF, b)  # IEEE total order
    ids = np.argsort(-key, axis=1, kind="stable")[:, :top]
    return lp, ent, ids, np.take_along_axis(logp, ids, axis=1)


def compare(got, logits, tokens, top):
    lp, ent, ids, tops = reference(logits, tokens, top)
    z = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        finite = np.where(np.isfinite(z), z, 0)
        span = np.ptp(finite, axis=1) + 20
    tol = CHAIN * EPS + 4 * EPS * span
    assert got[2].tolist() == ids.tolist()

    def near(a, b, t):
        a = a.astype(np.float64)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isneginf(a), np.isneginf(b))
        ok = np.isfinite(b)
        assert np.isfinite(a[ok]).all()
        t = np.broadcast_to(t.reshape(t.shape + (1,) * (b.ndim - 1)), b.shape)
        assert np.all(np.abs(a[ok] - b[ok]) <= t[ok]), np.abs(a[ok] - b[ok]).max()

    near(got[0], lp, tol)
    near(got[1], ent, tol * (1 + np.where(np.isnan(ent), 0, ent)))
    near(got[3], tops, tol)


def buf(dev, values):
    b = dev.alloc(values.size)
    dev.write(b, values.reshape(-1))
    return b


def test_null_handles_are_errors():
    for name, args in (("tb200_scorer_new", (None, 1, 1, 0, None)), ("tb200_score_enqueue", (None, None, None, 0)),
                       ("tb200_score", (None, None, None, 0, None, None, None, None)),
                       ("tb200_scorer_data", (None, None, None, None, None))):
        with pytest.raises(tb.DeviceError, match="null") as e:
            _lib.call(name, *args)
        assert e.value.code == _lib.TB200_ERR_ARG
    assert _lib.lib().tb200_scorer_free(None) == 0


def test_device_token_ids_are_checked_on_the_host():
    class Array:
        def __init__(self, **kw):
            self.__cuda_array_interface__ = {"shape": (4,), "typestr": "<i4", "data": (64, False), "version": 3} | kw

    assert tb.LogProbs._tokens(Array())[:2] == (64, 4)
    for bad in ({"typestr": "<i8"}, {"strides": (8,)}, {"shape": (2, 2), "strides": (16, 4)}):
        with pytest.raises(ValueError, match="32-bit"):
            tb.LogProbs._tokens(Array(**bad))


def test_host_token_ids_are_checked_and_copied():
    for bad in ([-1], [2 ** 32], [1.5], np.array([3, 2 ** 32 + 5])):
        with pytest.raises(ValueError, match="32 bits"):
            tb.LogProbs._tokens(bad)
    assert tb.LogProbs._tokens([])[1] == 0
    given = np.array([4, 2 ** 32 - 1], dtype=np.uint32)
    ptr, n, kept = tb.LogProbs._tokens(given)
    assert n == 2 and kept.tolist() == given.tolist() and ptr != given.ctypes.data


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 7, 7), (2, 64, 64), (5, 127, 10), (4, 128, 5),
                                            (33, 1000, 20), (2, 1024, 0), (700, 512, 3), (1, 5000, 64), (9, 32001, 1),
                                            (1, 151936, 20), (3, 151936, 64), (64, 151936, 5), (150, 40003, 8),
                                            (2, 262144, 40)])
@pytest.mark.parametrize("kind", ["normal", "peaked", "ties"])
def test_logprobs(b200, rows, vocab, top, kind):
    rng = np.random.default_rng(rows * 3 + vocab + top)
    x = rng.standard_normal((rows, vocab)).astype(F32) * F32(3)
    if kind == "peaked":  # nearly all of the probability on one token
        x[np.arange(rows), rng.integers(0, vocab, rows)] += F32(25)
    if kind == "ties":
        x = np.round(x).astype(F32)
        x[0] = F32(-2.5)  # every logit the same
    tokens = rng.integers(0, vocab, rows)
    tokens[::2] = x[::2].argmax(axis=1)
    s = tb.LogProbs(b200, rows, vocab, top)
    compare(s.score(buf(b200, x), tokens), x, tokens, top)


@pytest.mark.gpu
def test_one_token_has_almost_everything(b200):
    """The others' share keeps its relative error (CHAIN units), also below
    f32's distance from 1."""
    x = np.full((6, 4000), -30, dtype=F32)
    gaps = [1, 5, 10, 16, 20, 30]
    for i, g in enumerate(gaps):
        x[i, 77 * i] = F32(g - 30)
    s = tb.LogProbs(b200, 6, 4000)
    lp, ent, _, _ = s.score(buf(b200, x), [77 * i for i in range(6)])
    for i, g in enumerate(gaps):
        rest = 3999 * np.exp(-np.float64(g))
        logz = np.log1p(rest)
        assert abs(lp[i] + logz) <= 2 * CHAIN * EPS * logz
        h = logz + g * rest / (1 + rest)
        assert abs(ent[i] - h) <= 4 * CHAIN * EPS * h


@pytest.mark.gpu
@pytest.mark.parametrize("top", [1, 9])
@pytest.mark.parametrize("vocab", [40, 1000, 70001])
def test_rows_that_are_not_ordinary(b200, vocab, top):
    """Excluded tokens (-inf), rows of nothing else, NaN of either sign,
    infinities, zeros of either sign, the type's lowest and largest values."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((12, vocab)).astype(F32)
    x[0, : vocab // 2] = -np.inf
    x[1] = -np.inf
    x[2], x[2, 17] = -np.inf, 3.0
    x[3, 5] = np.nan
    x[4, 6] = np.inf
    x[5, 7], x[5, 8] = np.inf, np.inf
    x[6, 9] = -np.float32(np.nan)
    x[7] = np.where(np.arange(vocab) % 3 == 0, F32(0.0), F32(-0.0))
    x[8] = np.finfo(F32).min
    x[9], x[9, 3] = np.finfo(F32).min, 2.0
    x[10], x[10, 4], x[10, 5] = np.finfo(F32).max, 0.0, np.finfo(F32).min
    x[11, 1:] = -np.inf
    s = tb.LogProbs(b200, 12, vocab, top)
    for tokens in ([1] * 12, [17] * 12, [0] * 12, list(range(12))):
        got = s.score(buf(b200, x), tokens)
        lp, ent, ids, tops = reference(x, tokens, top)
        assert got[2].tolist() == ids.tolist()
        for g, e in ((got[0], lp), (got[1], ent), (got[3], tops)):
            assert np.array_equal(np.isnan(g), np.isnan(e))
            assert np.array_equal(np.isneginf(g), np.isneginf(e))
            ok = np.isfinite(e)
            # f32's lowest against ordinary numbers: relative to the difference
            assert np.all(np.abs(g[ok] - e[ok]) <= CHAIN * EPS * (2 + np.abs(e[ok])))


@pytest.mark.gpu
def test_orders_of_rising_and_falling_logits(b200):
    """All of the alternatives next to one another, at either end."""
    vocab = 151936
    x = np.stack([np.arange(vocab), -np.arange(vocab), np.arange(vocab) // 500]).astype(F32) * F32(1e-3)
    for top in (64, 20, 1):
        s = tb.LogProbs(b200, 3, vocab, top)
        compare(s.score(buf(b200, x), [5, 5, 5]), x, [5, 5, 5], top)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 1, 2, 30])
def test_many_rows_of_every_alignment(b200, top):
    """More rows than CTAs, rows that start anywhere within 16 bytes, ties
    between the parts of a row; twice the same bits."""
    rng = np.random.default_rng(top)
    x = np.round(rng.standard_normal((1301, 2053)) * 2).astype(F32)
    tokens = rng.integers(0, 2053, 1301)
    s, b = tb.LogProbs(b200, 1301, 2053, top), buf(b200, x)
    got = s.score(b, tokens)
    compare(got, x, tokens, top)
    for a, c in zip(got, s.score(b, tokens)):
        assert np.array_equal(a.view(np.int32), c.view(np.int32))


def row_kinds(vocab):
    """Rows of nine kinds, the alternatives spread, side by side, at either end, tied."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((9, vocab)).astype(F32) * F32(2)
    x[1] = np.round(x[1])
    x[2] = F32(0.5)  # every logit the same
    x[3] = np.sort(x[3])
    x[4] = np.sort(x[4])[::-1]
    x[5, vocab // 2:vocab // 2 + 300] += F32(12)
    x[6, rng.integers(0, vocab, 4)] += F32(25)
    x[7, rng.permutation(vocab)[vocab // 100:]] = -np.inf  # few are left, perhaps fewer than the alternatives
    x[8] = np.where(np.arange(vocab) % 128 < 40, x[8], x[8] - F32(30))
    return x


# Rows by a warp each in registers or step by step, by a CTA each, in pieces, in
# runs that end inside rows; one warp's share of a row is at most 64 steps of 16.
MANY_ROWS = [(9, 2045, 64), (1300, 2045, 7), (126, 2046, 64), (126, 2046, 2), (333, 2051, 0), (333, 2051, 1),
             (700, 5003, 1), (300, 5003, 20), (900, 16381, 40), (4200, 32765, 0), (1650, 32765, 5), (400, 32765, 5),
             (64, 32001, 0), (64, 32001, 5), (100, 33001, 1), (1, 20001, 3), (400, 40003, 3), (650, 40003, 0),
             (650, 40003, 1), (650, 40003, 6), (250, 300007, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,top", MANY_ROWS)
def test_ways_of_sharing_rows(b200, rows, vocab, top):
    torch = pytest.importorskip("torch")
    x = row_kinds(vocab)
    tokens = np.array([0, vocab - 1, 5, vocab - 1, 0, vocab // 2, 7, 8, 1])
    at = np.arange(rows) % 9
    b = b200.alloc(rows * vocab)
    given = torch.as_tensor(x, device="cuda")[torch.as_tensor(at, device="cuda")]
    torch.as_tensor(b, device="cuda").copy_(given.reshape(-1))
    torch.cuda.synchronize()
    got = tb.LogProbs(b200, rows, vocab, top).score(b, tokens[at])
    for first in {0, (rows - 1) // 18 * 9, (rows - 1) // 9 * 9}:
        part = slice(first, min(first + 9, rows))
        n = part.stop - part.start
        compare([g[part] for g in got], x[:n], tokens[:n], top)
    # Each row's alternatives whatever its place; its sums to twice the tolerance above, a span of 100 taken for all.
    for i in range(min(9, rows)):
        assert (got[2][i::9] == got[2][i]).all()
        for g in (got[0], got[1]):
            assert np.array_equal(np.isfinite(g[i::9]), np.full(len(g[i::9]), np.isfinite(g[i])))
            if np.isfinite(g[i]):
                assert np.abs(g[i::9] - g[i]).max() <= 2 * (CHAIN + 400) * EPS * (1 + abs(g[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,top", [(2101, 0), (2101, 1), (2101, 33), (9001, 5), (9001, 64)])
def test_many_rows_that_are_not_ordinary(b200, vocab, top):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((10, vocab)).astype(F32)
    x[0, : vocab // 2] = -np.inf
    x[1] = -np.inf
    x[2], x[2, 17] = -np.inf, 3.0
    x[3, vocab - 1] = np.nan
    x[4, 6] = np.inf
    x[5, 9] = -np.float32(np.nan)
    x[6] = np.where(np.arange(vocab) % 3 == 0, F32(0.0), F32(-0.0))
    x[7] = np.finfo(F32).min
    x[8], x[8, 4], x[8, 5] = np.finfo(F32).max, 0.0, np.finfo(F32).min
    x[9, 1:] = -np.inf
    rows = 1260
    at = np.arange(rows) % 10
    many = x[at]
    got = tb.LogProbs(b200, rows, vocab, top).score(buf(b200, many), at * 3)
    lp, ent, ids, tops = reference(x, np.arange(10) * 3, top)
    assert (got[2] == ids[at]).all()
    for g, e in ((got[0], lp), (got[1], ent), (got[3], tops)):
        e = e[at]
        assert np.array_equal(np.isnan(g), np.isnan(e))
        assert np.array_equal(np.isneginf(g), np.isneginf(e))
        ok = np.isfinite(e)
        assert np.all(np.abs(g[ok] - e[ok]) <= CHAIN * EPS * (2 + np.abs(e[ok])))


FAR = [-1e10, -1e20, -1e30, 1e7, 1e10, 1e30]


def far_rows(vocab, far):
    """Rows whose first, last, or only logits lie at `far`: finite mask values where it is negative, maxima alone,
    tied and a step apart where it is positive."""
    rng = np.random.default_rng(vocab)
    far, n = F32(far), min(vocab - 9, 4500)  # n: more than eight warps' first steps
    x = rng.standard_normal((9, vocab)).astype(F32) * F32(2)
    x[0, :n] = far
    x[1, vocab - n:] = far
    x[2] = far
    x[3], x[3, vocab // 2] = far, 1.5
    x[4], x[4, vocab - 5:] = far, x[5, :5]
    x[5, ::3] = far
    x[6, 7] = far
    x[7, [3, vocab // 2, vocab - 1]] = far
    x[8, 2:40:2], x[8, 1] = far, np.nextafter(far, F32(0))
    return x


def check_far(got, x, tokens, top, at):
    """Tolerances: the sums' CHAIN for log Z (twice for the entropy, which has T / (1 + S) as well), and two roundings
    relative to the result, which CHAIN covers too; see above. Exponents of shares that count are below 200, and
    their one rounding moves a share by at most 2^-24 of its exponent."""
    lp, ent, ids, tops = reference(x, tokens, top)
    assert (got[2] == ids[at]).all()
    for g, e in ((got[0], lp), (got[1], ent), (got[3], tops)):
        e = e[at]
        assert np.isfinite(e).all() and np.isfinite(g).all()
        assert np.all(np.abs(g - e) <= 2 * CHAIN * EPS * (1 + np.abs(e)))


# By a warp in registers, step by step, by CTAs for whole rows, for pieces, for runs that end inside rows.
@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,top", [(9, 500, 3), (9, 2045, 20), (1350, 5003, 0), (1350, 5003, 5),
                                            (1800, 9001, 1), (9, 9001, 1), (9, 70001, 0), (9, 70001, 1),
                                            (63, 151936, 5), (405, 40003, 3), (657, 40003, 1)])
@pytest.mark.parametrize("far", FAR)
def test_logits_far_from_zero(b200, rows, vocab, top, far):
    """Magnitudes past 2^20, where steps of f32(m log2 e) are no small numbers: whole and half-masked rows, and maxima
    with ties and neighbours."""
    torch = pytest.importorskip("torch")
    x = far_rows(vocab, far)
    tokens = np.array([vocab - 1, 0, 5, vocab // 2, vocab - 1, 1, 7, 3, 2])
    at = np.arange(rows) % 9
    b = b200.alloc(rows * vocab)
    b200.sync()
    given = torch.as_tensor(x, device="cuda")[torch.as_tensor(at, device="cuda")]
    torch.as_tensor(b, device="cuda").copy_(given.reshape(-1))
    torch.cuda.synchronize()
    check_far(tb.LogProbs(b200, rows, vocab, top).score(b, tokens[at]), x, tokens, top, at)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(9, 2000), (1350, 5003), (9, 70001)])
@pytest.mark.parametrize("base", [3e5, 9e5, 1.2e6, 5e6])
def test_ordinary_rows_moved_far(b200, rows, vocab, base):
    """Rows whose logits lie a few apart on both sides of the limit, on a coarse grid that f32 holds."""
    rng = np.random.default_rng(int(base))
    x = (np.round(rng.standard_normal((9, vocab)) * 6) / 2).astype(F32)
    x[1::2] = -F32(base) + x[1::2]
    x[::2] = F32(base) + x[::2]
    at = np.arange(rows) % 9
    tokens = rng.integers(0, vocab, 9)
    check_far(tb.LogProbs(b200, rows, vocab, 4).score(buf(b200, x[at]), tokens[at]), x, tokens, 4, at)


@pytest.mark.gpu
def test_rows_behind_the_last_stay(b200):
    """Fewer rows than the scorer holds; the same scorer again with others."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 300)).astype(F32)
    s, b = tb.LogProbs(b200, 5, 300, 2), buf(b200, x)
    s.score(b, [1, 2, 3, 4, 5])
    before = [torch.as_tensor(a, device="cuda").cpu().numpy().copy() for a in (s.logprob, s.entropy, s.top_ids)]
    y = rng.standard_normal((2, 300)).astype(F32)
    got = s.score(buf(b200, y), [7, 8])
    compare(got, y, [7, 8], 2)
    after = [torch.as_tensor(a, device="cuda").cpu().numpy() for a in (s.logprob, s.entropy, s.top_ids)]
    for a, c, g in zip(before, after, got):
        assert np.array_equal(a[2:], c[2:]) and np.array_equal(c[:2].view(np.int32), g.view(np.int32))
    assert s.score(b, [])[0].shape == (0,)


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(b200):
    """15000 rows of 151936 logits (2.3 G values): the last rows."""
    torch = pytest.importorskip("torch")
    rows, vocab = 15000, 151936
    b = b200.alloc(rows * vocab)
    rng = np.random.default_rng(8)
    x = rng.standard_normal((3, vocab)).astype(F32) * F32(2)
    for i, r in enumerate((0, 14200, 14999)):
        b200.copy(b, r * vocab, buf(b200, x[i]), 0, vocab)
    s = tb.LogProbs(b200, rows, vocab, 4)
    tokens = np.full(rows, 11)
    got = s.score(b, tokens)
    at = [0, 14200, 14999]
    compare([g[at] for g in got], x, [11] * 3, 4)
    # the other rows are zeros: uniform
    assert abs(got[0][1] + np.log(vocab)) <= CHAIN * EPS * 12 and got[2][1].tolist() == [0, 1, 2, 3]
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_tokens_on_the_device_and_captured(b200):
    """Ids in device memory (one past the vocabulary, one negative: NaN), and a
    captured call replayed with other logits and other ids."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(6)
    x = rng.standard_normal((4, 9000)).astype(F32)
    s, b = tb.LogProbs(b200, 4, 9000, 3), buf(b200, x)
    ids = torch.tensor([5, 9000, -1, 8999], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    tokens = [5, 9000, 2 ** 32 - 1, 8999]
    compare(s.score(b, ids), x, tokens, 3)
    stream, graph = torch.cuda.ExternalStream(b200.stream), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.enqueue(b, ids)
        with pytest.raises(tb.DeviceError, match="device memory"):
            s.enqueue(b, [1, 2, 3, 4])
    for seed in range(3):
        y = np.random.default_rng(seed).standard_normal((4, 9000)).astype(F32)
        b200.write(b, y.reshape(-1))
        ids.copy_(torch.tensor([seed, 1, 2, 3], dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        b200.sync()
        got = [torch.as_tensor(a, device="cuda").cpu().numpy() for a in (s.logprob, s.entropy, s.top_ids,
                                                                         s.top_logprobs)]
        compare(got, y, [seed, 1, 2, 3], 3)


@pytest.mark.gpu
def test_refusals(b200):
    for rows, vocab, top in ((0, 10, 1), (1, 0, 0), (1, 10, 11), (1, 1000, 65), (1, 2 ** 30 + 1, 0),
                             (2 ** 24 + 1, 10, 0)):
        with pytest.raises(tb.DeviceError, match="bad|top"):
            tb.LogProbs(b200, rows, vocab, top)
    s, b = tb.LogProbs(b200, 2, 100, 3), b200.alloc(200)
    with pytest.raises(tb.DeviceError, match="can't hold 3"):
        s.score(b200.alloc(300), [1, 2, 3])
    with pytest.raises(tb.DeviceError, match="fewer"):
        s.score(b200.alloc(199), [1, 2])
    with pytest.raises(tb.DeviceError, match="token 100 is past"):
        s.score(b, [1, 100])
    with pytest.raises(ValueError, match="32-bit"):
        torch = pytest.importorskip("torch")
        s.score(b, torch.zeros(2, dtype=torch.int64, device="cuda"))
    s.close()
    with pytest.raises(tb.DeviceError, match="null"):
        s.score(b, [1, 2])
