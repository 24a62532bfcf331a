"""ns_sample_tokens against its definition in 64 bits: sort, cut, draw.

Tokens have to be the definition's: the kernel's weights are within 2^-33 of themselves and their sums exact, so a random number falls between the two sides' borders once in some
10^6 rows of the largest vocabularies here.  The probability is one rounding to 32 bits (half a step, 2^-24) of a quotient of a weight and a sum of weights, each within
2^-33, and every weight is rounded to a multiple of 2^-42 of the largest, half a step 2^-43: 2^-24 + 2^-32 of it, and 2^-42 * vocabulary."""
import numpy as np
import pytest

from nn_b200 import native as N

from .test_rotary import bf16, refused


def define(x, temperature, k, p, least, u):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(temperature)))
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    run = np.cumsum(w[order])
    if p < 1:
        order = order[:min(len(order), 1 + int((run < p * run[-1]).sum()))] if p > 0 else order[:1]
    if least > 0:
        order = order[w[order] >= min(least, 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    target = min(max(u, 0.0), 1.0) * run[-1]
    i = int((run <= target).sum())
    if i >= len(kept):                     # u of 1: the last token that can be drawn
        i = int(np.flatnonzero(w[kept] > 0)[-1])
    return int(kept[i]), w[kept[i]] / run[-1]


def settings(rng, rows):
    pick = lambda *v: rng.choice(np.array(v, np.float32), rows).astype(np.float32)
    return dict(temperature=pick(0.0, 0.5, 0.7, 1.0, 1.0, 1.5, 20.0), top_k=rng.choice([0, 0, 1, 2, 40, 1000, 10 ** 9, -3], rows).astype(np.int32),
                top_p=pick(0.0, 0.1, 0.5, 0.9, 0.95, 1.0, 1.0, 2.0), min_p=pick(0.0, 0.0, 0.01, 0.2, 1.0, -1.0), u=rng.random(rows).astype(np.float32))


def sample(dev, x_bits_or_floats, dtype, rows, vocab, stride, s, probs=True, start=0):
    store = dev.from_numpy(x_bits_or_floats)
    up = {n: dev.from_numpy(a) for n, a in s.items() if a is not None}
    at = lambda n: up[n].ptr if n in up else 0
    ids, pr = dev.from_numpy(np.full(rows, -7, np.int32)), dev.from_numpy(np.full(rows, -7, np.float32))
    size = 4 if dtype == N.NS_F32 else 2
    N.call("ns_sample_tokens", dev.handle, store.ptr + start * size, dtype, stride, rows, vocab, at("temperature"), at("top_k"), at("top_p"), at("min_p"), at("u"), ids.ptr,
           pr.ptr if probs else 0)
    dev.synchronize()
    return ids.download(), pr.download()


def check(ids, probs, x, s):
    vocab = x.shape[1]
    get = lambda n, r, neutral: neutral if s.get(n) is None else s[n][r]
    for r in range(len(x)):
        i, p = define(x[r], get("temperature", r, 1.0), int(get("top_k", r, 0)), float(get("top_p", r, 1.0)), float(get("min_p", r, 0.0)), float(s["u"][r]))
        assert ids[r] == i, (r, ids[r], i, {n: a[r] for n, a in s.items() if a is not None})
        assert abs(probs[r] - p) <= (2.0 ** -24 + 2.0 ** -32) * p + 2.0 ** -42 * vocab, (r, probs[r], p)


# one CTA a row and clusters of 2, 4 and 8; vocabularies that fill no vector; rows in numbers that fill the machine or not
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [N.NS_F32, N.NS_BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (40, 1000), (9, 4097), (300, 517), (4, 32000), (20, 20011), (2, 131001), (100, 9000), (160, 6001)])
def test_draws(dev, rows, vocab, dtype):
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[rows // 2:] *= 0.1                              # flat rows: many tokens are kept
    bits, rounded = bf16(x)
    x = rounded if dtype == N.NS_BF16 else x
    s = settings(rng, rows)
    ids, probs = sample(dev, bits if dtype == N.NS_BF16 else x, dtype, rows, vocab, vocab, s)
    check(ids, probs, x, s)
    # the same rows without some settings, a row pitch, a start off a vector
    stride = vocab + 3
    wide = np.full(rows * stride + 5, np.inf, np.float32)
    wide[5:].reshape(rows, stride)[:, :vocab] = x
    for left_out in (("temperature", "top_k"), ("top_p",), ("min_p", "top_k", "top_p", "temperature")):
        t = {n: (None if n in left_out else a) for n, a in s.items()}
        ids, probs = sample(dev, bf16(wide)[0] if dtype == N.NS_BF16 else wide, dtype, rows, vocab, stride, t, start=5)
        check(ids, probs, x, t)


@pytest.mark.gpu
def test_equal_logits(dev):
    """Ties at every cutoff go to the lowest index."""
    rng = np.random.default_rng(1)
    for vocab in (8, 100, 3000, 40000):
        rows = 64
        x = rng.integers(-2, 2, (rows, vocab)).astype(np.float32)
        x[0], x[1, :] = 0.0, np.where(np.arange(vocab) % 2, 0.0, -0.0)
        s = settings(rng, rows)
        s["top_k"][:32] = rng.integers(2, vocab + 1, 32)
        # quarters of equal weights reach their share exactly
        s["top_p"][:2], s["top_k"][:2], s["temperature"][:2], s["min_p"][:2], s["u"][:2] = [0.25, 0.75], 0, 1.0, 0.0, 0.999
        ids, probs = sample(dev, x, N.NS_F32, rows, vocab, vocab, s)
        check(ids, probs, x, s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [N.NS_F32, N.NS_BF16])
@pytest.mark.parametrize("vocab", [16500, 50001])
def test_large_tokens_at_regular_places(dev, vocab, dtype):
    """The largest tokens all at every 8th place, none of them there, side by side, in order, many of one value: what a guess from a part of the row takes for more or for fewer
    than there are."""
    rng = np.random.default_rng(vocab)
    places = [np.arange(0, 8 * 400, 8), np.arange(3, 3 + 8 * 400, 8), np.arange(100, 500), np.arange(vocab - 400, vocab), np.arange(0, 8 * 2000, 8)]
    rows, xs = [], []
    for where in places:
        for high in (6.0, 0.5):
            x = rng.standard_normal(vocab).astype(np.float32)
            x[where] = high + rng.standard_normal(len(where)).astype(np.float32) * 0.5
            xs.append(x)
    xs.append(np.sort(rng.standard_normal(vocab).astype(np.float32)))
    xs.append(xs[-1][::-1].copy())
    xs.append(np.where(np.arange(vocab) % 8 == 0, 1.0, 0.0).astype(np.float32))
    xs.append(np.where(np.arange(vocab) % 97 == 5, 3.0, -1.0).astype(np.float32))
    base = np.stack(xs)
    ks = [2, 20, 50, 128, 129, 300, 1000, vocab // 16, vocab // 16 + 1, vocab - 1]
    x = np.repeat(base, len(ks), axis=0)
    n = len(x)
    bits, rounded = bf16(x)
    x = rounded if dtype == N.NS_BF16 else x
    k = np.tile(np.array(ks, np.int32), len(base))
    for top_p, min_p, t in ((1.0, 0.0, 1.0), (0.9, 0.0, 0.7), (0.99, 0.05, 2.0)):
        s = dict(temperature=np.full(n, t, np.float32), top_k=k, top_p=np.full(n, top_p, np.float32), min_p=np.full(n, min_p, np.float32), u=rng.random(n).astype(np.float32))
        ids, probs = sample(dev, bits if dtype == N.NS_BF16 else x, dtype, n, vocab, vocab, s)
        check(ids, probs, x, s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [N.NS_F32, N.NS_BF16])
@pytest.mark.parametrize("vocab,equal", [(16400, 600), (30000, 1200), (131001, 1900), (40000, 2500)])
def test_more_equal_candidates_than_are_sorted(dev, vocab, equal, dtype):
    """Many tokens of one value, or of two, around the cutoffs."""
    rng = np.random.default_rng(equal)
    ks = [100, 128, 300, 512, 513, 900, 1024, 1025]
    rows = 2 * len(ks)
    x = np.full((rows, vocab), -6.0, np.float32) + rng.random((rows, vocab)).astype(np.float32)
    for r in range(rows):
        where = rng.permutation(vocab)[:equal]
        x[r, where] = 2.0
        if r >= len(ks):
            x[r, where[:equal // 3]] = 2.015625
            x[r, where[:7]] = 3.0 + rng.random(7).astype(np.float32)
    bits, rounded = bf16(x)
    x = rounded if dtype == N.NS_BF16 else x
    for top_p, least in ((1.0, 0.0), (0.5, 0.0), (0.9, 0.3)):
        s = dict(temperature=np.full(rows, 0.8, np.float32), top_k=np.tile(np.array(ks, np.int32), 2), top_p=np.full(rows, top_p, np.float32), min_p=np.full(rows, least, np.float32),
                 u=rng.random(rows).astype(np.float32))
        ids, probs = sample(dev, bits if dtype == N.NS_BF16 else x, dtype, rows, vocab, vocab, s)
        check(ids, probs, x, s)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,dtype", [(380000, N.NS_F32), (760000, N.NS_BF16), (262144, N.NS_F32), (524289, N.NS_BF16)])
def test_the_largest_vocabularies(dev, vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = 12
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    x[:, rng.integers(0, vocab, 30)] += 8
    x[rows // 2:] *= 0.25
    bits, rounded = bf16(x)
    x = rounded if dtype == N.NS_BF16 else x
    s = dict(temperature=np.tile(np.array([1.0, 0.7, 1.3], np.float32), 4), top_k=np.tile(np.array([0, 50, 1000, 40000], np.int32), 3), top_p=np.tile(np.array([0.9, 1.0], np.float32), 6),
             min_p=np.zeros(rows, np.float32), u=rng.random(rows).astype(np.float32))
    ids, probs = sample(dev, bits if dtype == N.NS_BF16 else x, dtype, rows, vocab, vocab, s)
    check(ids, probs, x, s)


@pytest.mark.gpu
def test_temperatures_and_logits_of_every_size(dev):
    rng = np.random.default_rng(7)
    vocab = 20000
    xs, ts = [], []
    for scale in (1e-38, 1e-20, 1.0, 1e20, 1e37):
        for t in (1e-37, 1e-20, 1e-3, 1.0, 1e6, 1e20, 3e38, np.inf):
            xs.append(rng.standard_normal(vocab).astype(np.float32) * np.float32(scale))
            ts.append(t)
    x = np.stack(xs)
    n = len(x)
    for k in (0, 30, 700):
        for top_p in (1.0, 0.8):
            s = dict(temperature=np.array(ts, np.float32), top_k=np.full(n, k, np.int32), top_p=np.full(n, top_p, np.float32), u=rng.random(n).astype(np.float32))
            ids, probs = sample(dev, x, N.NS_F32, n, vocab, vocab, s)
            check(ids, probs, x, s)


@pytest.mark.gpu
def test_values_that_are_no_numbers(dev):
    rng = np.random.default_rng(2)
    vocab = 5000
    x = rng.standard_normal((12, vocab)).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0], x[1], x[2] = -np.inf, np.nan, low
    x[3, :] = -np.inf
    x[3, 4321] = low
    x[4, ::2], x[5, 1::3], x[6, ::7] = -np.inf, np.nan, np.inf
    x[7, 100], x[7, 200] = np.inf, np.inf
    x[8] = np.float32(3e38) * np.where(np.arange(vocab) % 5, -1, 1)
    x[9] *= 1e-42
    x[10], x[11] = 65504.0, low
    x[11, 7] = -1.0
    for seed in range(4):
        s = settings(np.random.default_rng(seed), 12)
        if seed == 0:
            s["temperature"][:], s["top_k"][:], s["top_p"][:], s["min_p"][:] = 1.0, 0, 1.0, 0.0
        ids, probs = sample(dev, x, N.NS_F32, 12, vocab, vocab, s)
        check(ids, probs, x, s)
    # settings that are no numbers are those that keep everything, a temperature that is none takes the maximum; the ends of u
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    nan = np.float32(np.nan)
    s = dict(temperature=np.array([nan, np.inf, 1e-38, 1, 1, 1], np.float32), top_k=np.array([3, 0, 0, 0, 5, 0], np.int32), top_p=np.array([1, 1, 1, nan, 1, 0.9], np.float32),
             min_p=np.array([0, 0, 0, nan, 0, 0], np.float32), u=np.array([0.5, 0.25, 0.5, 0.999999, 1.0, 0.0], np.float32))
    ids, probs = sample(dev, x, N.NS_F32, 6, vocab, vocab, s)
    plain = {**s, "top_p": np.where(np.isnan(s["top_p"]), 1, s["top_p"]).astype(np.float32), "min_p": np.nan_to_num(s["min_p"])}
    check(ids, probs, x, plain)


@pytest.mark.gpu
def test_a_row_alone_draws_what_it_draws_in_a_batch(dev):
    rng = np.random.default_rng(9)
    rows, vocab = 200, 12345
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    s = settings(rng, rows)
    ids, probs = sample(dev, x, N.NS_F32, rows, vocab, vocab, s)
    again = sample(dev, x, N.NS_F32, rows, vocab, vocab, s)
    assert np.array_equal(ids, again[0]) and np.array_equal(probs.view(np.int32), again[1].view(np.int32))
    for r in range(0, rows, 13):
        i, p = sample(dev, x[r:r + 1], N.NS_F32, 1, vocab, vocab, {n: a[r:r + 1] for n, a in s.items()})
        assert i[0] == ids[r] and p.view(np.int32)[0] == probs.view(np.int32)[r]
    assert np.array_equal(sample(dev, x, N.NS_F32, rows, vocab, vocab, s, probs=False)[0], ids)


def test_refusals():
    A = 1 << 20
    good = dict(x=A, dtype=N.NS_F32, stride=1000, rows=2, vocab=1000, temperature=0, top_k=0, top_p=0, min_p=0, u=A, ids=A, probs=0)

    def call(text, **other):
        refused(text, "ns_sample_tokens", None, *{**good, **other}.values())

    call("device handle is null")
    call("device handle is null", rows=0)
    call("device handle is null", vocab=380000)
    call("device handle is null", vocab=760000, dtype=N.NS_BF16)
    for name in ("x", "u", "ids"):
        call("null argument", **{name: 0})
    call("dtype", dtype=N.NS_I8)
    call("bad shape", vocab=0)
    call("bad shape", rows=-1)
    call("bad shape", stride=-1)
    call("tokens of this type", vocab=420000)
    call("too many rows", rows=1 << 28)
    call("misaligned", x=A + 2)
    call("misaligned", top_k=A + 2)
