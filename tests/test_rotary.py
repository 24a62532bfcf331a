"""Rotary positions (ns_rotary) and the append to a paged cache that turns queries and keys on the way (ns_kv_append_rotary), against the formula in 64 bits.

Tolerance.  cos and sin of the 64-bit angle come with at most 2.5 float ulps (the function's own, its correction, the amplitude), the two products and their sum
add 1: below 4 * 2^-23 * amplitude * (|a| + |b|) for a pair (a, b).  A bf16 result adds half a bf16 step, 2^-8 of its value; a sum of slabs the half
steps of its additions."""
import ctypes as C

import numpy as np
import pytest

from nn_b200 import native as N

AMP = 1.125


def bf16(x):
    """float array -> (bits, values), round to nearest even"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    bits = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return bits, values(bits)


def values(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def frequencies(rot, base=10000.0):
    return (base ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)


def turn(x, pos, freq, halves, amplitude=AMP, sign=1.0):
    """x [rows, heads, dim] in 64 bits -> (turned, |a| + |b| of each turned column)"""
    x = x.astype(np.float64)
    half = len(freq)
    t = sign * pos.astype(np.float64)[:, None] * freq.astype(np.float64)
    c, s = amplitude * np.cos(t)[:, None], amplitude * np.sin(t)[:, None]
    y, size = x.copy(), np.zeros_like(x)
    ia, ib = (np.arange(half), np.arange(half) + half) if halves else (2 * np.arange(half), 2 * np.arange(half) + 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = abs(a) + abs(b)
    return y, size


def bound(y, size, dtype, amplitude=AMP):
    return 4 * 2.0 ** -23 * amplitude * size + (2.0 ** -8 * abs(y) if dtype == N.NS_BF16 else 0.0)


def put(dev, x, dtype):
    """-> (storage, the values it holds)"""
    if dtype == N.NS_BF16:
        bits, v = bf16(x)
        return dev.from_numpy(bits), v
    return dev.from_numpy(np.ascontiguousarray(x, np.float32)), np.asarray(x, np.float32)


def get(store, shape):
    a = store.download(shape)
    return values(a) if a.dtype == np.uint16 else a


SHAPES = [  # rows, heads, dim, rot
    (1, 1, 2, 2), (1, 40, 128, 128), (3, 5, 128, 64), (7, 2, 96, 32), (33, 3, 40, 26), (5, 1, 64, 30), (300, 2, 64, 64), (9, 17, 256, 256), (2, 3, 33, 6), (1200, 1, 32, 16),
    (2, 2, 4096, 4096), (64, 48, 128, 128), (4, 7, 80, 80),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [N.NS_F32, N.NS_BF16])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("rows,heads,dim,rot", SHAPES)
def test_rotary(dev, rows, heads, dim, rot, halves, dtype):
    rng = np.random.default_rng(rows * 1000 + dim + rot)
    x_store, x = put(dev, rng.standard_normal((rows, heads, dim)), dtype)
    pos = rng.integers(0, 500000, rows).astype(np.int32)
    if rows > 2:
        pos[1] = -1
    freq = frequencies(rot)
    f, ps = dev.from_numpy(freq), dev.from_numpy(pos)
    before, _ = put(dev, np.full((rows, heads, dim), 7.0), dtype)
    layout = N.ROTARY_HALVES if halves else N.ROTARY_PAIRS
    for inverse in (0, 1):
        want, size = turn(x, pos, freq, halves, sign=-1.0 if inverse else 1.0)
        want[pos < 0], size[pos < 0] = 7.0, 0.0
        N.call("ns_rotary", dev.handle, x_store.ptr, dtype, heads * dim, dim, ps.ptr, f.ptr, AMP, layout, inverse, rows, heads, dim, rot, before.ptr, heads * dim, dim)
        dev.synchronize()
        got = get(before, (rows, heads, dim)).astype(np.float64)
        assert (abs(got - want) <= bound(want, size, dtype)).all(), (inverse, abs(got - want).max())
        assert np.array_equal(got[..., rot:][pos >= 0], x[..., rot:].astype(np.float64)[pos >= 0])      # columns that are not turned keep their bits
    # in place: the same bits
    out = before.download()
    N.call("ns_rotary", dev.handle, x_store.ptr, dtype, heads * dim, dim, ps.ptr, f.ptr, AMP, layout, 1, rows, heads, dim, rot, x_store.ptr, heads * dim, dim)
    dev.synchronize()
    assert np.array_equal(x_store.download((rows, heads, dim))[pos >= 0], out.reshape(rows, heads, dim)[pos >= 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [N.NS_F32, N.NS_BF16])
def test_rotary_pitches_and_alignment(dev, dtype):
    """Heads inside rows, rows inside heads, a matrix that starts off a vector, and what lies between the heads."""
    rng = np.random.default_rng(3)
    rows, heads, dim, rot = 13, 4, 32, 16
    freq, pos = frequencies(rot), rng.integers(0, 9000, rows).astype(np.int32)
    f, ps = dev.from_numpy(freq), dev.from_numpy(pos)
    size = 4 if dtype == N.NS_F32 else 2
    for start, ld, head in ((0, heads * 40, 40), (1, heads * 33 + 1, 33), (2, 34, 34 * rows), (8, 32, 32 * rows)):
        count = start + max(ld * rows, head * heads) + dim
        store, flat = put(dev, rng.standard_normal(count), dtype)
        out, old = put(dev, rng.standard_normal(count), dtype)
        at = start + np.arange(rows)[:, None, None] * ld + np.arange(heads)[:, None] * head + np.arange(dim)
        want, mag = turn(flat[at], pos, freq, True)
        N.call("ns_rotary", dev.handle, store.ptr + start * size, dtype, ld, head, ps.ptr, f.ptr, AMP, N.ROTARY_HALVES, 0, rows, heads, dim, rot, out.ptr + start * size, ld, head)
        dev.synchronize()
        got = get(out, count)
        assert (abs(got[at] - want) <= bound(want, mag, dtype)).all()
        rest = np.ones(count, bool)
        rest[at] = False
        assert np.array_equal(got[rest], old[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
def test_rotary_gradient(dev, halves):
    """The inverse is the gradient: <R x, g> = <x, R' g>, and R' g by differences of the call's own outputs."""
    rng = np.random.default_rng(11)
    rows, heads, dim, rot = 6, 3, 24, 14
    freq, pos = frequencies(rot), rng.integers(0, 100000, rows).astype(np.int32)
    f, ps = dev.from_numpy(freq), dev.from_numpy(pos)

    def call(x, inverse):
        a, b = dev.from_numpy(np.ascontiguousarray(x, np.float32)), dev.empty(x.size)
        N.call("ns_rotary", dev.handle, a.ptr, N.NS_F32, heads * dim, dim, ps.ptr, f.ptr, AMP, N.ROTARY_HALVES if halves else N.ROTARY_PAIRS, inverse, rows, heads, dim, rot,
               b.ptr, heads * dim, dim)
        dev.synchronize()
        return b.download(x.shape).astype(np.float64)

    x, g = (rng.standard_normal((rows, heads, dim)).astype(np.float32) for _ in range(2))
    y, gx = call(x, 0), call(g, 1)
    # each column of y and gx is within 4 * 2^-23 * AMP * (|a| + |b|)
    slack = 8 * 2.0 ** -23 * AMP * 2 * np.abs(x).max() * np.abs(g).sum()
    assert abs((y * g).sum() - (x.astype(np.float64) * gx).sum()) <= slack
    want, _ = turn(g, pos, freq, halves, sign=-1.0)
    assert np.abs(gx - want).max() <= 4 * 2.0 ** -23 * AMP * 2 * np.abs(g).max()
    step = 0.5
    for at in [(0, 0, 0), (1, 2, rot // 2), (5, 1, rot - 1), (3, 0, dim - 1)]:
        moved = x.copy()
        moved[at] += step
        h = np.float64(moved[at]) - np.float64(x[at])
        slope = ((call(moved, 0) - y) * g).sum() / h
        assert abs(slope - gx[at]) <= (2 * 4 * 2.0 ** -23 * AMP * 2 * (np.abs(x).max() + step) * np.abs(g).max() * 2) / step + 4 * 2.0 ** -23 * AMP * 2 * np.abs(g).max()


class _Cache(C.Structure):
    """What a cache's handle points to, for refusals that need no device."""
    _fields_ = [(n, C.c_int) for n in ("ordinal", "num_pages", "page_size", "heads", "head_dim")] + [("k", C.c_void_p), ("v", C.c_void_p), ("owns", C.c_bool)]


def refused(text, name, *args):
    with pytest.raises(N.NsError) as e:
        N.call(name, *args)
    assert e.value.code == 2 and text in str(e.value), str(e.value)


def test_rotary_refusals():
    A = 1 << 20
    good = dict(x=A, dtype=N.NS_BF16, x_ld=256, x_head=128, pos=A, freq=A, amplitude=1.0, layout=0, inverse=0, rows=4, heads=2, dim=128, rot=64, y=A, y_ld=256, y_head=128)

    def call(text, **other):
        refused(text, "ns_rotary", None, *{**good, **other}.values())

    call("device handle is null")              # whatever is right gets that far
    call("device handle is null", rows=0)
    call("null argument", x=0)
    call("null argument", pos=0)
    call("null argument", freq=0)
    call("null argument", y=0)
    call("dtype", dtype=N.NS_I8)
    call("layout", layout=2)
    call("rot_dims", rot=3)
    call("rot_dims", rot=0)
    call("rot_dims", rot=130)
    call("bad shape", heads=0)
    call("bad shape", dim=4098)
    call("bad shape", rows=-1)
    call("aligned", x=A + 1)
    call("aligned", pos=A + 2)
    call("in place", y_ld=512, x_ld=256)
    call("overlap", y=2 * A, y_head=64)
    call("overlap", y=2 * A, y_ld=255)
    call("overlap", y=2 * A, y_ld=128, y_head=128)
    call("negative pitch", x_ld=-256)
    call("2^31", x_ld=1 << 31)
    call("2^19 columns", heads=8192, x_head=0, y=2 * A, y_head=128, y_ld=1 << 20)
    call("device handle is null", y=2 * A, y_ld=128, y_head=512)      # rows inside heads
    call("device handle is null", y=2 * A, x_ld=0)                    # one row for all


def test_append_refusals():
    A = 1 << 20
    cache = _Cache(0, 8, 16, 2, 64, A, A, False)
    good = dict(cache=C.addressof(cache), src=A, splits=1, dtype=N.NS_BF16, ld=512, q_col=0, k_col=256, v_col=384, heads=4, freq=A, amplitude=1.0, layout=1, rot=32,
                offset=0, pos=A, lens=0, table=A, max_pages=4, batch=2, steps=3, q=A, q_ld=256)

    def call(text, **other):
        refused(text, "ns_kv_append_rotary", None, *{**good, **other}.values())

    call("device handle is null")
    call("device handle is null", q=0, heads=0, q_ld=0)
    call("device handle is null", batch=0)
    call("cache is null", cache=None)
    for name in ("src", "freq", "pos", "table"):
        call("null argument", **{name: 0})
    call("bad source", splits=2)
    call("bad source", dtype=N.NS_I8)
    call("layout", layout=-1)
    call("rot_dims", rot=66)
    call("columns outside", v_col=400)
    call("columns outside", q_col=300)
    call("columns outside", k_col=-1)
    call("queries of no heads", heads=0)
    call("shorter", q_ld=255)
    call("misaligned", pos=A + 2)
    call("bad shape", max_pages=0)
    call("bad shape", batch=-1)
    call("bad shape", batch=1 << 16, steps=1 << 15)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,group,rot,halves,page,splits,batch,steps", [
    (128, 2, 4, 128, True, 16, 0, 5, 1), (128, 8, 4, 128, True, 64, 2, 3, 1), (64, 1, 1, 64, False, 1, 1, 2, 9), (32, 3, 2, 20, True, 4, 3, 4, 5), (64, 2, 3, 30, False, 32, 8, 7, 1),
    (128, 1, 8, 6, True, 8, 0, 3, 40), (32, 2, 1, 2, False, 16, 1, 300, 1), (128, 4, 1, 64, True, 128, 4, 130, 1),
])
def test_append(dev, dim, kv, group, rot, halves, page, splits, batch, steps):
    rng = np.random.default_rng(dim + kv + rot + batch)
    heads, most = kv * group, 50
    pages = (most + steps + page - 1) // page + 1
    pos = rng.integers(0, most, batch).astype(np.int32)
    lens = rng.integers(0, steps + 1, batch).astype(np.int32)
    lens[0] = steps
    width, gap = (heads + 2 * kv) * dim, 24
    dtype = N.NS_F32 if splits else N.NS_BF16
    # the three fields in another order than usual, with columns between them
    k_col, q_col = 8, kv * dim + 16
    v_col, ld = q_col + heads * dim, width + gap
    src_store, src = put(dev, rng.standard_normal((max(1, splits), batch * steps, ld)), dtype)
    table = rng.permutation(batch * pages).astype(np.int32).reshape(batch, pages)
    old = [bf16(rng.standard_normal((batch * pages, kv, page, dim)))[0] for _ in range(2)]
    cache = C.c_void_p()
    N.call("ns_kv_cache_create", dev.handle, batch * pages, page, kv, dim, C.byref(cache))
    pools = [C.c_uint64(), C.c_uint64()]
    N.call("ns_kv_cache_pools", cache, C.byref(pools[0]), C.byref(pools[1]), None)
    dev.synchronize()
    for p, bits in zip(pools, old):
        N.call("ns_h2d", dev.handle, p, bits.ctypes.data_as(C.c_void_p), bits.nbytes)
    freq = frequencies(rot)
    f, ps, ls, tb, off = (dev.from_numpy(a) for a in (freq, pos, lens, table, np.array([70000], np.int32)))
    q_ld = heads * dim + 8
    q = dev.from_numpy(np.full(batch * steps * q_ld, 0x40E0, np.uint16))      # 7

    def append(**o):
        a = dict(offset=off.ptr, lens=ls.ptr, q=q.ptr, heads=heads) | o
        N.call("ns_kv_append_rotary", dev.handle, cache, src_store.ptr, max(1, splits), dtype, ld, q_col, k_col, v_col, a["heads"], f.ptr, AMP,
               N.ROTARY_HALVES if halves else N.ROTARY_PAIRS, rot, a["offset"], ps.ptr, a["lens"], tb.ptr, pages, batch, steps, a["q"], q_ld)
        dev.synchronize()
        got = []
        for p in pools:
            bits = np.empty((batch * pages, kv, page, dim), np.uint16)
            N.call("ns_d2h", dev.handle, bits.ctypes.data_as(C.c_void_p), p, bits.nbytes)
            got.append(bits)
        return got, q.download((batch * steps, q_ld))

    total = src.astype(np.float64).sum(0)
    rounding = max(0, splits - 1) * 2.0 ** -23 * np.abs(src).astype(np.float64).sum(0).max()      # of the slabs' sum in 32 bits
    at = (pos[:, None] + np.arange(steps)).reshape(-1)
    live = (np.arange(steps) < lens[:, None]).reshape(-1)
    fields = [total[:, c:c + n * dim].reshape(-1, n, dim) for c, n in ((q_col, heads), (k_col, kv), (v_col, kv))]
    tq, sq = turn(fields[0], at + 70000, freq, halves)
    tk, sk = turn(fields[1], at + 70000, freq, halves)
    (k, v), qs = append()
    qs = qs[:, :].reshape(-1, q_ld)
    got_q = values(qs[:, :heads * dim]).reshape(-1, heads, dim)
    assert (abs(got_q - tq) <= bound(tq, sq, N.NS_BF16) + 2 * rounding + 2.0 ** -133)[live].all()
    assert (got_q[~live] == 7.0).all() and (values(qs[:, heads * dim:]) == 7.0).all()
    want = [values(b).astype(np.float64) for b in old]
    slack = [np.zeros(w.shape) for w in want]
    for r in np.flatnonzero(live):
        b = r // steps
        pg, row = table[b, at[r] // page], at[r] % page
        want[0][pg, :, row], want[1][pg, :, row] = tk[r], fields[2][r]
        slack[0][pg, :, row] = bound(tk[r], sk[r], N.NS_BF16) + 2 * rounding
        slack[1][pg, :, row] = 2.0 ** -8 * abs(fields[2][r]) + rounding
    for bits, w, t in zip((k, v), want, slack):
        assert (abs(values(bits) - w) <= t).all()
    # keys and values alone give the same pools; without an offset and lens every token goes in, turned to its own position
    assert all(np.array_equal(a, b) for a, b in zip(append(q=0, heads=0)[0], (k, v)))
    (k, v), qs = append(offset=0, lens=0)
    tq, sq = turn(fields[0], at, freq, halves)
    got_q = values(np.ascontiguousarray(qs[:, :heads * dim])).reshape(-1, heads, dim)
    assert (abs(got_q - tq) <= bound(tq, sq, N.NS_BF16) + 2 * rounding).all()
    r = batch * steps - 1
    row = values(np.ascontiguousarray(v[table[r // steps, at[r] // page], :, at[r] % page]))
    assert (abs(row - fields[2][r]) <= 2.0 ** -8 * abs(fields[2][r]) + rounding).all()
    N.call("ns_kv_cache_destroy", cache)


@pytest.mark.gpu
def test_append_outside_the_cache(dev):
    """A negative position, one behind the page table, pages that are none of the pool's: only those tokens are left out, and the next synchronisation says so."""
    dim, kv, heads, page, pages, batch, steps = 32, 1, 2, 4, 2, 5, 2
    rng = np.random.default_rng(5)
    ld = (heads + 2 * kv) * dim
    src_store, src = put(dev, rng.standard_normal((batch * steps, ld)), N.NS_F32)
    pos = np.array([-1, 7, 2, 3, -2 ** 31], np.int32)
    table = np.array([[0, 1], [2, 3], [4, 99], [-5, 5], [6, 7]], np.int32)
    cache = C.c_void_p()
    N.call("ns_kv_cache_create", dev.handle, 8, page, kv, dim, C.byref(cache))
    vp = C.c_uint64()
    N.call("ns_kv_cache_pools", cache, None, C.byref(vp), None)
    freq = frequencies(8)
    f, ps, tb, q = dev.from_numpy(freq), dev.from_numpy(pos), dev.from_numpy(table), dev.zeros(batch * steps * heads * dim, N.NS_BF16)
    dev.synchronize()
    N.call("ns_kv_append_rotary", dev.handle, cache, src_store.ptr, 1, N.NS_F32, ld, 0, heads * dim, (heads + kv) * dim, heads, f.ptr, 1.0, N.ROTARY_PAIRS, 8, 0, ps.ptr, 0,
           tb.ptr, pages, batch, steps, q.ptr, heads * dim)
    with pytest.raises(N.NsError) as e:
        dev.synchronize()
    assert e.value.code == 4
    dev.synchronize()
    bits = np.empty((8, kv, page, dim), np.uint16)
    N.call("ns_d2h", dev.handle, bits.ctypes.data_as(C.c_void_p), vp, bits.nbytes)
    want = np.zeros_like(bits)
    v = bf16(src[:, (heads + kv) * dim:])[0]
    # sequence 0: -1 out, 0 in; 1: 7 in, 8 behind the table; 2: positions 2, 3 in page 4; 3: 3 in page -5, 4 in page 5; 4: far below
    want[0, 0, 0], want[3, 0, 3], want[4, 0, 2], want[4, 0, 3], want[5, 0, 0] = v[1], v[2], v[4], v[5], v[7]
    assert np.array_equal(bits, want)
    N.call("ns_kv_cache_destroy", cache)
