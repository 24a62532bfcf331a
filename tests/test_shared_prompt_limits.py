"""The operators of a step over a shared prompt where their forms change: which kernel reads the prefix, with few rows, odd ends, scales that are not positive and tables
with room behind the lengths; caches and matrices of more than 2^31 elements.  Tolerances are those of the operators' own tests."""
import ctypes as C

import numpy as np
import pytest

from nn_b200 import native as N

from .test_attention_shared import Setup
from .test_rotary import AMP, bf16, bound, frequencies, turn, values


def on_the_tensor_cores(s):
    """Whether the prefix of a call of this shape is read by the tensor-core kernel, seen by its rounding of weights to bf16.  Even keys of the prefix weigh 1 and odd ones
    1 - 2^-12, whose nearest bf16 is 1, with values of 1 and -1 (a last one without a partner 0), own pages are not seen: the sum of weighted values is exactly 0 with weights
    rounded to bf16, and some 2^-13 with weights in two halves."""
    kept = s.k.copy(), s.v.copy(), s.q.copy(), s.pos.copy(), s.scale
    s.k[:], s.v[:], s.q[:] = 0, 0, 0
    s.q[..., 0], s.scale = 0x3F80, 1.0
    s.pos = np.full_like(s.pos, -s.steps)
    j = np.arange(s.prefix)
    page, row = s.prefix_table[j // s.page], j % s.page
    s.k[page, :, row, 0] = np.where(j % 2 == 0, 0, 0xB980)[:, None]                 # -2^-12
    s.v[page, :, row] = np.where(j % 2 == 0, 0x3F80, 0xBF80)[:, None, None]
    if s.prefix % 2:
        s.v[page[-1], :, row[-1]] = 0
    s.upload()
    got = values(s.call())
    s.k, s.v, s.q, s.pos, s.scale = kept
    assert (got == 0).all() or (abs(got - 2.0 ** -13) < 2.0 ** -16).all()
    return bool((got == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,group,page,batch,prefix", [
    (32, 2, 8, 16, 60, 7301), (32, 1, 8, 32, 120, 7303), (32, 2, 8, 16, 60, 7297), (32, 2, 8, 64, 60, 7423), (32, 2, 8, 256, 60, 7425),       # tails of 5, 7, 1, 127 and 1 keys
    (64, 2, 8, 16, 60, 3713), (64, 2, 8, 8, 60, 3839), (128, 2, 8, 32, 60, 1793), (128, 2, 8, 8, 60, 1919)])
def test_a_prefix_that_ends_inside_a_block(dev, dim, kv, group, page, batch, prefix):
    """The tensor-core kernel with an odd number of keys in its last block: what lies behind the prefix, NaN or infinite, reaches no row."""
    own = [1 + (7 * b) % 45 for b in range(batch)]
    s = Setup(dev, dim, kv, group, page, batch, 1, prefix, own)
    assert on_the_tensor_cores(s)
    s.upload()
    clean = s.call()
    s.check(clean)
    last, row = s.prefix_table[-1], (prefix - 1) % page + 1
    for bad in (0x7FC0, 0x7F80, 0xFF80):
        s.k[last, :, row:], s.v[last, :, row:] = bad, bad
        s.upload()
        assert np.array_equal(s.call(), clean)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,group,page,batch,prefix,tiles", [
    (128, 16, 17, 64, 1, 14800, True), (128, 16, 23, 64, 1, 11000, True), (64, 8, 12, 16, 2, 17800, True), (128, 8, 11, 8, 3, 6500, True), (128, 4, 9, 128, 7, 6800, True),
    (32, 16, 17, 32, 1, 59000, True), (32, 16, 33, 16, 1, 12903, True), (128, 16, 16, 64, 1, 20000, False), (128, 16, 17, 64, 1, 14500, False), (128, 8, 11, 4, 3, 6500, False)])
def test_few_rows_a_head(dev, dim, kv, group, page, batch, prefix, tiles):
    """17, 23, 24, 33 and 63 rows a key/value head on the tensor cores: rows that fill no warp, warps without rows.  16 rows, little work and small pages stay with the other kernel."""
    s = Setup(dev, dim, kv, group, page, batch, 1, prefix, [30] * batch)
    assert on_the_tensor_cores(s) == tiles
    s.upload()
    s.check(s.call())
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.125])
@pytest.mark.parametrize("dim,kv,group,batch,steps,prefix", [(64, 2, 3, 4, 3, 90), (128, 2, 8, 40, 1, 2700), (32, 2, 8, 60, 1, 7300)])
def test_scales_that_are_not_positive(dev, dim, kv, group, batch, steps, prefix, scale):
    s = Setup(dev, dim, kv, group, 16, batch, steps, prefix, [40] * batch)
    s.scale = scale
    s.upload()
    s.check(s.call())
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,group,page,batch,steps,prefix,own,room_prefix,room_own", [
    (64, 2, 4, 16, 3, 1, 500, 37, 0, 8192), (64, 2, 4, 16, 3, 1, 500, 37, 8192, 8192), (64, 16, 1, 16, 8, 5, 2500, 300, 2560, 4096), (64, 16, 1, 16, 8, 5, 1250, 300, 8192, 4096),
    (128, 2, 4, 64, 40, 1, 300, 90, 40000, 0), (128, 2, 4, 64, 40, 1, 6000, 90, 0, 30000), (32, 2, 8, 16, 50, 2, 1, 2, 30000, 9000), (128, 1, 4, 32, 16, 1, 512, 20, 512, 32768)])
def test_tables_with_room(dev, dim, kv, group, page, batch, steps, prefix, own, room_prefix, room_own):
    """Tables that hold far more positions than there are; the entries behind the lengths name no pages and are not read."""
    s = Setup(dev, dim, kv, group, page, batch, steps, prefix, [max(steps, own - 3 * b) for b in range(batch)])
    more = max(0, (room_prefix + page - 1) // page - s.prefix_pages)
    junk = lambda *shape: s.rng.choice(np.array([-1, s.n_pages, 2 ** 31 - 1, -2 ** 31], np.int64), shape).astype(np.int32)
    s.prefix_table = np.concatenate([s.prefix_table, junk(more)])
    more = max(0, (room_own + page - 1) // page - s.max_pages)
    # (a shorter sequence's pages behind its length are not read either)
    for b in range(batch):
        s.table[b, (s.pos[b] + steps + page - 1) // page:] = -1
    want_table = np.where(s.table < 0, 0, s.table)
    s.table = np.concatenate([s.table, junk(batch, more)], 1)
    s.prefix_pages, s.max_pages = len(s.prefix_table), s.table.shape[1]
    s.upload()
    got = s.call()                             # (a page that is none, were it read, would be reported here)
    s.prefix_table, s.table = s.prefix_table[:(prefix + page - 1) // page], want_table
    s.check(got)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,splits", [(N.NS_BF16, 1), (N.NS_F32, 2)])
def test_append_to_a_pool_of_more_than_2_31_elements(dev, dtype, splits):
    """The last pages of such a pool, and the first ones, which a wrapped index would reach."""
    rng = np.random.default_rng(8)
    dim, kv, heads, page, batch, steps = 128, 8, 16, 64, 3, 70
    n = 2 ** 31 // (kv * page * dim) + 64
    cache, pools = C.c_void_p(), [C.c_uint64(), C.c_uint64()]
    N.call("ns_kv_cache_create", dev.handle, n, page, kv, dim, C.byref(cache))
    N.call("ns_kv_cache_pools", cache, C.byref(pools[0]), C.byref(pools[1]), None)
    dev.synchronize()
    table = (n - 1 - np.arange(batch * 2, dtype=np.int32)).reshape(batch, 2)
    pos = np.array([0, 10, 58], np.int32)
    ld = (heads + 2 * kv) * dim
    x = rng.standard_normal((splits, batch * steps, ld))
    bits, rounded = bf16(x)
    x = rounded if dtype == N.NS_BF16 else x.astype(np.float32)
    freq = frequencies(dim)
    src, f, ps, tb, q = dev.from_numpy(bits if dtype == N.NS_BF16 else x), dev.from_numpy(freq), dev.from_numpy(pos), dev.from_numpy(table), dev.zeros(batch * steps * heads * dim, N.NS_BF16)
    size = kv * page * dim * 2
    zero = np.zeros((64, kv, page, dim), np.uint16)
    for p in pools:
        for first in (0, n - 64):
            N.call("ns_h2d", dev.handle, p.value + first * size, zero.ctypes.data_as(C.c_void_p), zero.nbytes)
    N.call("ns_kv_append_rotary", dev.handle, cache, src.ptr, splits, dtype, ld, 0, heads * dim, (heads + kv) * dim, heads, f.ptr, AMP, N.ROTARY_HALVES, dim, 0, ps.ptr, 0, tb.ptr, 2,
           batch, steps, q.ptr, heads * dim)
    dev.synchronize()
    total = x.astype(np.float64).sum(0)
    rounding = (splits - 1) * 2.0 ** -23 * np.abs(x).astype(np.float64).sum(0).max()
    at = (pos[:, None] + np.arange(steps)).reshape(-1)
    tk, sk = turn(total[:, heads * dim:(heads + kv) * dim].reshape(-1, kv, dim), at, freq, True)
    tv = total[:, (heads + kv) * dim:].reshape(-1, kv, dim)
    for p, rows, slack in ((pools[0], tk, bound(tk, sk, N.NS_BF16) + 2 * rounding), (pools[1], tv, 2.0 ** -8 * abs(tv) + rounding)):
        got = np.empty((2, 64, kv, page, dim), np.uint16)
        for i, first in enumerate((0, n - 64)):
            N.call("ns_d2h", dev.handle, got[i].ctypes.data_as(C.c_void_p), p.value + first * size, got[i].nbytes)
        assert (got[0] == 0).all()
        want, tol = np.zeros((64, kv, page, dim)), np.zeros((64, kv, page, dim))
        for r in range(batch * steps):
            pg, row = table[r // steps, at[r] // page] - (n - 64), at[r] % page
            want[pg, :, row], tol[pg, :, row] = rows[r], slack[r]
        assert (abs(values(got[1]) - want) <= tol).all()
    N.call("ns_kv_cache_destroy", cache)


@pytest.mark.gpu
@pytest.mark.parametrize("heads_outside", [False, True])
def test_rotary_of_more_than_2_31_elements(dev, heads_outside):
    """In place, rows whose elements lie beyond 2^31; the others have negative positions and stay."""
    rng = np.random.default_rng(6)
    heads, dim = 4, 1024
    rows = 2 ** 31 // (heads * dim) + 1000
    x = dev.empty(rows * heads * dim, N.NS_BF16)
    ld, head = (dim, rows * dim) if heads_outside else (heads * dim, dim)
    some = np.array([0, 1, rows // 2, rows - 900, rows - 1])
    pos = np.full(rows, -1, np.int32)
    pos[some] = rng.integers(0, 100000, len(some))
    bits, rounded = bf16(rng.standard_normal((len(some), heads, dim)))
    freq = frequencies(dim)
    f, ps = dev.from_numpy(freq), dev.from_numpy(pos)
    for i, r in enumerate(some):
        for h in range(heads):
            N.call("ns_h2d", dev.handle, x.ptr + (int(r) * ld + h * head) * 2, bits[i, h].ctypes.data_as(C.c_void_p), dim * 2)
    # rows beside them, which stay
    beside = np.array([2, rows // 2 + 1, rows - 2])
    kept = np.full(dim, 0x40E0, np.uint16)
    for r in beside:
        for h in range(heads):
            N.call("ns_h2d", dev.handle, x.ptr + (int(r) * ld + h * head) * 2, kept.ctypes.data_as(C.c_void_p), dim * 2)
    N.call("ns_rotary", dev.handle, x.ptr, N.NS_BF16, ld, head, ps.ptr, f.ptr, AMP, N.ROTARY_HALVES, 0, rows, heads, dim, dim, x.ptr, ld, head)
    dev.synchronize()
    want, mag = turn(rounded, pos[some], freq, True)
    got = np.empty(dim, np.uint16)
    read = lambda r, h: N.call("ns_d2h", dev.handle, got.ctypes.data_as(C.c_void_p), x.ptr + (int(r) * ld + h * head) * 2, dim * 2)
    for i, r in enumerate(some):
        for h in range(heads):
            read(r, h)
            assert (abs(values(got) - want[i, h]) <= bound(want[i, h], mag[i, h], N.NS_BF16)).all()
    for r in beside:
        for h in range(heads):
            read(r, h)
            assert (got == 0x40E0).all()
