"""ns_attention_shared against softmax attention in 64 bits.

Tolerance of an output o = sum p_j v_j with normalised weights p: half a bf16 step of the result, 2^-8 |o|; the weights enter P.V rounded to bf16, half a step each,
2^-8 sum p_j |v_j|; a score is a 32-bit sum of dim products, off by (dim + 4) 2^-24 sum |q k| scale, which shifts weights and their sum by that fraction,
and exponentials, sums and folds add less than 2^-18: 2 ((dim + 4) 2^-24 max sum |q k| scale + 2^-18) sum p_j |v_j|."""
import ctypes as C

import numpy as np
import pytest

from nn_b200 import native as N

from .test_rotary import _Cache, bf16, refused, values

KEEP = 0x40E0      # 7: what an output holds before the call


class Setup:
    """A cache of random keys and values whose pages lie in any order, and what a call needs."""

    def __init__(self, dev, dim, kv, group, page, batch, steps, prefix, own, seed=0, spare=3, std=1.0):
        rng = self.rng = np.random.default_rng([dim, kv, group, page, batch, steps, prefix, max(own, default=0), seed])
        self.dev, self.dim, self.kv, self.heads, self.page, self.batch, self.steps, self.prefix = dev, dim, kv, kv * group, page, batch, steps, prefix
        self.pos = np.array(own, np.int32) - steps          # position of the first new token: the sequence has own[b] in all
        self.prefix_pages = (prefix + page - 1) // page
        self.max_pages = max((max(own, default=0) + page - 1) // page, 0)
        n = self.prefix_pages + batch * self.max_pages + spare
        order = rng.permutation(n).astype(np.int32)
        self.prefix_table, self.table = order[:self.prefix_pages], order[self.prefix_pages:self.prefix_pages + batch * self.max_pages].reshape(batch, self.max_pages)
        self.k, self.v = (bf16(std * rng.standard_normal((n, kv, page, dim)))[0] for _ in range(2))
        self.q = bf16(rng.standard_normal((batch * steps, self.heads, dim)))[0]
        self.scale = dim ** -0.5
        self.lens = None
        self.n_pages = n
        self.cache = C.c_void_p()
        N.call("ns_kv_cache_create", dev.handle, n, page, kv, dim, C.byref(self.cache))

    def upload(self):
        self.dev.synchronize()
        for p, bits in zip(self.pools(), (self.k, self.v)):
            N.call("ns_h2d", self.dev.handle, p, bits.ctypes.data_as(C.c_void_p), bits.nbytes)

    def pools(self):
        pools = [C.c_uint64(), C.c_uint64()]
        N.call("ns_kv_cache_pools", self.cache, C.byref(pools[0]), C.byref(pools[1]), None)
        return pools

    def args(self, o_pad=0):
        up = lambda a: self.dev.from_numpy(np.ascontiguousarray(a)) if a is not None and a.size else None
        self.kept = [up(a) for a in (self.q.reshape(-1), self.prefix_table, np.array([self.prefix], np.int32), self.table, self.pos, self.lens)]
        at = [0 if s is None else s.ptr for s in self.kept]
        self.o_ld = self.heads * self.dim + o_pad
        self.o = self.dev.from_numpy(np.full(self.batch * self.steps * self.o_ld, KEEP, np.uint16))
        own = self.max_pages > 0
        return (self.dev.handle, self.cache, at[0], self.heads * self.dim, self.o.ptr, self.o_ld, self.heads, at[1] if self.prefix_pages else 0, self.prefix_pages,
                at[2] if self.prefix_pages else 0, at[3] if own else 0, self.max_pages, at[4] if own else 0, at[5], self.batch, self.steps, self.scale)

    def call(self, o_pad=0):
        N.call("ns_attention_shared", *self.args(o_pad))
        self.dev.synchronize()
        return self.read()

    def read(self):
        bits = self.o.download((self.batch * self.steps, self.o_ld))
        assert (bits[:, self.heads * self.dim:] == KEEP).all()
        return bits[:, :self.heads * self.dim].reshape(self.batch, self.steps, self.heads, self.dim)

    def want(self):
        """-> (outputs, tolerance) in 64 bits; NaN where the row is padding"""
        k, v = values(self.k).astype(np.float64), values(self.v).astype(np.float64)
        rows = lambda pool, table: pool[table].transpose(1, 0, 2, 3).reshape(self.kv, -1, self.dim)
        q = values(self.q).astype(np.float64).reshape(self.batch, self.steps, self.kv, -1, self.dim)
        out = np.full((self.batch, self.steps, self.kv, q.shape[3], self.dim), np.nan)
        tol = np.zeros_like(out)
        pk, pv = (rows(x, self.prefix_table)[:, :self.prefix] for x in (k, v))
        for b in range(self.batch):
            ok, ov = (rows(x, self.table[b]) for x in (k, v))
            for i in range(self.steps):
                if self.lens is not None and i >= self.lens[b]:
                    continue
                n = max(0, int(self.pos[b]) + i + 1) if self.max_pages else 0
                kk, vv = np.concatenate([pk, ok[:, :n]], 1), np.concatenate([pv, ov[:, :n]], 1)
                if kk.shape[1] == 0:
                    out[b, i] = 0
                    continue
                s = np.einsum("kgd,kjd->kgj", q[b, i], kk) * self.scale
                size = np.einsum("kgd,kjd->kgj", abs(q[b, i]), abs(kk)).max() * abs(self.scale)
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[b, i] = w @ vv
                tol[b, i] = 2.0 ** -8 * abs(out[b, i]) + (2.0 ** -8 + 2 * ((self.dim + 4) * 2.0 ** -24 * size + 2.0 ** -18)) * (w @ abs(vv))
        shape = (self.batch, self.steps, self.heads, self.dim)
        return out.reshape(shape), tol.reshape(shape)

    def check(self, bits):
        want, tol = self.want()
        live = ~np.isnan(want)
        assert (bits[~live] == KEEP).all()
        got = values(bits).astype(np.float64)
        assert not np.isnan(got).any()
        far = np.where(live, abs(got - want) - tol, 0)
        assert far.max() <= 0, (np.argwhere(far > 0)[:5], far.max())

    def close(self):
        N.call("ns_kv_cache_destroy", self.cache)


CASES = [  # dim, kv heads, group, page, prefix, own positions of each sequence with the new ones, steps
    (128, 2, 4, 64, 300, [40, 1, 130], 1),
    (128, 1, 8, 16, 1, [1], 1),
    (64, 2, 1, 16, 500, [37, 2, 19, 64], 1),
    (32, 3, 2, 8, 129, [5, 200], 1),
    (32, 1, 3, 4, 77, [9] * 20, 1),
    (64, 1, 6, 1, 33, [3, 17], 2),
    (128, 2, 2, 2, 50, [11, 12, 13], 4),
    (64, 4, 4, 128, 1000, [130, 260, 7], 7),
    (128, 1, 4, 32, 2000, [33] * 40, 1),            # 160 rows: more than one tile of any kernel
    (128, 2, 8, 64, 700, [100] * 33, 1),            # 264 rows
    (64, 1, 16, 16, 513, [65, 31] * 10, 3),
    (32, 2, 4, 16, 4097, [300] * 16, 2),
    (128, 8, 1, 16, 63, [1] * 5, 1),
    (128, 1, 1, 16, 0, [100, 3], 1),                # no prefix
    (64, 2, 4, 64, 0, [4000, 1, 700], 1),
    (128, 2, 4, 16, 640, [], 1),                    # (filled in below: no pages of their own)
    (32, 1, 40, 16, 200, [20, 25], 1),              # groups of more heads than a tile has rows
    (128, 1, 2, 256, 900, [300, 20], 70),           # a portion of a prompt
    (64, 2, 3, 64, 3000, [90] * 50, 1),
    # work enough for the tensor-core kernel, 1 700 000 products of 128 columns, and some short of it
    (128, 1, 8, 64, 2000, [40, 1] * 32, 1),         # 512 rows: two tiles
    (128, 2, 4, 16, 3333, [17] * 32, 1),            # 128 rows: the groups take turns
    (128, 4, 2, 8, 2600, [5, 60] * 20, 1),          # 80 rows
    (64, 2, 8, 32, 4097, [33] * 33, 1),             # 264 rows: a group without rows
    (64, 8, 1, 128, 5000, [9, 200] * 16, 2),        # 64 rows, two tokens each
    (128, 1, 3, 256, 1153, [70] * 60, 5),           # 900 rows in groups of three
    (128, 1, 12, 64, 129, [1] * 600, 1),            # 7200 rows, two blocks
    (32, 2, 8, 16, 4099, [5, 33] * 16, 1),          # heads of 32 columns lie two keys a row
    (32, 1, 16, 64, 3001, [20] * 70, 1),
    (32, 4, 2, 256, 5000, [3] * 20, 4),
    (128, 2, 4, 16, 4001, [17] * 32, 1),            # 128 rows: the groups take turns
    (128, 4, 2, 8, 3300, [5, 60] * 20, 1),          # 80 rows
    (128, 1, 12, 64, 145, [1] * 600, 1),            # 7200 rows, two blocks
    (32, 2, 8, 16, 8200, [5, 33] * 16, 1),
    (32, 1, 16, 64, 3801, [20] * 70, 1),
    (32, 4, 2, 256, 6600, [3] * 20, 4),
    (128, 1, 8, 64, 3500, [40, 1] * 32, 1),
    (128, 2, 4, 16, 7000, [17] * 32, 1),
    (128, 4, 2, 8, 5500, [5, 60] * 20, 1),
    (64, 2, 8, 32, 7000, [33] * 33, 1),
    (64, 8, 1, 128, 7000, [9, 200] * 16, 2),
    (128, 1, 3, 256, 2050, [70] * 60, 5),
    (128, 1, 12, 64, 250, [1] * 600, 1),
    (32, 2, 8, 16, 13500, [5, 33] * 16, 1),
    (32, 1, 16, 64, 6200, [20] * 70, 1),
    (32, 4, 2, 256, 11000, [3] * 20, 4),
    (64, 1, 8, 16, 300, [], 1),                     # (filled in below: many sequences without pages of their own)
]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,group,page,prefix,own,steps", CASES)
def test_outputs(dev, dim, kv, group, page, prefix, own, steps):
    s = Setup(dev, dim, kv, group, page, len(own) or (700 if prefix == 300 else 6), steps, prefix, own)
    if not own:
        s.pos = np.zeros(s.batch, np.int32)
    s.upload()
    s.check(s.call())
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page,batch", [(128, 64, 3), (64, 16, 40), (32, 8, 3), (128, 16, 70), (64, 4, 5)])
def test_padding_and_rows_that_see_nothing(dev, dim, page, batch):
    """Padded rows stay as they are; negative positions leave the prefix, without one zeros; positions beyond a table do not count; outputs with a gap."""
    for prefix in (0, 75) if batch != 70 else (0, 1900):
        s = Setup(dev, dim, 2, 4, page, batch, 3, prefix, [41] * batch, seed=prefix)
        s.lens = s.rng.integers(0, 4, batch).astype(np.int32)
        s.pos = s.rng.integers(-4, 38, batch).astype(np.int32)
        s.pos[0], s.lens[:3], s.pos[1], s.pos[2] = -2, 3, -2 ** 31, -3
        s.upload()
        s.check(s.call(o_pad=24))
        s.pos[0], s.lens[:] = 2 ** 31 - 1, 3
        bits = s.call()
        s.pos[0] = s.max_pages * page - 1            # what it comes to: the whole table, for each of its tokens
        want, tol = s.want()
        assert (abs(values(bits[0, 0]) - want[0, 0]) <= tol[0, 0]).all()
        s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,group,page,batch,prefix", [(128, 2, 4, 64, 5, 300), (64, 1, 2, 16, 3, 65), (32, 2, 4, 4, 4, 130), (128, 1, 4, 16, 64, 1000), (64, 1, 4, 32, 50, 77),
                                                              (128, 1, 8, 16, 64, 1700), (64, 2, 8, 64, 40, 3001), (128, 2, 4, 64, 16, 6500), (128, 1, 8, 256, 60, 2050), (32, 2, 8, 16, 60, 3501), (32, 1, 8, 32, 120, 3333), (128, 1, 8, 16, 64, 2001), (64, 2, 8, 64, 40, 3301), (128, 2, 4, 64, 16, 8000),
                                                              (128, 1, 8, 256, 60, 2150), (32, 2, 8, 16, 60, 4400), (32, 1, 8, 32, 120, 4300), (128, 1, 8, 16, 64, 3500), (64, 2, 8, 64, 40, 5500),
                                                              (128, 2, 4, 64, 16, 14000), (128, 1, 8, 256, 60, 3700), (32, 2, 8, 16, 60, 7300), (32, 1, 8, 32, 120, 7300)])
def test_what_is_not_seen_does_not_count(dev, dim, kv, group, page, batch, prefix):
    """Behind the last position of the prefix and of every sequence, and in pages nobody names: NaN, infinities, the type's lowest value."""
    own = [1 + (7 * b) % 45 for b in range(batch)]
    s = Setup(dev, dim, kv, group, page, batch, 1, prefix, own)
    s.upload()
    clean = s.call()
    s.check(clean)
    kept_k, kept_v = s.k.copy(), s.v.copy()
    for bad in (0x7FC0, 0x7F80, 0xFF80, 0xFF7F):
        k, v = np.full_like(s.k, bad), np.full_like(s.v, bad)
        for table, n in [(s.prefix_table, prefix)] + [(s.table[b], own[b]) for b in range(batch)]:
            for j in range(n):
                k[table[j // page], :, j % page], v[table[j // page], :, j % page] = kept_k[table[j // page], :, j % page], kept_v[table[j // page], :, j % page]
        s.k, s.v = k, v
        s.upload()
        assert np.array_equal(s.call(), clean)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page,batch,prefix", [(128, 64, 2, 200), (64, 16, 40, 200), (128, 16, 70, 200), (32, 16, 5, 200), (128, 16, 70, 3000), (64, 64, 30, 14000), (32, 16, 250, 3300), (128, 16, 70, 3700),
                                                    (64, 64, 30, 17200), (32, 16, 250, 4200), (128, 16, 70, 6200), (64, 64, 30, 29000), (32, 16, 250, 7000)])
def test_scores_that_are_no_numbers(dev, dim, page, batch, prefix):
    """A NaN among the keys a row sees makes the row NaN, and only the rows that see it; a value of NaN too."""
    for where in ("prefix", "own"):
        for what in "kv":
            s = Setup(dev, dim, 1, 4, page, batch, 1, prefix, [50] * batch)
            table, j = (s.prefix_table, 130) if where == "prefix" else (s.table[1], 20)
            getattr(s, what)[table[j // page], 0, j % page, 3] = 0x7FC0
            s.upload()
            got = values(s.call())
            touched = np.zeros(batch, bool)
            touched[:] = where == "prefix"
            touched[1] = True
            assert np.isnan(got[touched][..., 3]).all() and (what == "v" or np.isnan(got[touched]).all())
            assert not np.isnan(got[~touched]).any()
            s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [0x7FC0, 0x7F80, 0xFF80])
@pytest.mark.parametrize("dim,group,steps,batch,prefix", [(128, 2, 3, 2, 40), (64, 4, 7, 3, 0), (32, 1, 20, 2, 77), (128, 4, 2, 40, 2600), (128, 4, 2, 40, 2900), (64, 8, 5, 4, 0)])
def test_a_later_token_of_the_call_does_not_reach_an_earlier_one(dev, dim, group, steps, batch, prefix, bad):
    """Keys and values of a token that are no numbers: the tokens before it in the same call do not see it."""
    for own in (steps, 37, 130):
        s = Setup(dev, dim, 2, group, 16, batch, steps, prefix, [own] * batch)
        s.upload()
        clean = s.call()
        s.check(clean)
        for i in (1, steps - 1):               # the call's i-th token
            for what in "kv":
                kept = getattr(s, what).copy()
                j = own - steps + i
                getattr(s, what)[s.table[0][j // 16], 1, j % 16] = bad
                s.upload()
                got = s.call()
                assert np.array_equal(got[1:], clean[1:]) and np.array_equal(got[0, :, :group], clean[0, :, :group])
                with np.errstate(invalid="ignore"):
                    want, tol = s.want()
                assert (abs(values(got[0, :i]) - want[0, :i]) <= tol[0, :i]).all()
                if bad == 0x7FC0:
                    assert np.isnan(values(got[0, i:, group:])).all()
                setattr(s, what, kept)
        s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page,batch,prefix", [(128, 16, 3, 100), (64, 64, 40, 500), (128, 32, 100, 1111), (32, 4, 4, 50), (128, 16, 40, 2600), (64, 8, 150, 1500), (128, 128, 64, 1600), (32, 16, 120, 3400),
                                                    (128, 16, 40, 3300), (64, 8, 150, 1800), (128, 128, 64, 2100), (32, 16, 120, 4400),
                                                    (128, 16, 40, 5500), (64, 8, 150, 2950), (128, 128, 64, 3400), (32, 16, 120, 7300)])
def test_pages_outside_the_pool(dev, dim, page, batch, prefix):
    """Positions of a page that is none are left out and reported."""
    s = Setup(dev, dim, 2, 4, page, batch, 1, prefix, [60] * batch)
    s.upload()
    gone_p, gone_o = s.prefix_pages // 2, 0
    s.prefix_table[gone_p] = s.n_pages
    s.table[1, gone_o] = -1
    N.call("ns_attention_shared", *s.args())
    with pytest.raises(N.NsError) as e:
        dev.synchronize()
    assert e.value.code == 4
    dev.synchronize()
    got = s.read()
    # the same without those positions: the tables closed up
    full_table, full_pos = s.table, s.pos.copy()
    s.prefix_table = np.delete(s.prefix_table, gone_p)
    s.prefix -= page
    want, tol = s.want()
    for b in range(0, batch, 7):
        assert b == 1 or (abs(values(got[b]) - want[b]) <= tol[b]).all()
    s.table = np.concatenate([np.delete(full_table[1], gone_o), full_table[1][gone_o:gone_o + 1] * 0]).reshape(1, -1).repeat(batch, 0)
    s.pos = full_pos - page if page <= 59 else np.full_like(full_pos, -1)
    want, tol = s.want()
    assert (abs(values(got[1]) - want[1]) <= tol[1]).all()
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group,batch,prefix", [(128, 4, 40, 900), (64, 1, 3, 900), (128, 4, 40, 6000), (64, 4, 100, 4100), (128, 4, 40, 11000), (64, 4, 100, 8600), (32, 8, 100, 9000)])
def test_values_alike(dev, dim, group, batch, prefix):
    """Weights add up to one: values that are all alike come back within the rounding of the weights and of the output."""
    s = Setup(dev, dim, 1, group, 64, batch, 1, prefix, [70] * batch)
    s.v[:] = bf16(np.broadcast_to(np.linspace(-3, 3, dim, dtype=np.float32), s.v.shape))[0]
    s.upload()
    got, want = values(s.call()).astype(np.float64), values(s.v[0, 0, 0]).astype(np.float64)
    assert (abs(got - want) <= (2 * 2.0 ** -8 + 2.0 ** -16) * abs(want)).all()
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,prefix", [(2, 200), (40, 200), (20, 1300), (40, 1400)])
def test_a_pool_of_more_than_2_31_elements(dev, batch, prefix):
    dim, kv, page = 128, 8, 64
    n = 2 ** 31 // (kv * page * dim) + 200
    s = Setup(dev, dim, kv, 4, page, batch, 1, prefix, [70] * batch)
    N.call("ns_kv_cache_destroy", s.cache)
    s.cache = C.c_void_p()
    N.call("ns_kv_cache_create", dev.handle, n, page, kv, dim, C.byref(s.cache))
    s.upload()                                       # the first pages
    want = s.call()
    s.check(want)
    # the same pages at the pool's end
    size = kv * page * dim * 2
    for p, bits in zip(s.pools(), (s.k, s.v)):
        N.call("ns_h2d", dev.handle, p.value + (n - s.n_pages) * size, bits.ctypes.data_as(C.c_void_p), bits.nbytes)
    s.prefix_table, s.table = s.prefix_table + (n - s.n_pages), s.table + (n - s.n_pages)
    assert np.array_equal(s.call(), want)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("longer", [False, True])
def test_replays_with_other_lengths(dev, longer):
    """A recorded call follows the device's positions, length and tables; two recorded calls share the scratch block in stream order."""
    sets = [Setup(dev, 128, 2, 4, 64, 6, 1, 500, [90] * 6, seed=1), Setup(dev, 64, 2, 4, 16, 40, 1, 300, [50] * 40, seed=2), Setup(dev, 128, 2, 4, 16, 48, 1, 2200, [50] * 48, seed=3),
            Setup(dev, 64, 1, 8, 64, 70, 1, 3000, [80] * 70, seed=4)]
    if longer:                                       # long enough for the tensor-core kernel, between two that are not
        for s in sets[2:]:
            s.close()
        sets[1:] = [Setup(dev, 128, 2, 4, 16, 48, 1, 4700, [50] * 48, seed=3), Setup(dev, 64, 1, 8, 64, 70, 1, 6300, [80] * 70, seed=4), Setup(dev, 128, 2, 2, 64, 40, 1, 5700, [30] * 40, seed=5),
                    Setup(dev, 32, 2, 8, 32, 70, 1, 6300, [80] * 70, seed=6), sets[1]]
    graphs = []
    for s in sets:
        s.upload()
        s.check(s.call())
    for s in sets:
        a = s.args()
        dev.capture_begin()
        N.call("ns_attention_shared", *a)
        graphs.append(dev.capture_end())
    for prefix, own in ((500, 90), (1, 1), (77, 30), (0, 3), (127, 9), (128, 9), (129, 50), (1025, 20), (9999, 50)):
        for s in sets:
            s.prefix, s.pos = min(prefix, s.prefix_pages * s.page), np.full(s.batch, min(own, s.max_pages * s.page) - 1, np.int32)
            s.kept[2].upload(np.array([s.prefix], np.int32))
            s.kept[4].upload(s.pos)
        for g in graphs:
            dev.graph_launch(g)
        dev.synchronize()
        for s in sets:
            s.check(s.read())
    for g in graphs:
        dev.graph_destroy(g)
    for s in sets:
        s.close()


@pytest.mark.gpu
def test_runs_repeat_bit_for_bit(dev):
    for batch in (3, 64, 20):
        s = Setup(dev, 128, 4, 4, 32, batch, 1, 3000, [200] * batch)
        s.upload()
        first = s.call()
        for _ in range(3):
            assert np.array_equal(s.call(), first)
        s.close()
    s = Setup(dev, 128, 4, 4, 32, 32, 1, 3600, [200, 3] * 16)
    s.upload()
    first = s.call()
    assert all(np.array_equal(s.call(), first) for _ in range(3))
    s.close()


def test_refusals():
    A = 1 << 20
    cache = _Cache(0, 8, 16, 2, 64, A, A, False)
    good = dict(cache=C.addressof(cache), q=A, q_stride=512, o=A, o_stride=512, heads=8, prefix_table=A, prefix_pages=3, prefix_len=A, table=A, max_pages=2, pos=A, lens=0,
                batch=2, steps=1, scale=0.1)

    def call(text, **other):
        refused(text, "ns_attention_shared", None, *{**good, **other}.values())

    call("device handle is null")
    call("device handle is null", batch=0)
    call("device handle is null", prefix_pages=0, prefix_table=0, prefix_len=0)
    call("device handle is null", max_pages=0, table=0, pos=0)
    call("cache is null", cache=None)
    call("null argument", q=0)
    call("null argument", o=0)
    call("without its table or length", prefix_table=0)
    call("without its table or length", prefix_len=0)
    call("without their table or positions", table=0)
    call("without their table or positions", pos=0)
    call("neither", prefix_pages=0, max_pages=0)
    call("bad shape", batch=-1)
    call("bad shape", prefix_pages=-1)
    call("query heads", heads=0)
    call("query heads", heads=7)
    call("2^31 positions", prefix_pages=1 << 27)
    call("2^31 positions", max_pages=1 << 27)
    call("too many rows", batch=1 << 15, steps=1 << 15)
    call("16-byte aligned", q=A + 8)
    call("16-byte aligned", q_stride=516)
    call("misaligned", pos=A + 2)
    call("misaligned", o=A + 1)
    call("shorter", q_stride=504)
    call("shorter", o_stride=511)
