"""A decoding step that samples many continuations of one prompt, as a host runs it: a fused projection's rows turned and appended to the sequences' pages
(ns_kv_append_rotary), attention over the prompt's pages and their own (ns_attention_shared), the output projection's logits (ns_matmul_bf16), the next
tokens from given random numbers (ns_sample_tokens), recorded in a graph whose positions advance on the device.  Every step is held to 64-bit arithmetic on
what the step before left on the device; the tolerances are those of the operators' own tests."""
import ctypes as C

import numpy as np
import pytest

from nn_b200 import native as N

from .test_rotary import AMP, bf16, bound, frequencies, turn, values
from .test_sample_tokens import define


class Step:
    """One attention layer over an embedding table, and a head."""

    def __init__(self, dev, batch, prompt, steps, dim=64, kv=2, group=3, page=16, vocab=520, seed=0):
        rng = np.random.default_rng(seed)
        self.dev, self.batch, self.prompt, self.steps, self.dim, self.kv, self.heads, self.page, self.vocab = dev, batch, prompt, steps, dim, kv, kv * group, page, vocab
        self.width = (self.heads + 2 * kv) * dim
        self.table = rng.standard_normal((vocab, self.width)).astype(np.float32)          # a token's projection
        self.head = bf16(rng.standard_normal((vocab, self.heads * dim)) * 0.6)[0]
        self.freq = frequencies(dim)
        self.tokens = rng.integers(0, vocab, prompt)
        self.first = rng.integers(0, vocab, batch)
        self.u = rng.random((steps, batch)).astype(np.float32)
        n_prompt, n_own = (prompt + page - 1) // page, (steps + page - 1) // page
        order = rng.permutation(n_prompt + batch * n_own + 2).astype(np.int32)
        self.prompt_table, self.own_table = order[:n_prompt], order[n_prompt:n_prompt + batch * n_own].reshape(batch, n_own)
        self.n_pages, self.n_own = len(order), n_own
        self.settings = dict(temperature=rng.choice([0.0, 0.7, 1.0], batch).astype(np.float32), top_k=rng.choice([0, 5, 50], batch).astype(np.int32),
                             top_p=rng.choice([0.8, 1.0], batch).astype(np.float32), min_p=rng.choice([0.0, 0.05], batch).astype(np.float32))
        up = dev.from_numpy
        self.cache = C.c_void_p()
        N.call("ns_kv_cache_create", dev.handle, self.n_pages, page, kv, dim, C.byref(self.cache))
        self.d = {n: up(np.ascontiguousarray(a)) for n, a in dict(
            table=self.table, freq=self.freq, head=self.head, prompt_table=self.prompt_table, own_table=self.own_table, prompt_len=np.array([prompt], np.int32),
            zero=np.zeros(batch, np.int32), pos=np.zeros(batch, np.int32), ids=self.first.astype(np.int32), u=self.u[0], **self.settings).items()}
        self.src, self.q = dev.empty(batch * self.width), dev.empty(max(prompt, batch) * self.heads * dim, N.NS_BF16)
        self.o, self.logits, self.probs = dev.empty(batch * self.heads * dim, N.NS_BF16), dev.empty(batch * vocab), dev.empty(batch)

    def append(self, src, offset, pos, table, pages, batch, steps):
        H, K, D = self.heads, self.kv, self.dim
        N.call("ns_kv_append_rotary", self.dev.handle, self.cache, src, 1, N.NS_F32, self.width, 0, H * D, (H + K) * D, H, self.d["freq"].ptr, AMP, N.ROTARY_HALVES, D, offset, pos, 0, table,
               pages, batch, steps, self.q.ptr, H * D)

    def read_prompt(self):
        rows = self.dev.from_numpy(self.table[self.tokens])
        self.append(rows.ptr, 0, self.d["zero"].ptr, self.d["prompt_table"].ptr, len(self.prompt_table), 1, self.prompt)
        self.dev.synchronize()

    def queue(self):
        h, d, D = self.dev.handle, self.d, self.heads * self.dim
        N.call("ns_embed_pos", h, d["ids"].ptr, d["table"].ptr, self.zeros_row().ptr, N.NS_F32, 0, self.batch, 1, self.width, self.vocab, 1, N.NS_F32, self.src.ptr)
        self.append(self.src.ptr, d["prompt_len"].ptr, d["pos"].ptr, d["own_table"].ptr, self.n_own, self.batch, 1)
        N.call("ns_attention_shared", h, self.cache, self.q.ptr, D, self.o.ptr, D, self.heads, d["prompt_table"].ptr, len(self.prompt_table), d["prompt_len"].ptr, d["own_table"].ptr,
               self.n_own, d["pos"].ptr, 0, self.batch, 1, self.dim ** -0.5)
        N.call("ns_matmul_bf16", h, self.o.ptr, d["head"].ptr, self.logits.ptr, 1, self.batch, self.vocab, D, 1, 0, 0, 0, N.EPI_NONE, N.NS_F32)
        N.call("ns_sample_tokens", h, self.logits.ptr, N.NS_F32, self.vocab, self.batch, self.vocab, d["temperature"].ptr, d["top_k"].ptr, d["top_p"].ptr, d["min_p"].ptr, d["u"].ptr,
               d["ids"].ptr, self.probs.ptr)

    def zeros_row(self):
        if not hasattr(self, "_zeros"):
            self._zeros = self.dev.zeros(self.width)
        return self._zeros

    def pools(self):
        got = []
        at = [C.c_uint64(), C.c_uint64()]
        N.call("ns_kv_cache_pools", self.cache, C.byref(at[0]), C.byref(at[1]), None)
        for p in at:
            bits = np.empty((self.n_pages, self.kv, self.page, self.dim), np.uint16)
            N.call("ns_d2h", self.dev.handle, bits.ctypes.data_as(C.c_void_p), p, bits.nbytes)
            got.append(values(bits).astype(np.float64))
        return got

    def check(self, t, ids_before):
        H, K, D = self.heads, self.kv, self.dim
        x = self.table[ids_before].astype(np.float64).reshape(self.batch, H + 2 * K, D)
        want, size = turn(x[:, :H + K], np.full(self.batch, self.prompt + t), self.freq, True)
        tol = bound(want, size, N.NS_BF16)
        q = values(self.q.download((self.batch, H, D), count=self.batch * H * D)).astype(np.float64)
        assert (abs(q - want[:, :H]) <= tol[:, :H]).all()
        k, v = self.pools()
        own = lambda pool, b: pool[self.own_table[b]].transpose(1, 0, 2, 3).reshape(K, -1, D)[:, :t + 1]
        prompt = lambda pool: pool[self.prompt_table].transpose(1, 0, 2, 3).reshape(K, -1, D)[:, :self.prompt]
        o = values(self.o.download((self.batch, H, D))).astype(np.float64)
        for b in range(self.batch):
            assert (abs(own(k, b)[:, -1] - want[b, H:]) <= tol[b, H:]).all() and (abs(own(v, b)[:, -1] - x[b, H + K:]) <= 2.0 ** -8 * abs(x[b, H + K:])).all()
            kk, vv = np.concatenate([prompt(k), own(k, b)], 1), np.concatenate([prompt(v), own(v, b)], 1)
            qq = q[b].reshape(K, H // K, D)
            s = np.einsum("kgd,kjd->kgj", qq, kk) * D ** -0.5
            most = np.einsum("kgd,kjd->kgj", abs(qq), abs(kk)).max() * D ** -0.5
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            wo = w @ vv
            slack = 2.0 ** -8 * abs(wo) + (2.0 ** -8 + 2 * ((D + 4) * 2.0 ** -24 * most + 2.0 ** -18)) * (w @ abs(vv))
            assert (abs(o[b].reshape(wo.shape) - wo) <= slack).all()
        logits = self.logits.download((self.batch, self.vocab))
        ids, probs = self.d["ids"].download(), self.probs.download()
        for b in range(self.batch):
            i, p = define(logits[b], *(self.settings[n][b] if n != "top_k" else int(self.settings[n][b]) for n in ("temperature", "top_k")), float(self.settings["top_p"][b]),
                          float(self.settings["min_p"][b]), float(self.u[t][b]))
            assert ids[b] == i and abs(probs[b] - p) <= (2.0 ** -24 + 2.0 ** -32) * p + 2.0 ** -42 * self.vocab
        return ids

    def close(self):
        N.call("ns_kv_cache_destroy", self.cache)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,prompt,dim,group,page", [(3, 70, 64, 3, 16), (40, 2600, 128, 4, 64), (130, 300, 32, 1, 4), (24, 5000, 64, 8, 128), (40, 3300, 128, 4, 64), (28, 5000, 64, 8, 128), (40, 5500, 128, 4, 64), (28, 8000, 64, 8, 128)])
def test_continuations_of_one_prompt(dev, batch, prompt, dim, group, page):
    steps = 20
    s = Step(dev, batch, prompt, steps, dim=dim, group=group, page=page)
    s.read_prompt()
    ids = s.first
    s.queue()                                    # the first step also sizes the scratch block
    dev.synchronize()
    ids = s.check(0, ids)
    dev.capture_begin()
    s.queue()
    graph = dev.capture_end()
    for t in range(1, steps):
        s.d["pos"].upload(np.full(batch, t, np.int32))
        s.d["u"].upload(s.u[t])
        dev.graph_launch(graph)
        dev.synchronize()
        now = s.d["ids"].download()
        if t in (1, 2, page - 1, page, steps - 1):
            now = s.check(t, ids)
        ids = now
    dev.graph_destroy(graph)
    # the same continuations again, without a graph: the same tokens
    s.d["ids"].upload(s.first.astype(np.int32))
    for t in range(steps):
        s.d["pos"].upload(np.full(batch, t, np.int32))
        s.d["u"].upload(s.u[t])
        s.queue()
        dev.synchronize()
    assert np.array_equal(s.d["ids"].download(), ids)
    s.close()


@pytest.mark.gpu
def test_two_device_objects_at_once(dev):
    """Steps queued on two streams of one GPU, not waited for in between, leave what each leaves alone."""
    from nn_b200.device import Device

    other = Device(0)
    steps = 12
    shapes = [dict(batch=40, prompt=5500, dim=128, group=4, page=64), dict(batch=28, prompt=8000, dim=64, group=8, page=128)]
    want = []
    for turn_ in range(2):
        both = [Step(d, c["batch"], c["prompt"], steps, dim=c["dim"], group=c["group"], page=c["page"], seed=3 + i) for i, (d, c) in enumerate(zip((dev, other), shapes))]
        for s in both:
            s.read_prompt()
            s.us = [s.dev.from_numpy(s.u[t]) for t in range(steps)]
            s.at = [s.dev.from_numpy(np.full(s.batch, t, np.int32)) for t in range(steps)]
            s.dev.synchronize()
        if turn_ == 0:
            order = [(s, t) for s in both for t in range(steps)]
        else:
            order = [(s, t) for t in range(steps) for s in both]
        for s, t in order:
            s.d["u"], s.d["pos"] = s.us[t], s.at[t]
            s.queue()
            if turn_ == 0:
                s.dev.synchronize()
        for s in both:
            s.dev.synchronize()
        got = [(s.d["ids"].download(), s.probs.download(), s.o.download((s.batch, s.heads * s.dim))) for s in both]
        if turn_ == 0:
            want = got
        else:
            assert all(np.array_equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
        for s in both:
            s.close()


@pytest.mark.gpu
def test_many_draws_from_one_row(dev):
    """A row pitch of 0: every draw of the first token reads the same logits."""
    rng = np.random.default_rng(4)
    vocab, rows = 3001, 500
    x = (rng.standard_normal(vocab) * 2).astype(np.float32)
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    store, us, ids = dev.from_numpy(x), dev.from_numpy(u), dev.zeros(rows, N.NS_I32)
    N.call("ns_sample_tokens", dev.handle, store.ptr, N.NS_F32, 0, rows, vocab, 0, 0, 0, 0, us.ptr, ids.ptr, 0)
    dev.synchronize()
    got = ids.download()
    assert all(got[r] == define(x, 1.0, 0, 1.0, 0.0, float(u[r]))[0] for r in range(rows)) and (np.diff(got) >= 0).all()
