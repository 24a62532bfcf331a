"""Operators of a serving step that samples many continuations of one prompt, as cases that can be timed and checked.

* ``rotary``    -- rotary positions of query and key heads: neighbouring pairs or halves, a part of the head, frequencies stretched for long contexts, forwards
  and backwards.
* ``append``    -- a token's queries, keys and values out of the fused projection: queries and keys turned to their positions, keys and values into the pages of
  a cache, every sequence at a position of its own.
* ``attention`` -- new positions against a prefix that all sequences share (its pages are read once for all of them) and against pages of their own.
* ``sample``    -- the next token of every row from a given random number, with a temperature, top-k, top-p and min-p of its own.

With ``own`` false everything is computed with elementary torch operations, else by the calls that a host program makes.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of one sequence: all its query and key heads, in place of a separate launch each
        {"name": "rotary 1 row", "kind": "rotary", "rows": 1, "heads": 40, "dim": 128, "rot": 128, "halves": True, "inverse": False, "dtype": "bf16", "far": 4000},
        # a prompt's portion at far positions, its query and key heads side by side
        {"name": "rotary 8192 rows", "kind": "rotary", "rows": 8192, "heads": 40, "dim": 128, "rot": 128, "halves": True, "inverse": False, "dtype": "bf16",
         "far": 500000},
        # the gradient of a partial rotation of neighbouring pairs, in 32 bits, rows that fill no tile
        {"name": "rotary f32 1777 rows", "kind": "rotary", "rows": 1777, "heads": 20, "dim": 96, "rot": 32, "halves": False, "inverse": True, "dtype": "f32",
         "far": 30000},
        # a step of a full batch, straight from the projection's partial sums
        {"name": "append 64 x 1", "kind": "append", "batch": 64, "steps": 1, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "halves": True, "splits": 2, "page": 64,
         "far": 4000, "ragged": False},
        # prompts of different lengths side by side
        {"name": "append 13 x 777", "kind": "append", "batch": 13, "steps": 777, "heads": 32, "kv": 8, "dim": 128, "rot": 64, "halves": False, "splits": 0, "page": 16,
         "far": 300, "ragged": True},
        # a few continuations of a short prompt: every launch counts
        {"name": "attention 3 x 500", "kind": "attention", "batch": 3, "steps": 1, "heads": 8, "kv": 2, "dim": 64, "page": 16, "prefix": 500, "own": 37},
        # drafted tokens of a few sequences, a key/value head for every query head
        {"name": "attention 8 x 5 x 2500", "kind": "attention", "batch": 8, "steps": 5, "heads": 16, "kv": 16, "dim": 64, "page": 16, "prefix": 2500, "own": 300},
        # the full batch of the benchmark over a system prompt
        {"name": "attention 64 x 4096", "kind": "attention", "batch": 64, "steps": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "prefix": 4096, "own": 512},
        # many continuations of one long document
        {"name": "attention 256 x 16384", "kind": "attention", "batch": 256, "steps": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "prefix": 16384, "own": 600},
        # an interactive user
        {"name": "sample 1 x 32000", "kind": "sample", "rows": 1, "vocab": 32000, "dtype": "f32"},
        # the full batch of the benchmark decoder
        {"name": "sample 64 x 32000", "kind": "sample", "rows": 64, "vocab": 32000, "dtype": "f32"},
        # many continuations, a large vocabulary of no round size, logits as a bf16 product leaves them
        {"name": "sample 256 x 131001", "kind": "sample", "rows": 256, "vocab": 131001, "dtype": "bf16"},
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["rotary", "append", "attention", "attention", "attention", "sample", "sample"])
    dim = rng.choice([32, 64, 128, 128])
    if kind == "rotary":
        dim = rng.choice([40, 64, 96, 128, 256])
        dtype = rng.choice(["bf16", "f32"])
        heads = spread(1, 40)
        rows = spread(1, max(1, min(8192, 8192 * 40 * 128 // (heads * dim * (2 if dtype == "f32" else 1)))))
        return {"kind": kind, "rows": rows, "heads": heads, "dim": dim, "rot": 2 * rng.randint(1, dim // 2), "halves": rng.random() < 0.5,
                "inverse": rng.random() < 0.3, "dtype": dtype, "far": spread(100, 1000000)}
    if kind == "append":
        kv = rng.choice([1, 2, 4, 8])
        batch, steps = (spread(1, 256), 1) if rng.random() < 0.5 else (spread(1, 13), spread(2, 777))
        return {"kind": kind, "batch": batch, "steps": steps, "heads": kv * rng.choice([1, 2, 4]), "kv": kv, "dim": dim, "rot": 2 * rng.randint(1, dim // 2),
                "halves": rng.random() < 0.5, "splits": rng.choice([0, 1, 2, 4] if steps == 1 else [0, 1]), "page": rng.choice([16, 32, 64, 128]),
                "far": spread(10, 4000), "ragged": rng.random() < 0.5}
    if kind == "attention":
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2] if kv > 8 else [1, 2, 4] if kv > 4 else [1, 3, 4, 8])
        batch = spread(1, 256)
        return {"kind": kind, "batch": batch, "steps": rng.choice([1, 1, 1, 2, 4]) if batch <= 64 else 1, "heads": heads, "kv": kv, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "prefix": spread(40, 16384), "own": spread(1, 300 if kv > 8 else 600)}
    dtype = rng.choice(["f32", "bf16"])
    return {"kind": kind, "rows": spread(1, 256 if dtype == "bf16" else 128), "vocab": spread(1000, 131001), "dtype": dtype}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return g


def _normal(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _integers(g, lo, hi, *shape):
    """lo .. hi, both among them"""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _frequencies(dims, stretch):
    """One for every pair of columns, slow ones stretched as for a context longer than the trained one."""
    f = 10000.0 ** (-np.arange(0, dims, 2) / dims)
    slow = np.clip((2 * math.pi / f - 256.0) / (4096.0 - 256.0), 0.0, 1.0)
    f = f * (1 - slow) + f / stretch * slow
    return torch.tensor(f.astype(np.float32), device="cuda")


def _tensors(case, seed):
    """The inputs of a case: a dict of tensors."""
    g, c = _generator(seed), case
    kind = c["kind"]
    if kind == "rotary":
        dtype = F32 if c["dtype"] == "f32" else BF16
        return {"x": _normal(g, c["rows"], c["heads"], c["dim"], dtype=dtype), "pos": _integers(g, 0, c["far"], c["rows"]),
                "freq": _frequencies(c["rot"], 4.0)}
    if kind == "append":
        B, T, H, K, D, S = c["batch"], c["steps"], c["heads"], c["kv"], c["dim"], c["page"]
        t = {"lens": _integers(g, 1, T, B) if c["ragged"] else torch.full((B,), T, dtype=torch.int32, device="cuda"), "pos": _integers(g, 0, c["far"], B),
             "freq": _frequencies(c["rot"], 4.0), "offset": _integers(g, 0, c["far"], 1)}
        width = (H + 2 * K) * D
        t["src"] = _normal(g, max(1, c["splits"]), B, T, width, dtype=F32 if c["splits"] else BF16, std=max(1, c["splits"]) ** -0.5)
        pages = (c["far"] + T + S - 1) // S + 1
        t["table"] = torch.randperm(B * pages, generator=g, device="cuda").to(torch.int32).reshape(B, pages)
        # the cache's other pages are another program part's; here the pools hold what the sequences can reach
        t["k"], t["v"] = (_normal(g, B * pages, K, S, D, dtype=BF16) for _ in range(2))
        t["q"] = torch.zeros(B, T, H, D, dtype=BF16, device="cuda")
        return t
    if kind == "attention":
        B, T, H, K, D, S, P, L = c["batch"], c["steps"], c["heads"], c["kv"], c["dim"], c["page"], c["prefix"], c["own"]
        # positions that the sequences have already: from none to L; the new ones follow
        t = {"pos": _integers(g, 0, L, B), "prefix_len": torch.full((1,), P, dtype=torch.int32, device="cuda")}
        n_prefix, n_own = (P + S - 1) // S, (L + T + S - 1) // S
        order = torch.randperm(n_prefix + B * n_own, generator=g, device="cuda").to(torch.int32)
        t["prefix_table"], t["table"] = order[:n_prefix].contiguous(), order[n_prefix:].reshape(B, n_own).contiguous()
        # keys lean towards a common direction, as trained ones do, so that scores are spread and not all alike
        lean = _normal(g, K, 1, D)
        t["k"] = (_normal(g, len(order), K, S, D) + 0.5 * lean).to(BF16)
        t["v"] = _normal(g, len(order), K, S, D, dtype=BF16)
        t["q"] = (_normal(g, B, T, H, D, std=1.2) + 0.3 * lean.repeat_interleave(H // K, 0).reshape(H, D)).to(BF16)
        return t
    R, V = c["rows"], c["vocab"]
    x = _normal(g, R, V, std=2.0)
    # a few likely tokens in every row
    x.scatter_add_(1, torch.randint(0, V, (R, 12), generator=g, device="cuda"), _normal(g, R, 12, std=2.0, mean=7.0))
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (R,), generator=g, device="cuda")]
    return {"x": x.to(F32 if c["dtype"] == "f32" else BF16), "temperature": pick(0.0, 0.6, 0.7, 1.0, 1.0, 1.3), "top_k": pick(0, 0, 20, 50, 200, 1000).to(torch.int32),
            "top_p": pick(0.8, 0.9, 0.95, 1.0, 1.0), "min_p": pick(0.0, 0.0, 0.02, 0.1), "u": torch.rand(R, generator=g, device="cuda")}


class State:
    """What the program keeps between calls."""

    def __init__(self, case, tensors):
        self.case = case
        self.__dict__.update(tensors)
        self.cache = None

    def __del__(self):
        if self.cache is not None:
            try:
                native().call("ns_kv_cache_destroy", self.cache)
            except Exception:
                pass


_device = None


def native():
    from nn_b200 import native as N

    return N


def device():
    global _device
    if _device is None:
        from nn_b200.device import Device

        _device = Device(0)
    return _device


def _own_cache(s):
    """A cache over the pools: its handle, once their contents lie in it."""
    import ctypes

    pools = s.k.clone(), s.v.clone()
    handle = ctypes.c_void_p()
    torch.cuda.synchronize()
    pages, heads, page, dim = s.k.shape
    native().call("ns_kv_cache_create_in", device().handle, pages, page, heads, dim, s.k.data_ptr(), s.v.data_ptr(), ctypes.byref(handle))
    device().synchronize()
    s.k.copy_(pools[0])
    s.v.copy_(pools[1])
    torch.cuda.synchronize()
    return handle


def prepare(case, seed):
    s = State(case, _tensors(case, seed))
    kind = case["kind"]
    if kind == "rotary":
        s.y = torch.empty_like(s.x)
    elif kind == "attention":
        s.o = torch.empty_like(s.q)
    elif kind == "sample":
        s.ids = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        s.probs = torch.empty(case["rows"], dtype=F32, device="cuda")
    if own and kind in ("append", "attention"):
        s.cache = _own_cache(s)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
AMPLITUDE = 1.125        # of the turned columns, as for stretched frequencies


def _turn(x, angle, rot, halves, sign):
    """x [..., heads, dim] in 32 bits; angle [..., 1, rot / 2] in 64, whose cosine and sine are rounded once."""
    cos, sin = (AMPLITUDE * angle.cos()).to(F32), (sign * AMPLITUDE * angle.sin()).to(F32)
    y = x.clone()
    if halves:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_rotary(s):
    c = s.case
    angle = (s.pos.double()[:, None] * s.freq.double())[:, None, :]
    s.y.copy_(_turn(s.x.to(F32), angle, c["rot"], c["halves"], -1.0 if c["inverse"] else 1.0))
    return s.y


def _plain_append(s):
    c = s.case
    B, T, H, K, D, S = c["batch"], c["steps"], c["heads"], c["kv"], c["dim"], c["page"]
    x = s.src.to(F32).sum(0).reshape(B, T, H + 2 * K, D)
    at = s.pos[:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
    angle = ((at + s.offset).double()[..., None] * s.freq.double())[:, :, None, :]
    turned = _turn(x[:, :, :H + K], angle, c["rot"], c["halves"], 1.0)
    live = torch.arange(T, device="cuda") < s.lens[:, None]
    b, i = live.nonzero(as_tuple=True)
    s.q[b, i] = turned[b, i, :H].to(BF16)
    page, row = s.table[b, at[b, i].long() // S].long(), at[b, i].long() % S
    s.k[page, :, row] = turned[b, i, H:].to(BF16)
    s.v[page, :, row] = x[b, i, H + K:].to(BF16)
    return {"q": s.q, "k": s.k, "v": s.v}


def _plain_attention(s):
    c = s.case
    B, T, H, K, D, S, P = c["batch"], c["steps"], c["heads"], c["kv"], c["dim"], c["page"], c["prefix"]
    rows = lambda pool, table: pool[table.long()].to(F32).transpose(-3, -2).reshape(*table.shape[:-1], -1, K, D)
    q = s.q.to(F32).reshape(B, T, K, H // K, D)
    n = s.table.shape[1] * S
    scores = torch.empty(B, T, K, H // K, P + n, device="cuda")
    # the shared part is one matrix product for each key/value head
    scores[..., :P] = torch.einsum("btkgd,jkd->btkgj", q, rows(s.k, s.prefix_table)[:P])
    scores[..., P:] = torch.einsum("btkgd,bjkd->btkgj", q, rows(s.k, s.table))
    scores *= D ** -0.5
    j, last = torch.arange(n, device="cuda"), s.pos[:, None] + torch.arange(T, device="cuda")
    scores[..., P:].masked_fill_((j > last[..., None])[:, :, None, None, :], -math.inf)
    w = (scores - scores.amax(-1, keepdim=True)).exp_()
    del scores
    total = w.sum(-1, keepdim=True)
    # (every page of a sequence holds numbers here, also behind its last position: a weight of zero leaves them out)
    o = torch.einsum("btkgj,jkd->btkgd", w[..., :P], rows(s.v, s.prefix_table)[:P]) + torch.einsum("btkgj,bjkd->btkgd", w[..., P:], rows(s.v, s.table))
    s.o.copy_((o / total).reshape(B, T, H, D))
    return s.o


def _plain_sample(s):
    x = s.x.double()
    greedy = s.temperature <= 0
    t = torch.where(greedy, 1.0, s.temperature.double())[:, None]
    # weights and their sums in 64 bits: a draw falls between two tokens' borders
    w = ((x - x.amax(1, keepdim=True)) / t).exp()
    V = x.shape[1]
    k = torch.where(greedy, 1, torch.where(s.top_k <= 0, V, s.top_k)).long().clamp(max=V)[:, None]
    sorted_x, order = x.sort(dim=1, descending=True, stable=True)      # equal ones by their index
    ws = w.gather(1, order)
    rank = torch.arange(V, device="cuda")
    ws = torch.where(rank < k, ws, 0.0)
    run_sum = ws.cumsum(1)
    before = run_sum - ws
    keep = (rank < k) & ((before < s.top_p.double()[:, None] * run_sum[:, -1:]) | (rank == 0)) & (ws >= s.min_p.double()[:, None])
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    run_sum = kept.cumsum(1)
    total = run_sum[:, -1:]
    ids = (run_sum > s.u.double()[:, None] * total).to(torch.int8).argmax(1, keepdim=True)
    s.ids.copy_(ids[:, 0])
    s.probs.copy_((kept.gather(1, ids) / total)[:, 0])
    return {"ids": s.ids, "probs": s.probs}


# ------------------------------------------------------------------------------------------------------------------ one pass
def _own_rotary(s):
    c, N = s.case, native()
    N.call("ns_rotary", device().handle, s.x.data_ptr(), N.NS_F32 if c["dtype"] == "f32" else N.NS_BF16, c["heads"] * c["dim"], c["dim"], s.pos.data_ptr(),
           s.freq.data_ptr(), AMPLITUDE, N.ROTARY_HALVES if c["halves"] else N.ROTARY_PAIRS, int(c["inverse"]), c["rows"], c["heads"], c["dim"], c["rot"],
           s.y.data_ptr(), c["heads"] * c["dim"], c["dim"])
    return s.y


def _own_append(s):
    c, N = s.case, native()
    H, K, D = c["heads"], c["kv"], c["dim"]
    N.call("ns_kv_append_rotary", device().handle, s.cache, s.src.data_ptr(), max(1, c["splits"]), N.NS_F32 if c["splits"] else N.NS_BF16, (H + 2 * K) * D,
           0, H * D, (H + K) * D, H, s.freq.data_ptr(), AMPLITUDE, N.ROTARY_HALVES if c["halves"] else N.ROTARY_PAIRS, c["rot"], s.offset.data_ptr(),
           s.pos.data_ptr(), s.lens.data_ptr(), s.table.data_ptr(), s.table.shape[1], c["batch"], c["steps"], s.q.data_ptr(), H * D)
    return {"q": s.q, "k": s.k, "v": s.v}


def _own_attention(s):
    c = s.case
    H, D = c["heads"], c["dim"]
    native().call("ns_attention_shared", device().handle, s.cache, s.q.data_ptr(), H * D, s.o.data_ptr(), H * D, H, s.prefix_table.data_ptr(), s.prefix_table.shape[0],
                  s.prefix_len.data_ptr(), s.table.data_ptr(), s.table.shape[1], s.pos.data_ptr(), 0, c["batch"], c["steps"], D ** -0.5)
    return s.o


def _own_sample(s):
    c, N = s.case, native()
    N.call("ns_sample_tokens", device().handle, s.x.data_ptr(), N.NS_F32 if c["dtype"] == "f32" else N.NS_BF16, c["vocab"], c["rows"], c["vocab"],
           s.temperature.data_ptr(), s.top_k.data_ptr(), s.top_p.data_ptr(), s.min_p.data_ptr(), s.u.data_ptr(), s.ids.data_ptr(), s.probs.data_ptr())
    return {"ids": s.ids, "probs": s.probs}


def run(s):
    kind = s.case["kind"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "attention": _own_attention, "sample": _own_sample}[kind](s)
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[kind](s)


# ------------------------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    c, kind = case, case["kind"]
    if kind == "rotary":
        n = c["rows"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * (4 if c["dtype"] == "f32" else 2) + 4 * c["rows"] + 2 * c["rot"], "flops": 3 * c["rows"] * c["heads"] * c["rot"]}
    if kind == "append":
        rows = c["batch"] * c["steps"] * (0.5 if c["ragged"] else 1.0)
        width = (c["heads"] + 2 * c["kv"]) * c["dim"]
        return {"bytes": rows * width * ((4 * c["splits"] if c["splits"] else 2) + 2) + 16 * c["batch"], "flops": rows * (c["heads"] + c["kv"]) * c["rot"] * 3}
    if kind == "attention":
        # a sequence has L / 2 positions of its own on average, and its new ones
        B, T, H, K, D, P = c["batch"], c["steps"], c["heads"], c["kv"], c["dim"], c["prefix"]
        mine = c["own"] / 2 + T
        return {"bytes": 4 * (P + B * mine) * K * D + 4 * B * T * H * D, "flops": 4 * B * T * H * D * (P + mine)}
    return {"bytes": c["rows"] * c["vocab"] * (4 if c["dtype"] == "f32" else 2) + 28 * c["rows"], "flops": 20 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_turn(x, angle, rot, halves, sign):
    """Complex numbers times amplitude * e^(+-i angle)."""
    x = x.double()
    pairs = torch.stack([x[..., :rot // 2], x[..., rot // 2:rot]], -1) if halves else x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, AMPLITUDE), sign * angle)
    turned = torch.cat([z.real, z.imag], -1) if halves else torch.view_as_real(z).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _exact_sample_row(x, temperature, k, p, least, u):
    """One row by its sorted tokens, on the CPU."""
    if temperature <= 0:
        return int(np.argmax(x)), 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[:k] if k > 0 else order
    w = np.exp((x[order] - x[order[0]]) / temperature)
    reached = np.cumsum(w)
    n = 1 + int(np.searchsorted(reached, p * reached[-1], side="left"))
    n = min(n, len(order), max(1, int(np.sum(w >= least))))
    tokens = np.argsort(order[:n])
    reached = np.cumsum(w[:n][tokens])
    i = min(int(np.searchsorted(reached, u * reached[-1], side="right")), n - 1)
    return int(order[tokens[i]]), float(w[tokens[i]] / reached[-1])


def exact(case, seed):
    c, t = case, _tensors(case, seed)
    kind = c["kind"]
    if kind == "rotary":
        angle = torch.outer(t["pos"].double(), t["freq"].double())[:, None, :].expand(-1, c["heads"], -1)
        return _exact_turn(t["x"], angle, c["rot"], c["halves"], -1.0 if c["inverse"] else 1.0)
    if kind == "append":
        H, K, D, S = c["heads"], c["kv"], c["dim"], c["page"]
        x = t["src"].double().sum(0)
        q, k, v = t["q"].double(), t["k"].double(), t["v"].double()
        for b, (n, first) in enumerate(zip(t["lens"].tolist(), t["pos"].tolist())):
            at = torch.arange(first, first + n, device="cuda")
            heads = x[b, :n].reshape(n, H + 2 * K, D)
            angle = torch.outer((at + t["offset"].long()).double(), t["freq"].double())[:, None, :].expand(-1, H + K, -1)
            turned = _exact_turn(heads[:, :H + K], angle, c["rot"], c["halves"], 1.0)
            q[b, :n] = turned[:, :H]
            page = t["table"][b].long()[at // S]
            k[page, :, at % S], v[page, :, at % S] = turned[:, H:], heads[:, H + K:]
        return {"q": q, "k": k, "v": v}
    if kind == "attention":
        B, T, H, K, D, P = c["batch"], c["steps"], c["heads"], c["kv"], c["dim"], c["prefix"]
        flat = lambda pool, table: pool[table.long()].permute(1, 0, 2, 3).reshape(K, -1, D).double()
        pk, pv = (flat(t[n], t["prefix_table"])[:, :P] for n in "kv")
        out = torch.empty(B, T, H, D, dtype=torch.float64, device="cuda")
        for b, first in enumerate(t["pos"].tolist()):
            ok, ov = (flat(t[n], t["table"][b]) for n in "kv")
            for i in range(T):
                n = first + i + 1
                q = t["q"][b, i].double().reshape(K, H // K, D) * D ** -0.5
                # the maximum and the sum over both parts together
                parts = [q @ pk.transpose(1, 2), q @ ok[:, :n].transpose(1, 2)]
                log_sum = torch.logsumexp(torch.cat(parts, 2), 2, keepdim=True)
                out[b, i] = ((parts[0] - log_sum).exp() @ pv + (parts[1] - log_sum).exp() @ ov[:, :n]).reshape(H, D)
        return out
    if c["rows"] * c["vocab"] > 1 << 26:
        return None
    x = t["x"].double().cpu().numpy()
    rows = [_exact_sample_row(x[r], *(t[n][r].double().item() if n != "top_k" else int(t[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u")))
            for r in range(c["rows"])]
    return {"ids": np.array([r[0] for r in rows], np.int32), "probs": np.array([r[1] for r in rows])}
