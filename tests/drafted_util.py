"""Plain 64-bit implementations of the drafted step's operators, and inputs for
their tests."""
import math
import os

import numpy as np

EMULATED = bool(os.environ.get("Q35_EMULATION_LIB"))
INT64 = np.int64


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def random_tree(rng, n, reach=6):
    """Parents before children; node 0 is the root."""
    i = np.arange(1, n)
    return np.concatenate([[-1], i - rng.integers(1, np.minimum(i, reach) + 1)]).astype(np.int32)


def ancestor_bits(parents):
    """[n, n] booleans: row i holds node i and the nodes above it."""
    n = len(parents)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def mask_words(bits, words):
    """Boolean rows as 64-bit words, bit j % 64 of word j / 64."""
    n, m = bits.shape
    full = np.zeros((n, 64 * words), np.uint8)
    full[:, :m] = bits
    return np.packbits(full, axis=1, bitorder="little").view(np.uint64).reshape(n, words)


def page_table(rng, lens, page_tokens, spare=0, width=None):
    """Requests' pages in any order; entries past a request's pages are -1."""
    need = [(int(n) + page_tokens - 1) // page_tokens for n in lens]
    total = max(1, sum(need) + spare)
    perm = rng.permutation(total).astype(np.int32)
    table = np.full((len(need), width or max(1, max(need))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


class TreeCase:
    """Inputs of attention_tree_paged on the host."""

    def __init__(self, seed, contexts, nodes, heads=8, kv_heads=2, head_dim=256, page_tokens=16, gated=True, bits=None,
                 q_scale=1.0, spare_rows=0, max_nodes=None, max_len=None):
        rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.head_dim, self.page_tokens = heads, kv_heads, head_dim, page_tokens
        self.contexts, self.nodes = np.asarray(contexts, np.int32), np.asarray(nodes, np.int32)
        self.batch = len(self.nodes)
        self.start = starts(self.nodes)
        self.rows = int(self.start[-1]) + spare_rows
        self.max_nodes = max_nodes or max(1, int(self.nodes.max()))
        lens = self.contexts + self.nodes
        self.max_len = max_len or max(1, int(lens.max()))
        words = (self.max_nodes + 63) // 64
        width = (self.max_len + page_tokens - 1) // page_tokens
        self.table, self.total_pages = page_table(rng, lens, page_tokens, spare=1, width=width)
        self.bits = bits or [ancestor_bits(random_tree(rng, int(n))) for n in self.nodes]
        self.masks = np.zeros((self.rows, words), np.uint64)
        for b, m in enumerate(self.bits):
            if len(m):
                self.masks[self.start[b]:self.start[b + 1]] = mask_words(m, words)
        shape = (self.total_pages, page_tokens, kv_heads, head_dim)
        # rows that belong to no request (spare pages, the ends of last pages) hold NaN
        self.k, self.v = np.full(shape, np.nan, np.float16), np.full(shape, np.nan, np.float16)
        for b in range(self.batch):
            for t in range(int(lens[b])):
                at = self.table[b, t // page_tokens], t % page_tokens
                self.k[at], self.v[at] = rng.standard_normal((2, kv_heads, head_dim)).astype(np.float16)
        self.q = (rng.standard_normal((self.rows, heads, head_dim)) * q_scale).astype(np.float32)
        self.gates = rng.standard_normal(self.q.shape).astype(np.float32) if gated else None
        self.scale = 1.0 / math.sqrt(head_dim)
        self.fill = -77.0

    def cache(self, b, pool):
        n = int(self.contexts[b] + self.nodes[b])
        t = np.arange(n)
        return pool[self.table[b, t // self.page_tokens], t % self.page_tokens].astype(np.float64)

    def run(self, q, ctx, workspace=None, arrays=None):
        """The operator's output [rows, heads, head_dim] (rows it leaves alone keep self.fill)."""
        d = arrays or self.device(ctx)
        self.call(q, ctx, d, workspace)
        return d["out"].download()

    def device(self, ctx):
        d = {n: ctx.array(getattr(self, n)) for n in ("q", "table", "contexts", "start", "masks")}
        d["k"], d["v"] = ctx.array(self.k.view(np.uint16)), ctx.array(self.v.view(np.uint16))
        d["gates"] = ctx.array(self.gates) if self.gates is not None else None
        d["out"] = ctx.array(np.full(self.q.shape, self.fill, np.float32))
        return d

    def call(self, q, ctx, d, workspace=None, **other):
        a = dict(total_pages=self.total_pages, max_pages=self.table.shape[1], page_tokens=self.page_tokens,
                 batch=self.batch, rows=self.rows, max_nodes=self.max_nodes, max_len=self.max_len, heads=self.heads,
                 kv_heads=self.kv_heads, head_dim=self.head_dim, scale=self.scale)
        a.update(other)
        q.attention_tree_paged(ctx, d["q"], d["gates"], d["k"], d["v"], a["total_pages"], d["table"], a["max_pages"],
                               a["page_tokens"], d["contexts"], d["start"], d["masks"], d["out"], a["batch"], a["rows"],
                               a["max_nodes"], a["max_len"], a["heads"], a["kv_heads"], a["head_dim"], a["scale"], workspace)

    def expected(self):
        """The formula in 64 bits, and how far an output in 32 bits may be from it.

        Scores: q enters as two binary16 parts (2^-22 of its largest value), its
        products with binary16 keys are exact and summed in fp32 (at most
        head_dim + 16 roundings of 2^-24 of the sum of magnitudes), then the
        scaling and the difference to the maximum (2^-22 of the score's size).
        An error e of every score moves p by at most a factor exp(2 e).
        Probabilities: exp2 (2^-22), two binary16 parts (2^-22), and sums over
        the rows in fp32: a wavefront adds at most len / 4 + 64 of them in a row,
        2^-24 each; the gate, the division and the joins: 2^-20 in all."""
        out, tol = np.full(self.q.shape, self.fill, np.float64), np.zeros(self.q.shape)
        group = self.heads // self.kv_heads
        for b in range(self.batch):
            r0, c, n = int(self.start[b]), int(self.contexts[b]), int(self.nodes[b])
            keys, values = self.cache(b, self.k), self.cache(b, self.v)
            for i in range(n):
                see = np.concatenate([np.ones(c, bool), np.asarray(self.bits[b][i][:n], bool)])
                for h in range(self.heads):
                    g = h // group
                    x = self.q[r0 + i, h].astype(np.float64)
                    if not see.any():
                        out[r0 + i, h] = 0.0
                        continue
                    k, v = keys[see, g], values[see, g]
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = k @ x * self.scale
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        y = p @ v
                        size = (np.abs(k) @ np.abs(x)).max() * self.scale + np.abs(k).max(axis=1).sum() * 0.0
                        e = size * ((self.head_dim + 16) * 2.0 ** -24 + 2.0 ** -22) + np.abs(s).max() * 2.0 ** -22
                        e += np.abs(x).max() * 2.0 ** -22 * np.abs(k).sum(axis=1).max() * self.scale
                        spread = p @ np.abs(v)
                    if self.gates is not None:
                        gate = 1.0 / (1.0 + np.exp(-self.gates[r0 + i, h].astype(np.float64)))
                        y, spread = y * gate, spread * gate
                    out[r0 + i, h] = y
                    tol[r0 + i, h] = spread * (np.expm1(2 * e) + (len(s) / 4 + 64) * 2.0 ** -24 + 3 * 2.0 ** -22 + 2.0 ** -20)
        return out, tol


def accept(start, parents, draft, sampled, width):
    batch = len(start) - 1
    path, count, token = np.full((batch, width), -1, np.int32), np.zeros(batch, np.int32), np.full(batch, -1, np.int32)
    for b in range(batch):
        r0, n = int(start[b]), int(start[b + 1] - start[b])
        at = 0 if n else None
        while at is not None:
            path[b, count[b]] = at
            count[b] += 1
            token[b] = sampled[r0 + at]
            below = [c for c in range(at + 1, n) if parents[r0 + c] == at and draft[r0 + c] == token[b]]
            at = below[0] if below else None
    return path, count, token


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, counts=None, penalty=1.0):
    """(token, probability) of one row."""
    x = np.array(logits, np.float32)
    if counts is not None and penalty > 1.0:
        hit = np.asarray(counts) > 0
        r = np.float32(penalty)
        x[hit] = np.where(x[hit] > 0, x[hit] / r, x[hit] * r)
    x[np.isnan(x)] = -np.inf
    order = np.lexsort((np.arange(x.size), -x.astype(np.float64)))
    order = order[x[order] > -np.inf]
    if order.size == 0:
        return -1, 0.0
    if not temperature > 1e-6:
        return int(order[0]), 1.0
    v = x[order].astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / np.float64(np.float32(temperature))))
    if 0 < top_k < order.size:
        w = w[:top_k]
    keep = len(w)
    run = np.cumsum(w)
    if top_p < 1.0:
        keep = min(keep, 1 + int(np.searchsorted(run, np.float64(np.float32(top_p)) * run[-1], side="left")))
    if min_p > 0.0:
        keep = min(keep, int((w >= min(1.0, np.float64(np.float32(min_p)))).sum()))
    keep = max(1, keep)
    mass = run[keep - 1]
    at = min(keep - 1, int(np.searchsorted(run[:keep], np.float64(np.float32(u)) * mass, side="right")))
    while w[at] == 0.0:
        at -= 1
    return int(order[at]), w[at] / mass
