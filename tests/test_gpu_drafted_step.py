"""A drafted step as it is used: the trees' attention over the cache, a token
sampled after every node, the accepted path, and its rows moved together behind
the context -- after which the cache serves the ordinary decode attention as if
the accepted tokens had been decoded one by one. Also: the same step captured
into graphs and replayed, calls of two contexts at once, and caches past 32-bit
offsets."""
import ctypes

import numpy as np
import pytest

from tests.drafted_util import EMULATED, TreeCase, accept, ancestor_bits, random_tree, sample

pytestmark = pytest.mark.gpu


def _step_inputs(seed, contexts, nodes, vocab, heads, kv_heads):
    """Trees with repeated tokens, and a head that favours them, so that paths of several nodes come about."""
    rng = np.random.default_rng(seed)
    parents = [random_tree(rng, n, reach=3) for n in nodes]
    case = TreeCase(seed, contexts, nodes, heads, kv_heads, 256, gated=True, bits=[ancestor_bits(p) for p in parents])
    rows = case.rows
    draft = rng.integers(0, 2, size=rows).astype(np.int32)
    logits = rng.standard_normal((rows, vocab)).astype(np.float32)
    logits[:, :2] += 9.0
    return case, np.concatenate(parents), draft, logits, rng.random(rows).astype(np.float32)


def test_a_drafted_step(q, ctx):
    contexts, nodes, vocab, heads, kv_heads = [37, 5, 100], [9, 4, 12], 3000, 4, 2
    case, parents, draft, logits, u = _step_inputs(18, contexts, nodes, vocab, heads, kv_heads)
    print("a drafted step", flush=True)
    d = case.device(ctx)
    token, path = ctx.array(shape=(case.rows,), dtype=np.int32), ctx.array(shape=(3, case.max_nodes), dtype=np.int32)
    count, following = ctx.array(shape=(3,), dtype=np.int32), ctx.array(shape=(3,), dtype=np.int32)
    case.call(q, ctx, d)
    q.sample_logits(ctx, ctx.array(logits), vocab, None, None, ctx.array(np.full(case.rows, 0.9, np.float32)), None,
                    ctx.array(np.full(case.rows, 0.95, np.float32)), None, ctx.array(u), case.rows, vocab, token)
    q.tree_accept(ctx, d["start"], ctx.array(parents), ctx.array(draft), token, path, case.max_nodes, count, following, 3,
                  case.rows, case.max_nodes)
    width = kv_heads * 256
    q.cache_compact_rows(ctx, d["k"], d["v"], 1, 0, case.total_pages, 16, width, d["table"], case.table.shape[1],
                         d["contexts"], path, case.max_nodes, count, 3)
    out = d["out"].download()
    want, tol = case.expected()
    assert (np.abs(out - want) <= tol).all()
    sampled = np.array([sample(logits[r], u[r], 0.9, 0, 0.95)[0] for r in range(case.rows)], np.int32)
    np.testing.assert_array_equal(token.download(), sampled)
    want_path = accept(case.start, parents, draft, sampled, case.max_nodes)
    got_path, got_count = path.download(), count.download()
    np.testing.assert_array_equal(got_path, want_path[0])
    np.testing.assert_array_equal(got_count, want_path[1])
    np.testing.assert_array_equal(following.download(), want_path[2])
    assert got_count.max() > 2
    # each accepted node's attention, decoded by position from the compacted cache
    for b in range(3):
        n = int(got_count[b])
        table = np.where(case.table[b] < 0, 0, case.table[b]).astype(np.int32)
        rows = case.start[b] + got_path[b, :n]
        lens = contexts[b] + 1 + np.arange(n, dtype=np.int32)
        one = ctx.array(shape=(n, heads, 256), dtype=np.float32)
        q.attention_decode_paged(ctx, ctx.array(case.q[rows]), ctx.array(case.gates[rows]), d["k"], d["v"],
                                 ctx.array(np.tile(table, (n, 1))), table.size, ctx.array(lens), 16, one, n, heads, kv_heads,
                                 256, case.scale)
        np.testing.assert_array_less(np.abs(one.download() - out[rows]), 2 * tol[rows] + 1e-30)


class _Graph:
    """The calls made between enter and exit on a context's stream, as a graph (the HIP runtime behind the library)."""

    def __init__(self, q, ctx):
        self.hip, self.stream = q.lib, ctypes.c_void_p(q.lib.q35_context_stream(ctx.handle))
        self.exec = None

    def _ok(self, status):
        assert status == 0, status

    def __enter__(self):
        self._ok(self.hip.hipStreamBeginCapture(self.stream, 1))  # this thread's calls
        return self

    def __exit__(self, *exc):
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self._ok(self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)))
        if exc[0] is None:
            self._ok(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)))
        self._ok(self.hip.hipGraphDestroy(graph))

    def replay(self):
        self._ok(self.hip.hipGraphLaunch(self.exec, self.stream))

    def close(self):
        self._ok(self.hip.hipGraphExecDestroy(self.exec))


@pytest.mark.skipif(EMULATED, reason="graphs need the device")
def test_captured_steps(q, ctx):
    """Two graphs of the whole step with workspaces of their own, replayed in turn between eager calls of
    other sizes: every replay gives the eager result on the inputs it finds."""
    contexts, nodes, vocab, heads, kv_heads = [400, 5, 900], [9, 4, 12], 9000, 4, 2

    class Step:
        def __init__(self, seed, ctx):
            self.case, parents, draft, logits, self.numbers = _step_inputs(seed, contexts, nodes, vocab, heads, kv_heads)
            c, self.ctx = self.case, ctx
            self.d = c.device(ctx)
            self.parents, self.draft, self.logits, self.u = (ctx.array(a) for a in (parents, draft, logits, self.numbers))
            self.token, self.p = ctx.array(shape=(c.rows,), dtype=np.int32), ctx.array(shape=(c.rows,), dtype=np.float32)
            self.path, self.count, self.next = (ctx.array(shape=n, dtype=np.int32) for n in ((3, c.max_nodes), (3,), (3,)))
            self.work = [ctx.array(shape=(max(1, n),), dtype=np.uint8) for n in (
                q.attention_tree_workspace(ctx, 3, c.rows, c.max_nodes, c.max_len, heads, kv_heads, 256),
                q.sample_workspace(ctx, c.rows, vocab))]
            self.spare = int(np.setdiff1d(np.arange(c.total_pages), c.table)[0])

        def run(self, own=False):
            c, d, ctx = self.case, self.d, self.ctx
            w = [None, None] if own else self.work
            c.call(q, ctx, d, w[0])
            q.sample_logits(ctx, self.logits, vocab, None, None, None, None, None, None, self.u, c.rows, vocab, self.token,
                            self.p, w[1])
            q.tree_accept(ctx, d["start"], self.parents, self.draft, self.token, self.path, c.max_nodes, self.count, self.next,
                          3, c.rows, c.max_nodes)
            q.cache_compact_rows(ctx, d["k"], d["v"], 1, 0, c.total_pages, 16, kv_heads * 256, d["table"], c.table.shape[1],
                                 d["contexts"], self.path, c.max_nodes, self.count, 3)
            q.cache_copy_pages(ctx, d["k"], d["v"], 1, 0, c.total_pages, 16, kv_heads * 256, [int(c.table[0, 0])], [self.spare])

        def reset(self):
            self.d["k"].upload(self.case.k.view(np.uint16))
            self.d["v"].upload(self.case.v.view(np.uint16))
            for a in (self.d["out"], self.token, self.p, self.path, self.count, self.next):
                a.upload(np.zeros(a.shape, a.dtype))

        def result(self):
            return [a.download() for a in (self.d["out"], self.token, self.p, self.path, self.count, self.next, self.d["k"],
                                           self.d["v"])]

    steps = [Step(5, ctx), Step(18, ctx)]
    eager, graphs = [], []
    for s in steps:
        s.reset()
        s.run()
        eager.append(s.result())
    for s in steps:
        with _Graph(q, ctx) as g:
            s.run()
        graphs.append(g)
    with pytest.raises(q.Q35Error, match="workspace of its own"):
        with _Graph(q, ctx):
            steps[0].run(own=True)
    # a second context on the same stream, whose own workspace grows between the replays
    other = q.Context(0, q.lib.q35_context_stream(ctx.handle))
    larger = Step(7, other)
    for turn in range(4):
        print("replay", turn, flush=True)
        for i in ((0, 1) if turn % 2 == 0 else (1, 0)):
            steps[i].reset()
            graphs[i].replay()
            for got, want in zip(steps[i].result(), eager[i]):
                np.testing.assert_array_equal(got, want)
            larger.reset()
            larger.run(own=True)
        ctx.synchronize()
    # other inputs in the same buffers
    steps[0].u.upload((1.0 - steps[0].numbers).astype(np.float32))
    steps[0].reset()
    steps[0].run()
    want = steps[0].result()
    assert not np.array_equal(want[1], eager[0][1])
    steps[0].reset()
    graphs[0].replay()
    for got, w in zip(steps[0].result(), want):
        np.testing.assert_array_equal(got, w)
    for g in graphs:
        g.close()
    other.close()


def test_two_contexts_at_once(q, ctx):
    """Calls of two contexts (two streams) in flight together, each on its own workspace."""
    import threading
    other = q.Context(0)
    cases = [TreeCase(20, [300, 40], [5, 9], 4, 2, 64), TreeCase(21, [129, 260], [16, 2], 4, 2, 64)]
    rng = np.random.default_rng(1)
    x, u = rng.standard_normal((2, 5000)).astype(np.float32), rng.random(2).astype(np.float32)
    got = [None, None]

    def work(i, c):
        d = cases[i].device(c)
        token, logits, number = c.array(np.zeros(1, np.int32)), c.array(x[i:i + 1]), c.array(u[i:i + 1])
        for _ in range(1 if EMULATED else 20):
            cases[i].call(q, c, d)
            q.sample_logits(c, logits, 5000, None, None, None, None, None, None, number, 1, 5000, token)
        got[i] = d["out"].download(), token.download()
    if EMULATED:  # the host build runs one launch at a time
        for i, c in enumerate((ctx, other)):
            work(i, c)
    else:
        threads = [threading.Thread(target=work, args=a) for a in ((0, ctx), (1, other))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    for i in range(2):
        want, tol = cases[i].expected()
        assert (np.abs(got[i][0] - want) <= tol).all()
        assert got[i][1][0] == sample(x[i], u[i])[0]
    other.close()


@pytest.mark.skipif(EMULATED, reason="13 GB of cache")
def test_offsets_past_32_bits(q, ctx):
    """Pools of more than 2^32 bytes and 2^31 values: attention, copies and compaction on their last pages."""
    kv_heads, hd, page = 2, 256, 16
    width = kv_heads * hd
    pages = (2 ** 31) // (page * width) + 5000
    small = TreeCase(30, [50, 20], [4, 9], 4, kv_heads, hd)
    high = pages - small.total_pages  # the case's pages at the pools' end
    k, v = (ctx.array(shape=(pages, page, kv_heads, hd), dtype=np.uint16) for _ in range(2))
    offset = high * page * width * 2
    for pool, host in ((k, small.k), (v, small.v)):
        bits = np.ascontiguousarray(host.view(np.uint16))
        ctx.check(q.lib.q35_memcpy_h2d(ctx.handle, ctypes.c_void_p(pool.address + offset), ctypes.c_void_p(bits.ctypes.data),
                                       bits.nbytes), "h2d")
    d = small.device(ctx)
    table = np.where(small.table < 0, -1, small.table + high).astype(np.int32)
    d["k"], d["v"], d["table"] = k, v, ctx.array(table)
    small.call(q, ctx, d, total_pages=pages)
    want, tol = small.expected()
    assert (np.abs(d["out"].download() - want) <= tol).all()
    # the path 0, 2 of each tree, then the first page of request 0 to a page at the start
    path, count = np.array([[0, 2], [0, 5]], np.int32), np.array([2, 2], np.int32)
    q.cache_compact_rows(ctx, k, v, 1, 0, pages, page, width, d["table"], table.shape[1], d["contexts"], ctx.array(path), 2,
                         ctx.array(count), 2)
    q.cache_copy_pages(ctx, k, v, 1, 0, pages, page, width, [table[0, 0], table[1, 0]], [3, pages // 2])

    def read(pool, first, n):
        out = np.empty((n, page, kv_heads, hd), np.uint16)
        ctx.check(q.lib.q35_memcpy_d2h(ctx.handle, ctypes.c_void_p(out.ctypes.data),
                                       ctypes.c_void_p(pool.address + first * page * width * 2), out.nbytes), "d2h")
        return out
    for pool, host in ((k, small.k), (v, small.v)):
        host = host.view(np.uint16).copy()
        for b in range(2):
            f, t = int(small.contexts[b] + path[b, 1]), int(small.contexts[b] + 1)
            host[small.table[b, t // 16], t % 16] = host[small.table[b, f // 16], f % 16]
        np.testing.assert_array_equal(read(pool, high, small.total_pages), host)
        np.testing.assert_array_equal(read(pool, 3, 1)[0], host[small.table[0, 0]])
        np.testing.assert_array_equal(read(pool, pages // 2, 1)[0], host[small.table[1, 0]])
