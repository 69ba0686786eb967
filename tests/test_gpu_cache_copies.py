"""Copies inside the paged cache (q35_cache_copy_pages, q35_cache_compact_rows,
q35_page_copy, q35_page_fork) against the same moves on host arrays, bit for
bit, and the acceptance of drafted trees (q35_tree_accept) against its walk."""
import numpy as np
import pytest

from tests.drafted_util import EMULATED, accept, page_table, random_tree, starts
from tests.model_util import build_small_model, small_dims, upload_model

pytestmark = pytest.mark.gpu


def _pools(rng, layers, pages, page_tokens, width, spare=0):
    """K and V bits; `spare` elements lie between the layers."""
    shape = (layers, pages * page_tokens * width + spare)
    return [rng.integers(0, 1 << 16, size=shape, dtype=np.uint16) for _ in range(2)]


def _layers(pool, pages, page_tokens, width):
    return pool[:, :pages * page_tokens * width].reshape(-1, pages, page_tokens, width)


# widths that take 16-byte, 4-byte and 2-byte pieces
@pytest.mark.parametrize("layers,page_tokens,width,spare", [(1, 16, 512, 0), (6, 16, 512, 0), (2, 4, 60, 0), (3, 5, 7, 0),
                                                            (2, 16, 128, 8), (2, 16, 128, 2), (2, 64, 64, 1)])
@pytest.mark.parametrize("whole", [True, False])
def test_copy_pages(q, ctx, layers, page_tokens, width, spare, whole):
    rng = np.random.default_rng(layers * width)
    pages = 24
    k, v = _pools(rng, layers, pages, page_tokens, width, spare)
    ids = rng.permutation(pages)
    src, dst = np.concatenate([ids[:5], ids[:2]]), ids[5:12]  # two sources read twice
    tokens = None if whole else rng.integers(0, page_tokens + 1, size=7)
    dk, dv = ctx.array(k), ctx.array(v)
    print(f"copy pages layers={layers} page={page_tokens} width={width} spare={spare}", flush=True)
    q.cache_copy_pages(ctx, dk, dv, layers, k.shape[1], pages, page_tokens, width, src, dst, tokens)
    for pool, got in ((k, dk.download()), (v, dv.download())):
        want = pool.copy()
        at = _layers(want, pages, page_tokens, width)
        for i in range(7):
            n = page_tokens if whole else int(tokens[i])
            at[:, dst[i], :n] = _layers(pool, pages, page_tokens, width)[:, src[i], :n]
        np.testing.assert_array_equal(got, want)


def test_copy_many_pages(q, ctx):
    """More pairs than one launch takes."""
    rng = np.random.default_rng(1)
    pages = 1300
    k, v = _pools(rng, 1, pages, 2, 8)
    ids = rng.permutation(pages)
    src, dst = ids[:600], ids[600:1200]
    dk, dv = ctx.array(k), ctx.array(v)
    q.cache_copy_pages(ctx, dk, dv, 1, 0, pages, 2, 8, src, dst)
    for pool, got in ((k, dk.download()), (v, dv.download())):
        at = _layers(pool, pages, 2, 8)
        at[:, dst] = at[:, src]
        np.testing.assert_array_equal(got, pool)


def test_unaligned_pools(q, ctx):
    """Pools that begin between 16-byte addresses."""
    import ctypes
    rng = np.random.default_rng(2)
    for shift in (2, 4, 8):
        k, v = (rng.integers(0, 1 << 16, size=shift // 2 + 6 * 16 * 16, dtype=np.uint16) for _ in range(2))
        dk, dv = ctx.array(k), ctx.array(v)

        class At:
            def __init__(self, a):
                self.ptr = ctypes.c_void_p(a.address + shift)
        q.cache_copy_pages(ctx, At(dk), At(dv), 1, 0, 6, 16, 16, [1, 4], [0, 5], [16, 3])
        for pool, got in ((k, dk.download()), (v, dv.download())):
            at = pool[shift // 2:].reshape(6, 16, 16)
            at[0] = at[1]
            at[5, :3] = at[4, :3]
            np.testing.assert_array_equal(got, pool)


@pytest.mark.skipif(EMULATED, reason="pages of 140 MB")
def test_copy_a_large_page(q, ctx):
    """More pieces in a page than a launch has workgroups' worth (2-byte pieces)."""
    rng = np.random.default_rng(5)
    page_tokens, width = 2 ** 20, 67
    k = rng.integers(0, 1 << 16, size=2 * page_tokens * width + 3, dtype=np.uint16)
    v = k[::-1].copy()
    dk, dv = ctx.array(k), ctx.array(v)
    tokens = page_tokens - 3
    q.cache_copy_pages(ctx, dk, dv, 1, 0, 2, page_tokens, width, [1], [0], [tokens])
    for pool, got in ((k, dk.download()), (v, dv.download())):
        pool[:tokens * width] = pool[page_tokens * width:(page_tokens + tokens) * width]
        assert np.array_equal(got, pool)


def test_copy_refusals(q, ctx):
    rng = np.random.default_rng(3)
    k, v = _pools(rng, 2, 8, 4, 16)
    dk, dv = ctx.array(k), ctx.array(v)

    def call(src, dst, tokens=None, layers=2, stride=8 * 4 * 16, pages=8, page_tokens=4, width=16):
        q.cache_copy_pages(ctx, dk, dv, layers, stride, pages, page_tokens, width, src, dst, tokens)
    for args, what in [((([0], [8])), "outside"), (([-1], [2]), "outside"), (([0], [2], [5]), "more tokens"),
                       (([0], [2], [-1]), "more tokens"), (([0, 1], [2, 2]), "written twice"), (([0, 2], [2, 3]), "both read"),
                       (([1], [1]), "both read")]:
        with pytest.raises(q.Q35Error, match=what):
            call(*args)
    for kw, what in [(dict(layers=0), "empty"), (dict(pages=0), "empty"), (dict(page_tokens=0), "empty"), (dict(width=0), "empty"),
                     (dict(stride=8 * 4 * 16 - 1), "overlap"), (dict(pages=2 ** 31), "2\\^31")]:
        with pytest.raises(q.Q35Error, match=what):
            call([0], [1], **kw)
    with pytest.raises(ValueError):
        call([0, 1], [2])
    call([], [])
    np.testing.assert_array_equal(dk.download(), k)
    np.testing.assert_array_equal(dv.download(), v)


@pytest.mark.parametrize("pairs", [16, 17, 31, 32, 33, 63, 64, 65, 300])
def test_copy_refusals_among_many_pairs(q, ctx, pairs):
    rng = np.random.default_rng(pairs)
    pages = 2 * pairs + 3
    k, v = _pools(rng, 1, pages, 2, 8)
    dk, dv = ctx.array(k), ctx.array(v)
    ids = rng.permutation(pages)
    for first, last in [(0, pairs - 1), (pairs - 2, 1)]:
        src, dst = ids[:pairs].copy(), ids[pairs:2 * pairs].copy()
        dst[first] = dst[last]
        with pytest.raises(q.Q35Error, match="written twice"):
            q.cache_copy_pages(ctx, dk, dv, 1, 0, pages, 2, 8, src, dst)
        src, dst = ids[:pairs].copy(), ids[pairs:2 * pairs].copy()
        src[first] = dst[last]
        with pytest.raises(q.Q35Error, match="both read"):
            q.cache_copy_pages(ctx, dk, dv, 1, 0, pages, 2, 8, src, dst)
    np.testing.assert_array_equal(dk.download(), k)
    np.testing.assert_array_equal(dv.download(), v)


def _compact(pool, table, contexts, path, count, page_tokens):
    for b in range(len(contexts)):
        for j in range(int(count[b])):
            f, t = int(contexts[b] + path[b, j]), int(contexts[b]) + j
            pool[:, table[b, t // page_tokens], t % page_tokens] = pool[:, table[b, f // page_tokens], f % page_tokens]


@pytest.mark.parametrize("layers,page_tokens,width", [(1, 16, 512), (6, 16, 512), (2, 4, 60), (2, 1, 7), (1, 64, 24)])
def test_compact_rows(q, ctx, layers, page_tokens, width):
    rng = np.random.default_rng(layers + width)
    contexts = np.array([0, 3, 15, 16, 77, 5], np.int32)
    paths = [[0], [0, 1, 2, 3], [0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12], [0, 2, 3, 9, 10, 30], [], [3, 4, 20]]
    count = np.array([len(p) for p in paths], np.int32)
    path = np.full((6, 12), -1, np.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = p
    table, pages = page_table(rng, contexts + 31, page_tokens)
    k, v = _pools(rng, layers, pages, page_tokens, width)
    dk, dv = ctx.array(k), ctx.array(v)
    print(f"compact layers={layers} page={page_tokens} width={width}", flush=True)
    q.cache_compact_rows(ctx, dk, dv, layers, k.shape[1], pages, page_tokens, width, ctx.array(table), table.shape[1],
                         ctx.array(contexts), ctx.array(path), 12, ctx.array(count), 6)
    for pool, got in ((k, dk.download()), (v, dv.download())):
        _compact(_layers(pool, pages, page_tokens, width), table, contexts, path, count, page_tokens)
        np.testing.assert_array_equal(got, pool)


@pytest.mark.parametrize("count", [255, 256, 257, 512, 600])
@pytest.mark.parametrize("bad", [None, 0, 254, -1])
def test_compact_long_paths(q, ctx, count, bad):
    """Paths of more steps than a workgroup has threads, and one bad step among
    them, which leaves its request as it is."""
    rng = np.random.default_rng(count)
    page_tokens, context = 16, 21
    path = np.arange(count, dtype=np.int32) + np.sort(rng.integers(0, 40, size=count)).astype(np.int32)
    paths = np.stack([path, path])
    contexts = np.full(2, context, np.int32)
    table, pages = page_table(rng, np.full(2, context + count + 40), page_tokens)
    k, v = _pools(rng, 1, pages, page_tokens, 24)
    dk, dv = ctx.array(k), ctx.array(v)
    if bad is not None:
        paths[1, bad] = table.shape[1] * page_tokens - context  # the first row past the table
    q.cache_compact_rows(ctx, dk, dv, 1, k.shape[1], pages, page_tokens, 24, ctx.array(table), table.shape[1],
                         ctx.array(contexts), ctx.array(paths), count, ctx.array(np.full(2, count, np.int32)), 2)
    moved = np.array([count, count if bad is None else 0])
    for pool, got in ((k, dk.download()), (v, dv.download())):
        _compact(_layers(pool, pages, page_tokens, 24), table, contexts, paths, moved, page_tokens)
        np.testing.assert_array_equal(got, pool)


def test_compact_out_of_bounds(q, ctx):
    """Requests that the device refuses are left as they are; the others move."""
    rng = np.random.default_rng(4)
    contexts = np.array([8, 8, 8, 8, 8, -1, 8, 8], np.int32)
    path = np.tile(np.array([0, 2, 5], np.int32), (8, 1))
    path[1] = [0, 0, 5]     # before its place
    path[2] = [0, 2, 1000]  # past the table
    path[3] = [0, -1, 5]
    count = np.array([3, 3, 3, 3, 4, 3, 3, 3], np.int32)  # request 4: more than a path row
    table, pages = page_table(rng, np.full(8, 20), 4)
    table[6, 3] = pages  # request 6: a page outside the pool under path[2]
    k, v = _pools(rng, 2, pages, 4, 8)
    dk, dv = ctx.array(k), ctx.array(v)
    q.cache_compact_rows(ctx, dk, dv, 2, k.shape[1], pages, 4, 8, ctx.array(table), table.shape[1], ctx.array(contexts),
                         ctx.array(path), 3, ctx.array(count), 8)
    moved = np.array([3, 0, 0, 0, 0, 0, 0, 3], np.int32)
    for pool, got in ((k, dk.download()), (v, dv.download())):
        _compact(_layers(pool, pages, 4, 8), table, contexts, path, moved, 4)
        np.testing.assert_array_equal(got, pool)


def test_compact_refusals(q, ctx):
    rng = np.random.default_rng(5)
    k, v = _pools(rng, 1, 4, 4, 8)
    dk, dv = ctx.array(k), ctx.array(v)
    table, one = ctx.array(np.arange(4, dtype=np.int32).reshape(1, 4)), ctx.array(np.array([0], np.int32))

    class Nothing:
        ptr = None
    good = dict(table=table, lens=one, path=one, count=one, page_tokens=4, max_pages=4, stride=1, batch=1)
    for other, what in [(dict(table=Nothing), "missing"), (dict(lens=Nothing), "missing"), (dict(path=Nothing), "missing"),
                        (dict(count=Nothing), "missing"), (dict(page_tokens=3), "power-of-two"), (dict(max_pages=0), "missing"),
                        (dict(stride=0), "missing"), (dict(batch=65536), "65535")]:
        a = {**good, **other}
        with pytest.raises(q.Q35Error, match=what):
            q.cache_compact_rows(ctx, dk, dv, 1, 0, 4, a["page_tokens"], 8, a["table"], a["max_pages"], a["lens"], a["path"],
                                 a["stride"], a["count"], a["batch"])
    q.cache_compact_rows(ctx, dk, dv, 1, 0, 4, 4, 8, table, 4, one, one, 1, one, 0)
    np.testing.assert_array_equal(dk.download(), k)


@pytest.mark.parametrize("nodes", [[1], [2, 1, 5], [64, 65, 63, 128], [256, 3, 200], [7, 0, 9]])
def test_accept(q, ctx, nodes):
    rng = np.random.default_rng(len(nodes) + sum(nodes))
    start = starts(nodes)
    rows, width = int(start[-1]), max(nodes)
    parents = np.concatenate([random_tree(rng, n) if n else np.zeros(0, np.int32) for n in nodes]).astype(np.int32)
    draft = rng.integers(0, 4, size=rows).astype(np.int32)  # few tokens: siblings often hold the same one
    sampled = rng.integers(0, 4, size=rows).astype(np.int32)
    print(f"accept nodes={nodes}", flush=True)
    out = [ctx.array(np.full((len(nodes), width + 2), 99, np.int32)), ctx.array(np.full(len(nodes), 99, np.int32)),
           ctx.array(np.full(len(nodes), 99, np.int32))]
    q.tree_accept(ctx, ctx.array(start), ctx.array(parents), ctx.array(draft), ctx.array(sampled), out[0], width + 2, out[1],
                  out[2], len(nodes), rows, width)
    path, count, token = (a.download() for a in out)
    want = accept(start, parents, draft, sampled, width)
    np.testing.assert_array_equal(path[:, :width], want[0])
    np.testing.assert_array_equal(path[:, width:], 99)
    np.testing.assert_array_equal(count, want[1])
    np.testing.assert_array_equal(token, want[2])


def test_accept_a_full_chain(q, ctx):
    """Every drafted token of a chain of 256 accepted."""
    n = 256
    draft = np.arange(n, dtype=np.int32)
    out = [ctx.array(np.zeros((1, n), np.int32)), ctx.array(np.zeros(1, np.int32)), ctx.array(np.zeros(1, np.int32))]
    q.tree_accept(ctx, ctx.array(starts([n])), ctx.array(draft - 1), ctx.array(draft), ctx.array(draft + 1), out[0], n, out[1],
                  out[2], 1, n, n)
    assert out[0].download()[0].tolist() == list(range(n))
    assert out[1].download().tolist() == [n] and out[2].download().tolist() == [n]


def test_accept_out_of_bounds(q, ctx):
    """Parents that come later, point outside or at themselves never match; row ranges outside give no nodes."""
    start = np.array([0, 4, 3, 9, 12], np.int32)
    parents = np.array([-1, 7, 2, 0, -1, 0, 1, -9, 3, 0, 0, 0], np.int32)
    draft = np.full(12, 5, np.int32)
    sampled = np.full(12, 5, np.int32)
    out = [ctx.array(np.zeros((4, 4), np.int32)), ctx.array(np.zeros(4, np.int32)), ctx.array(np.zeros(4, np.int32))]
    q.tree_accept(ctx, ctx.array(start), ctx.array(parents), ctx.array(draft), ctx.array(sampled), out[0], 4, out[1], out[2], 4,
                  12, 4)
    assert out[0].download().tolist() == [[0, 3, -1, -1], [-1] * 4, [-1] * 4, [0, 1, -1, -1]]
    assert out[1].download().tolist() == [2, 0, 0, 2]
    assert out[2].download().tolist() == [5, -1, -1, 5]


def test_accept_refusals(q, ctx):
    a = ctx.array(np.zeros(8, np.int32))

    class Nothing:
        ptr = None
    for i in range(7):
        args = [a] * 7
        args[i] = Nothing
        with pytest.raises(q.Q35Error, match="missing"):
            q.tree_accept(ctx, args[0], args[1], args[2], args[3], args[4], 4, args[5], args[6], 1, 4, 4)
    for batch, stride, nodes, what in [(0, 4, 4, "missing"), (1, 3, 4, "shorter"), (1, 4, 0, "missing"), (1, 300, 257, "256")]:
        with pytest.raises(q.Q35Error, match=what):
            q.tree_accept(ctx, a, a, a, a, a, stride, a, a, batch, 4, nodes)


@pytest.fixture(scope="module")
def runtime(q, ctx):
    dims, sched = small_dims()
    model = upload_model(q, ctx, dims, sched, build_small_model(dims, sched, seed=5))
    rt = q.Runtime(model, max_slots=2, max_batch=2, max_context=64, page_tokens=16, total_pages=12, max_step_rows=32)
    yield rt
    rt.close()
    model.close()


def test_page_fork(q, runtime):
    rt, lib = runtime, q.lib
    free = lib.q35_runtime_free_pages(rt.handle)
    pages = [rt.page_alloc() for _ in range(3)]
    out = rt.page_fork(pages, 37, 3)  # two full pages and five rows of the third
    assert out.shape == (3, 3) and (out[:, :2] == pages[:2]).all()
    copies = out[:, 2].tolist()
    assert len(set(copies + pages)) == 6
    assert [lib.q35_page_refcount(rt.handle, p) for p in pages] == [4, 4, 1]
    assert [lib.q35_page_refcount(rt.handle, p) for p in copies] == [1, 1, 1]
    whole = rt.page_fork(pages[:2], 32, 2)  # full pages only: nothing is copied
    assert (whole == pages[:2]).all() and lib.q35_page_refcount(rt.handle, pages[0]) == 6
    assert lib.q35_runtime_free_pages(rt.handle) == free - 6
    assert rt.page_fork([], 0, 4).size == 0
    for bad, tokens, children, what in [(pages, 33 + 16, 1, "cover"), (pages, 32, 1, "cover"), (pages, -1, 1, "cover"),
                                        ([pages[0], 99, pages[2]], 40, 1, "not allocated"), (pages, 40, 7, "exhausted")]:
        with pytest.raises(q.Q35Error, match=what):
            rt.page_fork(bad, tokens, children)
    assert lib.q35_runtime_free_pages(rt.handle) == free - 6
    assert [lib.q35_page_refcount(rt.handle, p) for p in pages] == [6, 6, 1]
    for row in out.tolist() + whole.tolist() + [pages]:
        for p in row:
            rt.page_release(p)
    assert lib.q35_runtime_free_pages(rt.handle) == free


def test_forked_requests_decode_as_their_own(q, ctx, runtime):
    """Two continuations of one prompt on forked pages give the tokens each gives alone."""
    rt = runtime
    prompt = np.arange(3, 24, dtype=np.int32)  # 21 positions: one full page, five rows of the next

    def prefill(slot, pages):
        table = np.array(pages + [0] * (rt.max_pages - len(pages)), np.int32)
        rt.prefill(slot, 0, prompt, table)

    def decode(slots, tables, tokens):
        out = []
        for step in range(3):
            pos = np.full(len(slots), prompt.size + step, np.int32)
            tokens = rt.step(slots, pos, tokens, tables)
            out.append(tokens.copy())
        return np.stack(out, 1)

    alone = []
    for first in (11, 29):
        slot, pages = rt.slot_alloc(prompt), [rt.page_alloc() for _ in range(2)]
        prefill(slot, pages)
        table = np.zeros((1, rt.max_pages), np.int32)
        table[0, :2] = pages
        alone.append(decode([slot], table, [first])[0])
        rt.slot_free(slot)
        for p in pages:
            rt.page_release(p)
    # one prompt's pages forked; its DeltaNet state comes from the same prompt in a second slot
    slots = [rt.slot_alloc(prompt), rt.slot_alloc(prompt)]
    pages, other = [rt.page_alloc() for _ in range(2)], [rt.page_alloc() for _ in range(2)]
    prefill(slots[0], pages)
    prefill(slots[1], other)
    forked = rt.page_fork(pages, prompt.size, 2)
    for p in pages + other:
        rt.page_release(p)
    tables = np.zeros((2, rt.max_pages), np.int32)
    tables[:, :2] = forked
    got = decode(slots, tables, [11, 29])
    np.testing.assert_array_equal(got, np.stack(alone))
    for s in slots:
        rt.slot_free(s)
    for p in forked.ravel().tolist():
        rt.page_release(p)
