"""Attention of drafted trees over the paged cache (q35_attention_tree_paged)
against the formula in 64 bits: tree and head shapes, page sizes, contexts from
none to several ranges, masks that leave a node nothing, infinities and NaN
where nobody looks, refused calls, and requests the device refuses."""
import ctypes

import numpy as np
import pytest

from tests.drafted_util import EMULATED, TreeCase, ancestor_bits, random_tree

pytestmark = pytest.mark.gpu


def _check(q, ctx, case, workspace=None):
    print(f"tree attention: contexts {case.contexts.tolist()} nodes {case.nodes.tolist()} heads {case.heads}/{case.kv_heads} "
          f"dim {case.head_dim} page {case.page_tokens}", flush=True)
    got = case.run(q, ctx, workspace).astype(np.float64)
    want, tol = case.expected()
    assert np.isfinite(want).all()
    np.testing.assert_array_equal(np.isfinite(got), True)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / np.maximum(tol, 1e-300))
    return got


# (contexts, nodes): single nodes, empty contexts, tile borders (32 rows), trees
# across them, requests without nodes between others, several ranges (128 rows)
SIZES = [([0], [1]), ([1], [1]), ([31, 32, 33], [1, 1, 1]), ([0, 5], [3, 9]), ([30, 64, 100], [5, 0, 17]),
         ([127, 200, 300], [8, 1, 13])]


@pytest.mark.parametrize("contexts,nodes", SIZES)
def test_sizes(q, ctx, contexts, nodes):
    _check(q, ctx, TreeCase(3, contexts, nodes))


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(2, 2, 64), (6, 2, 64), (5, 1, 128), (8, 8, 128), (16, 1, 64),
                                                     (3, 3, 256), (40, 1, 64)])
def test_heads(q, ctx, heads, kv_heads, head_dim):
    _check(q, ctx, TreeCase(4, [45, 3], [7, 11], heads, kv_heads, head_dim))


@pytest.mark.parametrize("page_tokens", [1, 2, 4, 64, 256])
def test_page_sizes(q, ctx, page_tokens):
    _check(q, ctx, TreeCase(5, [70, 2], [6, 6], 4, 2, 64, page_tokens))


@pytest.mark.parametrize("nodes,context", [(64, 10), (65, 0), (130, 17), (256, 1), (100, 96)])
def test_wide_trees(q, ctx, nodes, context):
    """Masks of several words, their tiles beginning at any bit of a word."""
    _check(q, ctx, TreeCase(6, [context], [nodes], 2, 1, 64))


def test_without_gates(q, ctx):
    _check(q, ctx, TreeCase(7, [50], [4], gated=False))


def test_bounds_above_the_sizes(q, ctx):
    """max_nodes and max_len are bounds only; rows past the last request stay as they were."""
    case = TreeCase(8, [40, 9], [3, 6], 4, 2, 64, max_nodes=70, max_len=1000, spare_rows=5)
    got = _check(q, ctx, case)
    assert np.all(got[-5:] == case.fill)


@pytest.mark.skipif(EMULATED, reason="long for the host build")
@pytest.mark.parametrize("contexts,nodes,heads,kv_heads", [([2000, 3], [12, 40], 8, 2), ([5000], [33], 4, 4),
                                                           ([700] * 9, [9, 1, 30, 2, 16, 5, 8, 8, 3], 16, 4)])
def test_long(q, ctx, contexts, nodes, heads, kv_heads):
    _check(q, ctx, TreeCase(9, contexts, nodes, heads, kv_heads))


def test_nothing_seen(q, ctx):
    """Masks without a bit and no context: zeros. Bits past the request's nodes do not count."""
    bits = [np.zeros((4, 64), bool), ancestor_bits(random_tree(np.random.default_rng(1), 3))]
    bits[0][1, 2] = True   # sees node 2 alone
    bits[0][2, 40] = True  # a bit past the nodes
    case = TreeCase(10, [0, 20], [4, 3], 4, 2, 64, bits=bits, max_nodes=64)
    got = _check(q, ctx, case)
    assert np.all(got[[0, 2, 3]] == 0.0) and np.any(got[1] != 0.0)


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_special_values_reach_only_who_sees_them(q, ctx, where, value):
    """A drafted node whose key or value is not finite: the nodes that do not see it are as without it."""
    parents = np.array([-1, 0, 0, 1, 2, 4], np.int32)
    case = TreeCase(11, [43], [6], 4, 2, 64, bits=[ancestor_bits(parents)])
    clean, tol = case.expected()
    t = int(case.contexts[0]) + 2
    pool = case.k if where == "k" else case.v
    pool[case.table[0, t // 16], t % 16, 1, 5] = value
    got = case.run(q, ctx)
    seen = np.zeros((6, 4), bool)
    seen[[2, 4, 5], 2:] = True  # nodes 2, 4, 5 of KV head 1
    # (such a tile sums its products in fp32 as they are, in another order: both
    # ways are within the formula's bound, neither has the other's bits)
    assert (np.abs(got - clean) <= tol)[~seen].all()
    with np.errstate(invalid="ignore"):
        want, _ = case.expected()
    if where == "v":
        np.testing.assert_array_equal(np.isfinite(got), np.isfinite(want))
        assert np.array_equal(got[~np.isfinite(got) & ~np.isnan(got)], want[~np.isfinite(want) & ~np.isnan(want)])
    elif np.isnan(value):
        assert np.isnan(got[seen]).all()
    # (an infinite key makes a score of who sees it infinite or NaN: either is
    # allowed there, as the two parts of a query may differ in sign)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-3, 300.0, 3e4, 1e30])
def test_query_magnitudes(q, ctx, q_scale):
    """Queries of any fp32 size keep 22 bits under their largest value."""
    case = TreeCase(12, [60], [5], 4, 2, 64, q_scale=q_scale)
    case.scale /= max(q_scale, 1.0)
    _check(q, ctx, case)


def test_lowest_and_infinite_scores(q, ctx):
    """Scores of fp32's lowest size on some rows leave the others' weights."""
    case = TreeCase(13, [40], [3], 2, 1, 64)
    case.q[:] = 0.0
    case.q[:, :, 0] = 1.0
    case.k[..., 0] = np.where(np.isnan(case.k[..., 0]), np.nan, -65504.0)
    t = 7
    case.k[case.table[0, t // 16], t % 16, :, 0] = 0.0
    case.scale = 1e33  # every other score overflows to -inf
    got = case.run(q, ctx)
    gate = 1.0 / (1.0 + np.exp(-case.gates.astype(np.float64)))
    want = case.v[case.table[0, t // 16], t % 16].astype(np.float64) * gate
    np.testing.assert_allclose(got, want, rtol=2.0 ** -20)


def test_requests_out_of_bounds(q, ctx):
    """Refused on the device: NaN in the rows of a request that breaks a bound, the others as without it."""
    case = TreeCase(14, [20, 30, 40, 10], [3, 4, 2, 5], 4, 2, 64)
    want, tol = case.expected()
    for what in ("context", "negative", "page", "nodes"):
        print("tree attention out of bounds:", what, flush=True)
        d = case.device(ctx)
        other = {}
        if what == "context":
            d["contexts"] = ctx.array(np.array([20, 100000, 40, 10], np.int32))
        elif what == "negative":
            d["contexts"] = ctx.array(np.array([20, -1, 40, 10], np.int32))
        elif what == "page":
            table = case.table.copy()
            table[1, 0] = case.total_pages
            d["table"] = ctx.array(table)
        else:
            other["max_nodes"] = 4  # the last request has 5
        case.call(q, ctx, d, **other)
        got = d["out"].download()
        bad = slice(9, 14) if what == "nodes" else slice(3, 7)
        assert np.isnan(got[bad]).all(), what
        ok = np.ones(case.rows, bool)
        ok[bad] = False
        assert (np.abs(got - want) <= tol)[ok].all(), what


def test_node_ranges_out_of_bounds(q, ctx):
    """Row ranges that leave the rows or run backwards: nothing is written for them."""
    case = TreeCase(15, [20, 30, 40], [3, 4, 2], 4, 2, 64)
    d = case.device(ctx)
    d["start"] = ctx.array(np.array([0, 3, 100, 9], np.int32))
    case.call(q, ctx, d)
    got = d["out"].download()
    want, tol = case.expected()
    assert (np.abs(got - want) <= tol)[:3].all() and np.all(got[3:] == case.fill)


def test_page_outside_where_nobody_looks(q, ctx):
    """A table entry outside the pool counts only for the nodes that see its rows."""
    bits = [np.eye(20, dtype=bool)]
    case = TreeCase(16, [0], [20], 4, 2, 64, page_tokens=4, bits=bits)
    want, tol = case.expected()
    d = case.device(ctx)
    table = case.table.copy()
    table[0, 2] = -5  # nodes 8 .. 11
    d["table"] = ctx.array(table)
    case.call(q, ctx, d)
    got = d["out"].download()
    ok = np.ones(20, bool)
    ok[8:12] = False
    assert np.isnan(got[~ok]).all() and (np.abs(got - want) <= tol)[ok].all()


def test_workspaces(q, ctx):
    case = TreeCase(17, [600, 300], [3, 9], 2, 1, 64)
    size = q.attention_tree_workspace(ctx, case.batch, case.rows, case.max_nodes, case.max_len, 2, 1, 64)
    assert size > 0
    own = _check(q, ctx, case)
    given = case.run(q, ctx, ctx.array(shape=(size,), dtype=np.uint8))
    np.testing.assert_array_equal(given, own.astype(np.float32))
    with pytest.raises(q.Q35Error, match="workspace too small"):
        case.run(q, ctx, ctx.array(shape=(size - 1,), dtype=np.uint8))


def test_refusals(q, ctx):
    case = TreeCase(18, [20], [3], 4, 2, 64)
    for other, what in [(dict(head_dim=96), "head_dim"), (dict(heads=3), "heads % kv_heads"), (dict(heads=0), "empty shape"),
                        (dict(kv_heads=0), "empty shape"), (dict(batch=0), "empty shape"), (dict(max_nodes=0), "empty shape"),
                        (dict(max_nodes=257), "256 nodes"), (dict(page_tokens=12), "power-of-two"),
                        (dict(page_tokens=0), "power-of-two"), (dict(max_len=1000), "page table"),
                        (dict(total_pages=0), "empty pool"), (dict(scale=float("nan")), "scale"),
                        (dict(batch=65536), "65535"), (dict(total_pages=2 ** 31), "pool")]:
        d = case.device(ctx)
        with pytest.raises(q.Q35Error, match=what):
            case.call(q, ctx, d, **other)
        assert np.all(d["out"].download() == case.fill), other
    for missing in ("q", "k", "v", "table", "contexts", "start", "masks", "out"):
        d = case.device(ctx)

        class Nothing:
            ptr = None
        d[missing] = Nothing
        with pytest.raises(q.Q35Error, match="missing buffer"):
            case.call(q, ctx, d)
    d = case.device(ctx)

    class Odd:
        ptr = ctypes.c_void_p(d["q"].address + 4)
    d["q"] = Odd
    with pytest.raises(q.Q35Error, match="alignment"):
        case.call(q, ctx, d)
    case.call(q, ctx, case.device(ctx), rows=0)  # no rows: nothing to do
    ctx.synchronize()


def test_sizes_past_the_work_units(q, ctx):
    """Bounds whose workgroup shares would no longer be exact."""
    assert q.attention_tree_workspace(ctx, 65535, 65535, 1, 2 ** 31 - 2000, 2, 2, 64) > 0
    for batch, heads in [(65535, 8), (1, 65)]:
        with pytest.raises(q.Q35Error, match="too large"):
            q.attention_tree_workspace(ctx, batch, 65535, 1, 2 ** 31 - 2000, heads, heads, 64)
