"""Pools of the cache copies that share memory: refused where the moves of one
would meet the other's, served where the layers only alternate."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PAGES, PAGE, WIDTH = 6, 4, 8
ELEMS = PAGES * PAGE * WIDTH  # of a layer


class _At:
    def __init__(self, array, elems):
        self.ptr = ctypes.c_void_p(array.address + 2 * elems)


def _calls(q, ctx, k, v, layers, stride):
    table, context = ctx.array(np.array([[4, 1, 5, 0]], np.int32)), ctx.array(np.array([3], np.int32))
    path, count = ctx.array(np.array([[0, 2, 5]], np.int32)), ctx.array(np.array([3], np.int32))
    return (lambda: q.cache_copy_pages(ctx, k, v, layers, stride, PAGES, PAGE, WIDTH, [1, 4], [0, 3], [4, 2]),
            lambda: q.cache_compact_rows(ctx, k, v, layers, stride, PAGES, PAGE, WIDTH, table, 4, context, path, 3, count, 1))


@pytest.mark.parametrize("layers,stride,offset", [(1, 0, 1), (1, 0, ELEMS - 8), (1, 0, 8 - ELEMS), (3, ELEMS, ELEMS), (3, ELEMS, -2 * ELEMS),
                                                  (3, 2 * ELEMS, ELEMS - 1), (3, 2 * ELEMS, 5 * ELEMS - 1), (3, 2 * ELEMS, 4 * ELEMS),
                                                  (3, 2 * ELEMS, 3 * ELEMS + 8)])
def test_overlapping_pools(q, ctx, layers, stride, offset):
    rng = np.random.default_rng(1)
    host = rng.integers(0, 1 << 16, size=16 * ELEMS, dtype=np.uint16)
    pool = ctx.array(host)
    for call in _calls(q, ctx, _At(pool, 5 * ELEMS), _At(pool, 5 * ELEMS + offset), layers, stride):
        with pytest.raises(q.Q35Error, match="pools overlap"):
            call()
    np.testing.assert_array_equal(pool.download(), host)


def test_one_pool_for_both(q, ctx):
    """The same pool as K and V: a page is copied, rows are not moved twice."""
    rng = np.random.default_rng(2)
    host = rng.integers(0, 1 << 16, size=ELEMS, dtype=np.uint16)
    pool = ctx.array(host)
    copy, compact = _calls(q, ctx, pool, pool, 1, 0)
    copy()
    with pytest.raises(q.Q35Error, match="pools overlap"):
        compact()
    at = host.reshape(PAGES, PAGE, WIDTH)
    at[0], at[3, :2] = at[1], at[4, :2]
    np.testing.assert_array_equal(pool.download(), host)


@pytest.mark.parametrize("layers,stride,offset", [(3, 2 * ELEMS, ELEMS), (3, 2 * ELEMS, -ELEMS), (3, 2 * ELEMS, 5 * ELEMS), (1, 0, ELEMS),
                                                  (2, 3 * ELEMS, ELEMS + 8)])
def test_alternating_layers(q, ctx, layers, stride, offset):
    rng = np.random.default_rng(3)
    host = rng.integers(0, 1 << 16, size=16 * ELEMS, dtype=np.uint16)
    pool = ctx.array(host)
    copy, compact = _calls(q, ctx, _At(pool, 5 * ELEMS), _At(pool, 5 * ELEMS + offset), layers, stride)
    copy()
    compact()
    table = [4, 1, 5, 0]
    for start in (5 * ELEMS, 5 * ELEMS + offset):
        for l in range(layers):
            at = host[start + l * stride:][:ELEMS].reshape(PAGES, PAGE, WIDTH)
            at[0], at[3, :2] = at[1].copy(), at[4, :2].copy()
            for j, p in enumerate((0, 2, 5)):
                f, t = 3 + p, 3 + j
                at[table[t // PAGE], t % PAGE] = at[table[f // PAGE], f % PAGE]
    np.testing.assert_array_equal(pool.download(), host)
