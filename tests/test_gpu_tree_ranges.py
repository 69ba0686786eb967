"""Attention of drafted trees (q35_attention_tree_paged) over the range of
scales, scores and special values: large scores, scale 0 and scales that
underflow, values that are not finite in requests cut into several parts."""
import numpy as np
import pytest

from tests.drafted_util import TreeCase

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("top", [2.0 ** 23, 2.0 ** 24, 1.03 * 2.0 ** 25, 1.03 * 2.0 ** 26, 1.7 * 2.0 ** 27, 2.0 ** 28, 1.3 * 2.0 ** 29])
def test_large_scores(q, ctx, top, scale):
    """Scores (in binades) that fp32 holds no fraction of, or not every whole
    number: a row each ahead of the others by more than they can be off by, and
    rows of equal scores."""
    case = TreeCase(31, [70, 9], [5, 6], 4, 2, 64)
    rng = np.random.default_rng(5)
    sign = 1.0 if scale > 0 else -1.0
    case.scale = scale
    case.q[:] = 0.0
    case.q[:, :, 3] = top * 0.6931471805599453 / abs(scale)
    case.k[..., 3] = np.where(np.isnan(case.k[..., 3]), np.nan, sign * rng.choice([0.0, 0.25, 0.5], size=case.k.shape[:-1]))
    for b in range(2):  # position 2 of both requests, and 3 of the second, stand out
        for t in (2, 3)[:b + 1]:
            case.k[case.table[b, t // 16], t % 16, :, 3] = sign
    got = case.run(q, ctx).astype(np.float64)
    gate = 1.0 / (1.0 + np.exp(-case.gates.astype(np.float64)))
    for b, n in ((0, 1), (1, 2)):
        rows = slice(int(case.start[b]), int(case.start[b + 1]))
        v = case.cache(b, case.v)[2:2 + n].mean(axis=0)  # [kv_heads, head_dim]
        want = np.repeat(v, 2, axis=0) * gate[rows]
        # equal weights and the gate: two binary16 parts and a few fp32 roundings
        np.testing.assert_allclose(got[rows], want, rtol=2.0 ** -20, atol=2.0 ** -20)


@pytest.mark.parametrize("size", [1e7, 3e7, 1e8, 1e9])
def test_random_queries_of_large_scores(q, ctx, size):
    """Random queries with the scale as it is: one row leads by more than the
    others can weigh wherever scores are this large, but for close pairs."""
    case = TreeCase(32, [90, 200], [9, 12], 4, 2, 64, q_scale=size)
    case.scale = 0.125
    assert np.isfinite(case.run(q, ctx)).all()


def _check_scale(q, ctx, case, scale):
    """_check for a scale of either sign (the formula of -scale is that of -q)."""
    case.scale = scale
    got = case.run(q, ctx).astype(np.float64)
    case.scale = abs(scale)
    if scale < 0:
        case.q = -case.q
    want, tol = case.expected()
    assert np.isfinite(want).all() and np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / np.maximum(tol, 1e-300))


@pytest.mark.parametrize("scale,q_scale", [(0.0, 1.0), (-0.0, 1.0), (0.0, 1e-30), (1e-25, 1e-25), (-1e-25, 1e-25), (1e-38, 1e-36),
                                           (1e-44, 1.0), (1e-44, 1e-30), (-1e-30, 1e-9)])
def test_scales_that_vanish(q, ctx, scale, q_scale):
    """Scores of zero, or that round to it: an even average over the seen rows,
    in tiles that hold hidden rows and in others."""
    _check_scale(q, ctx, TreeCase(33, [10, 70, 0, 700], [3, 9, 5, 2], 4, 2, 64, q_scale=q_scale), scale)


@pytest.mark.parametrize("scale", [-0.2, -1.0])
def test_negative_scale(q, ctx, scale):
    _check_scale(q, ctx, TreeCase(34, [10, 70, 700], [3, 9, 2], 4, 2, 64), scale)


@pytest.mark.parametrize("scale,q_scale", [(3e38, 0.0), (3e38, 1e4), (1e38, 1e30), (-3e38, 1e4)])
def test_scales_that_overflow(q, ctx, scale, q_scale):
    """Keys of zero, or queries: a score of zero is one whatever the scale."""
    case = TreeCase(35, [10, 70], [3, 9], 4, 2, 64, q_scale=q_scale)
    case.k[~np.isnan(case.k)] = 0.0
    _check_scale(q, ctx, case, scale)


@pytest.mark.parametrize("scale,q_scale", [(1e37, 1e-38), (3e37, 1e-41), (-1e38, 1e-43), (1e30, 1e-31), (3e30, 1e-30)])
def test_queries_of_the_smallest_size(q, ctx, scale, q_scale):
    """Queries down to fp32's smallest, brought to scores of ordinary size by the scale."""
    _check_scale(q, ctx, TreeCase(36, [60, 200], [5, 9], 4, 2, 64, q_scale=q_scale), scale)
