"""Attention of drafted trees (q35_attention_tree_paged) over the range of
scales, scores and special values: large scores, scale 0 and scales that
underflow, values that are not finite in requests cut into several parts."""
import numpy as np
import pytest

from tests.drafted_util import TreeCase
from tests.test_gpu_tree_attention import _check

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
