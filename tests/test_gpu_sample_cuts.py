"""Sampling (q35_sample_logits) where a row's cut lies far below its largest
value: few tokens left by a mask or by a short last slice, a small top-k, low
temperatures, and workspaces that hold other bytes. Tolerances and the seeds'
distance from borders as in the tests of the options."""
import numpy as np
import pytest

from tests.drafted_util import EMULATED
from tests.test_gpu_sample_logits import _check, _logits

pytestmark = pytest.mark.gpu


def _filled(q, ctx, rows, vocab, byte):
    return ctx.array(np.full(q.sample_workspace(ctx, rows, vocab), byte, np.uint8))


# the top_k-th key 48 octaves and more below the largest (3.3 logits at a
# temperature of 0.1), so that it lies in the bin that takes all the rest
@pytest.mark.parametrize("byte", [0, 255])
@pytest.mark.parametrize("top_k", [20, 64, 300, 512])
@pytest.mark.parametrize("temperature", [0.05, 0.1, 0.3])
def test_few_tokens_left(q, ctx, temperature, top_k, byte):
    """Slices of 700, 1000, 400 and 900 tokens under a mask, and one of 37."""
    rng = np.random.default_rng(top_k)
    x = np.full((2, 4 * 4096 + 37), -np.inf, np.float32)
    for r in range(2):
        for s, n in enumerate((700, 1000, 400, 900)):
            at = 4096 * s + rng.choice(4096, size=n, replace=False)
            x[r, at] = (rng.standard_normal(n) * 2.2 - 4.0 * s).astype(np.float32)
        x[r, 4 * 4096:] = rng.standard_normal(37).astype(np.float32)
        x[r, 5 + r] = 12.0
    _check(q, ctx, x, np.array([0.37, 0.9999], np.float32), temperature, top_k, workspace=_filled(q, ctx, 2, x.shape[1], byte))
    _check(q, ctx, x, np.array([0.37, 0.9999], np.float32), temperature, top_k, 0.9, 0.01,
           workspace=_filled(q, ctx, 2, x.shape[1], byte))


@pytest.mark.parametrize("byte", [0, 255])
@pytest.mark.parametrize("last", [25, 513, 1000, 1024])
def test_a_short_last_slice(q, ctx, last, byte):
    rng = np.random.default_rng(last)
    x = _logits(rng, 3, 4096 + last, peaks=3)
    x[:, 4096:] -= 9.0
    x[1, :4096] = -np.inf
    x[1, 100:112] = 20.0 + np.arange(12)
    for top_k in (20, 200, 512):
        _check(q, ctx, x, np.array([0.1, 0.6, 0.99], np.float32), 0.1, top_k, workspace=_filled(q, ctx, 3, x.shape[1], byte))


def test_calls_that_share_a_workspace(q, ctx):
    """What the call before left in the workspace reaches no result: tokens, and
    probabilities of at most 1."""
    rng = np.random.default_rng(41)
    vocab = 8192
    work = _filled(q, ctx, 8, vocab, 0)
    for turn in range(2):
        x = _logits(rng, 8, vocab)
        for r in range(8):
            x[r, rng.permutation(vocab)[400:]] = -np.inf
        _check(q, ctx, x, rng.random(8).astype(np.float32), 0.1, 20, workspace=work)
        _check(q, ctx, _logits(rng, 8, vocab), rng.random(8).astype(np.float32), 1.0, 0, 0.9, workspace=work)


@pytest.mark.skipif(EMULATED, reason="long for the host build")
@pytest.mark.parametrize("masked", [0.95, 0.999])
def test_masked_vocabulary(q, ctx, masked):
    rng = np.random.default_rng(42)
    vocab = 248320
    x = _logits(rng, 4, vocab, peaks=24)
    x[rng.random(x.shape) < masked] = -np.inf
    for temperature in (0.05, 0.1, 0.3):
        _check(q, ctx, x, rng.random(4).astype(np.float32), temperature, 20, workspace=_filled(q, ctx, 4, vocab, 255))


@pytest.mark.parametrize("options", [dict(), dict(top_p=0.3), dict(top_k=4001), dict(top_p=0.77, min_p=0.9)])
@pytest.mark.parametrize("temperature,size", [(np.inf, 1e-42), (1e30, 1e-17), (1e30, 1e-12), (100.0, 1e-44), (1.0, 1e-44)])
def test_values_around_zero(q, ctx, temperature, size, options):
    """Thousands of values so near to zero that their products with the bins'
    scale round to it, from both sides: every weight is 1."""
    rng = np.random.default_rng(43)
    x = (rng.standard_normal((2, 13000)) * size).astype(np.float32)
    assert (x < 0).sum() > 3000 and (x > 0).sum() > 3000
    _check(q, ctx, x, np.array([0.902, 0.3117], np.float32), temperature, **options)
