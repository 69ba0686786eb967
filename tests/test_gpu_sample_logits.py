"""Sampling from given random numbers (q35_sample_logits) against the order and
running weights in 64 bits: every option alone and together, ties, masked rows,
special values, odd vocabularies, strides, refusals.

Tokens must be equal. The device sums weights as whole numbers of 2^-43 (a
token's rounding is at most 2^-44, n of them differ from the exact sum by less
than n 2^-44), so a draw could differ only where u times the kept weight lies
that near a border; the seeds here keep away from borders, except where the
weights are equal and their sums exact on both sides. Probabilities are rounded
once to fp32 (2^-24) after a quotient whose parts are off by n 2^-44 in all."""
import numpy as np
import pytest

from tests.drafted_util import EMULATED, sample

pytestmark = pytest.mark.gpu


def _logits(rng, rows, vocab, sigma=2.2, peaks=6):
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * np.float32(sigma)
    for r in range(rows):
        at = rng.integers(0, vocab, size=peaks)
        x[r, at] += rng.uniform(4.0, 10.0, size=peaks).astype(np.float32)
    return x


def _run(q, ctx, x, u, temperature=None, top_k=None, top_p=None, min_p=None, counts=None, penalty=None, stride=None,
         workspace=None):
    rows, vocab = x.shape
    print(f"sample rows={rows} vocab={vocab} T={temperature} k={top_k} p={top_p} min={min_p}", flush=True)
    stride = stride or vocab
    held = np.full((rows, stride), np.nan, np.float32)
    held[:, :vocab] = x

    def per_row(v, dtype):
        return ctx.array(np.broadcast_to(np.asarray(v, dtype), (rows,)).copy()) if v is not None else None
    token, p = ctx.array(np.full(rows, -9, np.int32)), ctx.array(np.full(rows, -9, np.float32))
    q.sample_logits(ctx, ctx.array(held), stride, ctx.array(counts) if counts is not None else None,
                    per_row(penalty, np.float32), per_row(temperature, np.float32), per_row(top_k, np.int32),
                    per_row(top_p, np.float32), per_row(min_p, np.float32), per_row(u, np.float32), rows, vocab, token, p,
                    workspace)
    return token.download(), p.download()


def _check(q, ctx, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, counts=None, penalty=1.0, **kw):
    rows, vocab = x.shape
    token, p = _run(q, ctx, x, u, temperature, top_k, top_p, min_p, counts, penalty, **kw)

    def at(v, r):
        return np.broadcast_to(np.asarray(v), (rows,))[r].item()
    for r in range(rows):
        want, prob = sample(x[r], at(u, r), at(temperature, r), at(top_k, r), at(top_p, r), at(min_p, r),
                            counts[r] if counts is not None else None, at(penalty, r))
        assert token[r] == want, (r, token[r], want)
        assert abs(p[r] - prob) <= prob * (2.0 ** -24 + vocab * 2.0 ** -44) + 2.0 ** -149, (r, p[r], prob)
    return token


VOCABS = [1, 2, 63, 64, 257, 1000, 4096, 4097, 9001]


@pytest.mark.parametrize("vocab", VOCABS)
def test_vocabularies(q, ctx, vocab):
    rng = np.random.default_rng(vocab)
    _check(q, ctx, _logits(rng, 3, vocab), rng.random(3).astype(np.float32))


@pytest.mark.parametrize("options", [dict(temperature=0.7), dict(temperature=2.5), dict(top_k=1), dict(top_k=5),
                                     dict(top_k=700), dict(top_p=0.1), dict(top_p=0.9), dict(top_p=0.9999), dict(top_p=0.0),
                                     dict(min_p=0.02), dict(min_p=0.5), dict(min_p=1.0), dict(min_p=1e-6), dict(min_p=2.0),
                                     dict(temperature=0.6, top_k=40, top_p=0.95, min_p=0.01),
                                     dict(temperature=1.3, top_k=2000, top_p=0.8), dict(top_p=0.7, min_p=0.2),
                                     dict(temperature=0.0), dict(temperature=float("nan")), dict(top_k=-3), dict(top_p=1.5)])
def test_options(q, ctx, options):
    rng = np.random.default_rng(21)
    _check(q, ctx, _logits(rng, 4, 5000), np.array([0.013, 0.37, 0.71, 0.9993], np.float32), **options)


def test_options_per_row(q, ctx):
    rng = np.random.default_rng(22)
    _check(q, ctx, _logits(rng, 6, 4500), rng.random(6).astype(np.float32), temperature=[0.0, 0.5, 1.0, 1.0, 3.0, 0.9],
           top_k=[0, 3, 0, 50, 0, 1], top_p=[0.5, 1.0, 0.4, 0.9, 1.0, 0.2], min_p=[0.0, 0.1, 0.0, 0.0, 0.3, 0.9])


def test_missing_options(q, ctx):
    rng = np.random.default_rng(23)
    x, u = _logits(rng, 3, 700), rng.random(3).astype(np.float32)
    token, p = _run(q, ctx, x, u)
    for r in range(3):
        want, prob = sample(x[r], u[r])
        assert token[r] == want and abs(p[r] - prob) <= 2.0 ** -23


@pytest.mark.parametrize("penalty", [1.0, 1.05, 3.0])
def test_penalty(q, ctx, penalty):
    rng = np.random.default_rng(24)
    counts = (rng.random((3, 4300)) < 0.3).astype(np.int32) * rng.integers(1, 4, size=(3, 4300), dtype=np.int32)
    _check(q, ctx, _logits(rng, 3, 4300), rng.random(3).astype(np.float32), top_p=0.9, counts=counts, penalty=penalty)


def test_equal_logits(q, ctx):
    """All weights equal, their sums exact: positions at the borders themselves."""
    n = 5000
    x = np.full((7, n), 1.25, np.float32)
    u = np.array([0.0, 0.5, 0.25, 0.125, 1 - 2.0 ** -24, 1.0 / 3.0, 0.75], np.float32)
    _check(q, ctx, x, u)
    _check(q, ctx, x, u, top_k=1024)
    _check(q, ctx, x, u, top_p=0.5)
    _check(q, ctx, x, u, min_p=1.0, temperature=0.3)


@pytest.mark.parametrize("options", [dict(), dict(min_p=1.0), dict(min_p=0.3, top_p=0.5), dict(top_k=7), dict(top_k=600, min_p=1.0)])
def test_infinite_temperature(q, ctx, options):
    """Every weight is 1, whatever the logits."""
    x = _logits(np.random.default_rng(17), 3, 5000)
    _check(q, ctx, x, np.array([0.0, 0.3, 0.999], np.float32), temperature=np.inf, **options)


# around the number of keys that a row's cuts are found among at once (2048):
# n tokens close to the largest (some equal), all others far below
@pytest.mark.parametrize("n", [1023, 1024, 1025, 2047, 2048, 2049, 2600])
@pytest.mark.parametrize("options", [dict(top_k=400), dict(top_k=512, top_p=0.6), dict(top_k=513, min_p=0.99, top_p=0.9),
                                     dict(min_p=0.95), dict(top_p=0.97), dict(top_p=0.8, min_p=0.9), dict()])
def test_many_keys_before_a_cut(q, ctx, n, options):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((2, 9001)) - 40).astype(np.float32)
    for r in range(2):
        near = np.round(rng.uniform(5.0, 5.1, size=n) * 4096) / 4096
        x[r, rng.choice(9001, size=n, replace=False)] = near.astype(np.float32)
    _check(q, ctx, x, np.array([0.37, 0.93], np.float32), **options)


def test_ties_take_the_lower_token(q, ctx):
    x = np.zeros((4, 4200), np.float32)
    x[:, [4100, 17, 2000]] = 3.0
    x[1, 5] = -0.0  # equal to 0
    token = _check(q, ctx, x, np.array([0.1, 0.9, 0.5, 0.2], np.float32), top_k=2)
    assert set(token.tolist()) <= {17, 2000}
    _check(q, ctx, x[:, :9], np.array([0.05, 0.6, 0.3, 0.95], np.float32), temperature=5.0)


def test_many_ties_at_the_cut(q, ctx):
    """More equal values at a cut than are settled at once, over several slices."""
    rng = np.random.default_rng(25)
    x = np.round(rng.standard_normal((2, 13000)) * 2).astype(np.float32)
    for k in (300, 5000, 12999):
        _check(q, ctx, x, np.array([0.4321, 0.98765], np.float32), top_k=k)
    _check(q, ctx, x, np.array([0.4321, 0.98765], np.float32), top_p=0.61803, temperature=2.0)


def test_flat_rows(q, ctx):
    """Bins of thousands of different values: the draw's position among them."""
    rng = np.random.default_rng(26)
    x = (1.0 + 1e-3 * rng.random((2, 12500))).astype(np.float32)
    for kw in (dict(), dict(top_p=0.5), dict(top_k=6001), dict(min_p=0.9995)):
        _check(q, ctx, x, np.array([0.5432, 0.0712], np.float32), **kw)


def test_masked_rows(q, ctx):
    rng = np.random.default_rng(27)
    x = _logits(rng, 5, 8500)
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2, :8192] = -np.inf
    x[3, rng.random(8500) < 0.99] = -np.inf
    x[4] = np.finfo(np.float32).min  # the lowest value is a value
    token = _check(q, ctx, x, np.array([0.5, 0.5, 0.7, 0.2, 0.25], np.float32), top_k=100)
    assert token[0] == -1 and token[1] == 0 and token[2] >= 8192 and token[4] == 25


def test_special_values(q, ctx):
    x = np.zeros((5, 600), np.float32)
    x[0, :] = np.nan
    x[0, 7] = -3.0
    x[1, [3, 9]] = np.inf
    x[2, :] = -np.inf
    x[2, 4] = np.nan
    x[3, 10] = np.finfo(np.float32).max
    x[4, ::2] = np.finfo(np.float32).min
    token = _check(q, ctx, x, np.array([0.9, 0.6, 0.1, 0.3, 0.999], np.float32))
    assert token.tolist()[:4] == [7, 9, -1, 10]
    _check(q, ctx, x, np.array([0.9, 0.6, 0.1, 0.3, 0.999], np.float32), top_p=0.9, min_p=0.1, top_k=50)


@pytest.mark.parametrize("temperature", [1.1e-6, 1e-4, 50.0, 1e30, float("inf")])
def test_extreme_temperatures(q, ctx, temperature):
    rng = np.random.default_rng(28)
    _check(q, ctx, _logits(rng, 2, 3000, peaks=2), np.array([0.3, 0.8], np.float32), temperature=temperature)


def test_numbers_outside_the_range(q, ctx):
    """u below 0 or NaN draws as 0, u of 1 or more as the last kept token."""
    x = np.log(np.array([[4.0, 3.0, 2.0, 1.0]] * 4, np.float32))
    token, p = _run(q, ctx, x, np.array([-1.0, np.nan, 1.0, 7.0], np.float32))
    assert token.tolist() == [0, 0, 3, 3]


def test_strides_and_workspace(q, ctx):
    rng = np.random.default_rng(29)
    x, u = _logits(rng, 3, 4111), rng.random(3).astype(np.float32)
    first = _check(q, ctx, x, u, stride=4500, top_p=0.9)
    size = q.sample_workspace(ctx, 3, 4111)
    work = ctx.array(shape=(size,), dtype=np.uint8)
    np.testing.assert_array_equal(_check(q, ctx, x, u, top_p=0.9, workspace=work), first)
    # a smaller call after it finds what the larger left in the workspace
    _check(q, ctx, x[:1, :900], u[:1], top_k=3, workspace=work)
    with pytest.raises(q.Q35Error, match="workspace too small"):
        _check(q, ctx, x, u, workspace=ctx.array(shape=(size - 256,), dtype=np.uint8))


def test_without_probability(q, ctx):
    rng = np.random.default_rng(30)
    x = _logits(rng, 2, 300)
    token = ctx.array(np.zeros(2, np.int32))
    q.sample_logits(ctx, ctx.array(x), 300, None, None, None, None, None, None, ctx.array(np.array([0.2, 0.8], np.float32)), 2,
                    300, token)
    assert token.download().tolist() == [sample(x[0], 0.2)[0], sample(x[1], 0.8)[0]]


def test_refusals(q, ctx):
    x = ctx.array(np.zeros((2, 8), np.float32))
    u, token = ctx.array(np.zeros(2, np.float32)), ctx.array(np.full(2, 5, np.int32))

    class Nothing:
        ptr = None
    for args, what in [((x, 8, u, 0, 8, token), "no rows"), ((x, 8, u, 2, 0, token), "no tokens"),
                       ((x, 8, u, 65536, 8, token), "65535"), ((x, 2 ** 21, u, 2, 2 ** 20 + 1, token), "1048576"),
                       ((x, 7, u, 2, 8, token), "overlap"), ((Nothing, 8, u, 2, 8, token), "missing"),
                       ((x, 8, Nothing, 2, 8, token), "missing"), ((x, 8, u, 2, 8, Nothing), "missing")]:
        logits, stride, uniforms, rows, vocab, out = args
        with pytest.raises(q.Q35Error, match=what):
            q.sample_logits(ctx, logits, stride, None, None, None, None, None, None, uniforms, rows, vocab, out)
    assert token.download().tolist() == [5, 5]


@pytest.mark.skipif(EMULATED, reason="long for the host build")
@pytest.mark.parametrize("vocab,rows", [(248320, 5), (1 << 20, 2), (100003, 9)])
def test_large_vocabularies(q, ctx, vocab, rows):
    rng = np.random.default_rng(vocab)
    x, u = _logits(rng, rows, vocab, peaks=24), rng.random(rows).astype(np.float32)
    for kw in (dict(temperature=0.7, top_k=20, top_p=0.95), dict(top_p=0.95, min_p=0.02), dict(temperature=1.3), dict(top_k=3000)):
        _check(q, ctx, x, u, **kw)


@pytest.mark.skipif(EMULATED, reason="long for the host build")
def test_runs_agree(q, ctx):
    """The same call gives the same tokens and probabilities every time."""
    rng = np.random.default_rng(31)
    x, u = np.round(_logits(rng, 8, 248320), 1), rng.random(8).astype(np.float32)
    first = _run(q, ctx, x, u, top_p=0.97, temperature=1.5)
    for _ in range(5):
        again = _run(q, ctx, x, u, top_p=0.97, temperature=1.5)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1].view(np.uint32), again[1].view(np.uint32))
