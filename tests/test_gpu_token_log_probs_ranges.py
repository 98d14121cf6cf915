"""cml_token_log_probs: answers stay inside their ranges (no log probability above 0, no entropy below 0), a row with one token left has exactly 0 and 0, and NaN logits
take no other token's place among the best.

The best token's own term of the sum is 2^0 up to a factor that both ends know, so with nothing else in the row no rounding is left: equality is asked for.  Elsewhere the
tolerance of the other scoring tests: 1e-5.
"""
import numpy as np
import pytest

from camelid_amd import binding as B
from camelid_amd.binding import check, lib
from tests import gpu_util as G
from tests.test_gpu_token_log_probs import compare, score
from tests.typed_rows import Rows, from_bits, to_bits

pytestmark = pytest.mark.gpu


def one_left(t, n, vocab, scale, seed=0):
    rng = np.random.default_rng(seed)
    v = np.full((n, vocab), -np.inf, np.float32)
    at = rng.integers(vocab, size=n)
    v[np.arange(n), at] = scale * rng.standard_normal(n)
    return to_bits(v, t), at


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab", [(5000, 1), (4100, 130), (1500, 3001), (700, 9001), (40, 32003), (1, 128256), (3, 128257)])
@pytest.mark.parametrize("scale", [0.01, 20.0, 1000.0])
def test_one_token_left(t, n, vocab, scale):
    bits, at = one_left(t, n, vocab, scale, seed=n)
    p, rank, h, ids, lps = score(t, bits, at, 2)
    assert np.all(p == 0) and np.all(h == 0), (np.abs(p).max(), np.abs(h).max())
    assert np.all(rank == 1) and np.array_equal(ids[:, 0], at) and np.all(ids[:, 1] == -1)
    assert np.all(lps[:, 0] == 0) and np.all(lps[:, 1] == -np.inf)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab", [(4100, 130), (1500, 3001), (700, 9001), (40, 32003), (2, 128257)])
@pytest.mark.parametrize("scale", [0.1, 5.0, 20.0, 300.0])
def test_ranges(t, n, vocab, scale):
    rng = np.random.default_rng(vocab)
    v = to_bits(scale * rng.standard_normal((n, vocab)), t)
    best = from_bits(v, t).argmax(axis=1)
    p, _, h, _, lps = score(t, v, best, 4)
    assert p.max() <= 0 and lps.max() <= 0 and h.min() >= 0, (p.max(), lps.max(), h.min())
    assert np.array_equal(p, lps[:, 0])
    few = slice(0, min(n, 20))
    compare(t, v[few], best[few], 4)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_two_tokens_left(t):
    """The second of them from as likely as the first to far below it."""
    n, vocab, rng = 64, 5000, np.random.default_rng(8)
    v = np.full((n, vocab), -np.inf, np.float32)
    at = np.array([rng.choice(vocab, 2, replace=False) for _ in range(n)])
    first = rng.integers(-64, 64, n) / 4.0
    v[np.arange(n), at[:, 0]] = first
    v[np.arange(n), at[:, 1]] = first - np.arange(n) / 2.0
    bits = to_bits(v, t)
    compare(t, bits, at[:, 0], 3)
    p, _, h, _, lps = score(t, bits, at[:, 0], 3)
    assert np.all(p <= 0) and np.all(lps <= 0) and np.all(h >= 0)
    d = np.float64(from_bits(bits, t)[np.arange(n), at[:, 1]]) - from_bits(bits, t)[np.arange(n), at[:, 0]]
    assert np.all(np.abs(p + np.log1p(np.exp(-np.abs(d)))) <= 5 * 2.0 ** -23)  # (the term, the sum of 1 and it, the quotient, the logarithm, its product)


@pytest.mark.parametrize("n", [1, 3, 1500, 5000])
@pytest.mark.parametrize("top", [1, 5, 20])
@pytest.mark.parametrize("lanes", [1, 3, 4, 40, 60])
def test_nan_logits_take_no_place(n, top, lanes):
    """Whole lanes' logits of the first batch are NaN (eight neighbouring ones, 512 apart); the best of the others are all in that batch."""
    rng, vocab = np.random.default_rng(lanes), 3000 if n > 3 else 40000
    v = rng.standard_normal((n, vocab)).astype(np.float32)
    v[:, :1024] += 20
    for base in (0, 512):
        v[:, base:base + 8 * lanes] = np.nan
    p, _, h, ids, _ = score("f32", v.view(np.uint32), np.full(n, 1000), top)
    assert np.all(np.isnan(p)) and np.all(np.isnan(h))
    order = np.argsort(-np.where(np.isnan(v), -np.inf, v), axis=1, kind="stable")[:, :top]
    assert np.array_equal(ids, order)
