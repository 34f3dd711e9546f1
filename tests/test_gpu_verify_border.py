"""Draws whose number falls on the border between two parts of a row, where
sums of the same weights in another order may fall on either side."""
from bisect import bisect_right
from itertools import accumulate
from math import ldexp

import numpy as np
import pytest

from test_gpu_verify_draft import make, run, softmax

pytestmark = pytest.mark.gpu

NO = 0xFFFFFFFF


def border(w, u):
    """First and last token that a draw of the f64 weights w at u may give: the
    lowest whose running sum exceeds u times the whole sum, each of the two off by
    at most len(w) additions of half a unit in the last place of the whole sum
    (sums as integers, in 2^-200)."""
    run = list(accumulate(int(ldexp(x, 200)) for x in map(float, w)))
    num, den = float(u).as_integer_ratio()
    cut, slack = run[-1] * num // den, 2 * len(w) * run[-1] // 2 ** 53 + 1
    has = np.flatnonzero(w)
    at = [bisect_right(run, cut + d) for d in (-slack, slack)]
    return tuple(int(has[-1]) if x > has[-1] else x for x in at)


@pytest.mark.parametrize("vocab,period,us", [(32768, 16384, [0.5]), (32768, 4096, [k / 8 for k in range(8)]),
                                             (4096, 2048, [0.5]), (8192, 2048, [0.25, 0.5, 0.75])])
def test_draw_at_the_border_of_repeated_parts(gpu, vocab, period, us):
    """Rows made of equal parts, u on the parts' borders, from one sequence (eight
    CTAs each) to as many as one CTA serves: every sequence draws one token, and
    one that the rounding of the sums allows."""
    for n in (1, 18, 40, 150 if vocab < 8192 else 60):
        rng = np.random.default_rng(vocab + period + n)
        p = np.tile(softmax(2.5 * rng.standard_normal((n, 1, period))), (1, 1, vocab // period))
        u = np.resize(np.asarray(us, np.float32), (n, 1))
        tok, cnt = run(gpu, p, p[:, :0], np.zeros((n, 0), np.uint32), None, u)
        assert np.all(cnt == 1)
        for i in range(n):
            lo, hi = border(p[i, 0], u[i, 0])
            assert lo <= int(tok[i, 0]) <= hi and p[i, 0, tok[i, 0]] > 0, (i, tok[i, 0], lo, hi)


def test_residual_at_the_border_of_repeated_parts(gpu):
    """The same after a rejection: the weights max(p - q, 0) repeat."""
    vocab, n = 32768, 18
    rng = np.random.default_rng(7)
    p = np.tile(softmax(2.5 * rng.standard_normal((n, 2, vocab // 8))), (1, 1, 8))
    q = np.tile(softmax(2.5 * rng.standard_normal((n, 1, vocab // 8))), (1, 1, 8))
    drafts = np.full((n, 1), NO, np.uint32)  # outside the vocabulary: rejected
    u = np.stack([np.zeros(n), np.arange(n) % 8 / 8], 1).astype(np.float32)
    tok, cnt = run(gpu, p, q, drafts, None, u)
    assert np.all(cnt == 1) and np.all(tok[:, 1] == NO)
    for i in range(n):
        w = np.maximum(p[i, 0].astype(np.float64) - q[i, 0].astype(np.float64), 0)
        lo, hi = border(w, u[i, 1])
        assert lo <= int(tok[i, 0]) <= hi and w[tok[i, 0]] > 0


def test_one_token_per_sequence_over_many_numbers(gpu):
    """Rows of 32000, the numbers next to every border between the parts that
    threads add up: one token each, within rounding of the running sum."""
    vocab, n = 32000, 18
    p, _, _, _ = make(n, 0, vocab, 3)
    c = np.cumsum(p[:, 0].astype(np.float64), -1)
    for step in range(1, 8):
        at = np.minimum(np.arange(1, n + 1) * 128 * (2 * step + 1), vocab - 1)
        u = (c[np.arange(n), at - 1] / c[:, -1]).astype(np.float32)[:, None]
        tok, cnt = run(gpu, p, p[:, :0], np.zeros((n, 0), np.uint32), None, u)
        assert np.all(cnt == 1)
        for i in range(n):
            lo, hi = border(p[i, 0], u[i, 0])
            assert lo <= int(tok[i, 0]) <= hi
