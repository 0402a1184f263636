"""GPU: orator_token_logprobs against the formulas in float64.  Ids are exact.  With u = 2^-24, a
log probability is (x - m) - log S: x - m is rounded once (u |x - m|), a term of S is off by that,
by its exponential (4 u) and by its rounding, the sum by at most 64 roundings in a row (sums are
taken by threads and joined in trees), the logarithm by 4 u, the difference by u of the result."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_helpers import down, empty, say, up
from helpers import SplitMix64
from orator_amd import asr_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
CHAIN = 256  # roundings in a row of a sum, at most


def model(x, tokens, k):
    x = x.astype(np.float64)
    rows, n = x.shape
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        ref = np.where(np.isneginf(m), 0, m)
        d = x - ref
        e = np.exp(d)
        S = e.sum(1, keepdims=True)
        logS = np.log(S)
        de = np.where(np.isneginf(d), 0, d)
        T = (e * de).sum(1, keepdims=True)
        lp = np.where(S == 0, -np.inf, d - logS)
        logS = np.where(S == 0, 0, logS)
        ent = np.where(S == 0, 0, logS - T / np.where(S == 0, 1, S))[:, 0]
        # |T| terms weigh their own roundings
        term = U * (np.abs(de) + CHAIN + 8)
        dS = ((e * term).sum(1, keepdims=True) / np.where(S == 0, 1, S))
        dlp = dS + 4 * U * np.abs(logS) + 2 * U * (np.abs(de) + np.abs(np.where(np.isneginf(lp), 0, lp)))
        dT = (e * np.abs(de) * (term + 2 * U)).sum(1, keepdims=True) / np.where(S == 0, 1, S)
        dent = (dS + 4 * U * np.abs(logS) + dT + np.abs(T / np.where(S == 0, 1, S)) * dS)[:, 0] + 4 * U * np.abs(ent)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :k]
    tok = np.clip(tokens, 0, n - 1)
    r = np.arange(rows)
    logp = np.where((tokens >= 0) & (tokens < n), lp[r, tok], np.nan)
    return (logp, dlp[r, tok], ent, dent, ids, np.take_along_axis(lp, ids, 1),
            np.take_along_axis(dlp, ids, 1))


def run(x, tokens, k, stride=None, off=0, stream=None):
    rows, n = x.shape
    stride = stride or n
    wide = np.full((rows, stride), 1e30, np.float32)
    wide[:, :n] = x
    flat = np.concatenate([np.full(off, np.nan, np.float32), wide.ravel()])
    dx = up(flat)
    lp, en = empty((rows,), np.float32), empty((rows,), np.float32)
    ids, top = empty((rows, max(k, 1)), np.int32), empty((rows, max(k, 1)), np.float32)
    asr_ops.TokenLogprobs(dx.ptr + 4 * off, stride, up(np.asarray(tokens, np.int32)), rows, n, k, lp,
                          en, ids, top, stream)
    return (down(lp, (rows,)), down(en, (rows,)), down(ids, (rows, max(k, 1)), np.int32)[:, :k],
            down(top, (rows, max(k, 1)))[:, :k])


def same(got, want, tol):
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(got[fine].astype(np.float64) - want[fine])
    assert (off <= tol[fine] + 1e-37).all(), off.max()


def check(x, tokens, k, **kw):
    say("logprobs", x.shape, k, kw)
    got = run(x, tokens, k, **kw)
    lp, dlp, en, den, ids, top, dtop = model(x, np.asarray(tokens), k)
    np.testing.assert_array_equal(got[2], ids)
    same(got[0], lp, dlp)
    same(got[1], en, den)
    same(got[3], top, dtop)


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 2, 2), (3, 5, 5), (2, 31, 7), (4, 32, 32),
                                      (2, 63, 8), (5, 64, 20), (3, 65, 1), (2, 255, 5),
                                      (2, 256, 32), (3, 257, 3), (2, 1000, 10), (1, 4096, 20),
                                      (9, 4097, 5), (2, 12289, 32), (1, 151936, 5),
                                      (3, 151936, 20), (33, 2051, 0)])
def test_shapes(rows, n, k):
    r = SplitMix64(rows * 31 + n)
    x = r.normal((rows, n), 3.0)
    check(x, (r.uniform(rows) * n).astype(np.int32), k)


@pytest.mark.parametrize("off,more", [(1, 0), (0, 1), (3, 2), (2, 5)])
def test_strides_and_alignment(off, more):
    n = 5003
    r = SplitMix64(off * 10 + more)
    check(r.normal((4, n), 2.0), [0, n - 1, 17, 4], 6, stride=n + more, off=off)


@pytest.mark.parametrize("n", [40, 1027, 20000, 151936])
def test_ties_go_to_the_lowest_id(n):
    """Equal logits everywhere, many equal ones at the top, steps of a sixteenth, both zeros."""
    r = SplitMix64(n)
    x = np.zeros((5, n), np.float32)
    x[1] = np.rint(r.normal((n,)) * 2) / 16
    x[2, ::7] = 1.0
    x[3, n // 2:] = -0.0
    x[4] = -3.0
    x[4, [n - 1, n // 3]] = 5.0
    check(x, [0, 1, 7, n - 1, n - 1], 32)


@pytest.mark.parametrize("n", [33, 3000, 151936])
def test_orders_that_the_rows_may_have(n):
    """Ascending, descending, all of the best ones side by side, one far above the rest."""
    x = np.zeros((5, n), np.float32)
    x[0] = np.linspace(-20, 20, n)
    x[1] = np.linspace(20, -20, n)
    x[2, n - 33:] = 10 + np.arange(33)
    x[3, n // 2] = 80.0
    x[4] = np.where(np.arange(n) % 64 == 5, 9.0, -9.0) + np.arange(n) * 1e-6
    check(x, [n - 1, 0, n - 1, 0, 5], 20)


@pytest.mark.parametrize("n", [48, 9001, 151936])
def test_banned_ids(n):
    """Entries of -infinity and of the type's lowest value; a row of one id; a row of none."""
    r = SplitMix64(n)
    x = r.normal((6, n), 2.0)
    x[0, 1::2] = -np.inf
    x[1, :] = -np.inf
    x[2, :] = -np.inf
    x[2, n - 2] = 1.5
    x[3, ::3] = np.finfo(np.float32).min
    x[4, :] = np.finfo(np.float32).min
    x[5, 5:] = -np.inf
    check(x, [1, 3, n - 2, 3, 0, 2], 12)


def test_nan_and_infinity():
    n = 3000
    r = SplitMix64(2)
    x = r.normal((4, n))
    x[0, 7] = np.nan
    x[1, 9] = np.inf
    x[2, 100:] = np.nan
    say("logprobs nan")
    lp, en, ids, top = run(x, [3, 3, 3, 3], 8)
    assert np.isnan(lp[:3]).all() and np.isnan(en[:3]).all() and np.isnan(top[:3]).all()
    y = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    np.testing.assert_array_equal(ids, np.argsort(-y, axis=1, kind="stable")[:, :8])
    want = model(x[3:], np.array([3]), 8)
    same(lp[3:], want[0], want[1])
    # fewer numbers than alternatives: the NaN entries follow, the lowest id first
    z = np.full((1, 40), np.nan, np.float32)
    z[0, 30], z[0, 20] = -np.inf, 1.0
    np.testing.assert_array_equal(run(z, [0], 5)[2], [[20, 30, 0, 1, 2]])


def test_tokens_outside_and_outputs_left_out():
    n = 700
    r = SplitMix64(14)
    x = r.normal((5, n))
    check(x, [-1, n, 2147483647, -2147483648, n - 1], 3)
    full = run(x, [1, 2, 3, 4, 5], 4)
    dx, tok = up(x), up(np.array([1, 2, 3, 4, 5], np.int32))
    lp, en, ids, top = (empty((5,), np.float32), empty((5,), np.float32), empty((5, 4), np.int32),
                        empty((5, 4), np.float32))
    say("logprobs partial outputs")
    asr_ops.TokenLogprobs(dx, n, tok, 5, n, 0, lp, None, None, None)
    asr_ops.TokenLogprobs(dx, n, None, 5, n, 9, None, en, None, None)
    asr_ops.TokenLogprobs(dx, n, None, 5, n, 4, None, None, ids, top)
    np.testing.assert_array_equal(down(lp, (5,)), full[0])
    np.testing.assert_array_equal(down(en, (5,)), full[1])
    np.testing.assert_array_equal(down(ids, (5, 4), np.int32), full[2])
    np.testing.assert_array_equal(down(top, (5, 4)), full[3])


def test_the_best_alternative_is_what_argmax_takes():
    """A step as it is used: ArgmaxBanned's token is scored, and leads the alternatives."""
    n = 151936
    r = SplitMix64(15)
    x = r.normal((1, n), 4.0)
    dx, tok = up(x), empty((1,), np.int32)
    lp, en, ids, top = (empty((1,), np.float32), empty((1,), np.float32), empty((1, 5), np.int32),
                        empty((1, 5), np.float32))
    say("argmax then logprobs")
    asr_ops.ArgmaxBanned(dx, n, -1, -1, tok)
    asr_ops.TokenLogprobs(dx, n, tok, 1, n, 5, lp, en, ids, top)
    assert down(ids, (1, 5), np.int32)[0, 0] == down(tok, (1,), np.int32)[0] == x.argmax()
    assert down(top, (1, 5))[0, 0] == down(lp, (1,))[0]


@pytest.mark.parametrize("rows,n", [(1300, 9000), (5000, 300), (300, 5000)])
def test_many_rows(rows, n):
    """Rows that a launch takes in several rounds, and more than one launch takes."""
    r = SplitMix64(rows)
    check(r.normal((rows, n), 2.0), (r.uniform(rows) * n).astype(np.int32), 4)


def test_a_long_vocabulary_and_few_numbers_left():
    """A million entries; rows with 3 numbers above -infinity, near the end and far apart."""
    n = 1000003
    r = SplitMix64(16)
    x = np.full((3, n), -np.inf, np.float32)
    x[0] = r.normal((n,), 3.0)
    x[1, [5, 700001, n - 1]] = [0.5, 2.0, 1.0]
    x[2, n - 40:] = np.arange(40)
    check(x, [77, n - 1, n - 1], 32)
