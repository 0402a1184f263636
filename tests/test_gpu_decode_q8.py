"""GPU: decode attention over the 8-bit cache (orator_gqa_decode_q8[_paged]) against the softmax
formula in float64 on the values the cache holds, within q8_model.attend's derived bound."""
from __future__ import annotations

import math

import numpy as np
import pytest

import q8_model as qm
from gpu_helpers import down, empty, say, up
from helpers import SplitMix64
from orator_amd import decoder_attn as da
from orator_amd.runtime import DeviceBuffer
from test_gpu_kv_q8 import upload

pytestmark = pytest.mark.gpu


def close(got, want, tol):
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.abs(got - want)[bad].max(), tol[bad].min(), np.argwhere(bad)[:4])


def run_paged(q, c, table, n_pages, pos, scale, stream=None):
    B, Hq, Dh = q.shape
    out = up(np.full(q.shape, 7.0, np.float32))
    da.GqaDecodeAttnQ8Paged(up(q), *upload(c), up(table), table.shape[1], c.ps, n_pages,
                            up(np.asarray(pos, np.int32)), out, B, Hq, c.Hkv, Dh, scale, stream)
    return down(out, q.shape)


@pytest.mark.parametrize("Hq,Hkv,Dh,ps", [(16, 8, 128, 16), (8, 8, 128, 32), (16, 4, 64, 16),
                                          (8, 1, 128, 64), (10, 2, 64, 16), (16, 1, 128, 16),
                                          (20, 1, 128, 16), (7, 1, 64, 128), (6, 2, 48, 16),
                                          (4, 4, 256, 16), (2, 1, 16, 16)])
def test_shapes(Hq, Hkv, Dh, ps):
    lens = [1, 17, 64, 65, 200, 513]
    r = SplitMix64(Hq * 7 + Dh + ps)
    B = len(lens)
    max_pages = -(-max(lens) // ps)
    table, n_pages = qm.table_of(r, B, max_pages, spare=2)
    c = qm.Cache(n_pages, ps, Hkv, Dh, rng=r)
    q = r.normal((B, Hq, Dh), 2.0)
    scale = 1 / math.sqrt(Dh)
    pos = [n - 1 for n in lens]
    want, tol = qm.attend(q, *c.values64(), table, pos, scale, max_pages * ps)
    say("decode q8", Hq, Hkv, Dh, ps)
    close(run_paged(q, c, table, n_pages, pos, scale), want, tol)


@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1301,
                               2047, 2048, 2049, 4097])
def test_lengths_contiguous(S):
    Hq, Hkv, Dh = 16, 8, 128
    cap = (S + 15) // 16 * 16 + (0 if S % 2 else 48)
    r = SplitMix64(S)
    c = qm.Cache(1, cap, Hkv, Dh, rng=r)
    q = r.normal((1, Hq, Dh), 2.0)
    scale = 1 / math.sqrt(Dh)
    table = np.zeros((1, 1), np.int32)
    want, tol = qm.attend(q, *c.values64(), table, [S - 1], scale, cap)
    # the keys past the last one hold what no output may take up
    c.ks[0, :, S:] = np.nan
    c.vs[0, :, S:] = np.inf
    out = empty(q.shape, np.float32)
    say("decode q8 contiguous", S, cap)
    da.GqaDecodeAttnQ8(up(q), *upload(c), out, Hq, Hkv, Dh, up(np.array([S - 1], np.int32)), cap,
                       scale)
    close(down(out, q.shape), want, tol)


def test_no_keys_unmapped_pages_and_positions_past_the_table():
    """d_pos < 0 and tables without a mapped page give zeros; unmapped pages are left out wherever
    they lie; positions past the table attend what it holds."""
    Hq, Hkv, Dh, ps, max_pages, n_pages = 4, 2, 128, 16, 6, 8
    r = SplitMix64(4)
    table = np.array([[0, 1, 2, 3, 4, 5], [-1, 8, 2147483647, -2147483648, -1, -1],
                      [7, -1, 3, 9, 0, 6], [0, 1, 2, 3, 4, 5], [-1, -1, -1, -1, 2, -1],
                      [5, 4, 3, 2, 1, 0], [6, 7, -1, -1, -1, -1]], np.int32)
    pos = np.array([-1, 95, 95, -2147483648, 70, 2147483647, 40], np.int32)
    c = qm.Cache(n_pages, ps, Hkv, Dh, rng=r)
    q = r.normal((len(pos), Hq, Dh))
    want, tol = qm.attend(q, *c.values64(), table, pos, 0.2, max_pages * ps)
    assert (want[[0, 1, 3]] == 0).all() and (want[[2, 4, 5, 6]] != 0).any()
    say("decode q8 unmapped")
    got = run_paged(q, c, table, n_pages, pos, 0.2)
    close(got, want, tol)


def test_scales_far_apart_zero_rows_and_large_scores():
    """V scales over 12 orders of magnitude, rows of zeros, scores far from one another, a negative
    and a zero softmax scale."""
    Hq, Hkv, Dh, ps, L = 16, 8, 128, 16, 300
    r = SplitMix64(8)
    max_pages = -(-L // ps)
    table, n_pages = qm.table_of(r, 1, max_pages)
    c = qm.Cache(n_pages, ps, Hkv, Dh, rng=r)
    c.vs[:] *= 10 ** (r.normal(c.vs.shape) * 4)
    c.vs[:, 0] = 0
    c.ks[:, 1] = 0
    q = r.normal((1, Hq, Dh), 8.0)
    q[0, 4] = 0
    q[0, 5] *= 1e-30
    for scale in (1.0, -0.3, 0.0, 1e-3):
        want, tol = qm.attend(q, *c.values64(), table, [L - 1], abs(scale), max_pages * ps)
        if scale < 0:
            want, _ = qm.attend(-q, *c.values64(), table, [L - 1], -scale, max_pages * ps)
            _, tol = qm.attend(-q, *c.values64(), table, [L - 1], -scale, max_pages * ps)
        say("decode q8 scales", scale)
        close(run_paged(q, c, table, n_pages, [L - 1], scale), want, tol)


def test_a_row_that_is_nan_reaches_its_own_heads_only():
    Hq, Hkv, Dh, ps = 4, 2, 128, 16
    r = SplitMix64(10)
    table, n_pages = qm.table_of(r, 3, 4)
    c = qm.Cache(n_pages, ps, Hkv, Dh, rng=r)
    q = r.normal((3, Hq, Dh))
    c.ks[table[0, 1], 0, 3] = np.nan   # stream 0, head 0, K
    c.vs[table[1, 2], 1, 15] = np.nan  # stream 1, head 1, V
    q[2, 3, 5] = np.inf                # stream 2, q head 3
    pos = [60, 60, 60]
    want, tol = qm.attend(q, *c.values64(), table, pos, 0.1, 64)
    say("decode q8 nan")
    got = run_paged(q, c, table, n_pages, pos, 0.1)
    nan = np.zeros((3, Hq), bool)
    nan[0, :2] = nan[1, 2:] = nan[2, 3] = True
    assert np.isnan(got[nan]).all()
    close(got[~nan], want[~nan], tol[~nan])


def test_write_then_attend():
    """A run of the cache's operators: a prompt and then single tokens written, each step attended."""
    B, Hq, Hkv, Dh, ps, T = 3, 16, 8, 128, 16, 30
    r = SplitMix64(12)
    table, n_pages = qm.table_of(r, B, 3)
    c = qm.Cache(n_pages, ps, Hkv, Dh)
    bufs = upload(c)
    k, v = r.normal((B, T, Hkv, Dh)), r.normal((B, T, Hkv, Dh))
    dt = up(table)

    def write(k, v, at):
        n = k.shape[1]
        da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *bufs, dt, 3, ps, n_pages, B, n, Hkv, Dh,
                               up(np.full(B, at, np.int32)))
        kc, ks = qm.quantise(k)
        vc, vs = qm.quantise(v)
        for b in range(B):
            for t in range(n):
                p = at + t
                c.write(table[b, p // ps], p % ps, slice(None), kc[b, t], ks[b, t], vc[b, t], vs[b, t])

    write(k, v, 0)
    for step in range(4):
        at = T + step
        write(r.normal((B, 1, Hkv, Dh)), r.normal((B, 1, Hkv, Dh)), at)
        q = r.normal((B, Hq, Dh), 2.0)
        out = empty(q.shape, np.float32)
        say("write then attend", step)
        da.GqaDecodeAttnQ8Paged(up(q), *bufs, dt, 3, ps, n_pages, up(np.full(B, at, np.int32)), out,
                                B, Hq, Hkv, Dh, 0.09)
        want, tol = qm.attend(q, *c.values64(), table, [at] * B, 0.09, 48)
        close(down(out, q.shape), want, tol)


@pytest.mark.parametrize("B,Hq,Hkv,Dh", [(64, 2, 1, 64), (65, 2, 1, 64), (130, 8, 2, 128),
                                         (1, 600, 600, 64), (3, 40, 2, 64)])
def test_many_streams_and_heads(B, Hq, Hkv, Dh):
    """Batches that share the workgroups by lengths (64 streams at most) and those that do not; very
    unequal lengths, empty streams among them."""
    r = SplitMix64(B + Hq)
    lens = [(0, 1, 700, 33, 64, 257, 5, 130)[b % 8] for b in range(B)] if B > 1 else [100]
    max_pages = -(-max(lens) // 32)
    table, n_pages = qm.table_of(r, B, max_pages)
    c = qm.Cache(n_pages, 32, Hkv, Dh, rng=r)
    q = r.normal((B, Hq, Dh), 2.0)
    pos = [n - 1 for n in lens]
    want, tol = qm.attend(q, *c.values64(), table, pos, 0.1, max_pages * 32)
    say("decode q8 many", B, Hq, Hkv, Dh)
    close(run_paged(q, c, table, n_pages, pos, 0.1), want, tol)


def test_table_far_longer_than_the_streams():
    """A table of 131072 positions, streams of a few: what the capacity sizes is not used up."""
    B, Hq, Hkv, Dh, ps, max_pages = 3, 4, 2, 64, 16, 8192
    r = SplitMix64(18)
    table = np.full((B, max_pages), -1, np.int32)
    table[:, :20] = np.arange(B * 20, dtype=np.int32).reshape(B, 20)
    c = qm.Cache(B * 20, ps, Hkv, Dh, rng=r)
    q = r.normal((B, Hq, Dh))
    pos = [310, 0, 65]
    want, tol = qm.attend(q, *c.values64(), table, pos, 0.1, max_pages * ps)
    say("decode q8 long table")
    close(run_paged(q, c, table, B * 20, pos, 0.1), want, tol)


def test_a_pool_past_32_bits():
    """Pages whose codes lie more than 2^31 bytes into the pool: written, attended, read back."""
    Hkv, Dh, ps, T = 8, 128, 128, 300
    n_pages = (1 << 31) // (Hkv * ps * Dh) + 8
    r = SplitMix64(19)
    cache = [DeviceBuffer(n_pages * Hkv * ps * n) for n in (Dh, 4, Dh, 4)]
    table = np.array([[n_pages - 1, 0, n_pages - 3]], np.int32)
    k, v = r.normal((1, T, Hkv, Dh)), r.normal((1, T, Hkv, Dh))
    paging = (up(table), 3, ps, n_pages)
    say("decode q8 past 32 bits", n_pages)
    da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *cache, *paging, 1, T, Hkv, Dh,
                           up(np.zeros(1, np.int32)))
    c = qm.Cache(3, ps, Hkv, Dh)
    kc, ksc = qm.quantise(k)
    vc, vsc = qm.quantise(v)
    for t in range(T):
        c.write(t // ps, t % ps, slice(None), kc[0, t], ksc[0, t], vc[0, t], vsc[0, t])
    q = r.normal((1, Hkv * 2, Dh))
    out, ko, vo = empty(q.shape, np.float32), empty(k.shape, np.float32), empty(v.shape, np.float32)
    da.GqaDecodeAttnQ8Paged(up(q), *cache, *paging, up(np.array([T - 1], np.int32)), out, 1, Hkv * 2,
                            Hkv, Dh, 0.1)
    da.ReadKvCacheQ8Paged(*cache, *paging, ko, vo, False, 1, T, Hkv, Dh, up(np.zeros(1, np.int32)))
    want, tol = qm.attend(q, *c.values64(), np.arange(3, dtype=np.int32)[None], [T - 1], 0.1, 3 * ps)
    close(down(out, q.shape), want, tol)
    kv, vv = c.values()
    np.testing.assert_array_equal(down(ko, k.shape)[0], kv.reshape(-1, Hkv, Dh)[:T])
    np.testing.assert_array_equal(down(vo, v.shape)[0], vv.reshape(-1, Hkv, Dh)[:T])
