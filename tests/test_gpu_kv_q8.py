"""GPU: the 8-bit KV cache, written and read back (orator_kv_write_q8[_paged],
orator_kv_read_q8[_paged]).  Codes and scales are those of the real quotient (q8_model.quantise in
float64), bit for bit, and every byte that no row owns stays as it was; values read back equal
fl32(code * scale), and its bf16 rounding."""
from __future__ import annotations

import numpy as np
import pytest

import oracle_lib as orc
import q8_model as qm
from gpu_helpers import down, empty, say, up
from helpers import SplitMix64
from orator_amd import decoder_attn as da

pytestmark = pytest.mark.gpu


def upload(c):
    return [up(x) for x in (c.kq, c.ks, c.vq, c.vs)]


def check_cache(bufs, want):
    for buf, w in zip(bufs, (want.kq, want.ks, want.vq, want.vs)):
        np.testing.assert_array_equal(down(buf, w.shape, w.dtype), w)


@pytest.mark.parametrize("B,Tq,Hkv,Dh,ps,pos", [
    (1, 1, 8, 128, 16, [0]), (1, 1, 1, 16, 16, [15]), (5, 1, 8, 128, 16, [0, 15, 16, 31, 47]),
    (3, 1, 2, 64, 32, [31, 32, 63]), (1, 16, 8, 128, 16, [0]), (1, 16, 8, 128, 16, [3]),
    (2, 37, 2, 128, 64, [0, 21]), (2, 65, 3, 48, 16, [7, 0]), (1, 130, 2, 256, 128, [1]),
    (4, 50, 8, 64, 16, [16, 0, 15, 30]), (1, 100, 1, 80, 32, [28])])
def test_write_paged(B, Tq, Hkv, Dh, ps, pos):
    r = SplitMix64(B * 1000 + Tq * 10 + Dh)
    max_pages = -(-(max(pos) + Tq) // ps) + 1
    table, n_pages = qm.table_of(r, B, max_pages, spare=2)
    k, v = r.normal((B, Tq, Hkv, Dh)), r.normal((B, Tq, Hkv, Dh), 3.0)
    want = qm.Cache(n_pages, ps, Hkv, Dh, fill=77)
    kc, ks = qm.quantise(k)
    vc, vs = qm.quantise(v)
    for b in range(B):
        for t in range(Tq):
            p = pos[b] + t
            want.write(table[b, p // ps], p % ps, slice(None), kc[b, t], ks[b, t], vc[b, t],
                       vs[b, t])
    bufs = upload(qm.Cache(n_pages, ps, Hkv, Dh, fill=77))
    say("write q8 paged", B, Tq, Hkv, Dh, ps, pos)
    da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *bufs, up(table), max_pages, ps, n_pages, B, Tq,
                           Hkv, Dh, up(np.array(pos, np.int32)))
    check_cache(bufs, want)


@pytest.mark.parametrize("Tq,stride_more,pos", [(1, 0, 0), (1, 3, 95), (33, 5, 20), (96, 0, 0)])
def test_write_contiguous_strided(Tq, stride_more, pos):
    """Rows of a wider array (k and v as slices of a fused projection), at an odd element offset."""
    Hkv, Dh, cap = 2, 64, 96
    r = SplitMix64(Tq + pos)
    stride = Hkv * Dh + stride_more
    k, v = r.normal((Tq, stride)), r.normal((Tq, stride))
    want = qm.Cache(1, cap, Hkv, Dh, fill=5)
    kc, ks = qm.quantise(k[:, :Hkv * Dh].reshape(Tq, Hkv, Dh))
    vc, vs = qm.quantise(v[:, :Hkv * Dh].reshape(Tq, Hkv, Dh))
    for t in range(Tq):
        want.write(0, pos + t, slice(None), kc[t], ks[t], vc[t], vs[t])
    off = 1 if stride_more else 0
    dk, dv = (up(np.concatenate([np.zeros(off, np.float32), x.ravel()])) for x in (k, v))
    bufs = upload(qm.Cache(1, cap, Hkv, Dh, fill=5))
    say("write q8 strided", Tq, stride, pos)
    da.WriteKvCacheQ8(dk.ptr + 4 * off, dv.ptr + 4 * off, stride, *bufs, Tq, Hkv, Dh,
                      up(np.array([pos], np.int32)), cap)
    check_cache(bufs, want)


def test_write_values_at_the_borders():
    """Rows of zeros, of the smallest and largest magnitudes, with infinities and NaN, and values on
    and next to the border of two codes."""
    Hkv, Dh, cap = 1, 128, 16
    r = SplitMix64(9)
    rows = r.normal((14, 1, Dh))
    rows[0] = 0.0
    rows[1] = 0.0
    rows[1, 0, 3] = -0.0
    rows[2] *= np.float32(2.0 ** -126)  # the scale would be subnormal: zeros
    rows[3] = np.sign(rows[3]) * np.float32(2.0 ** -119)  # 127 * 2^-126 and a little more
    rows[4] = rows[4] / np.abs(rows[4]).max() * np.float32(3.0e38)
    rows[5, 0, 7] = np.inf
    rows[6, 0, 127] = np.nan
    rows[7, 0, 0] = -np.inf
    rows[8] = 2.0 ** -149
    s = np.float32(0.75)  # amax 127 * 0.75: quotients of k + 1/2 or next to it
    half = (np.arange(Dh, dtype=np.float32) - 64 + np.float32(0.5)) * s
    rows[9, 0], rows[10, 0], rows[11, 0] = half, np.nextafter(half, np.float32(1e9)), np.nextafter(
        half, np.float32(-1e9))
    rows[9:12, 0, 0] = 127 * s
    s = np.float32(1) / np.float32(3)  # an odd scale: (k + 1/2) * s rounded
    rows[12, 0] = ((np.arange(Dh) - 64 + 0.5) * np.float64(s)).astype(np.float32)
    rows[12, 0, 0] = np.float32(127) * s
    rows[13] = np.float32(-1.0)
    rows = rows.astype(np.float32)
    bufs = upload(qm.Cache(1, cap, Hkv, Dh, fill=1))
    want = qm.Cache(1, cap, Hkv, Dh, fill=1)
    c, sc = qm.quantise(rows)
    assert np.isnan(sc[5:8]).all() and (sc[[0, 1, 2, 8]] == 0).all() and sc[3, 0] > 0
    for t in range(len(rows)):
        want.write(0, t, slice(None), c[t], sc[t], c[t], sc[t])
    say("write q8 borders")
    da.WriteKvCacheQ8(up(rows), up(rows), Dh, *bufs, len(rows), Hkv, Dh, up(np.zeros(1, np.int32)),
                      cap)
    check_cache(bufs, want)


def test_codes_of_many_values_are_the_quotients():
    """2 million values, scales of every mantissa: not one code off the nearest."""
    Hkv, Dh, T = 4, 128, 4096
    r = SplitMix64(77)
    k = r.normal((T, Hkv, Dh)) * np.exp(r.normal((T, Hkv, 1)) * 4).astype(np.float32)
    # every third value moved to the border of two codes
    c, s = qm.quantise(k)
    edge = ((c.astype(np.float64) + 0.5) * s[..., None]).astype(np.float32)
    keep = np.abs(edge) < np.abs(k).max(-1, keepdims=True)
    k = np.where((np.arange(Dh) % 3 == 1) & keep, edge, k).astype(np.float32)
    c, s = qm.quantise(k)
    want = qm.Cache(1, T, Hkv, Dh)
    want.kq[0], want.ks[0] = c.transpose(1, 0, 2), s.T
    want.vq[:] = want._to_v(want.kq)
    want.vs[0] = s.T
    bufs = upload(qm.Cache(1, T, Hkv, Dh))
    say("write q8 many")
    da.WriteKvCacheQ8(up(k), up(k), Hkv * Dh, *bufs, T, Hkv, Dh, up(np.zeros(1, np.int32)), T)
    check_cache(bufs, want)


def test_write_outside_is_dropped():
    """Positions before 0 and past the table, unmapped pages (-1, n_pages, large), leave every byte."""
    B, Tq, Hkv, Dh, ps, max_pages, n_pages = 5, 20, 2, 128, 16, 3, 6
    r = SplitMix64(3)
    k, v = r.normal((B, Tq, Hkv, Dh)), r.normal((B, Tq, Hkv, Dh))
    table = np.array([[0, 1, 2], [3, -1, 4], [5, 6, 5], [2147483647, -2147483648, 7], [0, 1, 2]],
                     np.int32)
    pos = np.array([-18, 10, 12, 0, 2147483640], np.int32)
    want = qm.Cache(n_pages, ps, Hkv, Dh, fill=9)
    kc, ks = qm.quantise(k)
    vc, vs = qm.quantise(v)
    for b in range(B):
        for t in range(Tq):
            p = int(pos[b]) + t
            if 0 <= p < max_pages * ps and 0 <= table[b, p // ps] < n_pages:
                want.write(table[b, p // ps], p % ps, slice(None), kc[b, t], ks[b, t], vc[b, t],
                           vs[b, t])
    bufs = upload(qm.Cache(n_pages, ps, Hkv, Dh, fill=9))
    say("write q8 outside")
    da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *bufs, up(table), max_pages, ps, n_pages, B, Tq,
                           Hkv, Dh, up(pos))
    check_cache(bufs, want)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,Tq,Hkv,Dh,ps,pos", [
    (1, 1, 8, 128, 16, [0]), (3, 1, 2, 16, 16, [0, 15, 16]), (2, 33, 8, 128, 16, [0, 9]),
    (1, 70, 3, 64, 64, [5]), (2, 40, 1, 256, 32, [31, 2]), (2, 17, 2, 112, 16, [1, 16])])
def test_read_paged(B, Tq, Hkv, Dh, ps, pos, bf16):
    r = SplitMix64(B * 100 + Tq + Dh)
    max_pages = -(-(max(pos) + Tq) // ps)
    table, n_pages = qm.table_of(r, B, max_pages, spare=1)
    c = qm.Cache(n_pages, ps, Hkv, Dh, rng=r)
    kv, vv = c.values()
    j = np.array(pos)[:, None] + np.arange(Tq)
    page = np.take_along_axis(table, j // ps, 1)
    dt = np.uint16 if bf16 else np.float32
    dk, dv = empty((B, Tq, Hkv, Dh), dt), empty((B, Tq, Hkv, Dh), dt)
    say("read q8", B, Tq, Hkv, Dh, ps, pos, bf16)
    da.ReadKvCacheQ8Paged(*upload(c), up(table), max_pages, ps, n_pages, dk, dv, bf16, B, Tq, Hkv,
                          Dh, up(np.array(pos, np.int32)))
    for buf, val in ((dk, kv), (dv, vv)):
        want = val[page, j % ps]
        if bf16:
            want = orc.to_bf16(np.ascontiguousarray(want))
        np.testing.assert_array_equal(down(buf, (B, Tq, Hkv, Dh), dt), want)


def test_read_leaves_rows_outside_and_contiguous():
    Hkv, Dh, cap, Tq = 2, 64, 48, 30
    r = SplitMix64(21)
    c = qm.Cache(1, cap, Hkv, Dh, rng=r)
    kv, _ = c.values()
    for pos in (-7, 0, 30):
        dk, dv = up(np.full((Tq, Hkv, Dh), 3.0, np.float32)), up(np.full((Tq, Hkv, Dh), 3.0, np.float32))
        say("read q8 contiguous", pos)
        da.ReadKvCacheQ8(*upload(c), dk, dv, False, Tq, Hkv, Dh, up(np.array([pos], np.int32)), cap)
        want = np.full((Tq, Hkv, Dh), 3.0, np.float32)
        for t in range(Tq):
            if 0 <= pos + t < cap:
                want[t] = kv[0, pos + t]
        np.testing.assert_array_equal(down(dk, want.shape), want)


def test_written_rows_read_back_within_half_a_scale():
    """A run of the two: |value - x| <= scale / 2 plus the rounding of the product."""
    B, Tq, Hkv, Dh, ps = 3, 25, 8, 128, 16
    r = SplitMix64(31)
    k, v = r.normal((B, Tq, Hkv, Dh)), r.normal((B, Tq, Hkv, Dh), 0.01)
    table, n_pages = qm.table_of(r, B, 3)
    pos = np.array([0, 5, 16], np.int32)
    bufs = upload(qm.Cache(n_pages, ps, Hkv, Dh))
    dk, dv = empty(k.shape, np.float32), empty(k.shape, np.float32)
    say("write then read q8")
    da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *bufs, up(table), 3, ps, n_pages, B, Tq, Hkv,
                           Dh, up(pos))
    da.ReadKvCacheQ8Paged(*bufs, up(table), 3, ps, n_pages, dk, dv, False, B, Tq, Hkv, Dh, up(pos))
    for x, buf in ((k, dk), (v, dv)):
        s = np.abs(x).max(-1, keepdims=True).astype(np.float64) / 127
        # the scale's and the product's roundings: each 2^-24 of at most 127 scales
        assert (np.abs(down(buf, x.shape) - x.astype(np.float64)) <= s * (0.5 + 127 * 2 * qm.U)).all()


@pytest.mark.parametrize("bf16,off", [(False, 4), (True, 2), (True, 8)])
def test_read_into_unaligned_outputs(bf16, off):
    """Outputs at their natural alignment only."""
    Tq, Hkv, Dh, cap = 37, 2, 128, 64
    r = SplitMix64(41)
    c = qm.Cache(1, cap, Hkv, Dh, rng=r)
    kv, vv = c.values()
    dt = np.uint16 if bf16 else np.float32
    n = Tq * Hkv * Dh * np.dtype(dt).itemsize
    dk, dv = empty((n + 16,), np.uint8), empty((n + 16,), np.uint8)
    say("read q8 unaligned", bf16, off)
    da.ReadKvCacheQ8(*upload(c), dk.ptr + off, dv.ptr + off, bf16, Tq, Hkv, Dh,
                     up(np.array([5], np.int32)), cap)
    for buf, val in ((dk, kv), (dv, vv)):
        want = np.ascontiguousarray(val[0, 5:5 + Tq])
        got = down(buf, (n + 16,), np.uint8)[off:off + n].view(dt).reshape(want.shape)
        np.testing.assert_array_equal(got, orc.to_bf16(want) if bf16 else want)


def test_a_stream_of_a_padded_batch_writes_nothing():
    B, Tq, Hkv, Dh, ps = 3, 20, 2, 64, 16
    r = SplitMix64(43)
    k, v = r.normal((B, Tq, Hkv, Dh)), r.normal((B, Tq, Hkv, Dh))
    table, n_pages = qm.table_of(r, B, 2)
    want = qm.Cache(n_pages, ps, Hkv, Dh, fill=3)
    kc, ks = qm.quantise(k)
    vc, vs = qm.quantise(v)
    for t in range(Tq):
        want.write(table[1, (7 + t) // ps], (7 + t) % ps, slice(None), kc[1, t], ks[1, t], vc[1, t],
                   vs[1, t])
    bufs = upload(qm.Cache(n_pages, ps, Hkv, Dh, fill=3))
    say("write q8 padded")
    da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *bufs, up(table), 2, ps, n_pages, B, Tq, Hkv, Dh,
                           up(np.array([-Tq, 7, -2147483648], np.int32)))
    check_cache(bufs, want)


@pytest.mark.parametrize("B,Tq,Hkv,Dh", [(9, 70, 8, 128), (9, 71, 8, 64), (40, 9, 16, 128), (3, 2000, 1, 64)])
def test_calls_on_both_sides_of_the_block_kernels(B, Tq, Hkv, Dh):
    """Large calls from odd positions, and the same rows written one stream at a time."""
    r = SplitMix64(Tq)
    ps, max_pages = 32, -(-(Tq + 40) // 32)
    table, n_pages = qm.table_of(r, B, max_pages)
    pos = np.array([(7 * b) % 33 for b in range(B)], np.int32)
    k, v = r.normal((B, Tq, Hkv, Dh)), r.normal((B, Tq, Hkv, Dh))
    bufs, dt = upload(qm.Cache(n_pages, ps, Hkv, Dh, fill=2)), up(table)
    say("write q8 large", B, Tq, Hkv, Dh)
    da.WriteKvCacheQ8Paged(up(k), up(v), Hkv * Dh, *bufs, dt, max_pages, ps, n_pages, B, Tq, Hkv, Dh,
                           up(pos))
    other = upload(qm.Cache(n_pages, ps, Hkv, Dh, fill=2))
    for b in range(B):
        for t in range(0, Tq, 250):
            n = min(250, Tq - t)
            da.WriteKvCacheQ8Paged(up(k[b, t:t + n]), up(v[b, t:t + n]), Hkv * Dh, *other,
                                   up(table[b]), max_pages, ps, n_pages, 1, n, Hkv, Dh,
                                   up(pos[b:b + 1] + t))
    want = qm.Cache(n_pages, ps, Hkv, Dh)
    arrays = (want.kq, want.ks, want.vq, want.vs)
    for x, y, w in zip(bufs, other, arrays):
        np.testing.assert_array_equal(down(x, w.shape, w.dtype), down(y, w.shape, w.dtype))
    kc, ks = qm.quantise(k[B - 1])
    page, row = table[B - 1][(pos[B - 1] + np.arange(Tq)) // ps], (pos[B - 1] + np.arange(Tq)) % ps
    np.testing.assert_array_equal(down(bufs[0], want.kq.shape, np.int8)[page, :, row], kc)
    np.testing.assert_array_equal(down(bufs[1], want.ks.shape)[page, :, row], ks)
    dk, dv = empty(k.shape, np.float32), empty(v.shape, np.float32)
    da.ReadKvCacheQ8Paged(*bufs, dt, max_pages, ps, n_pages, dk, dv, False, B, Tq, Hkv, Dh, up(pos))
    for x, buf in ((k, dk), (v, dv)):
        c, s = qm.quantise(x)
        np.testing.assert_array_equal(down(buf, x.shape), c.astype(np.float32) * s[..., None])
