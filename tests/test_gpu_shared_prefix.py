"""GPU: decode of a batch behind one prefix (orator_gqa_decode_shared_paged, bf16 pool, and
_shared_q8_paged) against the softmax formula in float64, each stream's prefix read through
page-table row 0, within q8_model.attend's derived bound."""
from __future__ import annotations

import math

import numpy as np
import pytest

import oracle_lib as orc
import q8_model as qm
from gpu_helpers import down, say, up
from helpers import SplitMix64
from orator_amd import decoder_attn as da
from orator_amd.runtime import DeviceBuffer
from test_gpu_decode_q8 import close
from test_gpu_kv_q8 import upload

pytestmark = pytest.mark.gpu


class Bf16Pool:
    def __init__(self, n_pages, ps, Hkv, Dh, rng):
        self.ps, self.Hkv, self.Dh = ps, Hkv, Dh
        self.k = orc.to_bf16(rng.normal((n_pages, ps, Hkv, Dh)))
        self.v = orc.to_bf16(rng.normal((n_pages, ps, Hkv, Dh)))

    def values64(self):
        return orc.from_bf16(self.k).astype(np.float64), orc.from_bf16(self.v).astype(np.float64)


def run(q, pool, table, n_pages, pos, shared, scale, stream=None):
    B, Hq, Dh = q.shape
    out = up(np.full(q.shape, 7.0, np.float32))
    dt, dp, dq = up(table), up(np.asarray(pos, np.int32)), up(q)
    tail = (dt, table.shape[1], pool.ps, n_pages, dp, shared, out, B, Hq, pool.Hkv, Dh, scale, stream)
    if isinstance(pool, Bf16Pool):
        da.GqaDecodeAttnSharedPaged(dq, up(pool.k), up(pool.v), *tail)
    else:
        da.GqaDecodeAttnSharedQ8Paged(dq, *upload(pool), *tail)
    return down(out, q.shape)


def case(seed, q8, lens, shared, Hq, Hkv, Dh, ps):
    """Streams whose own pages past the prefix differ; table entries of rows b > 0 for pages wholly
    inside the prefix name no page at all."""
    r = SplitMix64(seed)
    B = len(lens)
    max_pages = max(1, -(-max(max(lens), shared) // ps))
    table, n_pages = qm.table_of(r, B, max_pages, spare=1)
    table[1:, :shared // ps] = -5
    pool = (qm.Cache(n_pages, ps, Hkv, Dh, rng=r) if q8 else Bf16Pool(n_pages, ps, Hkv, Dh, r))
    q = r.normal((B, Hq, Dh), 2.0)
    return q, pool, table, n_pages, [n - 1 for n in lens], 1 / math.sqrt(Dh)


def check(seed, q8, lens, shared, Hq=16, Hkv=8, Dh=128, ps=16):
    q, pool, table, n_pages, pos, scale = case(seed, q8, lens, shared, Hq, Hkv, Dh, ps)
    want, tol = qm.attend(q, *pool.values64(), table, pos, scale, table.shape[1] * ps, shared)
    say("shared", q8, lens[:6], len(lens), shared, Hq, Hkv, Dh, ps)
    close(run(q, pool, table, n_pages, pos, shared, scale), want, tol)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shared", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 255, 256, 513])
def test_prefix_lengths(q8, shared):
    check(shared, q8, [shared + n for n in (1, 2, 17, 64, 90)], shared)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,Dh,ps", [(8, 8, 128, 16), (16, 4, 64, 32), (8, 1, 128, 64),
                                          (6, 2, 64, 16), (12, 4, 128, 128), (20, 1, 128, 16),
                                          (6, 2, 48, 16), (2, 2, 256, 16)])
def test_shapes(q8, Hq, Hkv, Dh, ps):
    check(Hq + Dh, q8, [140, 131, 200, 190], 130, Hq, Hkv, Dh, ps)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B", [1, 2, 7, 8, 9, 16, 17, 33])
def test_batches(q8, B):
    check(B, q8, [97 + (5 * b) % 41 for b in range(B)], 96)


@pytest.mark.parametrize("q8", [False, True])
def test_long_prefix(q8):
    check(5, q8, [2049 + 37 * b for b in range(6)], 2047)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,Dh", [(2, 1, 128), (40, 1, 128), (3, 1, 64)])
def test_few_heads_and_groups_past_a_block_of_columns(q8, Hq, Hkv, Dh):
    """One kv head (many splits of the prefix and of a stream's own keys), groups that a block of 32
    query rows cuts, groups above 32."""
    check(11, q8, [1500, 1311, 2500, 1300, 1400], 1300, Hq, Hkv, Dh)


@pytest.mark.parametrize("q8", [False, True])
def test_thousands_of_streams(q8):
    check(12, q8, [33 + b % 3 for b in range(4100)], 32, 1, 1, 64)


@pytest.mark.parametrize("q8", [False, True])
def test_streams_shorter_than_the_prefix(q8):
    """Streams that attend part of the prefix, exactly the prefix, or nothing."""
    check(6, q8, [0, 1, 16, 40, 99, 100, 101, 180, -3], 100)


@pytest.mark.parametrize("q8", [False, True])
def test_nobody_past_the_prefix_and_unmapped_pages(q8):
    check(7, q8, [64, 64, 50], 64)
    q, pool, table, n_pages, pos, scale = case(8, q8, [150, 130, 160], 70, 16, 8, 128, 16)
    table[0, 1] = n_pages     # a page of the prefix
    table[0, 6] = -1          # stream 0's own
    table[1, 5:] = 1 << 30    # all that stream 1 has of its own but the page the prefix ends in
    want, tol = qm.attend(q, *pool.values64(), table, pos, scale, table.shape[1] * 16, 70)
    say("shared unmapped", q8)
    close(run(q, pool, table, n_pages, pos, 70, scale), want, tol)
    table[:] = -1
    assert (run(q, pool, table, n_pages, pos, 70, scale) == 0).all()


@pytest.mark.parametrize("q8", [False, True])
def test_keys_past_a_stream_are_not_taken_up(q8):
    """NaN and infinities behind a stream's last key, and in a prefix that a stream sees part of."""
    q, pool, table, n_pages, pos, scale = case(9, q8, [90, 81, 20], 80, 16, 8, 128, 16)
    want, tol = qm.attend(q, *pool.values64(), table, pos, scale, table.shape[1] * 16, 80)
    j = 85
    if q8:
        pool.ks[table[1, j // 16], :, j % 16] = np.nan
        pool.vs[table[1, j // 16], :, j % 16] = np.inf
    else:
        pool.k[table[1, j // 16], j % 16] = 0x7fc0
        pool.v[table[1, j // 16], j % 16] = 0x7f80
    say("shared masked nan", q8)
    close(run(q, pool, table, n_pages, pos, 80, scale), want, tol)
    # a NaN value inside the prefix: the streams that see it are NaN, the one that does not is not
    if q8:
        pool.vs[table[0, 2], :, 3] = np.nan
    else:
        pool.v[table[0, 2], 3] = 0x7fc0
    got = run(q, pool, table, n_pages, pos, 80, scale)
    assert np.isnan(got[:2]).all()
    close(got[2], want[2], tol[2])


def test_shared_equals_the_plain_paged_decode():
    """With every stream's table naming the same prefix pages, the batch gives what
    orator_gqa_decode_paged gives."""
    q, pool, table, n_pages, pos, scale = case(10, False, [300, 270, 290, 257], 256, 16, 8, 128, 16)
    table[1:, :16] = table[0, :16]
    got = run(q, pool, table, n_pages, pos, 256, scale)
    want, tol = qm.attend(q, *pool.values64(), table, pos, scale, table.shape[1] * 16)
    out = up(np.zeros(q.shape, np.float32))
    da.GqaDecodeAttnPaged(up(q), up(pool.k), up(pool.v), up(table), table.shape[1], 16,
                          up(np.asarray(pos, np.int32)), out, 4, 16, 8, 128, scale)
    close(got, want, tol)
    close(got, down(out, q.shape), 2 * tol)


def test_a_bf16_pool_past_32_bits():
    """Pages whose rows lie more than 2^32 bytes into the pool."""
    B, Hq, Hkv, Dh, ps, P = 2, 16, 8, 128, 128, 150
    n_pages = (1 << 32) // (ps * Hkv * Dh * 2) + 6
    r = SplitMix64(23)
    table = np.array([[n_pages - 1, n_pages - 2], [-1, n_pages - 5]], np.int32)
    small = Bf16Pool(3, ps, Hkv, Dh, r)
    small.v[2, :P % ps] = small.v[1, :P % ps]  # each stream's copy of the page the prefix ends in
    small.k[2, :P % ps] = small.k[1, :P % ps]
    pools = []
    for x in (small.k, small.v):
        pool = DeviceBuffer(n_pages * x[0].nbytes)
        for at, page in ((0, n_pages - 1), (1, n_pages - 2), (2, n_pages - 5)):
            pool.upload(x[at], page * x[0].nbytes)
        pools.append(pool)
    q = r.normal((B, Hq, Dh))
    pos = [200, 180]
    want, tol = qm.attend(q, *small.values64(), np.array([[0, 1], [0, 2]], np.int32), pos, 0.09, 256, P)
    out = up(np.zeros(q.shape, np.float32))
    say("shared past 32 bits", n_pages)
    da.GqaDecodeAttnSharedPaged(up(q), *pools, up(table), 2, ps,
                                n_pages, up(np.array(pos, np.int32)), P, out, B, Hq, Hkv, Dh, 0.09)
    close(down(out, q.shape), want, tol)


@pytest.mark.parametrize("q8", [False, True])
def test_infinities_in_q_reach_their_own_rows_only(q8):
    q, pool, table, n_pages, pos, scale = case(24, q8, [90, 81, 100], 70, 16, 8, 128, 16)
    want, tol = qm.attend(q, *pool.values64(), table, pos, scale, table.shape[1] * 16, 70)
    q = q.copy()
    q[1, 5, 3] = np.inf
    q[2, 0, 127] = np.nan
    say("shared q inf", q8)
    got = run(q, pool, table, n_pages, pos, 70, scale)
    hit = np.zeros(q.shape[:2], bool)
    hit[1, 5] = hit[2, 0] = True
    assert np.isnan(got[hit]).all()
    close(got[~hit], want[~hit], tol[~hit])


@pytest.mark.parametrize("q8,P", [(False, 1696), (True, 1696), (True, 0)])
def test_positions_up_to_the_largest(q8, P):
    """A table of 2^31 positions, of which the first page and the last are mapped: 1024 keys, and
    those of the last page that an int holds (768); the prefix ends in that page, or there is none."""
    ps, Hkv, Dh = 1024, 1, 64
    n = (1 << 31) // ps
    r = SplitMix64(31)
    pool = qm.Cache(3, ps, Hkv, Dh, rng=r) if q8 else Bf16Pool(3, ps, Hkv, Dh, r)
    q = r.normal((2, 2, Dh), 2.0)
    small = np.array([[0, 1], [0, 2]], np.int32)
    table = np.full((2, n), -1, np.int32)
    table[:, 0], table[:, -1] = small[:, 0], small[:, 1]
    far = (n - 2) * ps  # positions of the last page, less those of a table of two
    want, tol = qm.attend(q, *pool.values64(), small, [1791, 1750], 0.125, 1792, P)
    pos = [0x7fffffff, 1750 + far]
    say("largest positions", q8, P)
    close(run(q, pool, table, 3, pos, P + far if P else 0, 0.125), want, tol)
