"""The 8-bit KV cache and the attention over it, in numpy: what the kernels of kv_q8.hip,
decode_q8 and the shared-prefix decode are held to.  Quotients, scores and sums in float64."""
from __future__ import annotations

import numpy as np

BLOCK = 16
U = 2.0 ** -24  # half a step of fp32, relative


def quantise(x):
    """Codes (int8) and scales (fp32) of rows x [..., Dh] fp32."""
    x = np.asarray(x, np.float32)
    fine = np.isfinite(x).all(-1)
    amax = np.where(fine, np.abs(np.where(np.isfinite(x), x, 0)).max(-1), 0).astype(np.float32)
    s = (amax * (np.float32(1) / np.float32(127))).astype(np.float32)
    s = np.where(s >= np.float32(2.0 ** -126), s, np.float32(0))
    d = np.where(s > 0, s, 1).astype(np.float64)[..., None]
    c = np.clip(np.rint(np.where(fine[..., None], x, 0).astype(np.float64) / d), -127, 127)
    c = np.where((s > 0)[..., None], c, 0).astype(np.int8)
    return c, np.where(fine, s, np.float32(np.nan)).astype(np.float32)


class Cache:
    """A q8 pool [n_pages] of `ps` positions, in the library's layout, with random contents or a
    fill value (codes and scales both), so that a write out of place shows."""

    def __init__(self, n_pages, ps, Hkv, Dh, fill=None, rng=None):
        self.ps, self.Hkv, self.Dh = ps, Hkv, Dh
        self.kq = np.zeros((n_pages, Hkv, ps, Dh), np.int8)
        self.vq = np.zeros((n_pages, Hkv, ps // BLOCK, Dh, BLOCK), np.int8)
        self.ks = np.zeros((n_pages, Hkv, ps), np.float32)
        self.vs = np.zeros((n_pages, Hkv, ps), np.float32)
        if fill is not None:
            self.kq[:], self.vq[:], self.ks[:], self.vs[:] = fill, fill, fill, fill
        if rng is not None:
            for c, s, v in ((self.kq, self.ks, False), (self.vq, self.vs, True)):
                codes, scales = quantise(rng.normal((n_pages, Hkv, ps, Dh)))
                s[:] = scales
                c[:] = self._to_v(codes) if v else codes

    def _to_v(self, codes):
        n = codes.shape[0]
        return codes.reshape(n, self.Hkv, -1, BLOCK, self.Dh).transpose(0, 1, 2, 4, 3)

    def write(self, page, at, h, kc, ks, vc, vs):
        self.kq[page, h, at], self.ks[page, h, at] = kc, ks
        self.vq[page, h, at // BLOCK, :, at % BLOCK], self.vs[page, h, at] = vc, vs

    def values(self):
        """K and V values [n_pages, ps, Hkv, Dh] as fp32 products (what reads back)."""
        k = self.kq.astype(np.float32) * self.ks[..., None]
        v = self.vq.transpose(0, 1, 2, 4, 3).reshape(self.kq.shape).astype(np.float32)
        v = v * self.vs[..., None]
        return k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)

    def values64(self):
        k = self.kq.astype(np.float64) * self.ks[..., None]
        v = self.vq.transpose(0, 1, 2, 4, 3).reshape(self.kq.shape) * self.vs[..., None].astype(
            np.float64)
        return k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)


def stream_rows(table, ps, n_pages, S, b, shared=0):
    """(positions, page, row in the page) of the keys that stream b attends of its first S."""
    j = np.arange(S)
    row = np.where(j < shared, 0, b)
    page = table[row, j // ps]
    ok = (page >= 0) & (page < n_pages)
    return j[ok], page[ok], (j % ps)[ok]


def attend(q, kpages, vpages, table, pos, scale, capacity, shared=0):
    """Attention of q [B, Hq, Dh] over pages [n_pages, ps, Hkv, Dh] (float64) through table
    [B, max_pages], and a bound of a kernel's distance from it.

    The bound, with u = 2^-24: a score is a sum of Dh products in fp32 (or one that is at least as
    exact), then scaled twice: off by at most (Dh + 6) u sum|q k| scale, and by its own rounding
    against the maximum, 4 u |s - m|; the exponential adds 4 u.  A weight is off by twice that,
    relative (its own and the sum's), the sums of at most 600 terms in a row and the joins by
    608 u, the quotient and the value's scale by 4 u; all of sum_j p_j |v_j|."""
    B, Hq, Dh = q.shape
    n_pages, ps, Hkv, _ = kpages.shape
    G = Hq // Hkv
    out, tol = np.zeros((B, Hq, Dh)), np.zeros((B, Hq, Dh))
    for b in range(B):
        S = 0 if pos[b] < 0 else min(int(pos[b]), capacity - 1) + 1
        _, page, row = stream_rows(table, ps, n_pages, S, b, shared)
        if page.size == 0:
            continue
        k, v = kpages[page, row].astype(np.float64), vpages[page, row].astype(np.float64)
        for h in range(Hq):
            x = q[b, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = (k[:, h // G] @ x) * scale
                p = np.exp(s - s.max())
                out[b, h] = (p @ v[:, h // G]) / p.sum()
                ds = (Dh + 6) * U * (np.abs(k[:, h // G]) @ np.abs(x)) * scale
                ds = ds + 4 * U * np.abs(s - s.max()) + 4 * U
                rel = 2 * ds + (608 + 4) * U
                tol[b, h] = ((p * rel) @ np.abs(v[:, h // G]) +
                             (p @ rel) / p.sum() * (p @ np.abs(v[:, h // G]))) / p.sum()
    return out, tol


def table_of(rng, B, max_pages, spare=0):
    n = B * max_pages + spare
    return np.array(rng.uniform(n).argsort(), np.int32)[:B * max_pages].reshape(B, max_pages), n
