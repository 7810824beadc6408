"""Helpers of the tests of a paged cache of codes: pages filled from plain rows, the rotation with one rounding, and
attention in 64 bits over what the codes stand for."""
import ctypes

import numpy as np

from vvllm_amd import capi

NP = {capi.F16: np.float16, capi.F32: np.float32}


def rotate64(x, cs):
    """x [T, H, D] and cs [T, D / 2, 2] in 64 bits (products of fp32 values are exact there)."""
    h = x.shape[-1] // 2
    x, cs = x.astype(np.float64), cs.astype(np.float64)
    x0, x1, c, s = x[..., :h], x[..., h:], cs[:, None, :, 0], cs[:, None, :, 1]
    return np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], -1)


class PagesQ:
    """A paged cache of codes on the device; kp, vp (bytes), ks, vs ({scale, minimum}) and table are its host copies.
    Rows that no sequence has reached hold codes of all ones and NaN scales."""

    def __init__(self, rng, lens, page, KVH, D, group, kb, vb, dtype, spare=2, max_pages=None, offset=2.0):
        counts = [-(-max(n, 0) // page) for n in lens]
        width = max_pages or max(1, max(counts))
        pages = sum(counts) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(lens), width), -1, np.int32)
        self.page, self.KVH, self.D, self.group, self.kb, self.vb, self.dtype = page, KVH, D, group, kb, vb, dtype
        self.kp = np.full((pages, KVH, page, D * kb // 8), 255, np.uint8)
        self.vp = np.full((pages, KVH, page, D * vb // 8), 255, np.uint8)
        self.ks = np.full((pages, KVH, page, D // group, 2), np.nan, np.float16)
        self.vs = self.ks.copy()
        at = 0
        bias = rng.normal(0, offset, (1, KVH, D))
        for s, n in enumerate(lens):
            self.table[s, :counts[s]] = order[at:at + counts[s]]
            at += counts[s]
            if n > 0:
                j = np.arange(n)
                where = self.table[s, j // page], slice(None), j % page
                self.kp[where], self.ks[where] = capi.pack_paged_q(rng.normal(0, 1, (n, KVH, D)) + bias, kb, group, True)
                self.vp[where], self.vs[where] = capi.pack_paged_q(rng.normal(0, 1, (n, KVH, D)), vb, group, False)
        self.lens = np.array(lens, np.int32)
        self.upload()

    def upload(self):
        self.d_k, self.d_v, self.d_ks, self.d_vs, self.d_t, self.d_n = (
            capi.DevBuf.from_array(a) for a in (self.kp, self.vp, self.ks, self.vs, self.table, self.lens))

    def download(self):
        return (self.d_k.to_array(np.uint8, self.kp.shape), self.d_v.to_array(np.uint8, self.vp.shape),
                self.d_ks.to_array(np.uint16, self.ks.shape), self.d_vs.to_array(np.uint16, self.vs.shape))

    def cache(self, **kw):
        d = dict(k_pages=self.d_k.ptr, v_pages=self.d_v.ptr, k_scales=self.d_ks.ptr, v_scales=self.d_vs.ptr,
                 page_table=self.d_t.ptr, num_pages=len(self.kp), page_size=self.page, num_seqs=len(self.table),
                 max_pages=self.table.shape[1], num_kv_heads=self.KVH, head_dim=self.D, group=self.group, k_bits=self.kb,
                 v_bits=self.vb, dtype=self.dtype)
        return ctypes.byref(capi.PagedCacheQ(**{**d, **kw}))

    def where(self, s, n=None):
        """(pages, rows) of the positions that sequence s attends to."""
        j = np.arange(min(max(int(self.lens[s]) if n is None else n, 0), self.table.shape[1] * self.page))
        page = self.table[s, j // self.page]
        on = (page >= 0) & (page < len(self.kp))
        return page[on], j[on] % self.page

    def rows(self, s, n=None):
        """K and V rows of sequence s in 64 bits, [keys, KVH, D] each, and the sizes that their parts have:
        |s c| + |m|."""
        page, r = self.where(s, n)
        out = []
        for held, sm, bits, keys in ((self.kp, self.ks, self.kb, True), (self.vp, self.vs, self.vb, False)):
            out.append(capi.unpack_paged_q(held[page, :, r], sm[page, :, r], bits, keys))
            out.append(capi.unpack_paged_q(held[page, :, r], np.abs(sm[page, :, r]), bits, keys))
        return out[0], out[2], out[1], out[3]


def attention_q_ref(pages, q, scale, tol_out):
    """softmax(scale q K^T) V in 64 bits over the cache's values, and how far an element may be off: half a step of the
    output's type (tol_out); a score's D products with codes, group sums and minima (fp32, sizes |q| (|s c| + |m|)), twice
    in the exponential (numerator and sum), and fp32 queries to 2^-23 of their largest; sums of n weights, and weights
    of 2^-20 (parts of 11 bits, two roundings before)."""
    B, H, D = q.shape
    ref, tol = np.zeros((B, H, D)), np.zeros((B, H, D))
    for s in range(B):
        k, v, ka, va = pages.rows(s)
        if not len(k):
            continue
        for h in range(H):
            g = h // (H // pages.KVH)
            x = q[s, h].astype(np.float64) * scale
            sc = k[:, g] @ x
            p = np.exp(sc - sc.max())
            ref[s, h] = p @ v[:, g] / p.sum()
            d = ((D + 16) * 2.0 ** -24 * (ka[:, g] @ np.abs(x)) + 2.0 ** -23 * np.abs(x).max() * ka[:, g].sum(1)).max()
            tol[s, h] = (2 * d + (len(k) / 4 + 16) * 2.0 ** -24 + 2.0 ** -20) * va[:, g].max()
    return ref, tol + tol_out * np.abs(ref) + 2.0 ** -25
