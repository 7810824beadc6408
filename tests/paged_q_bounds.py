"""Attention over a cache of codes in 64 bits, with a bound of what the kernel's arithmetic may add that stays sharp where scores
are large, and keys that lead all others."""
import numpy as np

from vvllm_amd import capi


def attention_q_bounds(pages, q, scale, tol_out):
    """softmax(scale q K^T) V in 64 bits, and how far an element may be off, by the weights p_k: with score k off by e_k,
    |e_k| <= d_k, out - ref = sum p_k (exp(e_k) - 1) (v_k - ref) / sum p_k exp(e_k).  d_k: D products with codes, group sums and
    middles in fp32 (sizes |q| (2^bits |s| + |m|)), fp32 queries to 2^-23 of their largest, roundings of the scale and of the
    difference to the largest score, and 2^-21 for a weight's own (an exponential, a high and a low part).  Sums: two roundings
    each 16 keys and 64 at the end, of partial sums of sizes 2^bits |s| + |m|.  Weights times scales are kept to 2^-37 of the
    largest scale and weight, times codes of at most 2^(bits - 1); n such roundings, at random, to 8 deviations sqrt(n / 3)."""
    B, H, D = q.shape
    ref, tol = np.zeros((B, H, D)), np.zeros((B, H, D))
    for s in range(B):
        page, r = pages.where(s)
        if not len(page):
            continue
        k, v, _, _ = pages.rows(s)
        a, b = (np.abs(sm[page, :, r].astype(np.float64)) for sm in (pages.ks, pages.vs))
        ks, vs = (np.repeat(2.0 ** bits * x[..., 0] + x[..., 1], pages.group, -1) for x, bits in ((a, pages.kb), (b, pages.vb)))
        for h in range(H):
            g = h // (H // pages.KVH)
            x = q[s, h].astype(np.float64) * scale
            sc = k[:, g] @ x
            p = np.exp(sc - sc.max())
            p /= p.sum()
            ref[s, h] = p @ v[:, g]
            d = (D + 16) * 2.0 ** -24 * (ks[:, g] @ np.abs(x)) + 2.0 ** -22 * (sc.max() - sc) + 2.0 ** -21
            if pages.dtype == capi.F32:
                d += 2.0 ** -23 * np.abs(x).max() * ks[:, g].sum(1)
            with np.errstate(divide="ignore"):
                e = d + np.log(p)  # p_k (exp(d_k) - 1) without overflow
            off = np.where(d < 1, p * np.expm1(np.minimum(d, 1)), np.exp(np.minimum(e, 700)))
            least = (p * np.exp(-np.minimum(d, 700))).sum()
            tol[s, h] = off @ np.abs(v[:, g] - ref[s, h]) / least
            tol[s, h] += (len(p) / 8 + 64) * 2.0 ** -24 * (p @ vs[:, g])
            n = min(len(p), 8 * np.sqrt(len(p) / 3))
            tol[s, h] += n * p.max() * 2.0 ** -37 * b[:, g, :, 0].max() * 2.0 ** (pages.vb - 1)
    return ref, tol + tol_out * np.abs(ref) + 2.0 ** -25


def plant(pages, s, at, sign, lead):
    """Sequence s gets keys of at most `lead` in size, and of 2 * sign in all dims at position `at`: queries of positive dims
    score that one above (sign 1) or below (-1) all others."""
    page, r = pages.where(s)
    n = len(page)
    rng = np.random.default_rng(n)
    k = rng.uniform(-lead, lead, (n, pages.KVH, pages.D))
    k[at] = 2 * sign
    pages.kp[page, :, r], pages.ks[page, :, r] = capi.pack_paged_q(k, pages.kb, pages.group, True)
