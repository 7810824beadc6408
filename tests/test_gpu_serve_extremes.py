"""The batched decode operators at the ends of what their header allows: 65535 sequences, a sequence of 2^29 positions whose pages
are mostly gone, 65535 rows of logits, 4-bit linears of the most rows and the longest k."""
import ctypes

import numpy as np
import pytest

from q4_plan import plan
from serving import HALF, Pages, attention_ref
from test_gpu_logits_rules import Case as Rules
from test_gpu_paged import run_attention
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F32, 128), (F16, 40)])
@pytest.mark.parametrize("cap", [48, 1200])
def test_the_largest_batch(gpu, dtype, D, cap):
    """65535 sequences, one in two hundred with keys, the first and last among them; in one launch and split."""
    B, H, KVH = 65535, 2, 1
    print("[case] batch", dtype, D, cap, flush=True)
    rng = np.random.default_rng(cap + D)
    lens = np.where(rng.random(B) < 0.005, rng.integers(1, cap + 1, B), 0)
    lens[[0, 63, 64, B - 1]] = cap, 1, 2, cap - 1
    pg = Pages(rng, lens.tolist(), 16, KVH, D, dtype, max_pages=-(-cap // 16))
    q = rng.normal(0, 1, (B, H, D)).astype(NP[dtype])
    got = run_attention(pg, q)
    some = np.flatnonzero(lens)
    assert not got[lens == 0].any()
    pg.table, pg.lens = pg.table[some], pg.lens[some]
    ref, tol = attention_ref(pg, q[some], float(np.float32(1 / np.sqrt(D))), HALF[dtype])
    off = np.abs(got[some] - ref) / tol
    assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F16, 128), (F32, 96), (F16, 40)])
def test_the_longest_sequence(gpu, dtype, D):
    """2^29 - 5 positions in pages of 2^16, all given back but the first and the last two; then an append at its end."""
    page, pages, H, KVH = 1 << 16, 1 << 13, 4, 2
    n = page * pages - 5
    print("[case] longest", dtype, D, flush=True)
    rng = np.random.default_rng(D)
    pg = Pages(rng, [3 * page], page, KVH, D, dtype, spare=1, max_pages=3)
    table = np.full((1, pages), -1, np.int32)
    table[0, [0, -2, -1]] = pg.table[0]
    pg.table, pg.lens = table, np.array([n], np.int32)
    pg.upload()
    q = (rng.normal(0, 1, (1, H, D)) * 3).astype(NP[dtype])
    live = [0, pages - 2, pages - 1]
    k, v = (a[table[0, live]].reshape(-1, KVH, D)[:3 * page - 5].astype(np.float64) for a in (pg.kp, pg.vp))
    scale = float(np.float32(1 / np.sqrt(D)))
    got = run_attention(pg, q)[0]
    for h in range(H):
        x = k[:, h // 2] * q[0, h].astype(np.float64) * scale
        sc = x.sum(1)
        p = np.exp(sc - sc.max())
        ref = p @ v[:, h // 2] / p.sum()
        # attention_ref's terms: the scores' products, a sum of the weights, weights of 2^-20, the output's rounding
        tol = (2 * (D + 4) * 2.0 ** -24 * np.abs(x).sum(1).max() + (len(k) / 4 + 16) * 2.0 ** -24 + 2.0 ** -20) * np.abs(v[:, h // 2]).max()
        assert (np.abs(got[h] - ref) <= tol + HALF[dtype] * np.abs(ref) + 2.0 ** -25).all()
    new = rng.normal(0, 1, (2, 1, KVH, D)).astype(NP[dtype])
    dk, dv, dp = (capi.DevBuf.from_array(a) for a in (*new, np.array([n], np.int32)))
    capi.call("vvh_rope_append_paged", pg.cache(), None, None, dk.ptr, dv.ptr, None, dp.ptr, 1, 0, None, 0, None)
    capi.sync()
    for buf, a, row in zip((pg.d_k, pg.d_v), (pg.kp, pg.vp), new):
        a[table[0, -1], page - 5] = row[0]
        np.testing.assert_array_equal(buf.to_array(NP[dtype], a.shape), a)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 9, 100])
def test_the_most_rows_of_logits(gpu, dtype, n):
    Rules(65535, n, dtype, history=7, biases=2, mask="rows").check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("N", [3, 200])
def test_the_most_rows(gpu, act, N):
    """65535 passes of 16 rows (fp16 32768 of 32)."""
    M, K = 65535 * 16, 32
    print("[case] rows", act, N, flush=True)
    assert -(-M // plan(M, N, K, act == F32).rows) <= 65535
    rng = np.random.default_rng(N)
    x = rng.integers(-8, 9, (M, K)).astype(NP[act])  # products and sums exact
    codes, scales = rng.integers(0, 256, (N, K // 2), np.uint8), np.full((N, 1), 0.125, np.float16)
    d = [capi.DevBuf.from_array(a) for a in (x, codes, scales)]
    out = capi.DevBuf(M * N * 4)
    capi.call("vvh_linear_q4", out.ptr, d[0].ptr, d[1].ptr, d[2].ptr, None, None, None, M, N, K, 32, act, F32, None)
    capi.sync()
    w = (np.stack([codes & 15, codes >> 4], -1).reshape(N, K).astype(np.float32) - 8) * np.float32(0.125)
    np.testing.assert_array_equal(out.to_array(np.float32, (M, N)), x.astype(np.float32) @ w.T)


@pytest.mark.parametrize("M,act", [(1, F16), (4, F16), (1, F32), (4, F32), (5, F16), (17, F32)])
def test_the_longest_k(gpu, M, act):
    """2^24 activations, few of them not 0 (exact sums): the ends of every share and some between."""
    N, K = 3, 1 << 24
    p = plan(M, N, K, act == F32)
    print("[case] k", M, act, p.splits, flush=True)
    assert 1 < p.splits <= 65535
    rng = np.random.default_rng(M)
    ends = np.arange(0, K, p.seg * 256)
    at = np.unique(np.concatenate([ends, ends[1:] - 1, rng.integers(0, K, 2000), [K - 1]]))
    x = np.zeros((M, K), NP[act])
    x[:, at] = rng.integers(-4, 5, (M, len(at)))
    codes = rng.integers(0, 256, (N, K // 2), np.uint8)
    scales = rng.choice(np.array([0.25, 0.5, 1], np.float16), (N, K // 128))
    d = [capi.DevBuf.from_array(a) for a in (x, codes, scales)]
    out = capi.DevBuf(M * N * 4)
    capi.call("vvh_linear_q4", out.ptr, d[0].ptr, d[1].ptr, d[2].ptr, None, None, None, M, N, K, 128, act, F32, None)
    capi.sync()
    c = (codes[:, at // 2] >> (4 * (at % 2)).astype(np.uint8) & 15).astype(np.float64) - 8
    want = x[:, at].astype(np.float64) @ (c * scales[:, at // 128].astype(np.float64)).T
    np.testing.assert_array_equal(out.to_array(np.float32, (M, N)), want.astype(np.float32))
