"""The paged cache: vvh_rope_append_paged against vvh_rope_append's bits and a 64-bit rotation, and
vvh_attention_paged against attention in 64 bits, over page sizes, lengths from none to several thousand, pages that are
gone, rows that hold NaN where no sequence has been, and the two together with graphs and streams."""
import numpy as np
import pytest

from serving import HALF, Pages, Stream, attention_ref, put
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}


def case(*a):
    print("[case]", *a, flush=True)


def rope_table(positions, D, theta=1e4):
    t = capi.DevBuf(max(1, positions * D * 4))
    capi.call("vvh_rope_table", t.ptr, positions, D, theta, None)
    return t


# ---- the append ------------------------------------------------------------------------
def rotate(x, cs):
    """x [T, H, D] in 64 bits with cs [T, D / 2, 2]."""
    h = x.shape[-1] // 2
    x0, x1, c, s = x[..., :h], x[..., h:], cs[:, None, :, 0], cs[:, None, :, 1]
    return np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], -1)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("H,KVH,D,page", [(14, 2, 64, 16), (12, 2, 128, 64), (32, 8, 128, 1), (3, 3, 10, 24), (5, 1, 96, 7),
                                          (40, 8, 256, 16), (1, 1, 2, 3), (0, 2, 64, 16)])
def test_append_tokens_and_prompts(gpu, dtype, H, KVH, D, page):
    case("append", dtype, H, KVH, D, page)
    rng = np.random.default_rng(H + D)
    lens = [40, 1, 0, 33]
    pg = Pages(rng, lens, page, KVH, D, dtype, max_pages=60 // page + 1)
    seqs = [0] * 9 + [1, 3, 0, 2, 9, -1, 3, 3]
    pos = list(range(20, 29)) + [0, 32, 39, 5, 3, 3, -1, 58]    # sequence 2 has no pages; 9 and -1 are none; 58's page may be
    keep = [0 <= s < 4 and p >= 0 and pg.table[s, p // page] >= 0 for s, p in zip(seqs, pos)]
    assert sum(keep) in (12, 13)
    T = len(pos)
    q, k, v = (rng.normal(0, 1, (T, n, D)).astype(NP[dtype]) for n in (H, KVH, KVH))
    out0 = rng.normal(0, 1, (T, H, D)).astype(NP[dtype])
    table = rope_table(70, D)
    cs = table.to_array(np.float32, (70, D // 2, 2)).astype(np.float64)
    dq, dk, dv, do, ds, dp = (capi.DevBuf.from_array(a) for a in (q, k, v, out0, np.array(seqs, np.int32), np.array(pos, np.int32)))
    capi.call("vvh_rope_append_paged", pg.cache(), do.ptr, dq.ptr, dk.ptr, dv.ptr, ds.ptr, dp.ptr, T, H, table.ptr, 70, None)
    got = do.to_array(NP[dtype], q.shape)
    kp, vp = pg.d_k.to_array(NP[dtype], pg.kp.shape), pg.d_v.to_array(NP[dtype], pg.vp.shape)
    at = cs[np.clip(pos, 0, 69)]
    rq, rk = rotate(q.astype(np.float64), at), rotate(k.astype(np.float64), at)
    # two products and a sum in fp32, the output's rounding
    tol = lambda r, x: HALF[dtype] * np.abs(r) + 2.0 ** -25 + 3 * 2.0 ** -24 * 2 * np.abs(x.astype(np.float64)).max()  # noqa: E731
    touched = np.zeros(pg.kp.shape[:2], bool)
    for t in range(T):
        if not keep[t]:
            np.testing.assert_array_equal(got[t], out0[t])
            continue
        if H:
            assert (np.abs(got[t] - rq[t]) <= tol(rq[t], q)).all()
        p = pg.table[seqs[t], pos[t] // page], pos[t] % page
        touched[p] = True
        assert (np.abs(kp[p] - rk[t]) <= tol(rk[t], k)).all()
        np.testing.assert_array_equal(vp[p], v[t])
    np.testing.assert_array_equal(kp[~touched], pg.kp[~touched])
    np.testing.assert_array_equal(vp[~touched], pg.vp[~touched])
    np.testing.assert_array_equal(dk.to_array(NP[dtype], k.shape), k)
    # in place: the same bits
    capi.call("vvh_rope_append_paged", pg.cache(), dq.ptr, dq.ptr, dk.ptr, dv.ptr, ds.ptr, dp.ptr, T, H, table.ptr, 70, None)
    back = dq.to_array(NP[dtype], q.shape)
    for t in range(T):
        np.testing.assert_array_equal(back[t], got[t] if keep[t] else q[t])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_has_the_bits_of_rope_append(gpu, dtype):
    """A sequence appended page by page and in one contiguous cache: the same rotations, far positions among them."""
    rng = np.random.default_rng(5)
    T, H, KVH, D, pos0 = 70, 14, 2, 64, 30000
    q, k, v = (rng.normal(0, 1, (T, n, D)).astype(NP[dtype]) for n in (H, KVH, KVH))
    pg = Pages(rng, [T], 16, KVH, D, dtype, max_pages=pos0 // 16 + 10, fill=0)
    t = np.full((1, pos0 // 16 + 10), -1, np.int32)
    t[0, pos0 // 16:pos0 // 16 + 5] = pg.table[0, :5]
    put(pg.d_t, t)
    table = rope_table(pos0 + T, D)
    dq, dk, dv, ds, dp = (capi.DevBuf.from_array(a) for a in (q, k, v, np.zeros(T, np.int32), np.arange(pos0, pos0 + T, dtype=np.int32)))
    do = capi.DevBuf(q.nbytes)
    capi.call("vvh_rope_append_paged", pg.cache(), do.ptr, dq.ptr, dk.ptr, dv.ptr, ds.ptr, dp.ptr, T, H, table.ptr, pos0 + T, None)
    kc, vc = capi.DevBuf((pos0 + T) * KVH * D * 4), capi.DevBuf((pos0 + T) * KVH * D * 4)
    capi.call("vvh_rope_append", dq.ptr, dk.ptr, dv.ptr, kc.ptr, vc.ptr, T, H, KVH, D, pos0, 1e4, dtype, None)
    np.testing.assert_array_equal(do.to_array(NP[dtype], q.shape), dq.to_array(NP[dtype], q.shape))
    kp = pg.d_k.to_array(NP[dtype], pg.kp.shape)[pg.table[0, :5]].reshape(-1, KVH, D)[:T]
    np.testing.assert_array_equal(kp, dk.to_array(NP[dtype], k.shape))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 63])
def test_append_without_rotation(gpu, dtype, D):
    rng = np.random.default_rng(D)
    pg = Pages(rng, [5, 9], 4, 3, D, dtype)
    k, v = (rng.normal(0, 1, (2, 3, D)).astype(NP[dtype]) for _ in range(2))
    dk, dv, dp = (capi.DevBuf.from_array(a) for a in (k, v, np.array([3, 8], np.int32)))
    capi.call("vvh_rope_append_paged", pg.cache(), None, None, dk.ptr, dv.ptr, None, dp.ptr, 2, 0, None, 0, None)
    kp, vp = pg.d_k.to_array(NP[dtype], pg.kp.shape), pg.d_v.to_array(NP[dtype], pg.vp.shape)
    for s, p in ((0, 3), (1, 8)):
        pg.kp[pg.table[s, p // 4], p % 4], pg.vp[pg.table[s, p // 4], p % 4] = k[s], v[s]
    np.testing.assert_array_equal(kp, pg.kp)
    np.testing.assert_array_equal(vp, pg.vp)


def test_append_from_rows_that_are_not_aligned(gpu):
    """q, k and v two bytes past 16-byte addresses."""
    rng = np.random.default_rng(8)
    pg = Pages(rng, [30, 30], 16, 2, 64, F16)
    a = {n: rng.normal(0, 1, (2, h, 64)).astype(np.float16) for n, h in (("q", 14), ("k", 2), ("v", 2))}
    table, dp = rope_table(40, 64), capi.DevBuf.from_array(np.array([29, 17], np.int32))
    outs = []
    for shift in (0, 1):
        d = {n: capi.DevBuf.from_array(np.concatenate([np.zeros(shift, np.float16), x.ravel()])) for n, x in a.items()}
        o = capi.DevBuf(a["q"].nbytes + 2)
        capi.call("vvh_rope_append_paged", pg.cache(), o.addr(2 * shift), *(d[n].addr(2 * shift) for n in "qkv"), None, dp.ptr,
                  2, 14, table.ptr, 40, None)
        outs.append((o.to_array(np.float16, (2 * 14 * 64 + 1,))[shift:][:2 * 14 * 64], pg.d_k.to_array(np.uint16, pg.kp.shape),
                     pg.d_v.to_array(np.uint16, pg.vp.shape)))
    for x, y in zip(*outs):
        np.testing.assert_array_equal(x, y)


# ---- attention -------------------------------------------------------------------------
def run_attention(pg, q, out=None, max_len=0, scale=None, stream=None):
    B, H, D = q.shape
    scale = 1 / np.sqrt(D) if scale is None else scale
    dq, do = capi.DevBuf.from_array(q), out or capi.DevBuf(max(1, q.nbytes))
    capi.call("vvh_attention_paged", pg.cache(), do.ptr, dq.ptr, pg.d_n.ptr, max_len, H, float(scale), stream)
    capi.sync()
    return do.to_array(q.dtype, q.shape).astype(np.float64)


def check_attention(rng, lens, page, H, KVH, D, dtype, max_len=0, std=2.0, change=None, **kw):
    case("attention", lens[:8], page, H, KVH, D, dtype, max_len)
    pg = Pages(rng, lens, page, KVH, D, dtype, **kw)
    if change:
        change(pg)
        pg.upload()
    q = rng.normal(0, std, (len(lens), H, D)).astype(NP[dtype])
    ref, tol = attention_ref(pg, q, float(np.float32(1 / np.sqrt(D))), HALF[dtype])
    got = run_attention(pg, q, max_len=max_len)
    off = np.abs(got - ref) / tol
    assert (off <= 1).all(), off.max()
    return pg, q, got


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("H,KVH,D", [(14, 2, 64), (12, 2, 128), (8, 8, 64), (16, 1, 128), (20, 1, 64), (40, 1, 128), (33, 1, 96),
                                     (6, 2, 96), (3, 1, 256), (4, 2, 40), (2, 1, 7), (1, 1, 1)])
def test_lengths(gpu, dtype, H, KVH, D):
    """No key, one, the sides of a tile of 64, several hundred; pages that end inside a tile."""
    rng = np.random.default_rng(H * D)
    check_attention(rng, [0, 1, 2, 63, 64, 65, 127, 128, 129, 300, 513, 700], 16, H, KVH, D, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 100, 256])
@pytest.mark.parametrize("max_len", [0, 100, 5000])
def test_page_sizes_and_hints(gpu, dtype, page, max_len):
    rng = np.random.default_rng(page)
    check_attention(rng, [777, 64, 1, 1300, 0], page, 14, 2, 64, dtype, max_len)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,H,KVH,D", [([9000], 12, 2, 128), ([20001, 3, 0, 700], 7, 1, 64), ([1] * 300, 14, 2, 64),
                                          ([0] * 70 + [5000] + [0] * 70, 4, 4, 64), ([4096] * 5, 16, 4, 128),
                                          (list(range(0, 2000, 13)), 8, 2, 64), ([0, 0, 0], 8, 2, 64), ([33000, 1], 2, 2, 96),
                                          ([7] * 1100, 2, 1, 64)])
def test_ragged_batches(gpu, dtype, lens, H, KVH, D):
    """One long sequence, one among many that are empty, more sequences than lanes."""
    rng = np.random.default_rng(len(lens) + D)
    check_attention(rng, lens, 32, H, KVH, D, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,H,KVH,D", [([9000], 4, 2, 80), ([20001, 3, 0, 700], 2, 1, 256), ([1] * 300, 4, 2, 40), ([0, 5000] * 4, 3, 3, 112),
                                          ([64, 65, 63, 128, 4], 8, 2, 256), ([3000] * 3, 2, 1, 7)])
@pytest.mark.parametrize("max_len", [0, 64, 100])
def test_ragged_batches_of_other_head_dims(gpu, dtype, lens, H, KVH, D, max_len):
    rng = np.random.default_rng(len(lens) + D)
    check_attention(rng, lens, 24, H, KVH, D, dtype, max_len)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_pages_that_are_gone(gpu, dtype, D):
    """Entries below 0 and past the pool: their positions are left out, at the start, inside, everywhere."""
    def change(pg):
        pg.table[0, :10] = -1
        pg.table[1, 3:6] = [len(pg.kp), 2**31 - 1, -2**31]
        pg.table[2, :] = -1
        pg.table[3, -1] = -1
    rng = np.random.default_rng(D)
    pg, q, got = check_attention(rng, [500, 300, 200, 320], 16, 12, 2, D, dtype, change=change, max_pages=32)
    assert not got[2].any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_lengths_out_of_range(gpu, dtype):
    """Negative lengths are none, lengths past the table's capacity end there."""
    rng = np.random.default_rng(3)
    pg = Pages(rng, [160, 160, 160], 16, 2, 64, dtype)
    pg.lens[:] = [2**31 - 1, -5, 161]
    pg.upload()
    q = rng.normal(0, 2, (3, 14, 64)).astype(NP[dtype])
    ref, tol = attention_ref(pg, q, 0.125, HALF[dtype])
    assert (np.abs(run_attention(pg, q) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("fill", [np.inf, -np.inf])
def test_rows_not_reached_hold_infinities(gpu, dtype, D, fill):
    rng = np.random.default_rng(D)
    check_attention(rng, [70, 1, 0, 190], 24, 6, 2, D, dtype, fill=fill)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 40])
def test_seen_rows_that_are_not_finite(gpu, dtype, D):
    """A NaN key spoils its rows and no other; a key of -infinity weighs nothing where its score is -infinity."""
    rng = np.random.default_rng(4)
    pg = Pages(rng, [150, 150, 90], 16, 2, D, dtype)
    pg.kp[pg.table[0, 4], 3, 1] = np.nan
    pg.kp[pg.table[1, 2], 5, 0] = -np.inf
    pg.upload()
    q = np.abs(rng.normal(0, 1, (3, 4, D))).astype(NP[dtype]) + NP[dtype](0.01)
    with np.errstate(invalid="ignore", over="ignore"):
        ref, tol = attention_ref(pg, q, 0.125, HALF[dtype])
    got = run_attention(pg, q, scale=0.125)
    assert np.isnan(got[0, 2:]).all() and np.isfinite(got[0, :2]).all() and np.isfinite(got[1:]).all()
    pg.kp[pg.table[1, 2], 5, 0] = -60000
    ref, tol = attention_ref(pg, q, 0.125, HALF[dtype])
    wide = np.ones((3, 4, D), bool)
    wide[0, 2:] = False
    # the weight of that key is 0 either way: a tolerance without its score
    pg.kp[pg.table[1, 2], 5, 0] = 0
    tol = attention_ref(pg, q, 0.125, HALF[dtype])[1]
    assert (np.abs(got - ref)[wide] <= tol[wide]).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_scores_of_any_size(gpu, dtype, D):
    """One key far above the rest, and scores that are all far below zero."""
    rng = np.random.default_rng(D)
    def big(pg):
        pg.kp[pg.table[0, 2], 1] *= 30
        pg.kp[:, :, 0] = np.where(np.isnan(pg.kp[:, :, 0]), np.nan, -np.abs(pg.kp[:, :, 0]) - 3)
    pg = Pages(rng, [100, 500], 16, 2, D, dtype)
    big(pg)
    pg.upload()
    q = np.abs(rng.normal(0, 4, (2, 6, D))).astype(NP[dtype])
    ref, tol = attention_ref(pg, q, float(np.float32(1 / np.sqrt(D))), HALF[dtype])
    assert (np.abs(run_attention(pg, q) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("n", [500, 3000])
@pytest.mark.parametrize("at", [0, 250, 499])
def test_many_small_weights(gpu, dtype, D, n, at):
    """One key of value 0 whose weight is 2^25.3 times every other's: the outputs are the others' values.  All terms
    have one sign, so an output's relative error is that of the scores (their D products, in numerator and sum), of the
    exponentials and weights (2^-20) and of the sums."""
    rng = np.random.default_rng(D + n)
    pg = Pages(rng, [n], 16, 2, D, dtype)
    k, v = (a[pg.table[0, :-(-n // 16)]].reshape(-1, 2, D) for a in (pg.kp, pg.vp))
    k[:n], v[:n] = 0, rng.uniform(60, 64, (n, 2, D))
    k[at, :, 0], v[at] = 2.1923828125, 0
    for a, r in ((pg.kp, k), (pg.vp, v)):
        a[pg.table[0, :-(-n // 16)]] = r.reshape(-1, 16, 2, D)
    pg.upload()
    q = np.zeros((1, 6, D), NP[dtype])
    q[:, :, 0] = 8
    ref = attention_ref(pg, q, 1.0, HALF[dtype])[0]
    rel = HALF[dtype] + 2.0 ** -20 + 2 * (D + 4) * 2.0 ** -24 * 8 * 2.1923828125 + (n / 4 + 16) * 2.0 ** -24
    assert (np.abs(run_attention(pg, q, scale=1.0) - ref) <= rel * ref).all()


def test_offsets_past_32_bits(gpu):
    """A pool of more than 2^31 values: pages at its end, in fp16 (5.4 GB a pool)."""
    rng = np.random.default_rng(1)
    KVH, D, page, pages = 8, 128, 64, 41000
    n = page * KVH * D * 2
    small = Pages(rng, [200, 130], page, KVH, D, F16, fill=0)
    big_k, big_v = capi.DevBuf(pages * n), capi.DevBuf(pages * n)
    table = np.where(small.table >= 0, pages - 1 - small.table, -1).astype(np.int32)
    for s in range(2):
        for j in range(-(-int(small.lens[s]) // page)):
            for b, a in ((big_k, small.kp), (big_v, small.vp)):
                r = np.ascontiguousarray(a[small.table[s, j]])
                capi.call("vvh_memcpy_h2d", b.addr(int(table[s, j]) * n), r.ctypes.data, n)
    put(small.d_t, table)
    q = rng.normal(0, 2, (2, 16, D)).astype(np.float16)
    ref, tol = attention_ref(small, q, float(np.float32(1 / np.sqrt(D))), HALF[F16])
    dq, do = capi.DevBuf.from_array(q), capi.DevBuf(q.nbytes)
    cache = small.cache(k_pages=big_k.ptr, v_pages=big_v.ptr, num_pages=pages)
    capi.call("vvh_attention_paged", cache, do.ptr, dq.ptr, small.d_n.ptr, 0, 16, float(1 / np.sqrt(D)), None)
    assert (np.abs(do.to_array(np.float16, q.shape).astype(np.float64) - ref) <= tol).all()
    # and the append's
    k, v = (rng.normal(0, 1, (2, KVH, D)).astype(np.float16) for _ in range(2))
    dk, dv, dp = (capi.DevBuf.from_array(a) for a in (k, v, np.array([199, 129], np.int32)))
    capi.call("vvh_rope_append_paged", cache, None, None, dk.ptr, dv.ptr, None, dp.ptr, 2, 0, None, 0, None)
    capi.sync()
    for s, p in ((0, 199), (1, 129)):
        row = np.empty((KVH, D), np.float16)
        for b, a in ((big_k, k), (big_v, v)):
            capi.call("vvh_memcpy_d2h", row.ctypes.data, b.addr(int(table[s, p // page]) * n + p % page * KVH * D * 2), row.nbytes)
            np.testing.assert_array_equal(row, a[s])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 40])
def test_addresses_that_are_not_aligned(gpu, dtype, D):
    """q, out and the pages one value past 16-byte addresses."""
    rng = np.random.default_rng(D)
    pg = Pages(rng, [150, 33], 16, 2, D, dtype)
    q = rng.normal(0, 2, (2, 6, D)).astype(NP[dtype])
    ref, tol = attention_ref(pg, q, 0.125, HALF[dtype])
    e = q.itemsize
    shifted = lambda a: capi.DevBuf.from_array(np.concatenate([np.zeros(1, a.dtype), a.ravel()]))  # noqa: E731
    dk, dv, dq, do = shifted(pg.kp), shifted(pg.vp), shifted(q), capi.DevBuf(q.nbytes + e)
    for sk, sq, so in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        kv = dict(k_pages=dk.addr(e), v_pages=dv.addr(e)) if sk else {}
        qa = dq.addr(e) if sq else capi.DevBuf.from_array(q)
        capi.call("vvh_attention_paged", pg.cache(**kv), do.addr(e * so), qa if sq else qa.ptr, pg.d_n.ptr, 0, 6, 0.125, None)
        got = do.to_array(q.dtype, (q.size + 1,))[so:][:q.size].reshape(q.shape).astype(np.float64)
        assert (np.abs(got - ref) <= tol).all(), (sk, sq, so)


def test_repeats_give_the_same_bits(gpu):
    rng = np.random.default_rng(2)
    pg = Pages(rng, [3000, 17, 900, 0, 1500], 16, 2, 128, F16)
    q = rng.normal(0, 2, (5, 12, 128)).astype(np.float16)
    first = run_attention(pg, q)
    for _ in range(3):
        np.testing.assert_array_equal(run_attention(pg, q), first)


def test_sequences_that_share_pages(gpu):
    """Two sequences with a common prefix on the same pages."""
    rng = np.random.default_rng(6)
    def change(pg):
        pg.table[1, :8] = pg.table[0, :8]
    check_attention(rng, [200, 150], 16, 14, 2, 64, F16, change=change)


# ---- together: a captured step, several streams -------------------------------------------
@pytest.mark.parametrize("dtype", [F16, F32])
def test_captured_step_replayed_with_new_lengths(gpu, dtype):
    """Append and attention captured once, replayed while the sequences grow, end and begin; every replay against
    64 bits and against the eager calls' bits."""
    rng = np.random.default_rng(9)
    H, KVH, D, page, B, cap = 14, 2, 64, 16, 6, 40
    pg = Pages(rng, [200, 15, 16, 600, 0, 1], page, KVH, D, dtype, spare=80, max_pages=cap, fill=0)
    free = list(set(range(len(pg.kp))) - set(pg.table[pg.table >= 0].tolist()))
    table = rope_table(cap * page, D)
    d = {n: capi.DevBuf(B * h * D * 4) for n, h in (("q", H), ("k", KVH), ("v", KVH), ("r", H), ("o", H))}
    dp = capi.DevBuf.from_array(pg.lens - 1)
    st = Stream()

    def issue(s):
        capi.call("vvh_rope_append_paged", pg.cache(), d["r"].ptr, d["q"].ptr, d["k"].ptr, d["v"].ptr, None, dp.ptr, B, H,
                  table.ptr, cap * page, s)
        capi.call("vvh_attention_paged", pg.cache(), d["o"].ptr, d["r"].ptr, pg.d_n.ptr, cap * page, H, 0.125, s)

    issue(st.s)  # the workspace of this stream
    st.sync()
    put(pg.d_k, pg.kp)
    put(pg.d_v, pg.vp)
    replay = st.capture(issue)
    for step in range(4):
        pos = pg.lens.copy()  # the new token's position
        pos[4] = -1 if step < 2 else step - 2  # an empty row that begins later
        if step == 2:
            pos[3] = -1  # one that ended
        pg.lens = pos + 1
        for s in range(B):
            if pos[s] >= 0 and pg.table[s, pos[s] // page] < 0:
                pg.table[s, pos[s] // page] = free.pop()
        new = {n: rng.normal(0, 1, (B, h, D)).astype(NP[dtype]) for n, h in (("q", H), ("k", KVH), ("v", KVH))}
        for n, a in new.items():
            put(d[n], a)
        put(dp, pos)
        put(pg.d_n, pg.lens)
        put(pg.d_t, pg.table)
        capi.sync()
        case("replay", step)
        replay()
        got, rq = (d[n].to_array(NP[dtype], (B, H, D)) for n in "or")
        pg.kp, pg.vp = (b.to_array(NP[dtype], pg.kp.shape) for b in (pg.d_k, pg.d_v))
        ref, tol = attention_ref(pg, rq, 0.125, HALF[dtype])
        live = pos >= 0
        assert (np.abs(got.astype(np.float64) - ref)[live] <= tol[live]).all()
        assert not got[~live].any()
        issue(None)
        capi.sync()
        np.testing.assert_array_equal(d["o"].to_array(NP[dtype], (B, H, D)), got)
    st.close()


def test_two_streams_at_once(gpu):
    """Different batches on two streams, issued alternately without waiting: each stream has a workspace of its own."""
    rng = np.random.default_rng(10)
    sets = []
    for n in (2500, 1900):
        pg = Pages(rng, [n, 50, 1200], 16, 2, 128, F16)
        q = rng.normal(0, 2, (3, 12, 128)).astype(np.float16)
        sets.append((pg, q, capi.DevBuf.from_array(q), capi.DevBuf(q.nbytes), Stream(), run_attention(pg, q)))
    for _ in range(20):
        for pg, q, dq, do, st, _ in sets:
            capi.call("vvh_attention_paged", pg.cache(), do.ptr, dq.ptr, pg.d_n.ptr, 0, 12, float(1 / np.sqrt(128)), st.s)
    capi.sync()
    for pg, q, dq, do, st, want in sets:
        np.testing.assert_array_equal(do.to_array(np.float16, q.shape).astype(np.float64), want)
        st.close()


def test_two_graphs_of_one_stream(gpu):
    """Two captured batches that share the stream's workspace, replayed in turn, and after a larger call has outgrown the
    workspace that they hold."""
    rng = np.random.default_rng(11)
    st, sets = Stream(), []
    for lens, H, KVH, D in (([2500, 50], 12, 2, 128), ([1900, 700, 1], 14, 2, 64), ([4000], 4, 2, 80)):
        pg = Pages(rng, lens, 16, KVH, D, F16)
        q = rng.normal(0, 2, (len(lens), H, D)).astype(np.float16)
        dq, do = capi.DevBuf.from_array(q), capi.DevBuf(q.nbytes)

        def issue(s, pg=pg, dq=dq, do=do, H=H):
            capi.call("vvh_attention_paged", pg.cache(), do.ptr, dq.ptr, pg.d_n.ptr, 0, H, 0.1, s)

        issue(st.s)
        st.sync()
        sets.append((do, q.shape, do.to_array(np.float16, q.shape), issue))
    graphs = [st.capture(x[3]) for x in sets]
    big = Pages(rng, [3000] * 40, 64, 8, 128, F16)
    for step in range(3):
        for (do, shape, want, _), replay in zip(sets, graphs):
            capi.call("vvh_fill_normal", do.ptr, F16, want.size, 1, 0.0, 1.0, None)
            capi.sync()
            replay()
            np.testing.assert_array_equal(do.to_array(np.float16, shape), want)
        if step == 0:
            q = rng.normal(0, 2, (40, 128, 128)).astype(np.float16)
            run_attention(big, q, stream=st.s)
    st.close()
