"""The paged cache of codes on the device: vvh_rope_append_paged_q against the format's codes worked out in 64 bits (equal,
bit for bit), vvh_read_paged_q against what they stand for, and vvh_attention_paged_q against attention in 64 bits over
those values."""
import numpy as np
import pytest

from paged_q import NP, PagesQ, attention_q_ref, rotate64
from serving import HALF, Stream, put
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
# head_dim, group, bits of keys, bits of values
FORMATS = [(64, 32, 4, 4), (64, 64, 8, 4), (64, 32, 8, 8), (64, 64, 4, 4), (96, 32, 4, 4), (96, 32, 8, 4), (96, 32, 8, 8),
           (128, 32, 4, 4), (128, 64, 4, 4), (128, 128, 4, 4), (128, 32, 8, 4), (128, 128, 8, 4), (128, 64, 8, 8), (128, 32, 8, 8)]


def case(*a):
    print("[case]", *a, flush=True)


def rope_table(positions, D, theta=1e4):
    t = capi.DevBuf(max(1, positions * D * 4))
    capi.call("vvh_rope_table", t.ptr, positions, D, theta, None)
    return t


def bits_equal(a, b):
    np.testing.assert_array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8))


# ---- the append ------------------------------------------------------------------------
def check_append(rng, pg, seqs, pos, keep, H, positions=70, rope=True, change=None):
    T, dtype, D, KVH = len(pos), pg.dtype, pg.D, pg.KVH
    q, k, v = (rng.normal(0, 1, (T, n, D)).astype(NP[dtype]) for n in (H, KVH, KVH))
    k = (k + rng.normal(0, 2, (KVH, D))).astype(NP[dtype])
    if change:
        change(k, v)
    out0 = rng.normal(0, 1, (T, H, D)).astype(NP[dtype])
    table = rope_table(positions, D)
    cs = table.to_array(np.float32, (positions, D // 2, 2))
    dq, dk, dv, do, dp = (capi.DevBuf.from_array(a) for a in (q, k, v, out0, np.array(pos, np.int32)))
    ds = capi.DevBuf.from_array(np.array(seqs, np.int32)) if seqs is not None else None
    args = (dk.ptr, dv.ptr, ds.ptr if ds else None, dp.ptr, T, H, table.ptr if rope else None, positions if rope else 0, None)
    capi.call("vvh_rope_append_paged_q", pg.cache(), do.ptr if H else None, dq.ptr if H else None, *args)
    capi.sync()
    got = do.to_array(NP[dtype], q.shape)
    with np.errstate(invalid="ignore", over="ignore"):
        at = cs[np.clip(pos, 0, positions - 1)]
        rq, rk = rotate64(q, at), (rotate64(k, at) if rope else k.astype(np.float64)).astype(np.float32)
    want = [pg.kp.copy(), pg.vp.copy(), pg.ks.copy().view(np.uint16), pg.vs.copy().view(np.uint16)]
    for t in range(T):
        if not keep[t]:
            bits_equal(got[t], out0[t])
            continue
        if H:  # two products and a sum in fp32, the output's rounding
            tol = HALF[dtype] * np.abs(rq[t]) + 2.0 ** -25 + 6 * 2.0 ** -24 * np.abs(q[t].astype(np.float64)).max()
            assert (np.abs(got[t] - rq[t]) <= tol).all()
        s = t if seqs is None else seqs[t]
        w = pg.table[s, pos[t] // pg.page], slice(None), pos[t] % pg.page
        for i, (x, b, keys) in enumerate(((rk[t], pg.kb, True), (v[t].astype(np.float32), pg.vb, False))):
            held, sm = capi.pack_paged_q(x, b, pg.group, keys)
            want[i][w], want[2 + i][w] = held, sm.view(np.uint16)
    now = pg.download()
    for i in (0, 1):
        bits_equal(now[i], want[i])
    for i in (2, 3):  # NaN is NaN whatever its bits
        a, b = now[i].view(np.float16), want[i].view(np.float16)
        assert ((now[i] == want[i]) | (np.isnan(a) & np.isnan(b)) | ((a == 0) & (b == 0))).all()
    bits_equal(dk.to_array(NP[dtype], k.shape), k)
    if H:  # in place: the same bits
        capi.call("vvh_rope_append_paged_q", pg.cache(), dq.ptr, dq.ptr, *args)
        back = dq.to_array(NP[dtype], q.shape)
        for t in range(T):
            bits_equal(back[t], got[t] if keep[t] else q[t])
    return dict(ks=dk, vs=dv, seqs=ds, pos=dp, rk=rk, v=v)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
@pytest.mark.parametrize("H,KVH,page", [(14, 2, 16), (3, 3, 48), (0, 1, 32), (40, 8, 16)])
def test_append_tokens_and_prompts(gpu, dtype, D, group, kb, vb, H, KVH, page):
    case("append", dtype, D, group, kb, vb, H, KVH, page)
    rng = np.random.default_rng(H + D + kb)
    pg = PagesQ(rng, [40, 1, 0, 33], page, KVH, D, group, kb, vb, dtype, max_pages=60 // page + 1)
    seqs = [0] * 9 + [1, 3, 0, 2, 9, -1, 3, 3]
    pos = list(range(20, 29)) + [0, 32, 39, 5, 3, 3, -1, 58]  # sequence 2 has no pages; 9 and -1 are none; 58's page may be
    keep = [0 <= s < 4 and p >= 0 and pg.table[s, p // page] >= 0 for s, p in zip(seqs, pos)]
    assert sum(keep) in (12, 13)
    check_append(rng, pg, seqs, pos, keep, H)


def test_append_to_sequences_in_order_and_pages_out_of_range(gpu):
    rng = np.random.default_rng(2)
    pg = PagesQ(rng, [40, 17, 30, 33], 16, 2, 64, 32, 4, 4, F16)
    pg.table[1, 1], pg.table[2, 1] = len(pg.kp), 1 << 30  # no pages
    put(pg.d_t, pg.table)
    check_append(rng, pg, None, [39, 16, 29, 80], [True, False, False, False], 4)   # 80: past the rope table and the pages


@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_without_rotation(gpu, dtype):
    rng = np.random.default_rng(3)
    pg = PagesQ(rng, [20, 30], 16, 3, 96, 32, 8, 4, dtype)
    check_append(rng, pg, None, [19, 7], [True, True], 0, rope=False)


@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 8)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_special_groups(gpu, dtype, kb, vb):
    """Constants, zeros, halves between two codes, infinities and NaN in one group, the types' ends, tiny values."""
    rng = np.random.default_rng(4)
    T, KVH, D = 12, 2, 128
    pg = PagesQ(rng, [T + 3], 16, KVH, D, 32, kb, vb, dtype)
    top = 2 ** vb - 1

    def change(k, v):
        big = np.finfo(NP[dtype]).max
        for x in (k, v):
            x[0], x[1], x[2] = 0, 0.1, -3.3333
            x[3, 0, 5], x[3, 1, 70] = np.nan, np.inf
            x[4, 0, 100], x[4, 1, :32] = -np.inf, np.inf
            x[5, 0, 3], x[5, 1, 3], x[5, 1, 4] = big, big, -big
            x[6] = x[6] * NP[dtype](1e-6)
            x[7, 0] = NP[dtype](2.0 ** -24) * rng.integers(0, 9, D)
            x[8, 0] = 100 + x[8, 0] * NP[dtype](0.01)
            x[9] = rng.integers(0, 2 * top + 1, (KVH, D)) / 2     # every half: the even code
            x[9, :, ::32], x[9, :, 1::32] = 0, top
            x[10] = rng.integers(0, 4 * top + 1, (KVH, D)) / 4 - 9
            x[10, :, ::32], x[10, :, 1::32] = -9, top - 9

    check_append(rng, pg, [0] * T, list(range(T)), [True] * T, 0, rope=False, change=change)
    check_append(rng, pg, [0] * T, list(range(T)), [True] * T, 2, change=change)


# ---- the read --------------------------------------------------------------------------
def read_rows(pg, seqs, pos, k=True, v=True, fill=7.0):
    T = len(pos)
    shape = (T, pg.KVH, pg.D)
    dk, dv = (capi.DevBuf.from_array(np.full(shape, fill, NP[pg.dtype])) for _ in range(2))
    dp = capi.DevBuf.from_array(np.array(pos, np.int32))
    ds = capi.DevBuf.from_array(np.array(seqs, np.int32)) if seqs is not None else None
    capi.call("vvh_read_paged_q", pg.cache(), dk.ptr if k else None, dv.ptr if v else None, ds.ptr if ds else None, dp.ptr, T, None)
    capi.sync()
    return dk.to_array(NP[pg.dtype], shape), dv.to_array(NP[pg.dtype], shape)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
@pytest.mark.parametrize("KVH,page", [(1, 16), (2, 48), (8, 64), (20, 32)])
def test_read(gpu, dtype, D, group, kb, vb, KVH, page):
    case("read", dtype, D, group, kb, vb, KVH, page)
    rng = np.random.default_rng(D + KVH)
    lens = [200, 1, 0, 77]
    pg = PagesQ(rng, lens, page, KVH, D, group, kb, vb, dtype)
    seqs = [0] * 200 + [3] * 77 + [1, 2, 0, -1, 4, 0]
    pos = list(range(200)) + list(range(76, -1, -1)) + [0, 0, -1, 3, 3, 1 << 30]
    got = read_rows(pg, seqs, pos)
    for x, held, sm, bits, keys in ((got[0], pg.kp, pg.ks, kb, True), (got[1], pg.vp, pg.vs, vb, False)):
        for t, (s, p) in enumerate(zip(seqs, pos)):
            if not (0 <= s < 4 and 0 <= p < lens[s]):
                assert (x[t] == 7).all()  # left as it was
                continue
            w = pg.table[s, p // page], slice(None), p % page
            bits_equal(x[t], capi.unpack_paged_q(held[w], sm[w], bits, keys).astype(np.float32).astype(NP[dtype]))


def test_read_keys_or_values_alone_and_by_sequence(gpu):
    rng = np.random.default_rng(6)
    pg = PagesQ(rng, [33, 40, 50], 16, 2, 64, 32, 4, 4, F16)
    k, v = read_rows(pg, None, [32, 3, 49])
    assert not (k == 7).all() and not (v == 7).all()
    k1, v1 = read_rows(pg, None, [32, 3, 49], v=False)
    bits_equal(k1, k)
    assert (v1 == 7).all()
    k2, v2 = read_rows(pg, None, [32, 3, 49], k=False)
    bits_equal(v2, v)
    assert (k2 == 7).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_read_of_odd_scales(gpu, dtype):
    """Scales and minima that a packer may give: negative, the largest, subnormal, NaN, infinite."""
    rng = np.random.default_rng(7)
    pg = PagesQ(rng, [64], 16, 2, 128, 32, 8, 4, dtype)
    for a in (pg.ks, pg.vs):
        w = a[pg.table[0, :4]]
        w[0, 0, 0, :, 0], w[0, 0, 1, :, 0], w[0, 0, 2, :, 1] = -0.5, 65504, -65504
        w[1, 1, 3], w[1, 1, 4, 2, 0], w[1, 1, 5, 1, 1], w[1, 1, 6, 0, 1] = 2.0 ** -24, np.nan, np.inf, -np.inf
        a[pg.table[0, :4]] = w
    pg.upload()
    got = read_rows(pg, [0] * 64, list(range(64)))
    with np.errstate(invalid="ignore", over="ignore"):
        for x, held, sm, bits, keys in ((got[0], pg.kp, pg.ks, 8, True), (got[1], pg.vp, pg.vs, 4, False)):
            page, r = pg.where(0)
            np.testing.assert_array_equal(x, capi.unpack_paged_q(held[page, :, r], sm[page, :, r], bits, keys).astype(np.float32)
                                          .astype(NP[dtype]))


def test_read_of_many_heads_takes_several_launches(gpu):
    """A launch of 65535 kv heads holds 4096 tokens: those after them are still their own sequences'."""
    rng = np.random.default_rng(29)
    KVH, D, T = 65535, 64, 4100
    pg = PagesQ(rng, [16], 16, KVH, D, 64, 4, 4, F16, spare=0)
    table = np.full((T, 1), int(pg.table[0, 0]), np.int32)
    dt, dp = capi.DevBuf.from_array(table), capi.DevBuf.from_array((np.arange(T) % 16).astype(np.int32))
    table[4097] = -1  # its row stays as it was
    put(dt, table)
    out = capi.DevBuf(T * KVH * D * 2)
    row = KVH * D * 2
    keep = rng.normal(0, 1, (KVH, D)).astype(np.float16)
    capi.call("vvh_memcpy_h2d", out.addr(4097 * row), keep.ctypes.data, row)
    capi.call("vvh_read_paged_q", pg.cache(page_table=dt.ptr, num_seqs=T), out.ptr, None, None, dp.ptr, T, None)
    capi.sync()
    for t in (0, 31, 4095, 4096, 4097, 4098, 4099):
        got = np.empty((KVH, D), np.float16)
        capi.call("vvh_memcpy_d2h", got.ctypes.data, out.addr(t * row), row)
        w = pg.table[0, 0], slice(None), t % 16
        bits_equal(got, keep if t == 4097 else capi.unpack_paged_q(pg.kp[w], pg.ks[w], 4, True).astype(np.float32).astype(np.float16))


# ---- attention -------------------------------------------------------------------------
def run_attention(pg, q, out=None, max_len=0, scale=None, stream=None):
    B, H, D = q.shape
    scale = 1 / np.sqrt(D) if scale is None else scale
    dq, do = capi.DevBuf.from_array(q), out or capi.DevBuf(max(1, q.nbytes))
    capi.call("vvh_attention_paged_q", pg.cache(), do.ptr, dq.ptr, pg.d_n.ptr, max_len, H, float(scale), stream)
    capi.sync()
    return do.to_array(q.dtype, q.shape).astype(np.float64)


def check_attention(rng, lens, page, H, KVH, D, group, kb, vb, dtype, max_len=0, std=2.0, change=None, **kw):
    case("attention", lens[:8], page, H, KVH, D, group, kb, vb, dtype, max_len)
    pg = PagesQ(rng, lens, page, KVH, D, group, kb, vb, dtype, **kw)
    if change:
        change(pg)
        pg.upload()
    q = rng.normal(0, std, (len(lens), H, D)).astype(NP[dtype])
    ref, tol = attention_q_ref(pg, q, float(np.float32(1 / np.sqrt(D))), HALF[dtype])
    got = run_attention(pg, q, max_len=max_len)
    assert np.isfinite(got).all()
    off = np.abs(got - ref)
    assert (off <= tol).all(), (off.max(), (off / tol).max())
    return pg, q, got


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
def test_attention_formats(gpu, dtype, D, group, kb, vb):
    rng = np.random.default_rng(D + group + kb + vb)
    check_attention(rng, [300, 0, 1, 15, 16, 17, 63, 64, 65, 511], 16, 14, 2, D, group, kb, vb, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
def test_attention_formats_long(gpu, dtype, D, group, kb, vb):
    rng = np.random.default_rng(D + group + kb + vb + 1)
    check_attention(rng, [3000, 5, 0, 1999, 2500], 48, 6, 2, D, group, kb, vb, dtype)


def attention_fp32(pages, q, scale):
    """The cache's values in fp32, then products, exponentials and sums in fp32."""
    out = np.zeros(q.shape, np.float32)
    for s in range(len(q)):
        k, v, _, _ = pages.rows(s)
        for h in range(q.shape[1] if len(k) else 0):
            g = h // (q.shape[1] // pages.KVH)
            sc = (k[:, g].astype(np.float32) @ q[s, h].astype(np.float32)) * np.float32(scale)
            p = np.exp(sc - sc.max())
            out[s, h] = (p / p.sum()) @ v[:, g].astype(np.float32)
    return out


@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
@pytest.mark.parametrize("lens", [[1, 1, 1], [7, 60, 300], [2000, 3000]])
def test_attention_is_as_exact_as_fp32(gpu, D, group, kb, vb, lens):
    """fp32 rows: the error's norm is within three times that of fp32 arithmetic on the values, or 2^-20 of the output's
    (weights and queries of 22 bits, whose errors are 2^-22 at most each, and sums with codes of up to twice the values'
    size)."""
    rng = np.random.default_rng(D + kb + len(lens))
    pg = PagesQ(rng, lens, 16, 2, D, group, kb, vb, F32)
    q = rng.normal(0, 2, (len(lens), 8, D)).astype(np.float32)
    scale = float(np.float32(1 / np.sqrt(D)))
    ref, _ = attention_q_ref(pg, q, scale, 0)
    off = lambda y: np.linalg.norm(y - ref) / np.linalg.norm(ref)  # noqa: E731
    own, plain = off(run_attention(pg, q)), off(attention_fp32(pg, q, scale))
    case("errors", own, plain)
    assert own <= max(3 * plain, 2.0 ** -20)


@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
def test_attention_of_fp16_is_bound_by_its_rounding(gpu, D, group, kb, vb):
    """fp16 rows: the error's norm is at most a tenth above that of the exact output rounded to fp16."""
    rng = np.random.default_rng(D + kb)
    pg = PagesQ(rng, [1, 40, 700, 2500], 16, 2, D, group, kb, vb, F16)
    q = rng.normal(0, 2, (4, 8, D)).astype(np.float16)
    scale = float(np.float32(1 / np.sqrt(D)))
    ref, _ = attention_q_ref(pg, q, scale, 0)
    own, best = (np.linalg.norm(y - ref) / np.linalg.norm(ref) for y in (run_attention(pg, q), ref.astype(np.float16)))
    case("errors", own, best)
    assert own <= 1.1 * best


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("H,KVH", [(1, 1), (2, 2), (8, 1), (5, 1), (16, 1), (17, 1), (20, 1), (33, 1), (34, 2), (32, 8), (24, 3)])
def test_attention_heads(gpu, dtype, H, KVH):
    rng = np.random.default_rng(H)
    check_attention(rng, [70, 1300, 9], 16, H, KVH, 64, 32, 4, 4, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens", [[90, 17], [1300, 5]])
def test_attention_many_kv_heads(gpu, dtype, lens):
    rng = np.random.default_rng(31)
    check_attention(rng, lens, 16, 600, 600, 64, 32, 4, 4, dtype)


@pytest.mark.parametrize("page", [16, 32, 48, 80, 256, 1024])
def test_attention_pages(gpu, page):
    rng = np.random.default_rng(page)
    check_attention(rng, [1, page - 1, page, page + 1, 3 * page + 5, 2000], page, 8, 2, 128, 64, 4, 4, F16)


@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 4), (8, 8)])
@pytest.mark.parametrize("max_len", [0, 1, 100, 3000, 1 << 40])
def test_attention_whatever_length_was_expected(gpu, max_len, kb, vb):
    rng = np.random.default_rng(max_len % 97)
    check_attention(rng, [700, 2, 0, 2100], 16, 8, 2, 64, 32, kb, vb, F16, max_len=max_len, max_pages=200)


def test_attention_many_sequences(gpu):
    rng = np.random.default_rng(12)
    lens = [int(n) for n in rng.integers(0, 400, 200)]
    lens[3], lens[70], lens[199] = 0, 1900, 1
    check_attention(rng, lens, 16, 4, 1, 64, 32, 4, 4, F16)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 8)])
def test_attention_with_pages_that_are_gone(gpu, dtype, kb, vb):
    def change(pg):
        pg.table[0, 3], pg.table[0, 7], pg.table[0, 8] = -1, len(pg.kp), 1 << 30
        pg.table[1] = -1          # nothing left
        pg.table[2, :50] = -1     # the oldest
        pg.table[3, 40:] = -1

    rng = np.random.default_rng(13)
    pg, q, got = check_attention(rng, [200, 100, 1000, 2000, 16], 16, 6, 2, 96, 32, kb, vb, dtype, change=change)
    assert (got[1] == 0).all()


def test_attention_lengths_out_of_range(gpu):
    def change(pg):
        pg.lens[:] = [-5, 10 ** 9, 2 ** 31 - 1, 17]
        for a in (pg.ks, pg.vs):  # every row of the pages may be reached
            a[np.isnan(a)] = 0.25

    rng = np.random.default_rng(14)
    check_attention(rng, [30, 40, 700, 17], 16, 4, 2, 64, 32, 4, 4, F16, change=change)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("std", [0.0, 2.0 ** -20, 1e-3, 100.0, 3000.0])
def test_attention_queries_of_any_size(gpu, dtype, std):
    rng = np.random.default_rng(15)
    check_attention(rng, [300, 1200], 16, 4, 2, 64, 32, 4, 4, dtype, std=std)


def test_attention_fp32_queries_past_fp16(gpu):
    rng = np.random.default_rng(16)
    pg = PagesQ(rng, [300, 1200], 16, 2, 128, 32, 4, 4, F32)
    for std in (1e30, 1e-30):
        q = rng.normal(0, std, (2, 4, 128)).astype(np.float32)
        scale = float(np.float32(0.1 / std))
        ref, tol = attention_q_ref(pg, q, scale, HALF[F32])
        assert (np.abs(run_attention(pg, q, scale=scale) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("vb", [4, 8])
def test_attention_values_of_very_different_scales(gpu, dtype, vb):
    """Groups of 2^-24 to 65504 / 15 a step along a context, in an order that grows, falls and mixes."""
    def change(pg):
        rng = np.random.default_rng(1)
        for s, order in enumerate((1, -1, 0)):
            page, r = pg.where(s)
            e = np.linspace(-24, 4, len(r))
            e = e[::order] if order else rng.permutation(e)
            sc = 2.0 ** e[:, None, None]
            pg.vs[page, :, r, :, 0] = sc
            pg.vs[page, :, r, :, 1] = -7 * sc * (-1) ** np.arange(len(r))[:, None, None]

    rng = np.random.default_rng(17)
    check_attention(rng, [700, 700, 1500], 16, 4, 2, 128, 64, 8, vb, dtype, change=change)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 8)])
def test_attention_over_negative_scales(gpu, dtype, kb, vb):
    """Groups that a packer counted down from their largest value."""
    def change(pg):
        rng = np.random.default_rng(2)
        for a, b in ((pg.ks, kb), (pg.vs, vb)):
            down = rng.random(a.shape[:-1]) < 0.5
            with np.errstate(invalid="ignore"):
                a[..., 1] = np.where(down, a[..., 1] + a[..., 0] * (2 ** b - 1), a[..., 1])
            a[..., 0] = np.where(down, -a[..., 0], a[..., 0])

    rng = np.random.default_rng(26)
    check_attention(rng, [300, 1500, 70], 16, 6, 2, 64, 32, kb, vb, dtype, change=change)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [-0.125, 0.0, -3e-5, 40.0])
def test_attention_of_any_scale(gpu, dtype, scale):
    rng = np.random.default_rng(27)
    pg = PagesQ(rng, [300, 1500, 0, 7], 16, 2, 64, 32, 4, 4, dtype)
    q = rng.normal(0, 1, (4, 6, 64)).astype(NP[dtype])
    ref, tol = attention_q_ref(pg, q, float(np.float32(scale)), HALF[dtype])
    got = run_attention(pg, q, scale=scale)
    assert (np.abs(got - ref) <= tol).all() and (got[2] == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [np.nan, np.inf, -np.inf])
def test_attention_of_a_scale_that_is_not_finite(gpu, dtype, scale):
    """Rows that have a key are NaN, as the softmax of such scores; the others zeros."""
    for lens in ([1, 0, 40], [3000, 0, 1]):
        pg = PagesQ(np.random.default_rng(28), lens, 16, 2, 64, 32, 4, 4, dtype)
        q = np.ones((3, 14, 64), NP[dtype])
        got = run_attention(pg, q, scale=scale)
        assert np.isnan(got[[0, 2]]).all() and (got[1] == 0).all()


def test_attention_scores_that_differ_by_hundreds(gpu):
    rng = np.random.default_rng(18)
    check_attention(rng, [900, 2000], 16, 4, 2, 64, 32, 8, 4, F32, std=60.0)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [100, 2500])
def test_attention_nan_groups(gpu, dtype, n):
    """A NaN group of a value gives its dims NaN, one of a key its heads; other heads and sequences stay as they are."""
    rng = np.random.default_rng(19)
    lens = [n, n, n]
    pg = PagesQ(rng, lens, 16, 2, 128, 32, 4, 4, dtype)
    q = rng.normal(0, 2, (3, 8, 128)).astype(NP[dtype])
    clean = run_attention(pg, q)
    page, r = pg.where(0)
    pg.vs[page[n // 2], 1, r[n // 2], 2] = np.nan
    page, r = pg.where(1)
    pg.ks[page[n - 1], 0, r[n - 1], 3, 0] = np.nan
    pg.upload()
    got = run_attention(pg, q)
    nan = np.zeros(got.shape, bool)
    nan[0, 4:, 64:96] = True
    nan[1, :4] = True
    np.testing.assert_array_equal(np.isnan(got), nan)
    np.testing.assert_array_equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_queries_that_are_not_finite(gpu, dtype):
    rng = np.random.default_rng(20)
    pg = PagesQ(rng, [90, 1500, 40], 16, 2, 64, 32, 8, 4, dtype)
    q = rng.normal(0, 2, (3, 6, 64)).astype(NP[dtype])
    clean = run_attention(pg, q)
    q[0, 1, 5], q[1, 4, 9], q[1, 0, 63] = np.nan, np.inf, -np.inf
    got = run_attention(pg, q)
    bad = np.zeros((3, 6), bool)
    bad[0, 1] = bad[1, 4] = bad[1, 0] = True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[~bad])


def test_attention_twice_the_same_bits(gpu):
    rng = np.random.default_rng(21)
    pg = PagesQ(rng, [3000, 100, 4000, 0], 16, 2, 128, 32, 4, 4, F16)
    q = rng.normal(0, 2, (4, 12, 128)).astype(np.float16)
    np.testing.assert_array_equal(run_attention(pg, q), run_attention(pg, q))


# ---- graphs, streams, far pages -----------------------------------------------------------
def test_captured_step_replayed_with_new_values(gpu):
    """Append, attention and read of a step in one graph; lengths, positions and rows change between replays."""
    rng = np.random.default_rng(22)
    lens = [1000, 17, 0, 2000]
    H, KVH, D = 6, 2, 64
    pg = PagesQ(rng, lens, 16, KVH, D, 32, 8, 4, F16, max_pages=140)
    for s in range(4):  # a free page each
        used = set(pg.table[pg.table >= 0].tolist())
        free = [p for p in range(len(pg.kp)) if p not in used]
        n = -(-lens[s] // 16)
        if lens[s] % 16 == 0 and free:
            pg.table[s, n] = free[0]
    put(pg.d_t, pg.table)
    table = rope_table(2200, D)
    bufs = {n: capi.DevBuf(4 * h * D * 2) for n, h in (("q", H), ("r", H), ("a", H), ("k", KVH), ("v", KVH), ("ko", KVH), ("vo", KVH))}
    dpos = capi.DevBuf(16)

    def step(s):
        b = {n: x.ptr for n, x in bufs.items()}
        capi.call("vvh_rope_append_paged_q", pg.cache(), b["r"], b["q"], b["k"], b["v"], None, dpos.ptr, 4, H, table.ptr, 2200, s)
        capi.call("vvh_attention_paged_q", pg.cache(), b["a"], b["r"], pg.d_n.ptr, 0, H, 0.125, s)
        capi.call("vvh_read_paged_q", pg.cache(), b["ko"], b["vo"], None, dpos.ptr, 4, s)

    st, replay = Stream(), None
    for i in range(4):
        pos = np.array([lens[0] + i, lens[1] + i, -1 if i < 2 else i - 2, lens[3] + i], np.int32)
        put(dpos, pos)
        put(pg.d_n, pos + 1)
        for n, h in (("q", H), ("k", KVH), ("v", KVH)):
            put(bufs[n], rng.normal(0, 1, (4, h, D)).astype(np.float16))
        step(st.s)
        st.sync()
        names = [("r", H), ("a", H), ("ko", KVH), ("vo", KVH)]
        eager = [bufs[n].to_array(np.uint16, (4, h, D)) for n, h in names]
        held = pg.download()
        pg.kp, pg.vp, pg.ks, pg.vs, pg.lens = held[0], held[1], held[2].view(np.float16), held[3].view(np.float16), pos + 1
        ref, tol = attention_q_ref(pg, bufs["r"].to_array(np.float16, (4, H, D)), 0.125, HALF[F16])
        live = np.array([pg.table[s, pos[s] // 16] >= 0 if pos[s] >= 0 else False for s in range(4)])
        assert (np.abs(eager[1].view(np.float16) - ref) <= tol)[live].all()
        if replay is None:
            replay = st.capture(step)
        for _ in range(2):
            for n, h in names:
                capi.call("vvh_fill_normal", bufs[n].ptr, F16, 4 * h * D, 1, 0.0, 1.0, None)
            capi.sync()
            replay()
            for (n, h), e in zip(names, eager):
                x = bufs[n].to_array(np.uint16, (4, h, D))
                np.testing.assert_array_equal(x[live], e[live])
    st.close()


def test_two_graphs_of_one_stream(gpu):
    """Two captured calls that split, and so share the stream's workspace, replayed in turn."""
    rng = np.random.default_rng(28)
    st = Stream()
    pgs = [PagesQ(rng, lens, 16, 2, 128, 32, kb, 4, F16) for lens, kb in (([3000, 20, 2500], 4), ([1500] * 5, 8))]
    qs = [rng.normal(0, 2, (len(pg.lens), 12, 128)).astype(np.float16) for pg in pgs]
    dq, do = [capi.DevBuf.from_array(q) for q in qs], [capi.DevBuf(q.nbytes) for q in qs]

    def call(i):
        return lambda s: capi.call("vvh_attention_paged_q", pgs[i].cache(), do[i].ptr, dq[i].ptr, pgs[i].d_n.ptr, 0, 12,
                                   float(1 / np.sqrt(128)), s)

    out = lambda i: do[i].to_array(np.float16, qs[i].shape)  # noqa: E731
    eager = []
    for i in (0, 1):
        call(i)(st.s)
        st.sync()
        eager.append(out(i))
    replays = []
    for i in (0, 1):
        replays.append((st.capture(call(i)), st.keep))
    for i in (0, 1, 1, 0, 1, 0):
        capi.call("vvh_fill_normal", do[i].ptr, F16, qs[i].size, 1, 0.0, 1.0, None)
        capi.sync()
        replays[i][0]()
        np.testing.assert_array_equal(out(i), eager[i])
    for _, (g, e) in replays:
        st.hip.hipGraphExecDestroy(e)
        st.hip.hipGraphDestroy(g)
    del st.keep
    st.close()


def test_short_contexts_captured(gpu):
    """One launch, no workspace: captured on a stream that has made no call before, replayed with other lengths."""
    rng = np.random.default_rng(32)
    pg = PagesQ(rng, [500, 30, 0, 700], 16, 2, 128, 32, 8, 4, F16)
    q = rng.normal(0, 2, (4, 12, 128)).astype(np.float16)
    dq, do, st = capi.DevBuf.from_array(q), capi.DevBuf(q.nbytes), Stream()
    replay = st.capture(lambda s: capi.call("vvh_attention_paged_q", pg.cache(), do.ptr, dq.ptr, pg.d_n.ptr, 700, 12, 0.125, s))
    for lens in ([500, 30, 0, 700], [3, 0, 0, 64], [65, 17, -1, 640]):
        pg.lens = np.array(lens, np.int32)
        put(pg.d_n, pg.lens)
        ref, tol = attention_q_ref(pg, q, 0.125, HALF[F16])
        for _ in range(2):
            capi.call("vvh_fill_normal", do.ptr, F16, q.size, 1, 0.0, 1.0, None)
            capi.sync()
            replay()
            assert (np.abs(do.to_array(np.float16, q.shape) - ref) <= tol).all()
    st.close()


def test_two_streams_at_once(gpu):
    rng = np.random.default_rng(23)
    pgs = [PagesQ(rng, [3000, 900, 2500], 16, 2, 128, 64, 4, 4, F16) for _ in range(2)]
    qs = [rng.normal(0, 2, (3, 12, 128)).astype(np.float16) for _ in range(2)]
    alone = [run_attention(pg, q) for pg, q in zip(pgs, qs)]
    st = [Stream(), Stream()]
    dq = [capi.DevBuf.from_array(q) for q in qs]
    do = [capi.DevBuf(q.nbytes) for q in qs]
    for _ in range(10):
        for i in (0, 1):
            capi.call("vvh_attention_paged_q", pgs[i].cache(), do[i].ptr, dq[i].ptr, pgs[i].d_n.ptr, 0, 12, float(1 / np.sqrt(128)),
                      st[i].s)
    for i in (0, 1):
        st[i].sync()
        np.testing.assert_array_equal(do[i].to_array(np.float16, qs[i].shape).astype(np.float64), alone[i])
        st[i].close()


@pytest.mark.parametrize("D,group,kb,vb", [(64, 32, 4, 4), (128, 128, 8, 8)])
def test_pages_past_4_gb(gpu, D, group, kb, vb):
    """Pages whose bytes, and at head_dim 64 whose scales' bytes too, lie past 2^32: append, read and attention at the
    pool's end."""
    rng = np.random.default_rng(24)
    KVH, page = 16, 128
    per = D * kb // 8 * page * KVH
    pages = (1 << 32) // (D // group * 4 * page * KVH if D == 64 else per) + 5
    lens = [1500, 40]
    pg = PagesQ(rng, lens, page, KVH, D, group, kb, vb, F16)
    far = {int(p): pages - 1 - i for i, p in enumerate(pg.table[pg.table >= 0])}
    bufs = []
    for a in (pg.kp, pg.vp, pg.ks, pg.vs):
        one = a[0].nbytes
        b = capi.DevBuf(one * pages)
        for p, f in far.items():
            capi.call("vvh_memcpy_h2d", b.addr(f * one), np.ascontiguousarray(a[p]).ctypes.data, one)
        bufs.append(b)
    q = rng.normal(0, 2, (2, 32, D)).astype(np.float16)
    near = run_attention(pg, q)
    k0, v0 = read_rows(pg, [0] * 1500, list(range(1500)))
    kp, vp, ks, vs = pg.d_k, pg.d_v, pg.d_ks, pg.d_vs
    pg.table = np.array([[far.get(int(p), -1) for p in row] for row in pg.table], np.int32)
    put(pg.d_t, pg.table)
    cache = pg.cache
    pg.cache = lambda **kw: cache(**{**dict(k_pages=bufs[0].ptr, v_pages=bufs[1].ptr, k_scales=bufs[2].ptr, v_scales=bufs[3].ptr,
                                           num_pages=pages), **kw})
    np.testing.assert_array_equal(run_attention(pg, q), near)
    k1, v1 = read_rows(pg, [0] * 1500, list(range(1500)))
    bits_equal(k1, k0)
    bits_equal(v1, v0)
    x = rng.normal(0, 1, (1, KVH, D)).astype(np.float16)
    dx, dp = capi.DevBuf.from_array(x), capi.DevBuf.from_array(np.array([1499], np.int32))
    capi.call("vvh_rope_append_paged_q", pg.cache(), None, None, dx.ptr, dx.ptr, None, dp.ptr, 1, 0, None, 0, None)
    _, v2 = read_rows(pg, [0], [1499])
    want = capi.unpack_paged_q(*capi.pack_paged_q(x[0], vb, group, False), vb, False)
    bits_equal(v2[0], want.astype(np.float32).astype(np.float16))
    pg.d_k, pg.d_v, pg.d_ks, pg.d_vs = kp, vp, ks, vs


# ---- together --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", [(64, 32, 4, 4), (128, 64, 8, 4)])
def test_prompt_in_parts_then_decode(gpu, dtype, D, group, kb, vb):
    """A prompt appended in two parts, the second attending to both through the rows read back, then decode steps; the
    last row of the prompt's attention and a decode step's agree with 64 bits over the same cache."""
    rng = np.random.default_rng(25)
    H, KVH, page, n1, n2 = 6, 2, 16, 70, 45
    pg = PagesQ(rng, [0], page, KVH, D, group, kb, vb, dtype, spare=12, max_pages=12)
    pg.table[0] = rng.permutation(12)
    put(pg.d_t, pg.table)
    table = rope_table(200, D)
    scale = float(np.float32(1 / np.sqrt(D)))
    n = n1 + n2
    for a, b in ((0, n1), (n1, n)):
        T = b - a
        q, k, v = (capi.DevBuf.from_array(rng.normal(0, 1, (T, h, D)).astype(NP[dtype])) for h in (H, KVH, KVH))
        ds, dp = capi.DevBuf.from_array(np.zeros(T, np.int32)), capi.DevBuf.from_array(np.arange(a, b, dtype=np.int32))
        capi.call("vvh_rope_append_paged_q", pg.cache(), q.ptr, q.ptr, k.ptr, v.ptr, ds.ptr, dp.ptr, T, H, table.ptr, 200, None)
        ks, vs, o = capi.DevBuf(b * KVH * D * 4), capi.DevBuf(b * KVH * D * 4), capi.DevBuf(T * H * D * 4)
        ds, dp = capi.DevBuf.from_array(np.zeros(b, np.int32)), capi.DevBuf.from_array(np.arange(b, dtype=np.int32))
        capi.call("vvh_read_paged_q", pg.cache(), ks.ptr, vs.ptr, ds.ptr, dp.ptr, b, None)
        capi.call("vvh_attention", o.ptr, q.ptr, ks.ptr, vs.ptr, T, a + 1, H, KVH, D, scale, dtype, None)
        capi.sync()
        held = pg.download()
        pg.kp, pg.vp, pg.ks, pg.vs = held[0], held[1], held[2].view(np.float16), held[3].view(np.float16)
        rot = q.to_array(NP[dtype], (T, H, D))
        got = o.to_array(NP[dtype], (T, H, D))
        for t in (0, T // 2, T - 1):
            pg.lens = np.array([a + t + 1], np.int32)
            ref, tol = attention_q_ref(pg, rot[t:t + 1], scale, HALF[dtype])
            # the rows read back are rounded to the type: a score's and a value's sizes times half a step
            k_, v_, ka, va = pg.rows(0)
            more = 2 * HALF[dtype] * (np.abs(rot[t].astype(np.float64)).sum(1).max() * np.abs(k_).max() * scale + 1) * np.abs(v_).max()
            assert (np.abs(got[t] - ref[0]) <= tol[0] + more).all()
    for i in range(3):
        q, k, v = (capi.DevBuf.from_array(rng.normal(0, 1, (1, h, D)).astype(NP[dtype])) for h in (H, KVH, KVH))
        put(pg.d_n, np.array([n + i + 1], np.int32))
        dp = capi.DevBuf.from_array(np.array([n + i], np.int32))
        o = capi.DevBuf(H * D * 4)
        capi.call("vvh_rope_append_paged_q", pg.cache(), q.ptr, q.ptr, k.ptr, v.ptr, None, dp.ptr, 1, H, table.ptr, 200, None)
        capi.call("vvh_attention_paged_q", pg.cache(), o.ptr, q.ptr, pg.d_n.ptr, n + i + 1, H, scale, None)
        capi.sync()
        held = pg.download()
        pg.kp, pg.vp, pg.ks, pg.vs = held[0], held[1], held[2].view(np.float16), held[3].view(np.float16)
        pg.lens = np.array([n + i + 1], np.int32)
        ref, tol = attention_q_ref(pg, q.to_array(NP[dtype], (1, H, D)), scale, HALF[dtype])
        assert (np.abs(o.to_array(NP[dtype], (1, H, D)) - ref) <= tol).all()
