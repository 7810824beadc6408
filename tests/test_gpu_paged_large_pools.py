"""Pools whose offsets pass 32 bits: attention with 64-bit addresses in every type and head_dim of the matrix cores, in one
launch and split, and a pool between 2 and 4 GB by its 32-bit offsets; the live pages at the pool's end and start.  Memory that
no page table names is whatever it is."""
import ctypes

import numpy as np
import pytest

from serving import HALF, Pages, attention_ref, put
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}


def check(dtype, D, lens, gb, max_pages):
    rng = np.random.default_rng(D + len(lens))
    H, KVH, page = 12, 4, 64
    small = Pages(rng, lens, page, KVH, D, dtype, fill=0, max_pages=max_pages)
    e = np.dtype(NP[dtype]).itemsize
    n = page * KVH * D * e  # bytes of a page
    pages = int(gb * 2**30) // n + 1
    print("[case] pool", dtype, D, lens, pages, n * pages, flush=True)
    big = [capi.DevBuf(pages * n) for _ in range(2)]
    # every third page at the pool's start, the others at its end
    table = np.where(small.table < 0, -1, np.where(small.table % 3 == 0, small.table, pages - 1 - small.table)).astype(np.int32)
    for s, length in enumerate(lens):
        for j in range(-(-length // page)):
            for b, a in zip(big, (small.kp, small.vp)):
                r = np.ascontiguousarray(a[small.table[s, j]])
                capi.call("vvh_memcpy_h2d", b.addr(int(table[s, j]) * n), r.ctypes.data, n)
    put(small.d_t, table)
    q = rng.normal(0, 2, (len(lens), H, D)).astype(NP[dtype])
    scale = float(np.float32(1 / np.sqrt(D)))
    ref, tol = attention_ref(small, q, scale, HALF[dtype])
    dq, do = capi.DevBuf.from_array(q), capi.DevBuf(q.nbytes)
    cache = small.cache(k_pages=big[0].ptr, v_pages=big[1].ptr, num_pages=pages)
    capi.call("vvh_attention_paged", cache, do.ptr, dq.ptr, small.d_n.ptr, 0, H, scale, None)
    capi.sync()
    off = np.abs(do.to_array(NP[dtype], q.shape).astype(np.float64) - ref) / tol
    assert (off <= 1).all(), off.max()


def chunks(dtype, D):
    """Keys at a time, as the kernels take them; a block takes up to 16 chunks by itself."""
    return {F16: {64: 64}, F32: {128: 16}}[dtype].get(D, 32)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("way", ["four waves", "eight waves", "split"])
def test_offsets_past_32_bits(gpu, dtype, D, way):
    ch = chunks(dtype, D)
    cap = {"four waves": 4 * ch, "eight waves": 16 * ch, "split": 2048}[way]  # capacity decides
    lens = {"four waves": [cap, 1, cap - 3], "eight waves": [cap, cap // 2 + 1, 7], "split": [2000, 130, 0, 999]}[way]
    assert cap % 64 == 0 or way == "four waves"
    check(dtype, D, lens, 4.3, max(1, cap // 64))


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F16, 128), (F32, 96), (F32, 128)])
@pytest.mark.parametrize("gb", [2.1, 3.9])
def test_offsets_past_31_bits(gpu, dtype, D, gb):
    check(dtype, D, [1500, 77, 300], gb, 24)
    check(dtype, D, [64, 1, 50], gb, 1)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_values_past_32_bits(gpu, dtype):
    """The second look at values that are not finite finds them at the pool's end."""
    rng = np.random.default_rng(3)
    KVH, D, page, length = 4, 128, 64, 90
    e = np.dtype(NP[dtype]).itemsize
    n = page * KVH * D * e
    pages = int(4.3 * 2**30) // n + 1
    k, v = (rng.normal(0, 1, (2, page, KVH, D)).astype(NP[dtype]) for _ in range(2))
    v[1, 20, 2, 5], v[0, 3, 1, 100] = np.inf, -np.inf
    big = [capi.DevBuf(pages * n) for _ in range(2)]
    table = np.array([[pages - 1, pages - 2]], np.int32)
    for j in range(2):
        for b, a in zip(big, (k, v)):
            capi.call("vvh_memcpy_h2d", b.addr(int(table[0, j]) * n), np.ascontiguousarray(a[j]).ctypes.data, n)
    q = rng.normal(0, 1, (1, 8, D)).astype(NP[dtype])
    dq, do, dt, dn = (capi.DevBuf.from_array(a) for a in (q, q, table, np.array([length], np.int32)))
    c = capi.PagedCache(k_pages=big[0].ptr, v_pages=big[1].ptr, page_table=dt.ptr, num_pages=pages, page_size=page, num_seqs=1,
                        max_pages=2, num_kv_heads=KVH, head_dim=D, dtype=dtype)
    capi.call("vvh_attention_paged", ctypes.byref(c), do.ptr, dq.ptr, dn.ptr, 0, 8, 0.05, None)
    capi.sync()
    got = do.to_array(NP[dtype], q.shape)[0]
    want = np.zeros_like(got)
    want[4:6, 5], want[2:4, 100] = np.inf, -np.inf
    np.testing.assert_array_equal(np.where(np.isfinite(got), 0, got), want)
