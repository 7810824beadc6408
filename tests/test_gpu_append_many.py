"""vvh_rope_append_paged of more tokens than one launch holds (2^32 threads): every row of the cache is written, left-out
tokens among them, with and without rotation."""
import numpy as np
import pytest

from test_gpu_paged import rope_table
from vvllm_amd import capi
import ctypes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,heads", [(2, 0), (16, 1)])
def test_more_tokens_than_a_launch(gpu, D, heads):
    """One sequence whose tokens come in reverse order, its last page given back; D 16 takes the 16-byte pieces."""
    T, page = (1 << 24) + 1037, 1 << 16
    print("[case] append", T, D, heads, flush=True)
    pages = -(-T // page)
    k = (np.arange(T * D, dtype=np.int64) * 2654435761 >> 7 & 0x3BFF).astype(np.uint16).view(np.float16).reshape(T, D)
    pos = np.arange(T - 1, -1, -1, dtype=np.int32)
    table = np.arange(pages, dtype=np.int32)[::-1].copy()
    table[-1] = -1
    dk, dp, ds, dt = (capi.DevBuf.from_array(a) for a in (k, pos, np.zeros(T, np.int32), table))
    kp, vp = (capi.DevBuf.from_array(np.zeros((pages * page, D), np.float16)) for _ in range(2))
    c = capi.PagedCache(k_pages=kp.ptr, v_pages=vp.ptr, page_table=dt.ptr, num_pages=pages, page_size=page, num_seqs=1,
                        max_pages=pages, num_kv_heads=1, head_dim=D, dtype=capi.F16)
    rope = rope_table(1, D) if heads else None  # angles of position 0 only
    q = capi.DevBuf.from_array(np.full((T, D), 7, np.float16)) if heads else None
    if heads:  # all but the last token (position 0) are past the table of angles
        capi.call("vvh_rope_append_paged", ctypes.byref(c), q.ptr, q.ptr, dk.ptr, dk.ptr, ds.ptr, dp.ptr, T, heads, rope.ptr, 1, None)
    else:
        capi.call("vvh_rope_append_paged", ctypes.byref(c), None, None, dk.ptr, dk.ptr, ds.ptr, dp.ptr, T, 0, None, 0, None)
    capi.sync()
    row = table.astype(np.int64)[pos // page] * page + pos % page
    for buf in (kp, vp):
        want = np.zeros((pages * page, D), np.float16)
        some = slice(T - 1, T) if heads else slice(None)
        live = row[some] >= 0
        want[row[some][live]] = k[some][live]  # the rotation at position 0 is none
        np.testing.assert_array_equal(buf.to_array(np.float16, want.shape), want)
    if heads:
        got = q.to_array(np.float16, (T, D))
        assert (got == 7).all()
