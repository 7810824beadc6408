"""vvh_attention_paged over values that are not finite: in their dim an infinity gives itself, NaN where it meets one of
the other sign or a NaN, and every other dim is what it was; the same for each type, head_dim and alignment, in one
launch and split.  Finite dims against 64 bits with attention_ref's tolerance (the infinite values count as 0 there: they
are in no other dim's sum)."""
import numpy as np
import pytest

from serving import HALF, Pages, Stream, attention_ref, put
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}


def plant(pg, s, key, g, dim, value):
    pg.vp[pg.table[s, key // pg.page], key % pg.page, g, dim] = value


def want(pg, q, scale):
    """The 64-bit result: (values with NaN and infinities in place, tolerance of the finite ones)."""
    seen = pg.vp
    pg.vp = np.where(np.isfinite(seen), seen, 0)
    ref, tol = attention_ref(pg, q, scale, HALF[pg.dtype])
    pg.vp = seen
    for s in range(len(q)):
        _, v = pg.rows(s)
        for h in range(q.shape[1]):
            x = v[:, h // (q.shape[1] // pg.KVH)]
            up, down, nan = (x == np.inf).any(0), (x == -np.inf).any(0), np.isnan(x).any(0)
            ref[s, h, up], ref[s, h, down] = np.inf, -np.inf
            ref[s, h, nan | up & down] = np.nan
    return ref, tol


def check(got, ref, tol):
    odd = ~np.isfinite(ref)
    assert odd.any() and not odd.all()
    np.testing.assert_array_equal(got[odd], ref[odd])
    off = np.abs(got - ref)[~odd] / tol[~odd]
    assert (off <= 1).all(), off.max()


def attend(pg, q, scale, shift=False, max_len=0):
    e = q.itemsize
    at = lambda a: capi.DevBuf.from_array(np.concatenate([np.zeros(1, a.dtype), a.ravel()]))  # noqa: E731
    dq, do, dk, dv = at(q), capi.DevBuf(q.nbytes + e), None, None
    kv = {}
    if shift:  # the pages one value past their 16-byte addresses
        dk, dv = at(pg.kp), at(pg.vp)
        kv = dict(k_pages=dk.addr(e), v_pages=dv.addr(e))
    else:
        dq = capi.DevBuf.from_array(q)
    capi.call("vvh_attention_paged", pg.cache(**kv), do.ptr, dq.addr(e) if shift else dq.ptr, pg.d_n.ptr, max_len, q.shape[1],
              scale, None)
    capi.sync()
    return do.to_array(q.dtype, q.shape).astype(np.float64)


HEADS = [(14, 2, 64), (6, 2, 96), (12, 2, 128), (20, 1, 64), (4, 2, 40), (4, 2, 80), (2, 1, 256)]
LENS = [[100, 130, 1, 70], [3000, 200, 1, 2100], [700, 40000, 33, 65]]
# unaligned arrays: another route only where aligned ones take the matrix cores
ROUTES = [(h, n, shift) for h in HEADS for n in LENS for shift in (False, True) if not shift or h[2] in (64, 96, 128) and max(n) < 5000]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,lens,shift", ROUTES)
def test_infinite_values(gpu, dtype, heads, lens, shift):
    H, KVH, D = heads
    print("[case] infinities", dtype, H, KVH, D, lens, shift, flush=True)
    rng = np.random.default_rng(H + D + len(lens))
    pg = Pages(rng, lens, 24, KVH, D, dtype)
    plant(pg, 0, 5, 0, 3, np.inf)
    plant(pg, 0, lens[0] - 1, KVH - 1, 7, -np.inf)
    plant(pg, 1, 64, 0, 0, np.inf)          # both signs, far apart
    plant(pg, 1, lens[1] - 2, 0, 0, -np.inf)
    plant(pg, 1, 20, KVH - 1, D - 1, np.nan)
    plant(pg, 2, 0, 0, 1, -np.inf)          # one key
    pg.upload()
    q = rng.normal(0, 1, (len(lens), H, D)).astype(NP[dtype])
    scale = float(np.float32(1 / np.sqrt(D)))
    check(attend(pg, q, scale, shift), *want(pg, q, scale))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 96, 128, 40])
@pytest.mark.parametrize("n", [300, 3000])
@pytest.mark.parametrize("at", [0, 290])
def test_an_infinite_value_of_small_weight(gpu, dtype, D, n, at):
    """A weight of e^-40, far below what fp16 holds, and one that is the largest."""
    print("[case] small weight", dtype, D, n, at, flush=True)
    rng = np.random.default_rng(D + n)
    pg = Pages(rng, [n, n], 16, 2, D, dtype)
    q = np.zeros((2, 6, D), NP[dtype])
    q[:, :, 0] = 8
    for s in range(2):
        k = pg.kp[pg.table[s]].reshape(-1, 2, D)
        k[:n, :, 0] = 0
        k[at, :, 0] = (-5, 5)[s]  # a score of -40 and 40, the others' 0
        pg.kp[pg.table[s]] = k.reshape(-1, 16, 2, D)
    plant(pg, 0, at, 1, 2, -np.inf)
    plant(pg, 1, (at + 7) % 100, 0, 5, np.inf)
    pg.upload()
    check(attend(pg, q, 1.0), *want(pg, q, 1.0))


def test_infinite_values_come_and_go_in_a_graph(gpu):
    """A captured call: finite values have the eager call's bits before an infinity came and after it went."""
    rng = np.random.default_rng(7)
    pg = Pages(rng, [2500, 90], 16, 2, 128, F16)
    q = rng.normal(0, 1, (2, 12, 128)).astype(np.float16)
    scale = float(np.float32(1 / np.sqrt(128)))
    dq, do, st = capi.DevBuf.from_array(q), capi.DevBuf(q.nbytes), Stream()
    issue = lambda s: capi.call("vvh_attention_paged", pg.cache(), do.ptr, dq.ptr, pg.d_n.ptr, 0, 12, scale, s)  # noqa: E731
    issue(st.s)
    st.sync()
    plain = do.to_array(np.float16, q.shape)
    replay = st.capture(issue)
    clean = pg.vp.copy()
    for step in range(4):
        pg.vp = clean.copy()
        if step % 2:
            plant(pg, 0, 1111 * step // 2, 0, 9, np.inf)
            plant(pg, 1, 89, 1, 127, -np.inf)
        put(pg.d_v, pg.vp)
        capi.sync()
        replay()
        got = do.to_array(np.float16, q.shape)
        if step % 2:
            check(got.astype(np.float64), *want(pg, q, scale))
        else:
            np.testing.assert_array_equal(got, plain)
    st.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("H,KVH,D", [(14, 2, 64), (6, 2, 96), (12, 2, 128), (4, 2, 80)])
@pytest.mark.parametrize("lens", [[130, 64, 90], [3000, 1500, 700]])
def test_dims_and_rows_that_overflowed(gpu, dtype, H, KVH, D, lens):
    """A dim infinite for every key, one of NaN, a sequence whose keys are NaN next to them."""
    print("[case] overflowed", dtype, H, KVH, D, lens, flush=True)
    rng = np.random.default_rng(H * D)
    pg = Pages(rng, lens, 16, KVH, D, dtype)
    pages = lambda s: pg.table[s, :-(-lens[s] // 16)]  # noqa: E731
    pg.vp[pages(0), :, 0, 4] = -np.inf
    pg.vp[pages(0), :, KVH - 1, 9] = np.nan
    pg.vp[pages(1), ::2, 0, 6] = np.inf
    pg.kp[pages(2)] = np.nan
    pg.upload()
    q = rng.normal(0, 1, (3, H, D)).astype(NP[dtype])
    scale = float(np.float32(1 / np.sqrt(D)))
    pg.lens[2] = 0
    ref, tol = want(pg, q, scale)
    pg.lens[2] = lens[2]
    ref[2] = np.nan
    check(attend(pg, q, scale), ref, tol)
