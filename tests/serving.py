"""Helpers of the batched decode operators' GPU tests: streams and graphs through the HIP runtime, and a paged cache
filled from plain rows."""
import ctypes

import numpy as np

from vvllm_amd import capi

V = ctypes.c_void_p


def hip():
    for name in ("libamdhip64.so.7", "libamdhip64.so", "/opt/rocm/lib/libamdhip64.so"):
        try:
            lib = ctypes.CDLL(name)
            break
        except OSError:
            continue
    else:
        raise OSError("libamdhip64 not found")
    for name, args in dict(hipStreamCreate=[ctypes.POINTER(V)], hipStreamSynchronize=[V], hipStreamDestroy=[V],
                           hipStreamBeginCapture=[V, ctypes.c_int], hipStreamEndCapture=[V, ctypes.POINTER(V)],
                           hipGraphInstantiate=[ctypes.POINTER(V), V, V, V, ctypes.c_size_t], hipGraphLaunch=[V, V],
                           hipGraphExecDestroy=[V], hipGraphDestroy=[V]).items():
        getattr(lib, name).argtypes = args
    return lib


def ok(status):
    assert status == 0, f"hipError {status}"


class Stream:
    def __init__(self):
        self.hip, self.s = hip(), V()
        ok(self.hip.hipStreamCreate(ctypes.byref(self.s)))

    def sync(self):
        ok(self.hip.hipStreamSynchronize(self.s))

    def capture(self, issue):
        """issue(stream) captured; a function that replays it and waits."""
        g, e = V(), V()
        ok(self.hip.hipStreamBeginCapture(self.s, 0))
        issue(self.s)
        ok(self.hip.hipStreamEndCapture(self.s, ctypes.byref(g)))
        ok(self.hip.hipGraphInstantiate(ctypes.byref(e), g, None, None, 0))

        def replay():
            ok(self.hip.hipGraphLaunch(e, self.s))
            self.sync()

        self.keep = (g, e)
        return replay

    def close(self):
        if hasattr(self, "keep"):
            self.hip.hipGraphExecDestroy(self.keep[1])
            self.hip.hipGraphDestroy(self.keep[0])
        self.hip.hipStreamDestroy(self.s)


def put(buf, a):
    a = np.ascontiguousarray(a)
    capi.call("vvh_memcpy_h2d", buf.ptr, a.ctypes.data, a.nbytes)


class Pages:
    """A paged cache on the device; rows (kp, vp) and table are its host copies."""

    def __init__(self, rng, lens, page, KVH, D, dtype, spare=2, max_pages=None, fill=np.nan):
        self.np = np.float16 if dtype == capi.F16 else np.float32
        counts = [-(-max(n, 0) // page) for n in lens]
        width = max_pages or max(1, max(counts))
        pages = sum(counts) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(lens), width), -1, np.int32)
        self.kp = np.full((pages, page, KVH, D), fill, self.np)  # rows that no sequence has reached
        self.vp = self.kp.copy()
        at = 0
        for s, n in enumerate(lens):
            self.table[s, :counts[s]] = order[at:at + counts[s]]
            at += counts[s]
            for a in (self.kp, self.vp):
                flat = a[self.table[s, :counts[s]]].reshape(-1, KVH, D)
                flat[:max(n, 0)] = rng.normal(0, 1, (max(n, 0), KVH, D))
                a[self.table[s, :counts[s]]] = flat.reshape(-1, page, KVH, D)
        self.lens, self.page, self.KVH, self.D, self.dtype = np.array(lens, np.int32), page, KVH, D, dtype
        self.upload()

    def upload(self):
        self.d_k, self.d_v, self.d_t, self.d_n = (capi.DevBuf.from_array(a) for a in (self.kp, self.vp, self.table, self.lens))

    def cache(self, **kw):
        d = dict(k_pages=self.d_k.ptr, v_pages=self.d_v.ptr, page_table=self.d_t.ptr, num_pages=len(self.kp),
                 page_size=self.page, num_seqs=len(self.table), max_pages=self.table.shape[1], num_kv_heads=self.KVH,
                 head_dim=self.D, dtype=self.dtype)
        return ctypes.byref(capi.PagedCache(**{**d, **kw}))

    def rows(self, s, n=None):
        """K and V rows that sequence s attends to, in 64 bits: [keys, KVH, D] each."""
        j = np.arange(min(max(int(self.lens[s]) if n is None else n, 0), self.table.shape[1] * self.page))
        page = self.table[s, j // self.page]
        j, page = j[(page >= 0) & (page < len(self.kp))], page[(page >= 0) & (page < len(self.kp))]
        return (a[page, j % self.page].astype(np.float64) for a in (self.kp, self.vp))


def attention_ref(pages, q, scale, tol_out):
    """softmax(scale q K^T) V in 64 bits, and how far an element may be off: half a step of the output's type
    (tol_out), and in fp32 a score's D products (twice in the exponential: numerator and sum), a sum of n weights
    and weights of at least 2^-20."""
    B, H, D = q.shape
    ref, tol = np.zeros((B, H, D)), np.zeros((B, H, D))
    for s in range(B):
        k, v = pages.rows(s)
        if not len(k):
            continue
        for h in range(H):
            g = h // (H // pages.KVH)
            x = k[:, g] * q[s, h].astype(np.float64) * scale
            sc = x.sum(1)
            p = np.exp(sc - sc.max())
            ref[s, h] = p @ v[:, g] / p.sum()
            d = (D + 4) * 2.0 ** -24 * np.abs(x).sum(1).max()
            tol[s, h] = (2 * d + (len(k) / 4 + 16) * 2.0 ** -24 + 2.0 ** -20) * np.abs(v[:, g]).max()
    return ref, tol + tol_out * np.abs(ref) + 2.0 ** -25


HALF = {capi.F16: 2.0 ** -11, capi.F32: 2.0 ** -24}
