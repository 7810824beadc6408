"""vvh_linear_q4 against the same linear in 64 bits: rows from one to past a pass, groups, zero points, odd channel
counts, every pair of types, residual in place.

Tolerance per element: half a step of the output's type and K fp32 roundings of the largest sum that the codes can make,
K 2^-24 sum |x| s (c + z) (codes and zero points may be summed apart)."""
import numpy as np
import pytest

from serving import HALF, Stream
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}


class Case:
    def __init__(self, M, N, K, group, act, outd, zeros=False, bias=False, residual=False, seed=0):
        print("[case] q4", M, N, K, group, act, outd, zeros, bias, residual, flush=True)
        rng = np.random.default_rng(M + N + K + seed)
        self.M, self.N, self.K, self.group, self.act, self.outd = M, N, K, group, act, outd
        self.codes = rng.integers(0, 256, (N, K // 2), np.uint8)
        self.scales = rng.uniform(0.002, 0.01, (N, K // group)).astype(np.float16)
        self.zeros = rng.integers(0, 16, (N, K // group), np.uint8) if zeros else None
        self.bias = rng.normal(0, 0.1, N).astype(np.float32) if bias else None
        self.x = rng.normal(0, 1, (M, K)).astype(NP[act])
        self.res = rng.normal(0, 1, (M, N)).astype(NP[outd]) if residual else None
        self.d = {n: capi.DevBuf.from_array(a) for n, a in vars(self).items() if isinstance(a, np.ndarray)}
        self.d_out = capi.DevBuf(max(1, M * N * 4))

    def want(self):
        c = np.stack([self.codes & 15, self.codes >> 4], -1).reshape(self.N, -1, self.group).astype(np.float64)
        z = self.zeros.astype(np.float64)[..., None] if self.zeros is not None else 8.0
        s = self.scales.astype(np.float64)[..., None]
        x = self.x.astype(np.float64)
        flat = lambda w: w.reshape(self.N, self.K)  # noqa: E731
        y = x @ flat((c - z) * s).T
        most = np.abs(x) @ flat((c + z) * s).T
        if self.bias is not None:
            y = y + self.bias
            most = most + np.abs(self.bias)
        if self.res is not None:
            y = y + self.res
            most = most + np.abs(self.res.astype(np.float64))
        return y, HALF[self.outd] * np.abs(y) + 2.0 ** -25 + (self.K + 4) * 2.0 ** -24 * most

    def run(self, out=None, stream=None):
        p = lambda n: self.d[n].ptr if n in self.d else None  # noqa: E731
        out = out or self.d_out
        capi.call("vvh_linear_q4", out.ptr, p("x"), p("codes"), p("scales"), p("zeros"), p("bias"),
                  out.ptr if out is self.d.get("res") else p("res"), self.M, self.N, self.K, self.group, self.act, self.outd, stream)
        return out

    def got(self, out=None):
        return (out or self.d_out).to_array(NP[self.outd], (self.M, self.N))

    def check(self):
        y, tol = self.want()
        self.run()
        off = np.abs(self.got().astype(np.float64) - y) / tol
        assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 130])
def test_rows(gpu, act, M):
    Case(M, 200, 640, 64, act, act, zeros=M % 2 == 1, bias=M % 3 == 0, residual=M % 4 == 1).check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 896, 896), (1, 17, 128), (2, 1, 128), (7, 130, 4864), (1, 64, 8960), (16, 33, 1536),
                                   (40, 100, 384), (1, 2500, 256), (5, 16, 128 * 37)])
def test_groups_and_shapes(gpu, act, group, zeros, M, N, K):
    Case(M, N, K, group, act, act, zeros=zeros).check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("K,group", [(32, 32), (64, 32), (64, 64), (96, 32), (160, 32), (192, 64), (224, 32), (288, 32), (320, 64),
                                     (384, 128), (1056, 32), (2080, 32)])
@pytest.mark.parametrize("M", [1, 3, 20])
def test_short_and_odd_rows(gpu, act, K, group, M):
    """Rows that end inside a step, of one group and of odd numbers of groups (scales of odd addresses)."""
    Case(M, 37, K, group, act, act, zeros=K % 64 == 32).check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 40, 90112), (2, 33, 45056), (16, 130, 8960), (40, 100, 8960), (9, 1, 20480),
                                   (5, 200, 33280), (6, 17, 99968), (17, 130, 2176), (33, 260, 5120), (64, 40, 16640), (64, 4000, 3200)])
def test_rows_of_x_past_the_lds(gpu, act, M, N, K):
    """k shared by several blocks, whose sums a second launch adds."""
    Case(M, N, K, 128, act, act, zeros=True, bias=True, residual=True).check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M,N", [(1, 40000), (16, 20011), (33, 9000)])
def test_many_channels(gpu, act, M, N):
    """Blocks that take several groups of channels in turn."""
    Case(M, N, 96, 32, act, act, bias=True).check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("group,K", [(32, 32), (32, 224), (64, 256), (64, 448), (32, 512), (128, 640), (64, 960), (128, 1024)])
@pytest.mark.parametrize("M,N", [(5, 16390), (9, 16390), (16, 16300), (17, 8200), (23, 8200), (40, 16500), (65, 4100), (130, 2000)])
def test_many_rows_and_channels(gpu, act, group, K, M, N):
    """Steps of x in turn: one, even and odd numbers of them, rows that end inside one; passes of up to 16 and 32 rows."""
    Case(M, N, K, group, act, act, zeros=K % 3 == 1, bias=M % 2 == 1, residual=M % 3 == 1).check()


@pytest.mark.parametrize("act,outd", [(F16, F32), (F32, F16)])
def test_many_rows_and_channels_of_mixed_types(gpu, act, outd):
    Case(20, 8200, 512, 64, act, outd, zeros=True, bias=True, residual=True).check()


@pytest.mark.parametrize("act", [F16, F32])
def test_many_rows_in_place(gpu, act):
    """The residual's place for the output, row by row; rows with infinities and NaN leave the others alone."""
    c = Case(37, 8200, 320, 64, act, act, residual=True)
    c.x[3, 7], c.x[20, 300], c.x[36, 0] = np.inf, np.nan, -np.inf
    c.d["x"] = capi.DevBuf.from_array(c.x)
    with np.errstate(invalid="ignore", over="ignore"):
        y, tol = c.want()
    c.run(out=c.d["res"])
    got = c.got(c.d["res"]).astype(np.float64)
    rows = [m for m in range(37) if m not in (3, 20, 36)]
    assert (np.abs(got - y)[rows] <= tol[rows]).all()
    assert np.isnan(got[20]).all() and not np.isfinite(got[[3, 36]]).any()


@pytest.mark.parametrize("act,outd", [(F16, F32), (F32, F16)])
@pytest.mark.parametrize("M", [1, 4, 16, 40])
def test_mixed_types(gpu, act, outd, M):
    Case(M, 300, 896, 128, act, outd, bias=True, residual=True).check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M", [1, 6, 24])
def test_residual_in_place(gpu, act, M):
    c = Case(M, 500, 896, 64, act, act, residual=True, bias=True)
    y, tol = c.want()
    c.run()
    plain = c.got()
    c.run(out=c.d["res"])
    np.testing.assert_array_equal(c.got(c.d["res"]), plain)
    assert (np.abs(plain.astype(np.float64) - y) <= tol).all()


@pytest.mark.parametrize("act", [F16, F32])
def test_no_k(gpu, act):
    c = Case(3, 20, 0, 64, act, act, bias=True, residual=True)
    c.check()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M", [1, 5, 20])
def test_codes_and_scales_at_their_ends(gpu, act, M):
    """Codes 0 and 15, zero points 0 and 255, scales of 0, the smallest and the largest."""
    c = Case(M, 64, 512, 128, act, F32, zeros=True)
    c.codes[::2], c.codes[1::2] = 0, 255
    c.zeros[:32], c.zeros[32:] = 0, 255
    c.scales[:, 0], c.scales[:, 1], c.scales[:, 2] = 0, 6e-8, 65504
    c.d = {n: capi.DevBuf.from_array(a) for n, a in vars(c).items() if isinstance(a, np.ndarray)}
    c.check()


@pytest.mark.parametrize("M", [1, 4, 20])
def test_activations_of_any_size(gpu, M):
    """fp32 rows far from 1 and with values far apart; a row with infinities and NaN leaves the others alone."""
    c = Case(M, 50, 256, 64, F32, F32)
    c.x *= np.float32(1e20)
    c.x[-1] = np.float32(1e-30) * c.x[-1]
    c.x[0, 5] *= 1e4
    c.d["x"] = capi.DevBuf.from_array(c.x)
    c.check()
    if M > 1:
        c.x[1, 7], c.x[2, 9] = np.inf, np.nan
        c.d["x"] = capi.DevBuf.from_array(c.x)
        with np.errstate(invalid="ignore"):
            y, tol = c.want()
        c.run()
        rows = [m for m in range(M) if m not in (1, 2)]
        assert (np.abs(c.got().astype(np.float64) - y)[rows] <= tol[rows]).all()
        assert np.isnan(c.got()[2]).all() and not np.isfinite(c.got()[1]).any()


@pytest.mark.parametrize("M", [1, 20])
def test_an_infinity_next_to_large_values(gpu, M):
    """Infinite outputs where one activation is infinite, finite ones of the other sign next to it or not."""
    c = Case(M, 50, 512, 64, F32, F32)
    c.codes[:] = 0xCC  # every weight above 0
    c.x[:, 3::2] = -1e30
    c.x[:, 2] = np.inf
    c.x[:, 300] = 2e38
    c.d["x"], c.d["codes"] = capi.DevBuf.from_array(c.x), capi.DevBuf.from_array(c.codes)
    c.run()
    assert (c.got() == np.inf).all()


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M,N,K,group", [(1, 50, 96, 32), (3, 50, 640, 64), (20, 8200, 352, 32), (2, 50, 384, 128)])
def test_an_infinite_scale_in_the_last_group(gpu, act, M, N, K, group):
    """Rows that end inside a step: the infinity is met by its own group's sum, not by what is past the row."""
    c = Case(M, N, K, group, act, F32)
    c.codes[:] = 0xCC  # every weight above 0
    c.x = np.abs(c.x) + NP[act](0.1)
    c.scales[1::2, -1] = np.inf
    c.d = {n: capi.DevBuf.from_array(a) for n, a in vars(c).items() if isinstance(a, np.ndarray)}
    c.run()
    got = c.got()
    assert (got[:, 1::2] == np.inf).all() and np.isfinite(got[:, ::2]).all()


@pytest.mark.parametrize("act", [F16, F32])
def test_rows_of_a_large_call_are_the_small_calls(gpu, act):
    """Outputs next to the last row and channel stay as they were."""
    c = Case(5, 77, 320, 64, act, act)
    guard = np.full((6, 77), 7, NP[act])
    out = capi.DevBuf.from_array(guard)
    c.run(out=out)
    got = out.to_array(NP[act], (6, 77))
    assert (got[5] == 7).all()


def test_captured(gpu):
    st = Stream()
    cs = [Case(1, 896, 896, 64, F16, F16), Case(8, 500, 4864, 128, F16, F16, zeros=True), Case(3, 300, 640, 32, F32, F32),
          Case(40, 300, 640, 32, F32, F32), Case(40, 200, 4864, 64, F16, F16), Case(20, 8200, 320, 64, F16, F16)]
    for c in cs:
        c.run()
    eager = [c.got() for c in cs]
    for c in cs:
        c.run(stream=st.s)
    st.sync()
    replay = st.capture(lambda s: [c.run(stream=s) for c in cs])
    for _ in range(3):
        for c in cs:
            capi.call("vvh_fill_normal", c.d_out.ptr, F32, c.M * c.N // 2, 1, 0.0, 1.0, None)
        capi.sync()
        replay()
        for c, e in zip(cs, eager):
            np.testing.assert_array_equal(c.got(), e)
    st.close()


def test_quantized_weights(gpu):
    """Weights through the host packing: the linear is that of the weights they stand for."""
    rng = np.random.default_rng(1)
    w = rng.normal(0, 0.02, (300, 896)).astype(np.float32)
    c = Case(4, 300, 896, 64, F16, F16)
    c.codes, c.scales = capi.quantize_q4(w, 64)
    c.d["codes"], c.d["scales"] = capi.DevBuf.from_array(c.codes), capi.DevBuf.from_array(c.scales)
    c.check()
    y = c.x.astype(np.float64) @ w.astype(np.float64).T
    # half a step (absmax / 14, at most 0.1 / 14 here) per weight, each of its own sign
    assert np.abs(c.got() - y).max() <= 0.1 / 14 * 6 * np.sqrt(896 / 3)


def test_two_streams_at_once(gpu):
    """Calls that share out k, on two streams without waiting: each stream has a workspace of its own."""
    cs = [Case(16, 130, 8960, 128, F16, F16), Case(40, 100, 8960, 64, F16, F16, zeros=True), Case(2, 33, 45056, 128, F16, F16)]
    for c in cs:
        c.run()
    want = [c.got() for c in cs]
    streams = [Stream(), Stream()]
    outs = [[capi.DevBuf(c.M * c.N * 4) for c in cs] for _ in streams]
    for st, bufs in zip(streams, outs):  # the streams' workspaces
        for c, b in zip(cs, bufs):
            c.run(out=b, stream=st.s)
    for _ in range(10):
        for st, bufs in zip(streams, outs):
            for c, b in zip(cs, bufs):
                c.run(out=b, stream=st.s)
    for st, bufs in zip(streams, outs):
        st.sync()
        for c, b, w in zip(cs, bufs, want):
            np.testing.assert_array_equal(c.got(b), w)
        st.close()
