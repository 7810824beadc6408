"""vvh_linear_q4 where test_gpu_linear_q4.py does not come: blocks that take several groups of channels in turn (asserted by the
host rule), the rows of a call next to those of smaller calls, and streams whose calls hold different sums at once."""
import numpy as np
import pytest

from q4_plan import plan
from serving import HALF, Stream
from test_gpu_linear_q4 import NP, Case
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32


class Large(Case):
    """The 64-bit result by 2048 channels at a time."""

    def want(self):
        x = self.x.astype(np.float64)
        y, most = np.empty((self.M, self.N)), np.empty((self.M, self.N))
        for a in range(0, self.N, 2048):
            n = slice(a, min(a + 2048, self.N))
            c = np.stack([self.codes[n] & 15, self.codes[n] >> 4], -1).reshape(-1, self.K // self.group, self.group).astype(np.float64)
            z = self.zeros[n].astype(np.float64)[..., None] if self.zeros is not None else 8.0
            s = self.scales[n].astype(np.float64)[..., None]
            y[:, n] = x @ ((c - z) * s).reshape(-1, self.K).T
            most[:, n] = np.abs(x) @ ((c + z) * s).reshape(-1, self.K).T
        for add in (self.bias, self.res):
            if add is not None:
                y, most = y + add.astype(np.float64), most + np.abs(add.astype(np.float64))
        return y, HALF[self.outd] * np.abs(y) + 2.0 ** -25 + (self.K + 4) * 2.0 ** -24 * most


# act, (M, N, K, group), waves a tile, whether k is shared too, groups in turn; of some the last blocks take fewer
TURNS = [(F16, (4, 9054, 8576, 128), 4, False, 2), (F16, (4, 13090, 8576, 64), 4, False, 3), (F16, (4, 5018, 17408, 128), 4, True, 2),
         (F16, (4, 17126, 8576, 32), 2, False, 2), (F16, (4, 33270, 8576, 128), 1, False, 2), (F32, (4, 9054, 4352, 128), 4, False, 2),
         (F32, (4, 13090, 8576, 128), 2, True, 3), (F32, (4, 7036, 8576, 64), 4, True, 3), (F32, (4, 131143, 1056, 32), 1, False, 2),
         (F32, (4, 17126, 4352, 32), 2, False, 2), (F32, (8, 131143, 800, 32), 1, False, 2), (F32, (8, 98855, 1664, 128), 1, False, 3)]


@pytest.mark.parametrize("i,act,shape,ks,shared,turns", [(i, *t) for i, t in enumerate(TURNS)])
def test_groups_of_channels_in_turn(gpu, i, act, shape, ks, shared, turns):
    M, N, K, group = shape
    p = plan(M, N, K, act == F32)
    assert (p.kernel, p.ks, p.splits > 1, p.turns) == ("whole", ks, shared, turns)
    assert N % (16 * p.waves // p.ks)  # a last group that is not full
    c = Large(M, N, K, group, act, (act, F32)[i % 3 == 2], zeros=i % 2 == 0, bias=i % 3 != 0, residual=True)
    y, tol = c.want()
    c.run()
    plain = c.got()
    off = np.abs(plain.astype(np.float64) - y) / tol
    assert (off <= 1).all(), (off.max(), np.argwhere(off > 1)[:5])
    c.run(out=c.d["res"])  # in the residual's place: the same bits
    np.testing.assert_array_equal(c.got(c.d["res"]), plain)


@pytest.mark.parametrize("act", [F16, F32])
@pytest.mark.parametrize("M,N,K", [(5, 77, 320), (13, 8200, 640), (40, 300, 5120), (70, 4000, 3200), (4, 9054, 4352)])
def test_rows_of_a_call_and_of_smaller_calls(gpu, act, M, N, K):
    """Every row by itself and with others, a guard on both sides of the output; both within the 64-bit tolerance."""
    c = Case(M, N, K, 64, act, act, bias=True)
    y, tol = c.want()
    e = np.dtype(NP[act]).itemsize
    p = {n: b.ptr for n, b in c.d.items()}
    for step in (M, max(1, M // 3), 1):
        out = capi.DevBuf.from_array(np.full((M + 2, N), 7, NP[act]))
        for m in range(0, M, step):
            rows = min(step, M - m)
            capi.call("vvh_linear_q4", out.addr((1 + m) * N * e), c.d["x"].addr(m * K * e), p["codes"], p["scales"], None, p["bias"], None,
                      rows, N, K, 64, act, act, None)
        got = out.to_array(NP[act], (M + 2, N))
        assert (got[0] == 7).all() and (got[-1] == 7).all()
        assert (np.abs(got[1:-1].astype(np.float64) - y) <= tol).all(), step


def test_two_streams_with_different_sums(gpu):
    """Calls that share out k, each stream with inputs of its own and in another order: no workspace is another's."""
    shapes = [(16, 130, 8960, 128, F16), (40, 100, 8960, 64, F16), (2, 33, 45056, 128, F16), (64, 4000, 4096, 64, F16), (16, 300, 4864, 32, F32)]
    assert all(plan(M, N, K, a == F32).splits > 1 for M, N, K, _, a in shapes)
    sets = [[Case(M, N, K, g, a, a, zeros=i % 2 == 0, seed=10 * s) for i, (M, N, K, g, a) in enumerate(shapes)] for s in range(2)]
    sets[1].reverse()
    want = []
    for cs in sets:
        for c in cs:
            c.run()
        want.append([c.got() for c in cs])
    streams = [Stream(), Stream()]
    for st, cs in zip(streams, sets):  # the streams' workspaces
        for c in cs:
            c.run(stream=st.s)
    for _ in range(10):
        for a, b in zip(*sets):
            a.run(stream=streams[0].s)
            b.run(stream=streams[1].s)
    for st, cs, ws in zip(streams, sets, want):
        st.sync()
        for c, w in zip(cs, ws):
            np.testing.assert_array_equal(c.got(), w)
        st.close()
