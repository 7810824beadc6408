"""vvh_linear_q4 in graphs by its header's word on the workspace: up to the bounds a capture needs no call before it, past them
one; replays with new outputs every time, whole outputs compared with the eager call's bits."""
import numpy as np
import pytest

from q4_plan import plan
from serving import Stream
from test_gpu_linear_q4 import NP, Case
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32


def replays(cases, before):
    for c in cases:
        c.run()
    capi.sync()
    eager = [c.got() for c in cases]
    for c in cases:
        y, tol = c.want()
        assert (np.abs(c.got().astype(np.float64) - y) <= tol).all()
    st = Stream()
    capi.call("vvh_workspace_release", st.s)  # the handle may have been another stream's
    for c in cases if before else []:
        c.run(stream=st.s)
    st.sync()
    replay = st.capture(lambda s: [c.run(stream=s) for c in cases])
    for _ in range(3):
        for c in cases:
            capi.call("vvh_fill_normal", c.d_out.ptr, c.outd, c.M * c.N, 1, 0.0, 1.0, None)
        capi.sync()
        for c, e in zip(cases, eager):
            assert (c.got() != e).mean() > 0.9  # the earlier outputs are gone
        replay()
        for c, e in zip(cases, eager):
            np.testing.assert_array_equal(c.got(), e)
    st.close()


def test_captured_first(gpu):
    """No call before: sizes up to the header's bounds."""
    sizes = [(4, 300, 17152, F16), (1, 4000, 17152, F16), (4, 300, 8448, F32), (2, 4000, 8448, F32), (64, 4000, 2816, F16),
             (16, 900, 2816, F16), (16, 300, 1024, F32), (64, 4000, 1024, F32), (9, 100, 1024, F32)]
    assert not any(plan(M, N, K, act == F32).ws for M, N, K, act in sizes)
    replays([Case(M, N, K, 64, act, act, bias=True) for M, N, K, act in sizes], before=False)


@pytest.mark.parametrize("M,N,K,act", [(64, 4000, 4096, F16), (13, 18944, 3584, F16), (16, 300, 1088, F32), (33, 4000, 4096, F32),
                                       (3, 500, 23168, F16), (4, 500, 8512, F32)])
def test_captured_after_one_call(gpu, M, N, K, act):
    """k shared out, also where rows would fit a block."""
    assert plan(M, N, K, act == F32).splits > 1
    replays([Case(M, N, K, 64, act, F32 if act == F16 else F16, zeros=True, residual=True)], before=True)
