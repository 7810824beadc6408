"""When vvh_linear_q4 uses the stream's workspace: the bounds that its header names against the host rule."""
import os
import re

import pytest

from q4_plan import plan
from vvllm_amd import capi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(capi.__file__))), "include", "vvllm_hip.h")
NS = [1, 16, 100, 900, 2000, 4000, 8192, 9728, 16384, 18944, 40000, 151936]


def bounds():
    """(K of any call, K of calls of up to 4 rows) without a workspace, for fp16 and fp32 activations."""
    text = re.sub(r"\s+\*\s+", " ", open(HEADER).read())
    said = re.search(r"None is needed for K up to (\d+) \(fp16 activations; fp32 (\d+)\), and with up to 4 rows for K up to (\d+) "
                     r"\(fp32 (\d+)\)", text)
    assert said, "the header names no bounds"
    any16, any32, few16, few32 = map(int, said.groups())
    return {False: (any16, few16), True: (any32, few32)}


@pytest.mark.parametrize("f32", [False, True])
def test_header_bounds_of_the_workspace(f32):
    most, few = bounds()[f32]
    for M in list(range(1, 70)) + [100, 128, 200, 1000]:
        for N in NS:
            for K in range(32, (few if M <= 4 else most) + 1, 32):
                assert plan(M, N, K, f32).ws == 0, (M, N, K)
    # and they are the rule's: a group further on some call needs one
    assert any(plan(M, N, most + 32, f32).ws for M in range(5, 70) for N in NS)
    assert any(plan(M, N, few + 32, f32).ws for M in range(1, 5) for N in NS)


def test_splits_and_sizes():
    for f32 in (False, True):
        for M in (1, 3, 4, 5, 8, 9, 16, 17, 33, 64, 100):
            for N in NS:
                for K in (1056, 3200, 4096, 8960, 20480, 45056):
                    p = plan(M, N, K, f32)
                    assert p.ws == (p.splits * M * N if p.splits > 1 else 0)
                    assert M <= 4 or p.splits <= 12
    # k is shared although the rows fit: too few blocks for the device
    assert plan(64, 4000, 4096, False).splits == 2 and plan(13, 18944, 3584, False).splits == 2
