"""vvh_logits_rules in blocks of 512 and 1024 threads (spans of 4096 and 8192 logits), as large batches take them: the host
rule names the block, the rules are checked as in test_gpu_logits_rules.py."""
import numpy as np
import pytest

from test_gpu_logits_rules import NP, Case
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32


def threads(rows, n, cus=256):
    """As launch_logits_rules."""
    t = 1024
    while t > 256 and rows * -(-n // (8 * t)) < 2 * cus:
        t //= 2
    return t


WIDE = [(64, 151936, 1024), (256, 20001, 1024), (520, 8192, 1024), (520, 8191, 1024), (300, 5000, 512), (40, 65537, 512),
        (520, 7, 1024), (130, 16389, 512), (515, 8200, 1024)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows,n,block", WIDE)
def test_wide_blocks(gpu, dtype, rows, n, block):
    """History (past four tokens a thread), biases and masks at once, then in place: the same bits."""
    assert threads(rows, n) == block
    c = Case(rows, n, dtype, history=4 * block + 37, biases=min(40, n), mask="rows")
    plain = c.check()
    np.testing.assert_array_equal(c.run(out=c.d["logits"]), plain.astype(NP[dtype]))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows,n,block", [(300, 5003, 512), (256, 20001, 1024)])
@pytest.mark.parametrize("history,penalties,biases,mask", [(0, "", 0, None), (0, "", 30, None), (0, "", 0, "one"), (9000, "rfp", 0, None),
                                                           (3, "r", 0, "rows"), (100, "fp", 5, None)])
def test_each_rule_alone_in_wide_blocks(gpu, dtype, rows, n, block, history, penalties, biases, mask):
    assert threads(rows, n) == block
    c = Case(rows, n, dtype, history, penalties, biases, mask)
    plain = c.check()
    np.testing.assert_array_equal(c.run(out=c.d["logits"]), plain.astype(NP[dtype]))


def test_one_token_all_the_time(gpu):
    """Rows whose whole history, and every bias, is one token at a span's border."""
    rows, n = 520, 8200
    assert threads(rows, n) == 1024
    c = Case(rows, n, F32, history=4200, biases=50)
    c.tokens[:] = np.where(np.arange(rows)[:, None] % 2, 8191, 8192)
    c.ids[:] = 8192
    c.counts[:] = 4200
    c.prompts[:] = np.arange(rows) * 9
    c.upload()
    c.check()
