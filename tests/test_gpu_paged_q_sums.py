"""Attention over codes where a wave takes thousands of keys: what its sums keep.  Many sequences share the pages of a small
pool, each several times over, so that the softmax over a context is the one over the pool."""
import numpy as np
import pytest

from paged_q import NP, PagesQ, attention_q_ref
from serving import HALF
from test_gpu_paged_q import case, run_attention
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
FORMATS = [(64, 32, 4, 4), (64, 64, 8, 8), (64, 64, 8, 4), (128, 32, 4, 4), (128, 128, 8, 8), (96, 32, 8, 4)]


def many_of_one(pg, B, times):
    """B sequences of the pool's one context, `times` times over."""
    pg.table = np.tile(pg.table[0], (B, times))
    pg.lens = np.full(B, int(pg.lens[0]) * times, np.int32)
    pg.d_t, pg.d_n = (capi.DevBuf.from_array(a) for a in (pg.table, pg.lens))


@pytest.mark.parametrize("H", [8, 24, 80])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
@pytest.mark.parametrize("std", [0.0, 1.0])
def test_long_runs_of_fp16_are_bound_by_their_rounding(gpu, std, H, D, group, kb, vb):
    """64 contexts of 32768 keys, 8192 a wave.  Errors of sums in fp32 are independent of the output's rounding, whose norm is
    at least 2^-13 of the output's: 2^-17 of it (16 times the 2^-21 that fp32 rows have) make the whole 2^-9 larger at most."""
    case("long runs", std, H, D, group, kb, vb)
    rng = np.random.default_rng(D + kb + H)
    n = 2048
    pg = PagesQ(rng, [n], 64, 8, D, group, kb, vb, F16)
    q = rng.normal(0, std, (1, H, D)).astype(np.float16)
    scale = float(np.float32(1 / np.sqrt(D)))
    ref, _ = attention_q_ref(pg, q, scale, 0)
    many_of_one(pg, 64, 16)
    got = run_attention(pg, np.tile(q, (64, 1, 1)))
    own, best = (np.linalg.norm(y - ref) / np.linalg.norm(ref) for y in (got, np.tile(ref.astype(np.float16), (64, 1, 1))))
    own /= 8.0  # of 64 rows, the reference is one
    best /= 8.0
    case("errors", own, best)
    assert best >= 2.0 ** -13
    assert own <= (1 + 2.0 ** -9) * best


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("H", [8, 24])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
def test_values_that_cancel(gpu, dtype, H, D, group, kb, vb):
    """Equal weights, and values in pairs that add up to nearly nothing: what is left shows the sums' own errors.  A wave's
    8192 keys are added up in steps of at most 32, each rounded to 2^-24 of a partial sum: the codes' middles are half a step
    beside the groups', so that partial sums of pairs are at most half the largest step a key.  512 roundings (high and low
    parts) of at most 2^-25 of 8192 / 2 steps, at random: within 6 of their standard deviations sqrt(512 / 3)."""
    rng = np.random.default_rng(D + vb + H)
    n, top = 2048, 2 ** vb - 1
    pg = PagesQ(rng, [n], 64, 8, D, group, kb, vb, dtype)
    page, r = pg.where(0)
    s = (rng.random((n // 2, 8, D // group)) * 0.3 + 0.1).astype(np.float16).repeat(2, 0)
    pg.vs[page, :, r] = np.stack([s, (s * -(top / 2)).astype(np.float16)], -1)
    codes = rng.integers(0, 256, (n // 2, 8, D * vb // 8)).astype(np.uint8).repeat(2, 0)
    codes[1::2] = 255 - codes[1::2]  # each code's complement
    pg.vp[page, :, r] = codes
    pg.upload()
    q = np.zeros((1, H, D), NP[dtype])
    ref, _ = attention_q_ref(pg, q, 1.0, 0)
    many_of_one(pg, 64, 16)
    got = run_attention(pg, np.tile(q, (64, 1, 1)), scale=1.0)
    tol = HALF[dtype] * np.abs(ref) + 2.0 ** -25 + 6 * np.sqrt(512 / 3) * 2.0 ** -25 * 0.4 / 2
    off = np.abs(got - ref)
    case("cancel", dtype, H, D, group, kb, vb, off.max(), (off / tol).max())
    assert (off <= tol).all()
