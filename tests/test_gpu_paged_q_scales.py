"""Attention over codes whose groups' scales are far apart."""
import numpy as np
import pytest

from paged_q import NP, PagesQ
from test_gpu_paged_q import case
from test_gpu_paged_q_heads import check
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", [(128, 32, 4, 4), (128, 32, 8, 8), (96, 32, 8, 4), (64, 32, 8, 8), (128, 64, 8, 4)])
@pytest.mark.parametrize("G", [2, 7, 16])
@pytest.mark.parametrize("lens", [[60, 300], [1700, 900]])
@pytest.mark.parametrize("order", [1, -1, 0])
def test_groups_whose_scales_are_far_apart(gpu, dtype, D, group, kb, vb, G, lens, order):
    """Scales of a value's groups from fp16's largest down to 2^-20 of it, each 2^-10 of the one before, growing by 2^6 along the
    context, falling, or mixed: each group's dims are held by what its own values are, and 2^-37 of the largest scale."""
    case("apart", dtype, D, group, kb, vb, G, lens, order)
    rng = np.random.default_rng(D + G + vb)
    pg = PagesQ(rng, lens, 16, 2, D, group, kb, vb, dtype)
    ratio = 2.0 ** (-10 * (np.arange(D // group) % 3))
    for s, n in enumerate(lens):
        page, r = pg.where(s)
        e = np.linspace(-6, 0, n)
        e = e[::order] if order else rng.permutation(e)
        sc = (65504 * 2.0 ** e[:, None, None] * ratio * np.ones((1, 2, 1))).astype(np.float16)
        # values of at most fp16's range: codes 0 .. 2 around the minimum -scale
        pg.vs[page, :, r, :, 0], pg.vs[page, :, r, :, 1] = sc, -sc
        codes = rng.integers(0, 3, (n, 2, D)).astype(np.uint8)
        pg.vp[page, :, r] = codes if vb == 8 else codes[..., 0::2] | codes[..., 1::2] << 4
    pg.upload()
    check(pg, rng.normal(0, 2, (len(lens), 2 * G, D)).astype(NP[dtype]))
