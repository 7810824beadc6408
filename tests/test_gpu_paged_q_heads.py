"""Attention over codes with more than 8 query heads a kv head, where a column of the products holds all groups of its head, in
every format."""
import numpy as np
import pytest

from paged_q import NP, PagesQ
from paged_q_bounds import attention_q_bounds
from serving import HALF
from test_gpu_paged_q import FORMATS, case, run_attention
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
ALL = FORMATS + [(64, 32, 8, 4), (64, 64, 8, 8), (128, 64, 8, 4), (128, 128, 8, 8)]


def check(pg, q):
    scale = float(np.float32(1 / np.sqrt(pg.D)))
    ref, tol = attention_q_bounds(pg, q, scale, HALF[pg.dtype])
    for a in range(0, pg.D, pg.group):  # the bound of each group's dims would tell them from zeros
        assert np.median(tol[..., a:a + pg.group]) < 0.5 * np.sqrt((ref[..., a:a + pg.group] ** 2).mean())
    got = run_attention(pg, q, scale=scale)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref) / tol).max()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", ALL)
@pytest.mark.parametrize("G", [9, 16, 20])
@pytest.mark.parametrize("lens", [[70, 300, 9], [70, 1300, 9]])
def test_many_heads_of_a_kv_head(gpu, dtype, D, group, kb, vb, G, lens):
    case("heads", dtype, D, group, kb, vb, G, lens)
    rng = np.random.default_rng(D + G + kb)
    pg = PagesQ(rng, lens, 16, 2, D, group, kb, vb, dtype)
    check(pg, rng.normal(0, 2, (3, 2 * G, D)).astype(NP[dtype]))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", [f for f in ALL if f[0] > f[1]])
@pytest.mark.parametrize("G", [2, 16])
@pytest.mark.parametrize("n", [200, 2500])
def test_nan_groups(gpu, dtype, D, group, kb, vb, G, n):
    """A NaN group of a value gives its dims NaN, whether a column has one group or all of them, one of a key its heads; all
    else stays as it is."""
    case("nan", dtype, D, group, kb, vb, G, n)
    rng = np.random.default_rng(D + G)
    pg = PagesQ(rng, [n, n, n], 16, 2, D, group, kb, vb, dtype)
    q = rng.normal(0, 2, (3, 2 * G, D)).astype(NP[dtype])
    clean = run_attention(pg, q)
    page, r = pg.where(0)
    pg.vs[page[n // 2], 1, r[n // 2], 1] = np.nan
    page, r = pg.where(1)
    pg.ks[page[n - 1], 0, r[n - 1], -1, 0] = np.nan
    pg.upload()
    got = run_attention(pg, q)
    nan = np.zeros(got.shape, bool)
    nan[0, G:, group:2 * group] = True
    nan[1, :G] = True
    np.testing.assert_array_equal(np.isnan(got), nan)
    np.testing.assert_array_equal(got[~nan], clean[~nan])
