"""Attention over codes with scores of any size: where a score's last bit is a factor, past fp32's range, and with the same
result however a row is split."""
import numpy as np
import pytest

from paged_q import NP, PagesQ
from paged_q_bounds import attention_q_bounds, plant
from serving import HALF
from test_gpu_paged_q import case, read_rows, run_attention
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
FORMATS = [(64, 32, 4, 4), (96, 32, 8, 4), (128, 64, 8, 8), (128, 128, 4, 4)]
LENS = [[1], [40], [700], [3000], [9, 3000, 0, 64, 700, 1]]  # a wave, several, split, and together


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("scale", [1e38, 3.4e38, 1e30, 1e10, -1e38, -3.4e38, -1e20])
def test_the_best_key_whatever_the_scale(gpu, dtype, D, group, kb, vb, lens, scale):
    """One key leads by a score of at least a tenth of itself, far more than its rounding: it is all of the row."""
    case("best key", dtype, D, group, kb, vb, lens, scale)
    rng = np.random.default_rng(D + len(lens))
    pg = PagesQ(rng, lens, 16, 2, D, group, kb, vb, dtype)
    best = [int(rng.integers(0, max(n, 1))) for n in lens]
    for s, n in enumerate(lens):
        if n:
            plant(pg, s, best[s], np.sign(scale), 1.0)
    pg.upload()
    q = rng.uniform(1, 2, (len(lens), 6, D)).astype(NP[dtype])
    got = run_attention(pg, q, scale=scale)
    for s, n in enumerate(lens):
        if not n:
            assert (got[s] == 0).all()
            continue
        _, v, _, _ = pg.rows(s)
        want = np.repeat(v[best[s]], 3, 0)
        size = np.abs(v[best[s]]).max()  # high and low parts of a weight, and the groups' middles
        assert (np.abs(got[s] - want) <= HALF[dtype] * np.abs(want) + 2.0 ** -20 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [0.125, 2.0 ** 12, 2.0 ** 18, 1e30, 3e38, -2.0 ** 18, -3e38, 1e-40])
@pytest.mark.parametrize("lens", [[700], [3000], [20, 5000, 0, 1000]])
def test_equal_scores_of_any_size(gpu, dtype, lens, scale):
    """All keys alike: the plain average, also where values' scales grow along the context (parts whose weights are times other
    powers of two) and scores leave fp32."""
    case("equal", dtype, lens, scale)
    rng = np.random.default_rng(40)
    pg = PagesQ(rng, lens, 16, 2, 64, 32, 4, 4, dtype)
    for s, n in enumerate(lens):
        page, r = pg.where(s)
        pg.kp[page, :, r] = rng.integers(0, 256, (1, 2, 32))
        pg.ks[page, :, r] = [0.25, -1.0]
        if n:
            sc = (2.0 ** np.linspace(-18, 2, n)[:, None, None]).astype(np.float16)
            pg.vs[page, :, r, :, 0], pg.vs[page, :, r, :, 1] = sc, -7 * sc
    pg.upload()
    q = rng.normal(0, 100, (len(lens), 6, 64)).astype(NP[dtype])
    got = run_attention(pg, q, scale=scale)
    same, tol = attention_q_bounds(pg, np.zeros_like(q), 1.0, HALF[dtype])
    assert (np.abs(got - same) <= tol).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS)
@pytest.mark.parametrize("size", [1.0, 30.0, 1000.0, 3e4, 3e6, 3e9])
def test_large_scores_against_the_weights(gpu, dtype, D, group, kb, vb, size):
    """Queries of any size, whose scores reach 2^40: held by a bound that only keys with a weight can widen."""
    case("large", dtype, D, group, kb, vb, size)
    if dtype == F16 and size > 3e3:
        scale, std = size / 3e3, 3e3
    else:
        scale, std = 1 / np.sqrt(D), size
    scale = float(np.float32(scale))
    rng = np.random.default_rng(41)
    lens = [1, 40, 300, 700, 3000]
    pg = PagesQ(rng, lens, 16, 2, D, group, kb, vb, dtype)
    q = rng.normal(0, std, (len(lens), 6, D)).astype(NP[dtype])
    ref, tol = attention_q_bounds(pg, q, scale, HALF[dtype])
    # the bound says something: most rows' is far below what their values are spread over
    tight = [(tol[s] < 0.02 * pg.rows(s)[1].std()).all(-1).mean() for s in range(1, len(lens))]
    case("rows with a tight bound", tight)
    assert np.mean(tight) >= 0.5
    got = run_attention(pg, q, scale=scale)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref) / tol).max()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("lens", [[30, 900, 1], [3000, 0, 1500]])
def test_leading_keys_of_large_queries(gpu, dtype, lens, size):
    """A key that leads, in rows of large scores with others of growing size before it: its value, and no NaN."""
    rng = np.random.default_rng(42)
    pg = PagesQ(rng, lens, 16, 2, 128, 32, 8, 4, dtype)
    for s, n in enumerate(lens):
        if n:
            plant(pg, s, n - 1 if s % 2 == 0 else 0, 1, 1.9)
    pg.upload()
    std = size if dtype == F32 else 1e4
    q = (rng.uniform(1, 2, (3, 6, 128)) * std).astype(NP[dtype])
    got = run_attention(pg, q, scale=size / std)
    for s, n in enumerate(lens):
        want = np.repeat(pg.rows(s)[1][n - 1 if s % 2 == 0 else 0], 3, 0) if n else np.zeros((6, 128))
        assert (np.abs(got[s] - want) <= HALF[dtype] * np.abs(want) + 2.0 ** -20 * np.abs(want).max() + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [np.nan, np.inf, -np.inf, 1e38])
@pytest.mark.parametrize("n", [40, 3000])
def test_rows_whose_pages_are_all_gone(gpu, dtype, scale, n):
    """They have no position: zeros, whatever the scale."""
    rng = np.random.default_rng(43)
    pg = PagesQ(rng, [n, n], 16, 2, 64, 32, 4, 4, dtype)
    pg.table[0] = -1
    pg.upload()
    got = run_attention(pg, np.ones((2, 6, 64), NP[dtype]), scale=scale)
    assert (got[0] == 0).all()
    assert np.isnan(got[1]).all() if not np.isfinite(scale) else np.isfinite(got[1]).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS + [(64, 64, 8, 8), (128, 32, 4, 4)])
@pytest.mark.parametrize("G", [1, 3, 16])
@pytest.mark.parametrize("lens", [[1], [1] * 70, [1, 2000, 1, 0, 1]])
def test_rows_of_one_key_are_the_row_read_back(gpu, dtype, D, group, kb, vb, G, lens):
    """Its weight is 1, and m + s c fits fp32 where m and s come from values of one size: the same bits as vvh_read_paged_q."""
    case("one key", dtype, D, group, kb, vb, G, lens)
    rng = np.random.default_rng(44)
    pg = PagesQ(rng, lens, 16, 2, D, group, kb, vb, dtype)
    q = rng.normal(0, 2, (len(lens), 2 * G, D)).astype(NP[dtype])
    got = run_attention(pg, q)
    one = [s for s, n in enumerate(lens) if n == 1]
    _, v = read_rows(pg, one, [0] * len(one))
    np.testing.assert_array_equal(got[one], v.astype(np.float64).repeat(G, 1))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,group,kb,vb", FORMATS + [(64, 64, 8, 8), (128, 32, 8, 8)])
@pytest.mark.parametrize("G", [2, 16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_queries_that_are_not_finite(gpu, dtype, D, group, kb, vb, G, bad):
    """Their rows are NaN, in whichever group the value is, those without a position zeros, all others as they were."""
    case("queries", dtype, D, group, kb, vb, G, bad)
    rng = np.random.default_rng(45)
    pg = PagesQ(rng, [1, 70, 2000, 0], 16, 2, D, group, kb, vb, dtype)
    q = rng.normal(0, 2, (4, 2 * G, D)).astype(NP[dtype])
    clean = run_attention(pg, q)
    where = [(s, h, d) for s in range(4) for h, d in ((0, 0), (G, D - 1), (2 * G - 1, D // 2))]
    for s, h, d in where:
        q[s, h, d] = bad
    got = run_attention(pg, q)
    rows = np.zeros(got.shape[:2], bool)
    for s, h, _ in where:
        rows[s, h] = s < 3
    assert np.isnan(got[rows]).all()
    np.testing.assert_array_equal(got[~rows], clean[~rows])
