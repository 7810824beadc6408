"""The paged cache of codes on the host: what its calls refuse before any device use, and the format's rows packed and
unpacked."""
import ctypes

import numpy as np
import pytest

from vvllm_amd import capi

P = 0x1000  # never dereferenced: every call below ends on the host
F16, F32 = capi.F16, capi.F32
INVALID, NOT_INIT, UNSUPPORTED = 1, 5, 7


def cache(**kw):
    d = dict(k_pages=P, v_pages=P, k_scales=P, v_scales=P, page_table=P, num_pages=10, page_size=16, num_seqs=4, max_pages=3,
             num_kv_heads=2, head_dim=64, group=32, k_bits=4, v_bits=4, dtype=F16)
    return ctypes.byref(capi.PagedCacheQ(**{**d, **kw}))


def append(c, q_out=P, q=P, k=P, v=P, seqs=P, pos=P, tokens=4, heads=14, rope=P, positions=100):
    return capi.status_of("vvh_rope_append_paged_q", c, q_out, q, k, v, seqs, pos, tokens, heads, rope, positions, None)


def read(c, k=P, v=2 * P, seqs=P, pos=P, tokens=4):
    return capi.status_of("vvh_read_paged_q", c, k, v, seqs, pos, tokens, None)


def attention(c, out=P, q=2 * P, lens=P, max_len=0, heads=14):
    return capi.status_of("vvh_attention_paged_q", c, out, q, lens, max_len, heads, 0.125, None)


@pytest.mark.parametrize("kw,status", [
    (dict(k_pages=None), INVALID), (dict(v_pages=None), INVALID), (dict(k_scales=None), INVALID),
    (dict(v_scales=None), INVALID), (dict(page_table=None), INVALID), (dict(num_pages=0), INVALID), (dict(page_size=0), INVALID),
    (dict(page_size=24), INVALID), (dict(page_size=8), INVALID), (dict(max_pages=0), INVALID), (dict(num_kv_heads=0), INVALID),
    (dict(head_dim=0), INVALID), (dict(head_dim=80), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED), (dict(group=0), INVALID),
    (dict(group=16), INVALID), (dict(group=128), INVALID), (dict(head_dim=96, group=64), INVALID), (dict(k_bits=2), INVALID),
    (dict(k_bits=0, v_bits=0), INVALID), (dict(v_bits=16), INVALID), (dict(v_bits=8), UNSUPPORTED), (dict(dtype=2), INVALID),
    (dict(k_pages=P + 8), INVALID), (dict(v_pages=P + 4), INVALID), (dict(k_scales=P + 4), INVALID),
    (dict(v_scales=P + 8), INVALID), (dict(page_table=P + 2), INVALID),
    (dict(num_pages=1 << 27, page_size=16), UNSUPPORTED), (dict(num_pages=1 << 40), UNSUPPORTED),
    (dict(page_size=(1 << 64) - 16), UNSUPPORTED), (dict(max_pages=(1 << 25) + 1), UNSUPPORTED),
    (dict(num_seqs=65536), UNSUPPORTED), (dict(num_kv_heads=65536), UNSUPPORTED)])
def test_bad_caches(kw, status):
    heads = 14 if kw.get("num_kv_heads") != 65536 else 65536
    assert append(cache(**kw), heads=heads) == status
    assert read(cache(**kw)) == status
    assert attention(cache(**kw), heads=heads) == status


@pytest.mark.parametrize("D,group,kb,vb", [(64, 32, 4, 4), (64, 64, 8, 4), (96, 32, 8, 8), (128, 32, 4, 4), (128, 64, 8, 8),
                                           (128, 128, 8, 4)])
def test_every_format_reaches_the_device(D, group, kb, vb):
    c = cache(head_dim=D, group=group, k_bits=kb, v_bits=vb)
    assert append(c) == read(c) == attention(c) == NOT_INIT


def test_append_arguments():
    assert append(None) == INVALID
    for name in ("q_out", "q", "k", "v", "pos"):
        assert append(cache(), **{name: None}) == INVALID
        assert append(cache(), **{name: P + 2}) == INVALID
    assert append(cache(), seqs=None) == NOT_INIT
    assert append(cache(), seqs=None, tokens=5) == INVALID       # five tokens, four sequences
    assert append(cache(), seqs=P + 2) == INVALID
    assert append(cache(), rope=None) == INVALID                  # queries without angles
    assert append(cache(), rope=P + 8) == INVALID
    assert append(cache(), rope=None, heads=0, q=None, q_out=None) == NOT_INIT
    assert append(cache(), tokens=1 << 31) == UNSUPPORTED
    assert append(cache(), heads=65536) == UNSUPPORTED
    assert append(cache(), tokens=0, q=None, k=None, v=None, pos=None) == 0


def test_read_arguments():
    assert read(None) == INVALID
    assert read(cache(), k=None, v=None) == INVALID
    assert read(cache(), k=None) == NOT_INIT and read(cache(), v=None) == NOT_INIT
    assert read(cache(), k=2 * P) == INVALID                      # one array for both
    assert read(cache(), pos=None) == INVALID
    for name in ("k", "v", "pos", "seqs"):
        assert read(cache(), **{name: P + 2}) == INVALID
    assert read(cache(), seqs=None) == NOT_INIT
    assert read(cache(), seqs=None, tokens=5) == INVALID
    assert read(cache(), tokens=1 << 31) == UNSUPPORTED
    assert read(cache(), tokens=0, k=None, v=None, pos=None) == 0


def test_attention_arguments():
    assert attention(None) == INVALID
    for name in ("out", "q", "lens"):
        assert attention(cache(), **{name: None}) == INVALID
        assert attention(cache(), **{name: P + 2}) == INVALID
    assert attention(cache(), out=2 * P) == INVALID               # out is q
    assert attention(cache(), heads=15) == INVALID                # two kv heads
    assert attention(cache(), heads=65536) == UNSUPPORTED
    assert attention(cache(num_seqs=1025), heads=32768) == UNSUPPORTED and attention(cache(num_seqs=1024), heads=32768) == NOT_INIT
    assert attention(cache(), heads=0) == 0
    assert attention(cache(num_seqs=0), q=None) == 0


# ---- the format ----------------------------------------------------------------------------
@pytest.mark.parametrize("keys", [False, True])
@pytest.mark.parametrize("bits,group,D", [(4, 32, 64), (4, 32, 96), (8, 32, 96), (4, 128, 128), (8, 64, 128)])
def test_rows_come_back_to_half_a_step(keys, bits, group, D):
    rng = np.random.default_rng(D + bits)
    x = (rng.normal(0, 2, (7, 3, D)) + rng.normal(0, 5, (3, D))).astype(np.float32)
    held, sm = capi.pack_paged_q(x, bits, group, keys)
    assert held.shape == (7, 3, D * bits // 8) and held.dtype == np.uint8
    assert sm.shape == (7, 3, D // group, 2) and sm.dtype == np.float16
    y = capi.unpack_paged_q(held, sm, bits, keys)
    s, m = (np.repeat(sm[..., i].astype(np.float64), group, -1) for i in (0, 1))
    # half a step; at the ends what the roundings leave: m's half step, and s's half step times the codes
    ends = 2.0 ** -11 * np.abs(m) + 2.0 ** -11 * s * (2 ** bits - 1)
    assert (np.abs(y - x) <= s / 2 + ends).all()
    # packing what the rows stand for gives values within half a step of them again
    assert (np.abs(capi.unpack_paged_q(*capi.pack_paged_q(y, bits, group, keys), bits, keys) - y) <= s / 2 + 2 * ends).all()


def test_codes_are_where_the_header_says():
    D = 96
    x = np.zeros((1, D), np.float32)
    for d in range(D):
        x[:] = 0
        x[0, d] = 15
        for bits in (4, 8):
            top = 2 ** bits - 1
            held, sm = capi.pack_paged_q(x, bits, 32, False)
            place = d if bits == 8 else d // 2
            assert held[0, place] == (top if bits == 8 else top << d % 2 * 4) and np.count_nonzero(held) == 1
            assert sm[0, d // 32, 1] == 0 and sm[0, d // 32, 0] == np.float16(15 / top)
            held, _ = capi.pack_paged_q(x, bits, 32, True)
            j, i = d // 32, d % 32 // 8
            at = (i * (D // 32) + j) * 8 + d % 8
            assert held[0, at if bits == 8 else at // 2] == (top if bits == 8 else top << at % 2 * 4) and np.count_nonzero(held) == 1


def test_special_groups():
    x = np.zeros((6, 64), np.float32)
    x[1] = 0.1                      # a constant: the nearest fp16, s the rest
    x[2, 5] = np.nan
    x[3, 40] = np.inf
    x[4, :32] = np.linspace(-1e6, 1e6, 32)
    x[5, :32] = np.linspace(0, 7.5, 32) // 0.5 * 0.5
    x[5, 3], x[5, 4] = 1.25, 1.75   # halfway between levels of 0.5: the even codes, 2 and 4
    held, sm = capi.pack_paged_q(x, 4, 32, False)
    y = capi.unpack_paged_q(held, sm, 4, False)
    assert (y[0] == 0).all() and (sm[0] == 0).all()
    assert (np.abs(y[1] - np.float32(0.1)) <= 2.0 ** -24).all() or (np.abs(y[1] - 0.1) <= 0.1 * 2.0 ** -11).all()
    assert np.isnan(y[2, :32]).all() and (y[2, 32:] == 0).all()
    assert np.isnan(y[3, 32:]).all() and (y[3, :32] == 0).all()
    assert sm[4, 0, 1] == -65504 and sm[4, 0, 0] == 65504 and np.isfinite(y[4]).all()
    assert y[5, 3] == 1.0 and y[5, 4] == 2.0
