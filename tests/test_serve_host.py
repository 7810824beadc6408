"""Arguments of the batched decode operators that are refused on the host, before any device use, and the host
packing of 4-bit weights."""
import ctypes

import numpy as np
import pytest

from vvllm_amd import capi

P = 0x1000  # never dereferenced: every call below ends on the host
F16, F32 = capi.F16, capi.F32
INVALID, NOT_INIT, UNSUPPORTED = 1, 5, 7


def cache(**kw):
    d = dict(k_pages=P, v_pages=P, page_table=P, num_pages=10, page_size=16, num_seqs=4, max_pages=3, num_kv_heads=2,
             head_dim=64, dtype=F16)
    return ctypes.byref(capi.PagedCache(**{**d, **kw}))


def append(c, q_out=P, q=P, k=P, v=P, seqs=P, pos=P, tokens=4, heads=14, rope=P, positions=100):
    return capi.status_of("vvh_rope_append_paged", c, q_out, q, k, v, seqs, pos, tokens, heads, rope, positions, None)


def attention(c, out=P, q=2 * P, lens=P, max_len=0, heads=14):
    return capi.status_of("vvh_attention_paged", c, out, q, lens, max_len, heads, 0.125, None)


@pytest.mark.parametrize("kw,status", [
    (dict(k_pages=None), INVALID), (dict(v_pages=None), INVALID), (dict(page_table=None), INVALID),
    (dict(num_pages=0), INVALID), (dict(page_size=0), INVALID), (dict(max_pages=0), INVALID),
    (dict(num_kv_heads=0), INVALID), (dict(head_dim=0), INVALID), (dict(head_dim=258), INVALID), (dict(dtype=2), INVALID),
    (dict(k_pages=P + 1), INVALID), (dict(dtype=F32, v_pages=P + 2), INVALID), (dict(page_table=P + 2), INVALID),
    (dict(num_pages=1 << 27, page_size=16), UNSUPPORTED), (dict(num_pages=1 << 40), UNSUPPORTED),
    (dict(page_size=(1 << 64) - 1), UNSUPPORTED), (dict(max_pages=(1 << 25) + 1), UNSUPPORTED),
    (dict(num_seqs=65536), UNSUPPORTED), (dict(num_kv_heads=65536), UNSUPPORTED)])
def test_bad_caches(kw, status):
    heads = 14 if kw.get("num_kv_heads") != 65536 else 65536
    assert append(cache(**kw), heads=heads) == status
    assert attention(cache(**kw), heads=heads) == status


def test_append_arguments():
    assert append(None) == INVALID
    for name in ("q_out", "q", "k", "v", "pos"):
        assert append(cache(), **{name: None}) == INVALID
        assert append(cache(), **{name: P + 1}) == INVALID
    assert append(cache(), seqs=None) == NOT_INIT
    assert append(cache(), seqs=None, tokens=5) == INVALID       # five tokens, four sequences
    assert append(cache(), seqs=P + 2) == INVALID
    assert append(cache(head_dim=63)) == INVALID                  # pairs of an odd head
    assert append(cache(), rope=None) == INVALID                  # queries without angles
    assert append(cache(), rope=P + 4) == INVALID
    assert append(cache(head_dim=63), rope=None, heads=0, q=None, q_out=None) == NOT_INIT
    assert append(cache(), tokens=1 << 31) == UNSUPPORTED
    assert append(cache(), heads=65536) == UNSUPPORTED
    assert append(cache(), tokens=0, q=None, k=None, v=None, pos=None) == 0
    assert append(cache()) == NOT_INIT


def test_attention_arguments():
    assert attention(None) == INVALID
    for name in ("out", "q", "lens"):
        assert attention(cache(), **{name: None}) == INVALID
        assert attention(cache(), **{name: P + 1}) == INVALID
    assert attention(cache(), out=2 * P) == INVALID               # out is q
    assert attention(cache(), heads=15) == INVALID                # two kv heads
    assert attention(cache(), heads=65536) == UNSUPPORTED
    assert attention(cache(), heads=0) == 0
    assert attention(cache(num_seqs=0), q=None) == 0
    assert attention(cache()) == NOT_INIT


def test_rope_table_arguments():
    st = capi.status_of
    assert st("vvh_rope_table", P, 10, 63, 1e4, None) == INVALID
    assert st("vvh_rope_table", P, 10, 258, 1e4, None) == INVALID
    assert st("vvh_rope_table", None, 10, 64, 1e4, None) == INVALID
    assert st("vvh_rope_table", P + 4, 10, 64, 1e4, None) == INVALID
    assert st("vvh_rope_table", P, 1 << 31, 64, 1e4, None) == UNSUPPORTED
    assert st("vvh_rope_table", None, 0, 64, 1e4, None) == 0
    assert st("vvh_rope_table", P, 10, 64, 1e4, None) == NOT_INIT


def linear(out=P, inp=2 * P, w=P, s=P, z=None, b=None, r=None, M=1, N=16, K=128, group=64, act=F16, outd=F16):
    return capi.status_of("vvh_linear_q4", out, inp, w, s, z, b, r, M, N, K, group, act, outd, None)


def test_linear_q4_arguments():
    for name in ("out", "inp", "w", "s"):
        assert linear(**{name: None}) == INVALID
    for kw in (dict(inp=P + 8), dict(w=P + 8), dict(s=P + 1), dict(b=P + 2), dict(r=P + 1), dict(out=P + 1),
               dict(outd=F32, out=P + 2), dict(act=2), dict(outd=-1), dict(group=16), dict(group=48), dict(group=0),
               dict(K=96), dict(K=160, group=128), dict(N=1 << 40, K=1 << 40)):
        assert linear(**kw) == INVALID, kw
    assert linear(N=1 << 31) == UNSUPPORTED
    assert linear(out=2 * P) == INVALID                           # out is inp
    assert linear(K=1 << 31) == UNSUPPORTED and linear(K=(1 << 24) + 64) == UNSUPPORTED
    assert linear(M=1 << 19, N=1 << 22, K=64) == UNSUPPORTED
    assert linear(M=1 << 21) == UNSUPPORTED
    assert linear(M=0, out=None) == 0 and linear(N=0, out=None) == 0
    assert linear() == NOT_INIT and linear(z=P + 1, b=P, r=P) == NOT_INIT
    assert linear(K=0, inp=None, w=None, s=None) == NOT_INIT


def rules(out=P, logits=P, rows=2, n=100, dtype=F32, spec=True, **kw):
    return capi.status_of("vvh_logits_rules", out, logits, ctypes.byref(capi.LogitsRules(**kw)) if spec else None, rows, n,
                          dtype, None)


def test_logits_rules_arguments():
    assert rules(spec=False) == INVALID
    assert rules(out=None) == INVALID and rules(logits=None) == INVALID
    assert rules(dtype=2) == INVALID
    assert rules(out=P + 2) == INVALID and rules(dtype=F16, logits=P + 1) == INVALID
    assert rules(tokens=P, token_stride=4) == INVALID             # without counts
    for name in ("repetition", "frequency", "presence"):
        assert rules(**{name: P}) == INVALID                      # without tokens
        assert rules(tokens=P, token_stride=4, token_counts=P, **{name: P + 2}) == INVALID
    assert rules(bias_offsets=P, bias_count=3, bias_ids=P) == INVALID
    assert rules(mask=P, mask_stride=3) == INVALID                # 100 logits take 4 words
    assert rules(n=1 << 31) == UNSUPPORTED
    assert rules(rows=65536) == UNSUPPORTED
    assert rules(token_stride=(1 << 30) + 1) == UNSUPPORTED
    assert rules(rows=0, out=None) == 0 and rules(n=0, out=None) == 0
    assert rules() == NOT_INIT and rules(mask=P, mask_stride=0) == NOT_INIT and rules(bias_offsets=P) == NOT_INIT


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_q4(group):
    rng = np.random.default_rng(group)
    w = rng.normal(0, 0.02, (5, 3 * group)).astype(np.float32)
    w[1, :group] = 0
    codes, scales = capi.quantize_q4(w, group)
    assert codes.shape == (5, 3 * group // 2) and codes.dtype == np.uint8
    assert scales.shape == (5, 3) and scales.dtype == np.float16
    c = np.stack([codes & 15, codes >> 4], -1).reshape(5, 3, group).astype(np.float64)
    back = (c - 8) * scales.astype(np.float64)[..., None]
    # half a step, and the scale's rounding at the far codes
    assert (np.abs(back.reshape(w.shape) - w) <= np.repeat(scales.astype(np.float64), group, 1) * (0.5 + 7 * 2.0 ** -10)).all()
    assert scales[1, 0] == 0 and (codes[1, :group // 2] == 0x88).all()
    with pytest.raises(ValueError):
        capi.quantize_q4(w, 48)
    with pytest.raises(ValueError):
        capi.quantize_q4(w[:, :-1], group)


def test_quantize_q4_extreme_weights():
    w = np.zeros((3, 32), np.float32)
    w[0, 3], w[1, 4], w[2, 5] = 1e30, 1e-12, -7e-6
    codes, scales = capi.quantize_q4(w, 32)
    assert scales[0, 0] == 65504 and codes[0, 1] >> 4 == 15   # saturates
    assert scales[1, 0] == 0 and (codes[1] == 0x88).all()     # below the smallest scale
    assert scales[2, 0] > 0 and codes[2, 2] >> 4 == 1         # -7 steps
