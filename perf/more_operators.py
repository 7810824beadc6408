"""Measured cases of the operators of a paged key-value cache held in 8 and 4 bits: the append that rotates and quantises
(vvh_rope_append_paged_q), rows read back as values (vvh_read_paged_q) and attention of one new token per sequence over the
codes (vvh_attention_paged_q).

With ``own`` true a pass makes the library's calls (include/vvllm_hip.h); with ``own`` false it computes the same in
elementary torch operations in 32 bits, rounded once (keys' rotation and codes in 64: a code is a choice between two
neighbours).  ``exact`` is the definition in 64 bits.

A row's group of dims holds its minimum m and scale s in fp16, and codes c: m = fp16(min x), s = fp16(fp32((max x - m) /
(2^bits - 1))), c the nearest whole number to (x - m) / s, the even one of two, within 0 .. 2^bits - 1; it stands for m + s c.

Sizes come from Qwen2.5-0.5B (14 heads, 2 kv heads of 64) and the 1.5B shapes (12 heads, 2 kv heads of 128), or are
generic.
"""
from __future__ import annotations

import ctypes
import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
THETA = 1e6


def listed() -> list[dict]:
    return [
        # one new token of each of eight sequences, read back: the smallest append, where latency counts
        dict(name="append_tokens_k4v4_f16", op="append", tokens=8, prompts=0, heads=14, kv_heads=2, head_dim=64,
             group=32, k_bits=4, v_bits=4, page=16, span=1000, act="f16", shape=1),
        # one new token of each of a large batch, fp32, keys in more bits than values
        dict(name="append_batch_k8v4_f32", op="append", tokens=96, prompts=0, heads=12, kv_heads=2, head_dim=128,
             group=64, k_bits=8, v_bits=4, page=64, span=5000, act="f32", shape=2),
        # five prompts of different lengths that join a running batch together
        dict(name="append_prompts_k4v4_f16", op="append", tokens=4001, prompts=5, heads=32, kv_heads=8, head_dim=128,
             group=32, k_bits=4, v_bits=4, page=16, span=3000, act="f16", shape=3),
        # two prompts in fp32, heads of 96, both in 8 bits
        dict(name="append_prompts_k8v8_f32", op="append", tokens=777, prompts=2, heads=16, kv_heads=4, head_dim=96,
             group=32, k_bits=8, v_bits=8, page=48, span=1000, act="f32", shape=4),
        # one chat's context for the attention of its next prompt
        dict(name="read_chat_k4v4_f16", op="read", batch=1, heads=14, kv_heads=2, head_dim=64, group=32, k_bits=4, v_bits=4,
             page=16, span=1500, spread="full", gone=0.0, act="f16", shape=5),
        # long contexts in fp32
        dict(name="read_long_k8v8_f32", op="read", batch=3, heads=12, kv_heads=2, head_dim=128, group=128, k_bits=8,
             v_bits=8, page=128, span=20001, spread="even", gone=0.0, act="f32", shape=6),
        # a batch's contexts, many kv heads
        dict(name="read_batch_k4v4_f16", op="read", batch=40, heads=32, kv_heads=8, head_dim=128, group=64, k_bits=4,
             v_bits=4, page=32, span=2000, spread="log", gone=0.0, act="f16", shape=7),
        # a few chats with short contexts: latency
        dict(name="attention_chats_k4v4_f16", op="attention", batch=4, heads=14, kv_heads=2, head_dim=64, group=32, k_bits=4,
             v_bits=4, page=16, span=512, spread="even", gone=0.0, act="f16", shape=8),
        # a full server: ragged contexts from one token to 8192, some rows of the batch empty, the finest groups
        dict(name="attention_ragged_k4v4_f16", op="attention", batch=96, heads=32, kv_heads=8, head_dim=128, group=32,
             k_bits=4, v_bits=4, page=64, span=8192, spread="log", gone=0.0, act="f16", shape=9),
        # three long contexts in fp32, whose oldest pages were given back
        dict(name="attention_long_k8v4_f32", op="attention", batch=3, heads=12, kv_heads=2, head_dim=128, group=128, k_bits=8,
             v_bits=4, page=128, span=30001, spread="even", gone=0.1, act="f32", shape=10),
        # contexts of one length, a query head for each kv head, both in 8 bits
        dict(name="attention_full_k8v8_f16", op="attention", batch=32, heads=8, kv_heads=8, head_dim=128, group=64, k_bits=8,
             v_bits=8, page=32, span=4096, spread="full", gone=0.0, act="f16", shape=11),
        # heads of 96, a small batch
        dict(name="attention_96_k4v4_f32", op="attention", batch=16, heads=12, kv_heads=2, head_dim=96, group=32, k_bits=4,
             v_bits=4, page=16, span=4000, spread="even", gone=0.0, act="f32", shape=12),
    ]


# ---- drawn cases ------------------------------------------------------------
def _log(rng, lo: int, hi: int) -> int:
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng) -> dict:
    op = rng.choice(["append", "append", "read", "attention", "attention", "attention"])
    kv = rng.choice([1, 2, 4, 8])
    D = rng.choice([64, 64, 96, 128, 128])
    k_bits, v_bits = rng.choice([(4, 4), (4, 4), (8, 4), (8, 8)])
    c = dict(op=op, heads=kv * rng.choice([1, 2, 4, 5, 6, 7, 8, 16, 20]), kv_heads=kv, head_dim=D,
             group=rng.choice([g for g in (32, 64, 128) if D % g == 0]), k_bits=k_bits, v_bits=v_bits,
             page=rng.choice([16, 16, 32, 48, 64, 128, 256]), act=rng.choice(["f16", "f16", "f32"]),
             shape=rng.randrange(1 << 20))
    if op == "append":
        c["prompts"] = rng.choice([0, rng.randint(1, 8)])
        c["tokens"] = _log(rng, 8 * c["prompts"], 4000) if c["prompts"] else _log(rng, 1, 256)
        c["span"] = _log(rng, 16, 5000)
    elif op == "read":
        c.update(batch=_log(rng, 1, 40), span=_log(rng, 1, 20000), spread=rng.choice(["even", "log", "full"]), gone=0.0)
    else:
        c.update(batch=_log(rng, 1, 96), span=_log(rng, 1, 30000), spread=rng.choice(["even", "log", "full"]),
                 gone=rng.choice([0.0, 0.0, 0.1]))
    return c


def draw(rng) -> dict:
    most = {c["op"]: max(work(x)["bytes"] for x in listed() if x["op"] == c["op"]) for c in listed()}
    while True:
        c = _draw(rng)
        # the plain attention pads every context to the longest
        if c["op"] == "attention" and c["batch"] * c["span"] * max(c["kv_heads"] * c["head_dim"], 4 * c["heads"]) > 9e8:
            continue
        if work(c)["bytes"] <= most[c["op"]]:
            return c


# ---- what a case's shape number stands for -----------------------------------
def _append_shape(c):
    """(sequence, position) of every token: one new token per sequence, or whole prompts."""
    rng = random.Random(c["shape"])
    if not c["prompts"]:
        return [(s, rng.randrange(c["span"])) for s in range(c["tokens"])]
    cuts = sorted(rng.sample(range(1, c["tokens"]), c["prompts"] - 1))
    out = []
    for s, (a, b) in enumerate(zip([0] + cuts, cuts + [c["tokens"]])):
        past = rng.choice([0, rng.randrange(c["span"])])
        out += [(s, past + i) for i in range(b - a)]
    return out


def _lengths(c):
    """Context length of every row of the batch."""
    rng = random.Random(c["shape"])
    if c["spread"] == "full":
        return [c["span"]] * c["batch"]
    if c["spread"] == "even":
        out = [rng.randint((c["span"] + 1) // 2, c["span"]) for _ in range(c["batch"])]
    else:  # from empty rows (the padding of a captured batch) and single tokens to the longest
        out = [rng.choice([0, 1, c["span"]]) if rng.random() < 0.1 else _log(rng, 1, c["span"]) for _ in range(c["batch"])]
    out[rng.randrange(c["batch"])] = c["span"]
    return out


def _first_page(c, length):
    """Pages of a sequence that were given back: the oldest ones, all but the last page at most."""
    pages = -(-length // c["page"])
    return min(int(c["gone"] * pages), max(0, pages - 1))


def work(case) -> dict:
    c, e = case, 4 if case["act"] == "f32" else 2
    q, kv = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    held = kv * (c["k_bits"] + c["v_bits"]) // 8 + 8 * kv // c["group"]  # a position's codes, scales and minima
    if c["op"] == "append":
        t = c["tokens"]
        return {"bytes": t * (2 * q * e + 4 * kv * e + held + 4 * c["head_dim"]), "flops": t * (3 * q + 20 * kv)}
    keys = sum(n - _first_page(c, n) * c["page"] for n in _lengths(c))
    if c["op"] == "read":
        return {"bytes": keys * (held + 2 * kv * e + 8), "flops": 4 * keys * kv}
    return {"bytes": keys * held + 2 * c["batch"] * q * e, "flops": 4 * keys * q}


# ---- inputs -------------------------------------------------------------------
def _rand(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _angles(positions, head_dim):
    """cos and sin of every rotation pair at every position, [positions, head_dim / 2, 2]."""
    freq = THETA ** (-torch.arange(0, head_dim, 2, device=DEV, dtype=torch.float64) / head_dim)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * freq[None, :]
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _table(g, counts, width):
    """A page table with counts[s] pages of row s taken from a shuffled pool, and the pool's size."""
    need = sum(counts)
    pool = torch.randperm(need + 3, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
    n = torch.tensor(counts, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < n[:, None]] = pool[:need]
    return table, need + 3


def _codes(g, shape, bits):
    """Bytes whose codes are those of rows of normal values: the middle ones more often than the ends."""
    at = torch.special.ndtri((torch.arange(256, device=DEV, dtype=torch.float64) + 0.5) / 256)  # 256 quantiles
    top = 2 ** bits - 1
    level = (top / 2 * (1 + at / 2.1)).round().clamp(0, top).to(torch.uint8)
    if bits == 8:
        return level[torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8).int()]
    both = (level[:, None] | level[None, :] << 4).flatten()
    return both[torch.randint(0, 65536, shape, generator=g, device=DEV, dtype=torch.int32)]


def _scales(g, shape, bits):
    """{scale, minimum} of groups of normal values, [..., 2] fp16."""
    s = (torch.rand(shape, generator=g, device=DEV) * 0.4 + 0.8) * (4.2 / (2 ** bits - 1))
    m = -s * (2 ** bits - 1) * (0.5 + 0.1 * torch.randn(shape, generator=g, device=DEV))
    return torch.stack([s, m], -1).half()


def prepare(case, seed):
    c, g = case, _rand(seed)
    dt = torch.float16 if c["act"] == "f16" else torch.float32
    H, KVH, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    st = SimpleNamespace(case=c, dt=dt, calls=None)
    if c["op"] == "append":
        where = _append_shape(c)
        last = [0] * (1 + max(s for s, _ in where))
        for s, p in where:
            last[s] = max(last[s], p)
        counts = [p // P + 1 for p in last]
        st.angles = _angles(max(last) + 1, D)
        st.q = _normal(g, (c["tokens"], H, D), dtype=dt)
        # keys with some channels far from zero, as projections with a bias give them
        st.k = (_normal(g, (c["tokens"], KVH, D)) + _normal(g, (KVH, D), 2.0)).to(dt)
        st.v = _normal(g, (c["tokens"], KVH, D), dtype=dt)
        st.out = torch.empty_like(st.q)
    else:
        lens = _lengths(c)
        counts = [-(-n // P) for n in lens]
    if c["op"] == "read":
        where = [(s, p) for s, n in enumerate(lens) for p in range(n)]
    if c["op"] != "attention":
        st.seqs, st.positions = _ints([s for s, _ in where]), _ints([p for _, p in where])
        st.k_out, st.v_out = (torch.empty((len(where), KVH, D), dtype=dt, device=DEV) for _ in range(2))
    else:
        st.lens, st.longest, st.scale = _ints(lens), max(lens), 1.0 / math.sqrt(D)
        # scores of a few units, so that a query weighs some positions above others
        st.q = _normal(g, (c["batch"], H, D), 2.0, dt)
        st.out = torch.empty_like(st.q)
    width = max(1, max(counts))
    st.table, st.pool = _table(g, counts, width)
    if c["op"] == "attention":
        first = _ints([_first_page(c, n) for n in lens])
        st.table[torch.arange(width, device=DEV)[None, :] < first[:, None]] = -1
    rows = (st.pool, KVH, P)
    st.kp, st.vp = (_codes(g, rows + (D * b // 8,), b) for b in (c["k_bits"], c["v_bits"]))
    st.ks, st.vs = (_scales(g, rows + (D // c["group"],), b) for b in (c["k_bits"], c["v_bits"]))
    return st


# ---- the plain forms ------------------------------------------------------------
def _rotate(x, cs):
    """Split-half rotation of x [T, H, D] with cs [T, D / 2, 2]."""
    h = x.shape[-1] // 2
    x0, x1, co, si = x[..., :h], x[..., h:], cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([x0 * co - x1 * si, x1 * co + x0 * si], -1)


def _unit_order(x, keys, back=False):
    """Codes [..., D] in the order of a page row: keys' units of 8 dims, (32-dim step, unit) turned to (unit, step)."""
    if not keys:
        return x
    steps = x.shape[-1] // 32
    shape = (4, steps, 8) if back else (steps, 4, 8)
    return x.reshape(x.shape[:-1] + shape).transpose(-3, -2).reshape(x.shape)


def _pack(codes, bits, keys):
    x = _unit_order(codes, keys)
    return x if bits == 8 else x[..., 0::2] | x[..., 1::2] << 4


def _unpack(held, bits, keys):
    x = held if bits == 8 else torch.stack([held & 15, held >> 4], -1).flatten(-2)
    return _unit_order(x, keys, back=True)


def _quantise(x, bits, group, keys):
    """Page rows and {scale, minimum} of x [T, KVH, D] (fp32)."""
    top = 2 ** bits - 1
    g = x.unflatten(-1, (-1, group)).double()
    m = g.amin(-1).float().half()
    s = ((g.amax(-1) - m.double()) / top).float().half()
    level = (g - m.double()[..., None]) / torch.where(s == 0, 1.0, s.double())[..., None]
    c = torch.where(s[..., None] == 0, 0.0, level).round().clamp(0, top).to(torch.uint8)
    return _pack(c.flatten(-2), bits, keys), torch.stack([s, m], -1)


def _values(held, scales, bits, group, keys):
    """What page rows [..., bytes] with scales [..., groups, 2] stand for, in 32 bits."""
    c = _unpack(held, bits, keys).float().unflatten(-1, (-1, group))
    s = scales.float()
    return (s[..., 1:] + s[..., :1] * c).flatten(-2)


def _slots(st):
    p, P = st.positions.long(), st.case["page"]
    return st.table[st.seqs.long(), p // P].long(), p % P


def _plain_append(st):
    c = st.case
    cs = st.angles[st.positions.long()]
    page, row = _slots(st)
    k = _rotate(st.k.double(), cs.double()).float()
    st.kp[page, :, row], st.ks[page, :, row] = _quantise(k, c["k_bits"], c["group"], True)
    st.vp[page, :, row], st.vs[page, :, row] = _quantise(st.v.float(), c["v_bits"], c["group"], False)
    return [_rotate(st.q.float(), cs).to(st.dt)] + _plain_read(st)


def _plain_read(st):
    c = st.case
    page, row = _slots(st)
    return [_values(st.kp[page, :, row], st.ks[page, :, row], c["k_bits"], c["group"], True).to(st.dt),
            _values(st.vp[page, :, row], st.vs[page, :, row], c["v_bits"], c["group"], False).to(st.dt)]


def _plain_attention(st):
    """All contexts padded to the longest; keys past a context's end and on pages that are gone weigh nothing."""
    c = st.case
    B, H, KVH, D, P = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    width = st.table.shape[1]
    at = torch.arange(width * P, device=DEV)
    live = (at[None, :] < st.lens[:, None]) & (st.table >= 0).repeat_interleave(P, dim=1)
    page = st.table.clamp(min=0).long()

    def rows(held, scales, bits, keys):  # [B, KVH, width * P, D]
        x = _values(held[page], scales[page], bits, c["group"], keys)
        return x.transpose(1, 2).reshape(B, KVH, width * P, D)

    k = rows(st.kp, st.ks, c["k_bits"], True).transpose(2, 3).contiguous()
    s = torch.matmul(st.q.float().reshape(B, KVH, H // KVH, D), k) * st.scale
    del k
    s = s.masked_fill(~live[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    return torch.matmul(w, rows(st.vp, st.vs, c["v_bits"], False).contiguous()).reshape(B, H, D).to(st.dt)


# ---- the library's calls ----------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _calls(st):
    """The arguments of a state's calls, which a program keeps next to its buffers."""
    from vvllm_amd import capi

    capi.init(torch.cuda.current_device())
    c = st.case
    st.call = capi.call
    st.keep = capi.PagedCacheQ(
        k_pages=_p(st.kp), v_pages=_p(st.vp), k_scales=_p(st.ks), v_scales=_p(st.vs), page_table=_p(st.table), num_pages=st.pool,
        page_size=c["page"], num_seqs=st.table.shape[0], max_pages=st.table.shape[1], num_kv_heads=c["kv_heads"],
        head_dim=c["head_dim"], group=c["group"], k_bits=c["k_bits"], v_bits=c["v_bits"],
        dtype=capi.F16 if c["act"] == "f16" else capi.F32)
    cache = ctypes.byref(st.keep)
    if c["op"] == "attention":
        return [("vvh_attention_paged_q", cache, _p(st.out), _p(st.q), _p(st.lens), st.longest, c["heads"], st.scale)]
    read = ("vvh_read_paged_q", cache, _p(st.k_out), _p(st.v_out), _p(st.seqs), _p(st.positions), len(st.positions))
    if c["op"] == "read":
        return [read]
    return [("vvh_rope_append_paged_q", cache, _p(st.out), _p(st.q), _p(st.k), _p(st.v), _p(st.seqs), _p(st.positions),
             c["tokens"], c["heads"], _p(st.angles), st.angles.shape[0]), read]


def run(state):
    st, op = state, state.case["op"]
    if own:
        if st.calls is None:
            st.calls = _calls(st)
        stream = torch.cuda.current_stream().cuda_stream
        st.call(*st.calls[0], stream)
        if op == "append":
            st.call(*st.calls[1], stream)
        return st.out if op == "attention" else [st.out, st.k_out, st.v_out] if op == "append" else [st.k_out, st.v_out]
    return dict(append=_plain_append, read=_plain_read, attention=_plain_attention)[op](st)


# ---- the definitions in 64 bits, written apart ---------------------------------------
def _code_of(held, bits, keys, D):
    """Code of every dim: [..., D], dim by dim from the bytes."""
    d = torch.arange(D, device=DEV)
    at = (d % 32 // 8) * (D // 32 * 8) + d // 32 * 8 + d % 8 if keys else d
    if bits == 8:
        return held[..., at].double()
    byte = held[..., at // 2].int()
    return ((byte >> (at % 2 * 4).int()) % 16).double()


def _stands_for(held, scales, c, bits, keys):
    D = c["head_dim"]
    g = torch.arange(D, device=DEV) // c["group"]
    sm = scales.double()
    return torch.addcmul(sm[..., 1][..., g], sm[..., 0][..., g], _code_of(held, bits, keys, D))


def _nearest(x, c, bits):
    """The value of x's nearest level, group by group of x [T, KVH, D] in 64 bits."""
    out = torch.empty_like(x)
    for a in range(0, c["head_dim"], c["group"]):
        y = x[..., a:a + c["group"]]
        m = y.min(-1, keepdim=True).values.float().half().double()
        s = ((y.max(-1, keepdim=True).values - m) / (2 ** bits - 1)).float().half().double()
        level = torch.round(torch.nan_to_num((y - m) / s, nan=0.0, posinf=0.0, neginf=0.0))
        out[..., a:a + c["group"]] = m + s * level.clamp(min=0, max=2 ** bits - 1)
    return out


def _exact_append(st):
    c = st.case
    h = c["head_dim"] // 2
    z = torch.view_as_complex(st.angles.double())[st.positions.long()][:, None, :]  # e^(i angle)

    def turn(x):
        y = torch.view_as_complex(torch.stack([x[..., :h], x[..., h:]], -1).double().contiguous()) * z
        return torch.cat([y.real, y.imag], -1)

    return [turn(st.q), _nearest(turn(st.k).float().double(), c, c["k_bits"]), _nearest(st.v.double(), c, c["v_bits"])]


def _exact_read(st):
    c = st.case
    p = st.positions.long()
    page, row = st.table.long()[st.seqs.long(), torch.div(p, c["page"], rounding_mode="floor")], p % c["page"]
    return [_stands_for(held[page, :, row], sm[page, :, row], c, bits, keys)
            for held, sm, bits, keys in ((st.kp, st.ks, c["k_bits"], True), (st.vp, st.vs, c["v_bits"], False))]


def _exact_attention(st):
    """Sequence by sequence over its own keys."""
    c = st.case
    P, KVH = c["page"], c["kv_heads"]
    out = torch.zeros(st.q.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(c)):
        j = torch.arange(_first_page(c, n) * P, n, device=DEV)
        if not len(j):
            continue
        page = st.table[b].long()[j // P]
        k, v = (_stands_for(held[page, :, j % P], sm[page, :, j % P], c, bits, keys)  # [n, KVH, D]
                for held, sm, bits, keys in ((st.kp, st.ks, c["k_bits"], True), (st.vp, st.vs, c["v_bits"], False)))
        q = st.q[b].double().reshape(KVH, -1, c["head_dim"])
        w = torch.softmax(torch.matmul(q, k.permute(1, 2, 0).contiguous()) * st.scale, -1)
        out[b] = torch.matmul(w, v.transpose(0, 1).contiguous()).reshape(-1, c["head_dim"])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return dict(append=_exact_append, read=_exact_read, attention=_exact_attention)[case["op"]](st)
