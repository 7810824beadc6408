"""Measured cases of the operators behind a decode step of several sequences at once: the page append with RoPE
(vvh_rope_append_paged), attention of one new token per sequence over a paged key-value cache (vvh_attention_paged),
linears of 4-bit weights with group scales (vvh_linear_q4) and the rules between logits and sampler
(vvh_logits_rules).

With ``own`` true a pass makes the library's calls (include/vvllm_hip.h); with ``own`` false it computes the same
in elementary torch operations in 32 bits, rounded once.  ``exact`` is the definition in 64 bits.

Sizes come from Qwen2.5-0.5B (14 heads, 2 kv heads of 64, hidden 896, MLP 4864, vocabulary 151936) and the 1.5B
shapes (12 heads, 2 kv heads of 128, hidden 1536, MLP 8960), or are generic.
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
        # one new token of each of eight sequences: the smallest append, where latency counts
        dict(name="append_tokens_f16", op="append", tokens=8, prompts=0, heads=14, kv_heads=2, head_dim=64, page=16,
             span=1000, act="f16", shape=1),
        # one new token of each of a large batch, fp32
        dict(name="append_batch_f32", op="append", tokens=96, prompts=0, heads=12, kv_heads=2, head_dim=128, page=64,
             span=5000, act="f32", shape=2),
        # five prompts of different lengths that join a running batch together
        dict(name="append_prompts_f16", op="append", tokens=4001, prompts=5, heads=32, kv_heads=8, head_dim=128,
             page=16, span=3000, act="f16", shape=3),
        # a few chats with short contexts: latency
        dict(name="attention_chats_f16", op="attention", batch=4, heads=14, kv_heads=2, head_dim=64, page=16, span=512,
             spread="even", gone=0.0, act="f16", shape=4),
        # a full server: ragged contexts from one token to 8192, some rows of the batch empty
        dict(name="attention_ragged_f16", op="attention", batch=96, heads=32, kv_heads=8, head_dim=128, page=64,
             span=8192, spread="log", gone=0.0, act="f16", shape=5),
        # three long contexts in fp32, whose oldest pages were given back
        dict(name="attention_long_f32", op="attention", batch=3, heads=12, kv_heads=2, head_dim=128, page=128,
             span=30001, spread="even", gone=0.1, act="f32", shape=6),
        # one token's o projection, added to the residual: the smallest linear
        dict(name="linear_o_token_f16", op="linear", M=1, N=896, K=896, group=64, zeros=False, bias=False,
             residual=True, act="f16"),
        # thirteen sequences through the wide gate/up projection, weights with zero points
        dict(name="linear_gate_up_batch_f16", op="linear", M=13, N=17920, K=1536, group=128, zeros=True, bias=False,
             residual=False, act="f16"),
        # one token's LM head in fp32, the finest groups
        dict(name="linear_head_token_f32", op="linear", M=1, N=151936, K=896, group=32, zeros=False, bias=True,
             residual=False, act="f32"),
        # one chat whose answer has to follow a grammar
        dict(name="logits_grammar_f32", op="logits", rows=1, n=151936, history=700, biases=20, mask=True, act="f32",
             shape=7),
        # an odd vocabulary, penalties only
        dict(name="logits_penalties_f32", op="logits", rows=5, n=32003, history=300, biases=0, mask=False, act="f32",
             shape=8),
        # a batch with long histories, each row with its own grammar
        dict(name="logits_batch_f16", op="logits", rows=64, n=151936, history=4000, biases=300, mask=True, act="f16",
             shape=9),
    ]


# ---- drawn cases ------------------------------------------------------------
def _log(rng, lo: int, hi: int) -> int:
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng) -> dict:
    kv = rng.choice([1, 2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 4, 5, 6, 7, 8, 16]), kv_heads=kv, head_dim=rng.choice([64, 64, 96, 128, 128]))


def _draw(rng) -> dict:
    op = rng.choice(["append", "attention", "attention", "linear", "linear", "logits"])
    act = rng.choice(["f16", "f16", "f32"])
    page = rng.choice([16, 16, 24, 32, 64, 128, 256])
    shape = rng.randrange(1 << 20)
    if op == "append":
        prompts = rng.choice([0, rng.randint(1, 8)])
        tokens = _log(rng, 8 * prompts, 4000) if prompts else _log(rng, 1, 256)
        return dict(op=op, tokens=tokens, prompts=prompts, **_heads(rng), page=page, span=_log(rng, 16, 5000), act=act,
                    shape=shape)
    if op == "attention":
        return dict(op=op, batch=_log(rng, 1, 96), **_heads(rng), page=page, span=_log(rng, 1, 30000),
                    spread=rng.choice(["even", "log", "full"]), gone=rng.choice([0.0, 0.0, 0.1]), act=act, shape=shape)
    if op == "linear":
        g = rng.choice([32, 64, 128])
        N, K = rng.choice([(896, 896), (9728, 896), (896, 4864), (1536, 1536), (17920, 1536), (1536, 8960),
                           (_log(rng, 100, 40000), 32 * _log(rng, 1, 256))])
        return dict(op=op, M=_log(rng, 1, 64), N=N, K=K, group=g, zeros=rng.random() < 0.4, bias=rng.random() < 0.4,
                    residual=rng.random() < 0.4, act=act)
    return dict(op=op, rows=_log(rng, 1, 64), n=_log(rng, 1000, 151936), history=_log(rng, 1, 4000),
                biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5, act=act, shape=shape)


def draw(rng) -> dict:
    most = {c["op"]: max(work(x)["bytes"] for x in listed() if x["op"] == c["op"]) for c in listed()}
    while True:
        c = _draw(rng)
        if c["op"] == "linear" and (c["K"] % c["group"] or c["M"] * c["N"] * c["K"] > 4e9):
            continue
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


def _histories(c):
    """Tokens of each row, and how many of them are its prompt's."""
    rng = random.Random(c["shape"])
    counts = [rng.randint(0, c["history"]) for _ in range(c["rows"])]
    counts[rng.randrange(c["rows"])] = c["history"]
    return counts, [rng.randint(0, n) for n in counts]


def work(case) -> dict:
    c, e = case, 4 if case["act"] == "f32" else 2
    if c["op"] == "append":
        q, kv = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        t = c["tokens"]
        return {"bytes": t * (2 * (q + 2 * kv) * e + 4 * c["head_dim"]), "flops": 3 * t * (q + kv)}
    if c["op"] == "attention":
        keys = sum(n - _first_page(c, n) * c["page"] for n in _lengths(c))
        rows = 2 * c["batch"] * c["heads"] * c["head_dim"]
        return {"bytes": (2 * keys * c["kv_heads"] * c["head_dim"] + rows) * e,
                "flops": 4 * keys * c["heads"] * c["head_dim"]}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": N * K // 2 + N * K // c["group"] * (3 if c["zeros"] else 2) + M * K * e
                + M * N * e * (2 if c["residual"] else 1) + (4 * N if c["bias"] else 0), "flops": 2 * M * N * K}
    cells = c["rows"] * c["n"]
    return {"bytes": 2 * cells * e + (cells // 8 if c["mask"] else 0) + 4 * sum(_histories(c)[0])
            + 8 * c["rows"] * c["biases"], "flops": cells}


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


def _pages(g, counts, width):
    """A page table with counts[s] pages of row s taken from a shuffled pool, and the pool's size."""
    need = sum(counts)
    pool = torch.randperm(need + 3, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
    n = torch.tensor(counts, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < n[:, None]] = pool[:need]
    return table, need + 3


def prepare(case, seed):
    c, g = case, _rand(seed)
    dt = torch.float16 if c["act"] == "f16" else torch.float32
    st = SimpleNamespace(case=c, dt=dt, call=None)
    if c["op"] in ("append", "attention"):
        H, KVH, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
        if c["op"] == "append":
            where = _append_shape(c)
            seqs = 1 + max(s for s, _ in where)
            last = [0] * seqs
            for s, p in where:
                last[s] = max(last[s], p)
            counts = [p // P + 1 for p in last]
            st.seqs, st.positions = _ints([s for s, _ in where]), _ints([p for _, p in where])
            st.angles = _angles(max(last) + 1, D)
            st.q = _normal(g, (c["tokens"], H, D), dtype=dt)
            st.k, st.v = (_normal(g, (c["tokens"], KVH, D), dtype=dt) for _ in range(2))
        else:
            lens = _lengths(c)
            counts = [-(-n // P) for n in lens]
            st.lens, st.longest = _ints(lens), max(lens)
            st.scale = 1.0 / math.sqrt(D)
            # scores of a few units, so that a query weighs some positions above others
            st.q = _normal(g, (c["batch"], H, D), 2.0, dt)
        width = max(1, max(counts))
        st.table, st.pool = _pages(g, counts, width)
        if c["op"] == "attention":
            first = _ints([_first_page(c, n) for n in lens])
            st.table[torch.arange(width, device=DEV)[None, :] < first[:, None]] = -1
        st.kp, st.vp = (_normal(g, (st.pool, P, KVH, D), dtype=dt) for _ in range(2))
        st.out = torch.empty_like(st.q)
    elif c["op"] == "linear":
        M, N, K, G = c["M"], c["N"], c["K"], c["group"]
        st.codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
        st.scales = (torch.rand((N, K // G), generator=g, device=DEV) * 0.008 + 0.002).half()
        st.zeros = torch.randint(5, 11, (N, K // G), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None
        st.bias = _normal(g, (N,), 0.01) if c["bias"] else None
        st.x = _normal(g, (M, K), dtype=dt)
        st.res = _normal(g, (M, N), dtype=dt) if c["residual"] else None
        st.out = torch.empty((M, N), device=DEV, dtype=dt)
    else:
        rows, n = c["rows"], c["n"]
        counts, prompts = _histories(c)
        st.logits = _normal(g, (rows, n), 3.0, dt)
        # words come back: the tokens of a text are far from even over the vocabulary
        st.tokens = (torch.rand((rows, c["history"]), generator=g, device=DEV) ** 6 * n).to(torch.int32).clamp_(0, n - 1)
        st.counts, st.prompts = _ints(counts), _ints(prompts)
        st.repetition = 1.0 + 0.3 * torch.rand(rows, generator=g, device=DEV)
        st.frequency, st.presence = (torch.rand(rows, generator=g, device=DEV) for _ in range(2))
        st.bias_ids = torch.randint(0, n, (rows * c["biases"],), generator=g, device=DEV, dtype=torch.int32)
        st.bias_values = _normal(g, (rows * c["biases"],), 5.0)
        st.bias_offsets = _ints([c["biases"] * r for r in range(rows + 1)])
        st.mask = None
        if c["mask"]:
            st.mask = torch.randint(-2**31, 2**31, (rows, (n + 31) // 32), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
        st.out = torch.empty_like(st.logits)
    return st


# ---- the plain forms ------------------------------------------------------------
def _rotate(x, cs):
    """Split-half rotation of x [T, H, D] with cs [T, D / 2, 2]."""
    h = x.shape[-1] // 2
    x0, x1, co, si = x[..., :h], x[..., h:], cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([x0 * co - x1 * si, x1 * co + x0 * si], -1)


def _plain_append(st, k_pages, v_pages, wide):
    P, p = st.case["page"], st.positions.long()
    cs = st.angles[p].to(wide)
    page = st.table[st.seqs.long(), p // P].long()
    k_pages[page, p % P] = _rotate(st.k.to(wide), cs).to(k_pages.dtype)
    v_pages[page, p % P] = st.v.to(v_pages.dtype)
    return _rotate(st.q.to(wide), cs)


def _plain_attention(st, wide):
    """All contexts padded to the longest; keys past a context's end and on pages that are gone weigh nothing."""
    c = st.case
    B, H, KVH, D, P = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    width = st.table.shape[1]
    at = torch.arange(width * P, device=DEV)
    live = (at[None, :] < st.lens[:, None]) & (st.table >= 0).repeat_interleave(P, dim=1)
    page = st.table.clamp(min=0).long()
    k = st.kp[page].reshape(B, width * P, KVH, D).permute(0, 2, 3, 1).to(wide).contiguous()
    s = torch.matmul(st.q.to(wide).reshape(B, KVH, H // KVH, D), k) * st.scale
    del k
    s = s.masked_fill(~live[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    v = st.vp[page].reshape(B, width * P, KVH, D).permute(0, 2, 1, 3).to(wide).contiguous()
    return torch.matmul(w, v).reshape(B, H, D)


def _plain_linear(st, wide):
    c = st.case
    N, K, G = c["N"], c["K"], c["group"]
    codes = torch.stack([st.codes & 15, st.codes >> 4], -1).reshape(N, K // G, G).to(wide)
    zeros = st.zeros.to(wide)[..., None] if c["zeros"] else 8.0
    w = ((codes - zeros) * st.scales.to(wide)[..., None]).reshape(N, K)
    y = torch.matmul(st.x.to(wide), w.t())
    if c["bias"]:
        y = y + st.bias.to(wide)
    return y + st.res.to(wide) if c["residual"] else y


def _plain_logits(st, wide):
    c = st.case
    rows, n = c["rows"], c["n"]
    x = st.logits.to(wide)
    at = torch.arange(c["history"], device=DEV)[None, :]
    tokens = st.tokens.long()
    used = (at < st.counts[:, None]).int()
    said = used * (at >= st.prompts[:, None]).int()
    seen = torch.zeros((rows, n), dtype=torch.int32, device=DEV).scatter_add_(1, tokens, used) > 0
    times = torch.zeros((rows, n), dtype=torch.int32, device=DEV).scatter_add_(1, tokens, said)
    r = st.repetition.to(wide)[:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st.frequency.to(wide)[:, None] * times - st.presence.to(wide)[:, None] * (times > 0)
    if c["biases"]:
        # of a token that a row lists twice the last entry counts
        entry = torch.arange(rows * c["biases"], device=DEV)
        cell = entry // c["biases"] * n + st.bias_ids.long()
        last = torch.full((rows * n,), -1, dtype=torch.int64, device=DEV).scatter_reduce_(0, cell, entry, "amax").reshape(rows, n)
        x = x + torch.where(last >= 0, st.bias_values.to(wide)[last.clamp(min=0)], 0.0)
    if c["mask"]:
        i = torch.arange(n, device=DEV)
        x = x.masked_fill((st.mask[:, i // 32] >> (i % 32)[None, :].int()) & 1 == 0, -math.inf)
    return x


# ---- the library's calls ----------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _calls(st):
    """The arguments of a state's call, which a program keeps next to its buffers."""
    from vvllm_amd import capi

    capi.init(torch.cuda.current_device())
    c, dtype = st.case, capi.F16 if st.case["act"] == "f16" else capi.F32
    if c["op"] in ("append", "attention"):
        cache = capi.PagedCache(k_pages=_p(st.kp), v_pages=_p(st.vp), page_table=_p(st.table), num_pages=st.pool,
                                page_size=c["page"], num_seqs=st.table.shape[0], max_pages=st.table.shape[1],
                                num_kv_heads=c["kv_heads"], head_dim=c["head_dim"], dtype=dtype)
        st.keep = cache
        if c["op"] == "append":
            args = ("vvh_rope_append_paged", ctypes.byref(cache), _p(st.out), _p(st.q), _p(st.k), _p(st.v),
                    _p(st.seqs), _p(st.positions), c["tokens"], c["heads"], _p(st.angles), st.angles.shape[0])
        else:
            args = ("vvh_attention_paged", ctypes.byref(cache), _p(st.out), _p(st.q), _p(st.lens), st.longest,
                    c["heads"], st.scale)
    elif c["op"] == "linear":
        args = ("vvh_linear_q4", _p(st.out), _p(st.x), _p(st.codes), _p(st.scales), _p(st.zeros), _p(st.bias),
                _p(st.res), c["M"], c["N"], c["K"], c["group"], dtype, dtype)
    else:
        st.keep = rules = capi.LogitsRules(
            tokens=_p(st.tokens), token_stride=c["history"], token_counts=_p(st.counts), prompt_counts=_p(st.prompts),
            repetition=_p(st.repetition), frequency=_p(st.frequency), presence=_p(st.presence),
            bias_ids=_p(st.bias_ids) if c["biases"] else None, bias_values=_p(st.bias_values) if c["biases"] else None,
            bias_offsets=_p(st.bias_offsets) if c["biases"] else None, bias_count=c["rows"] * c["biases"],
            mask=_p(st.mask), mask_stride=(c["n"] + 31) // 32)
        args = ("vvh_logits_rules", _p(st.out), _p(st.logits), ctypes.byref(rules), c["rows"], c["n"], dtype)
    return capi.call, args


def run(state):
    st, op = state, state.case["op"]
    if own:
        if st.call is None:
            st.call, st.args = _calls(st)
        st.call(*st.args, torch.cuda.current_stream().cuda_stream)
        return [st.out, st.kp, st.vp] if op == "append" else st.out
    if op == "append":
        return [_plain_append(st, st.kp, st.vp, torch.float32).to(st.dt), st.kp, st.vp]
    plain = dict(attention=_plain_attention, linear=_plain_linear, logits=_plain_logits)[op]
    return plain(st, torch.float32).to(st.dt)


# ---- the definitions in 64 bits, written apart ---------------------------------------
def _exact_append(st):
    c = st.case
    P, h = c["page"], c["head_dim"] // 2
    p = st.positions.long()
    z = torch.view_as_complex(st.angles.double())[p][:, None, :]  # e^(i angle)
    turn = lambda x: torch.view_as_complex(torch.stack([x[..., :h], x[..., h:]], -1).double().contiguous()) * z  # noqa: E731
    flat = lambda y: torch.cat([y.real, y.imag], -1)  # noqa: E731
    slot = st.table.long()[st.seqs.long(), torch.div(p, P, rounding_mode="floor")] * P + p % P
    k, v = st.kp.double().flatten(0, 1), st.vp.double().flatten(0, 1)
    k[slot], v[slot] = flat(turn(st.k)), st.v.double()
    return [flat(turn(st.q)), k.reshape(st.kp.shape), v.reshape(st.vp.shape)]


def _exact_attention(st):
    """Sequence by sequence over its own keys."""
    c = st.case
    P, KVH, D = c["page"], c["kv_heads"], c["head_dim"]
    out = torch.zeros(st.q.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(c)):
        j = torch.arange(_first_page(c, n) * P, n, device=DEV)
        if not len(j):
            continue
        page = st.table[b].long()[j // P]
        k, v = st.kp[page, j % P].double(), st.vp[page, j % P].double()  # [n, KVH, D]
        q = st.q[b].double().reshape(KVH, -1, D)
        w = torch.softmax(torch.matmul(q, k.permute(1, 2, 0).contiguous()) * st.scale, -1)
        out[b] = torch.matmul(w, v.transpose(0, 1).contiguous()).reshape(-1, D)
    return out


def _exact_linear(st):
    """Group by group: the codes' sum and the zero points' share apart."""
    c = st.case
    M, N, K, G = c["M"], c["N"], c["K"], c["group"]
    y = torch.zeros((M, N), dtype=torch.float64, device=DEV)
    x = st.x.double()
    for k0 in range(0, K, G):
        xs, g = x[:, k0:k0 + G], k0 // G
        packed = st.codes[:, k0 // 2:(k0 + G) // 2]
        dot = torch.matmul(xs[:, 0::2].contiguous(), (packed % 16).double().t().contiguous())
        dot += torch.matmul(xs[:, 1::2].contiguous(), (packed // 16).double().t().contiguous())
        z = st.zeros[:, g].double() if c["zeros"] else torch.full((N,), 8.0, dtype=torch.float64, device=DEV)
        y += (dot - xs.sum(1, keepdim=True) * z) * st.scales[:, g].double()
    if c["bias"]:
        y += st.bias.double()
    if c["residual"]:
        y += st.res.double()
    return y


def _exact_logits(st):
    """Row by row, touching only the tokens that a rule names."""
    c = st.case
    x = st.logits.double()
    counts, prompts = _histories(c)
    for r in range(c["rows"]):
        row, rep = x[r], st.repetition[r].double()
        seen = torch.unique(st.tokens[r, :counts[r]].long())
        row[seen] = torch.where(row[seen] > 0, row[seen] / rep, row[seen] * rep)
        said, times = torch.unique(st.tokens[r, prompts[r]:counts[r]].long(), return_counts=True)
        row[said] -= st.frequency[r].double() * times + st.presence[r].double()
        if c["biases"]:
            a = c["biases"] * r
            named = dict(zip(st.bias_ids[a:a + c["biases"]].tolist(), st.bias_values[a:a + c["biases"]].tolist()))
            row[list(named)] += torch.tensor(list(named.values()), dtype=torch.float64, device=DEV)
        if c["mask"]:
            bits = (st.mask[r].view(torch.uint8)[:, None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1
            row[bits.flatten()[:c["n"]] == 0] = -math.inf
    return x


def exact(case, seed):
    st = prepare(case, seed)
    return dict(append=_exact_append, attention=_exact_attention, linear=_exact_linear, logits=_exact_logits)[case["op"]](st)
