"""The batched decode operators as a program uses them: steps of a small decoder of 4-bit linears over a paged cache, with
sequences of different lengths, one that joins and one that ends, from the hidden rows to the next tokens.  Every operator
of a step is held against 64 bits on the inputs it had; the captured step, replayed, against the eager one's bits."""
import ctypes

import numpy as np
import pytest

from serving import HALF, Pages, Stream, attention_ref, put
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}
B, HID, H, KVH, D, MLP, VOCAB, PAGE, PAGES, LAYERS, GROUP = 6, 320, 10, 2, 64, 448, 1003, 16, 80, 2, 64
SCALE = 0.125


class Linear:
    """A 4-bit linear and, with its input's and output's buffers, how far the output is off."""

    def __init__(self, rng, N, K, zeros=False):
        self.N, self.K = N, K
        self.codes, self.scales = capi.quantize_q4(rng.normal(0, K ** -0.5, (N, K)).astype(np.float32), GROUP)
        self.zeros = rng.integers(7, 10, (N, K // GROUP), np.uint8) if zeros else None
        self.d = [capi.DevBuf.from_array(a) if a is not None else None for a in (self.codes, self.scales, self.zeros)]

    def run(self, out, x, res, dtype, outd, stream):
        w, s, z = (a.ptr if a else None for a in self.d)
        capi.call("vvh_linear_q4", out.ptr, x.ptr, w, s, z, None, res.ptr if res else None, B, self.N, self.K, GROUP, dtype, outd,
                  stream)

    def check(self, out, x, res, dtype, outd):
        c = np.stack([self.codes & 15, self.codes >> 4], -1).reshape(self.N, -1, GROUP).astype(np.float64)
        z = 8.0 if self.zeros is None else self.zeros.astype(np.float64)[..., None]
        s = self.scales.view(np.float16).astype(np.float64)[..., None]
        a = x.to_array(NP[dtype], (B, self.K)).astype(np.float64)
        y = a @ ((c - z) * s).reshape(self.N, self.K).T
        most = np.abs(a) @ ((c + z) * s).reshape(self.N, self.K).T
        if res:
            r = res.to_array(NP[outd], (B, self.N)).astype(np.float64)
            y, most = y + r, most + np.abs(r)
        off = np.abs(out.to_array(NP[outd], (B, self.N)) - y)
        assert (off <= HALF[outd] * np.abs(y) + 2.0 ** -25 + (self.K + 4) * 2.0 ** -24 * most).all(), off.max()


class Decoder:
    def __init__(self, rng, dtype, lens):
        self.dtype = dtype
        buf = lambda n: capi.DevBuf(B * n * 4)  # noqa: E731
        self.norm = capi.DevBuf.from_array(rng.uniform(0.5, 1.5, HID).astype(np.float32))
        self.table = capi.DevBuf(PAGES * PAGE * D * 4)
        capi.call("vvh_rope_table", self.table.ptr, PAGES * PAGE, D, 1e6, None)
        self.layers = []
        for i in range(LAYERS):
            self.layers.append(dict(
                cache=Pages(rng, lens, PAGE, KVH, D, dtype, spare=8, max_pages=PAGES),
                w={n: Linear(rng, N, K, zeros=i == 1) for n, N, K in (("q", H * D, HID), ("k", KVH * D, HID), ("v", KVH * D, HID),
                                                                     ("o", HID, H * D), ("gate", MLP, HID), ("up", MLP, HID),
                                                                     ("down", HID, MLP))},
                b={n: buf(k) for n, k in (("x", HID), ("n", HID), ("q", H * D), ("r", H * D), ("k", KVH * D), ("v", KVH * D),
                                          ("a", H * D), ("o", HID), ("n2", HID), ("gate", MLP), ("up", MLP), ("m", MLP),
                                          ("down", HID))}))
        for lay in self.layers[1:]:  # one page table for all layers
            lay["cache"].table[:] = self.layers[0]["cache"].table
            lay["cache"].d_t = self.layers[0]["cache"].d_t
            for a in (lay["cache"].kp, lay["cache"].vp):
                a[np.isnan(a)] = 1
            lay["cache"].upload()
            lay["cache"].d_t = self.layers[0]["cache"].d_t
        self.head = Linear(rng, VOCAB, HID)
        self.fin, self.logits, self.ruled = buf(HID), buf(VOCAB), buf(VOCAB)
        self.pos, self.lens = capi.DevBuf(B * 4), self.layers[0]["cache"].d_n
        hist = PAGES * PAGE
        self.tokens = rng.integers(0, VOCAB, (B, hist), np.int32)
        self.counts = np.array(lens, np.int32)
        self.mask = rng.integers(0, 1 << 32, (1, (VOCAB + 31) // 32), np.uint32)
        self.pen = rng.uniform(0.1, 1.2, (3, B)).astype(np.float32)
        self.prompt = (self.counts // 2).astype(np.int32)
        self.d_tokens, self.d_counts, self.d_mask, self.d_pen, self.d_prompt = (
            capi.DevBuf.from_array(a) for a in (self.tokens, self.counts, self.mask, self.pen, self.prompt))
        self.next = capi.DevBuf(B * 4)
        self.spec = capi.LogitsRules(tokens=self.d_tokens.ptr, token_stride=hist, token_counts=self.d_counts.ptr,
                                     prompt_counts=self.d_prompt.ptr, repetition=self.d_pen.ptr,
                                     frequency=self.d_pen.addr(4 * B), presence=self.d_pen.addr(8 * B), mask=self.d_mask.ptr)

    def step(self, s):
        t = self.dtype
        for i, lay in enumerate(self.layers):
            b, w = lay["b"], lay["w"]
            x = b["x"] if i == 0 else self.layers[i - 1]["b"]["down"]
            capi.call("vvh_rms_norm", b["n"].ptr, x.ptr, self.norm.ptr, B, HID, 1e-6, t, s)
            for n in "qkv":
                w[n].run(b[n], b["n"], None, t, t, s)
            capi.call("vvh_rope_append_paged", lay["cache"].cache(), b["r"].ptr, b["q"].ptr, b["k"].ptr, b["v"].ptr, None,
                      self.pos.ptr, B, H, self.table.ptr, PAGES * PAGE, s)
            capi.call("vvh_attention_paged", lay["cache"].cache(), b["a"].ptr, b["r"].ptr, self.lens.ptr, 0, H, SCALE, s)
            w["o"].run(b["o"], b["a"], x, t, t, s)
            capi.call("vvh_rms_norm", b["n2"].ptr, b["o"].ptr, self.norm.ptr, B, HID, 1e-6, t, s)
            w["gate"].run(b["gate"], b["n2"], None, t, t, s)
            w["up"].run(b["up"], b["n2"], None, t, t, s)
            capi.call("vvh_eltwise", 3, b["m"].ptr, b["gate"].ptr, b["up"].ptr, B * MLP, t, s)
            w["down"].run(b["down"], b["m"], b["o"], t, t, s)
        capi.call("vvh_rms_norm", self.fin.ptr, self.layers[-1]["b"]["down"].ptr, self.norm.ptr, B, HID, 1e-6, t, s)
        self.head.run(self.logits, self.fin, None, t, F32, s)
        capi.call("vvh_logits_rules", self.ruled.ptr, self.logits.ptr, ctypes.byref(self.spec), B, VOCAB, F32, s)
        for r in range(B):
            capi.call("vvh_argmax", self.ruled.addr(r * VOCAB * 4), VOCAB, self.next.addr(4 * r), s)

    def rows(self, name, i, n):
        return self.layers[i]["b"][name].to_array(NP[self.dtype], (B, n, D))

    def check(self, pos, before):
        """Every operator on the inputs it had; `before`: the layers' pages before the step."""
        t, live = self.dtype, pos >= 0
        cs = self.table.to_array(np.float32, (PAGES * PAGE, D // 2, 2)).astype(np.float64)[np.maximum(pos, 0)][:, None]

        def rotated(x):
            x0, x1 = x[..., :D // 2].astype(np.float64), x[..., D // 2:].astype(np.float64)
            return np.concatenate([x0 * cs[..., 0] - x1 * cs[..., 1], x1 * cs[..., 0] + x0 * cs[..., 1]], -1)

        for i, lay in enumerate(self.layers):
            b, w, pg = lay["b"], lay["w"], lay["cache"]
            x = b["x"] if i == 0 else self.layers[i - 1]["b"]["down"]
            for n in "qkv":
                w[n].check(b[n], b["n"], None, t, t)
            kp, vp = pg.d_k.to_array(NP[t], pg.kp.shape), pg.d_v.to_array(NP[t], pg.vp.shape)
            for name, n, got in (("q", H, self.rows("r", i, H)), ("k", KVH, None)):
                src = self.rows(name, i, n)
                want = rotated(src)
                if got is None:
                    got = kp[pg.table[np.arange(B), np.maximum(pos, 0) // PAGE], np.maximum(pos, 0) % PAGE]
                tol = HALF[t] * np.abs(want) + 2.0 ** -25 + 6 * 2.0 ** -24 * np.abs(src.astype(np.float64)).max()
                assert (np.abs(got - want) <= tol)[live].all(), (name, i)
            # the step's rows, and no other, are new
            wrote = np.zeros(pg.kp.shape[:2], bool)
            wrote[pg.table[live, pos[live] // PAGE], pos[live] % PAGE] = True
            for now, old in ((kp, before[i][0]), (vp, before[i][1])):
                np.testing.assert_array_equal(now[~wrote], old[~wrote])
            np.testing.assert_array_equal(vp[pg.table[live, pos[live] // PAGE], pos[live] % PAGE], self.rows("v", i, KVH)[live])
            pg.kp, pg.vp = kp, vp
            pg.lens = pos + 1
            ref, tol = attention_ref(pg, self.rows("r", i, H), SCALE, HALF[t])
            assert (np.abs(self.rows("a", i, H) - ref) <= tol).all()
            w["o"].check(b["o"], b["a"], x, t, t)
            w["gate"].check(b["gate"], b["n2"], None, t, t)
            w["up"].check(b["up"], b["n2"], None, t, t)
            w["down"].check(b["down"], b["m"], b["o"], t, t)
        self.head.check(self.logits, self.fin, None, t, F32)
        z = self.logits.to_array(np.float32, (B, VOCAB)).astype(np.float64)
        most = np.abs(z)
        for r in range(B):
            n, p = int(self.counts[r]), int(self.prompt[r])
            seen, times = np.unique(self.tokens[r, :n]), np.bincount(self.tokens[r, p:max(n, p)], minlength=VOCAB)
            f = float(self.pen[0, r])
            z[r, seen] = np.where(z[r, seen] > 0, z[r, seen] / f, z[r, seen] * f)
            most[r] *= max(f, 1 / f)
            z[r] -= float(self.pen[1, r]) * times + float(self.pen[2, r]) * (times > 0)
            most[r] += 1.2 * (times + 1)
        z[:, np.unpackbits(self.mask.view(np.uint8), bitorder="little")[:VOCAB] == 0] = -np.inf
        got = self.ruled.to_array(np.float32, (B, VOCAB))
        with np.errstate(invalid="ignore"):
            assert ((got == z) | (np.abs(got - z) <= 6 * 2.0 ** -24 * most)).all()
        np.testing.assert_array_equal(self.next.to_array(np.int32, (B,)), got.argmax(1))

    def outputs(self):
        return self.ruled.to_array(np.uint32, (B, VOCAB)), self.next.to_array(np.int32, (B,))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_steps(gpu, dtype):
    rng = np.random.default_rng(21)
    d = Decoder(rng, dtype, [1100, 16, 15, 400, 0, 1])
    pg = d.layers[0]["cache"]
    free = sorted(set(range(len(pg.kp))) - set(pg.table[pg.table >= 0].tolist()))
    pos = np.array(pg.lens)
    st, replay = Stream(), None
    for step in range(4):
        if step == 0:
            pos[4] = -1           # padding
        elif step == 2:
            pos[4], pos[3] = 0, -1  # a sequence joins, one ends
        for s in range(B):
            if pos[s] >= 0 and pg.table[s, pos[s] // PAGE] < 0:
                pg.table[s, pos[s] // PAGE] = free.pop()
        for lay in d.layers:
            lay["cache"].table[:] = pg.table
        put(pg.d_t, pg.table)
        put(d.pos, pos)
        put(d.lens, pos + 1)
        put(d.d_tokens, d.tokens)
        put(d.d_counts, d.counts)
        put(d.layers[0]["b"]["x"], rng.normal(0, 1, (B, HID)).astype(NP[dtype]))
        before = [(lay["cache"].d_k.to_array(NP[dtype], pg.kp.shape), lay["cache"].d_v.to_array(NP[dtype], pg.vp.shape))
                  for lay in d.layers]
        print("[step]", step, flush=True)
        d.step(st.s)  # eager; the stream's workspace too
        st.sync()
        eager = d.outputs()
        d.check(pos, before)
        if replay is None:
            replay = st.capture(d.step)
        for _ in range(2):  # the same rows once more
            capi.call("vvh_fill_normal", d.ruled.ptr, F32, B * VOCAB, 1, 0.0, 1.0, None)
            capi.call("vvh_fill_normal", d.layers[0]["b"]["a"].ptr, dtype, B * H * D, 2, 0.0, 1.0, None)
            capi.sync()
            replay()
            for a, e in zip(d.outputs(), eager):
                np.testing.assert_array_equal(a, e)
        chosen = eager[1]
        for s in range(B):
            if pos[s] >= 0:
                d.tokens[s, d.counts[s]] = chosen[s]
                d.counts[s] += 1
                pos[s] += 1
    st.close()
