"""vvh_logits_rules against the same rules in 64 bits, token by token.

Tolerance per element: half a step of the output's type and one fp32 rounding for each of the five operations on the
largest value on the way."""
import ctypes

import numpy as np
import pytest

from serving import HALF, Stream, put
from vvllm_amd import capi

pytestmark = pytest.mark.gpu
F16, F32 = capi.F16, capi.F32
NP = {F16: np.float16, F32: np.float32}


class Case:
    def __init__(self, rows, n, dtype, history=50, penalties="rfp", biases=0, mask=None, seed=0):
        print("[case] rules", rows, n, dtype, history, penalties, biases, mask, flush=True)
        rng = self.rng = np.random.default_rng(rows + n + seed)
        self.rows, self.n, self.dtype = rows, n, dtype
        self.logits = rng.normal(0, 4, (rows, n)).astype(NP[dtype])
        self.tokens = rng.integers(0, n, (rows, history), np.int32) if history else None
        if history:
            self.tokens[:, ::3] = self.tokens[:, :1]  # one token many times
            self.counts = rng.integers(0, history + 1, rows, np.int32)
            self.counts[rng.integers(rows)] = history
            self.prompts = (self.counts * rng.random(rows)).astype(np.int32)
        self.rep = rng.uniform(0.8, 1.5, rows).astype(np.float32) if "r" in penalties else None
        self.freq = rng.uniform(-0.5, 1, rows).astype(np.float32) if "f" in penalties else None
        self.pres = rng.uniform(-0.5, 1, rows).astype(np.float32) if "p" in penalties else None
        self.ids = None
        if biases:
            self.offsets = np.concatenate([[0], np.cumsum(rng.integers(0, 2 * biases, rows))]).astype(np.int32)
            self.ids = rng.integers(0, n, self.offsets[-1], np.int32)
            self.values = rng.normal(0, 5, len(self.ids)).astype(np.float32)
        words = (n + 31) // 32
        self.mask = None
        self.stride = words + 3 if mask == "rows" else 0
        if mask:
            self.mask = rng.integers(0, 1 << 32, (rows if mask == "rows" else 1, self.stride or words), np.uint32)
        self.upload()

    def upload(self):
        self.d = {n: capi.DevBuf.from_array(a) for n, a in vars(self).items() if isinstance(a, np.ndarray)}
        self.d_out = capi.DevBuf(self.logits.nbytes)

    def spec(self):
        p = lambda n: self.d[n].ptr if n in self.d else None  # noqa: E731
        return capi.LogitsRules(tokens=p("tokens"), token_stride=self.tokens.shape[1] if self.tokens is not None else 0,
                                token_counts=p("counts"), prompt_counts=p("prompts"), repetition=p("rep"), frequency=p("freq"),
                                presence=p("pres"), bias_ids=p("ids"), bias_values=p("values"), bias_offsets=p("offsets"),
                                bias_count=len(self.ids) if self.ids is not None else 0, mask=p("mask"), mask_stride=self.stride)

    def run(self, out=None, stream=None):
        out = out or self.d_out
        capi.call("vvh_logits_rules", out.ptr, self.d["logits"].ptr, ctypes.byref(self.spec()), self.rows, self.n, self.dtype, stream)
        return out.to_array(NP[self.dtype], self.logits.shape)

    def want(self):
        y, most = self.logits.astype(np.float64), np.abs(self.logits.astype(np.float64))
        for r in range(self.rows):
            if self.tokens is not None:
                total = min(max(int(self.counts[r]), 0), self.tokens.shape[1])
                prompt = max(int(self.prompts[r]), 0) if "prompts" in self.d else 0
                inside = lambda t: t[(t >= 0) & (t < self.n)]  # noqa: E731
                seen = np.unique(inside(self.tokens[r, :total]))
                if self.rep is not None:
                    x, f = y[r, seen], float(self.rep[r])
                    y[r, seen] = np.where(x > 0, x / f, x * f)
                    most[r, seen] *= max(f, 1 / f)
                said, times = np.unique(inside(self.tokens[r, prompt:total]), return_counts=True)
                for rule, size in ((self.freq, times), (self.pres, 1)):
                    if rule is not None:
                        y[r, said] -= float(rule[r]) * size
                        most[r, said] += abs(float(rule[r])) * size
            if self.ids is not None:
                a, b = np.clip(self.offsets[r:r + 2], 0, len(self.ids))
                for i, v in dict(zip(self.ids[a:b].tolist(), self.values[a:b].tolist())).items():
                    if 0 <= i < self.n:
                        y[r, i] += v
                        most[r, i] += abs(v)
            if self.mask is not None:
                bits = np.unpackbits(self.mask[r if self.stride else 0].view(np.uint8), bitorder="little")[:self.n]
                y[r, bits == 0] = -np.inf
        with np.errstate(invalid="ignore"):
            tol = HALF[self.dtype] * np.where(np.isfinite(y), np.abs(y), 0) + 2.0 ** -25 + 5 * 2.0 ** -24 * most
        return y, tol

    def check(self, got=None):
        y, tol = self.want()
        got = (self.run() if got is None else got).astype(np.float64)
        gone = np.isneginf(y)
        np.testing.assert_array_equal(np.isneginf(got), gone)
        off = np.abs(got - y)[~gone] / tol[~gone]
        assert (off <= 1).all(), off.max()
        return got


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (2, 2047), (2, 2048), (2, 2049), (5, 32003), (1, 151936), (9, 8191), (70, 1000),
                                    (3, 65537)])
@pytest.mark.parametrize("mask", [None, "rows", "one"])
def test_all_rules(gpu, dtype, rows, n, mask):
    Case(rows, n, dtype, history=200, biases=5, mask=mask).check()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("history,penalties,biases,mask", [(0, "", 0, None), (0, "", 9, None), (0, "", 0, "rows"), (30, "r", 0, None),
                                                           (30, "f", 0, None), (30, "p", 0, None), (30, "", 0, None),
                                                           (5000, "rfp", 0, "one"), (1, "rp", 3, None)])
def test_each_rule_alone(gpu, dtype, history, penalties, biases, mask):
    Case(4, 5000, dtype, history, penalties, biases, mask).check()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [5000, 4097])
def test_in_place(gpu, dtype, n):
    for kw in (dict(biases=4, mask="rows"), dict(biases=4), dict(penalties="", history=0, mask="one"), dict(penalties="", history=0)):
        c = Case(3, n, dtype, **kw)
        plain = c.check()
        np.testing.assert_array_equal(c.run(out=c.d["logits"]), plain.astype(NP[dtype]))


def test_no_prompt_counts(gpu):
    c = Case(3, 3000, F32)
    c.prompts = None
    c.upload()
    c.check()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_ids_and_counts_out_of_range(gpu, dtype):
    """Tokens and ids outside the vocabulary are ignored; counts and offsets are clamped."""
    c = Case(4, 700, dtype, history=60, biases=20, mask="rows")
    c.tokens[:, 1::5] = [-1, 700, 2**31 - 1, -2**31] * 3
    c.counts[:] = [-3, 1000, 0, 60]
    c.prompts[:] = [5, -7, 4, 90]
    c.ids[::3] = -1
    c.ids[1::7] = 700
    c.offsets[-1] += 50
    c.upload()
    c.check()


def test_logits_that_are_not_finite(gpu):
    """-infinity stays, NaN stays unless masked, a masked NaN or infinity is -infinity."""
    c = Case(2, 3000, F32, mask="rows")
    c.logits[:, 5:400:7], c.logits[:, 6:400:7], c.logits[:, 8:400:7] = -np.inf, np.nan, np.inf
    c.upload()
    got = c.run()
    bits = np.unpackbits(c.mask.view(np.uint8), axis=1, bitorder="little")[:, :3000].astype(bool)
    assert np.isneginf(got[~bits]).all()
    assert np.isnan(got[:, 6:400:7][bits[:, 6:400:7]]).all()
    assert (got[:, 8:400:7][bits[:, 8:400:7]] == np.inf).all()
    assert np.isneginf(got[:, 5:400:7]).all()
    c.mask[:] = 0
    c.upload()
    assert np.isneginf(c.run()).all()


def test_then_sampled(gpu):
    """The rules and the sampler in one captured step: the only allowed token, then the best that is left."""
    n = 151936
    c = Case(1, n, F32, history=64, biases=3, mask="rows")
    c.mask[:] = 0xFFFFFFFF
    c.upload()
    st, idx = Stream(), capi.DevBuf(4)

    def issue(s):
        capi.call("vvh_logits_rules", c.d_out.ptr, c.d["logits"].ptr, ctypes.byref(c.spec()), 1, n, F32, s)
        capi.call("vvh_argmax", c.d_out.ptr, n, idx.ptr, s)

    issue(st.s)
    st.sync()
    replay = st.capture(issue)
    for step in range(3):
        if step == 1:
            c.mask[:] = 0
            c.mask[0, 1234 // 32] = 1 << 1234 % 32
        if step == 2:
            c.mask[:] = 0xFFFFFFFF
            c.logits[0, 777] = 1e5
            put(c.d["logits"], c.logits)
        put(c.d["mask"], c.mask)
        capi.sync()
        replay()
        y, _ = c.want()
        assert idx.to_array(np.int32, (1,))[0] == (1234 if step == 1 else np.argmax(y[0]))
    st.close()
