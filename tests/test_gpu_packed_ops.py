"""mk_attention_packed, mk_lora_rows and mk_rope_rows against their definitions in 64 bits.

Tolerances. u = 2^-24 is half a step of fp32, H(t) half a step of type t relative to the value: 2^-8 (bf16), 2^-11 (half; 2^-25
absolute below its normal range), 0 added for fp32 outputs beyond the sums' own.
- attention: a score sums d exact products of 16-bit values in chains of at most d additions: |ds| <= (d + 8) u scale sum|q k|; the
  scale, the cap (its slope is at most 1, its own roundings 16 u cap) and the bias (the distance is exact below 2^24) add 4 u |s| +
  16 u cap + 8 u |bias|. exp(s - m) then is off by e = ds + 8 u (|s| + |m|) + 8 u of itself, and so are the weights' sum and, after H(in) for
  the weight's own rounding, each weight: |do| <= H(out) |o| + (H(in) + 2 max e + n u) sum p |v| / l with n keys. Half weights below
  2^-14 of the largest (l >= 1 in its units) lose 2^-25 each.
- adapters: t sums K products in chains of at most K / 8 + 16; as two 16-bit values it keeps H^2, rank products more, and the
  scale and the base one rounding each.
- rotary: the norm's sum over d values and its root 16 u, cosine and sine 4 u absolute and the angle's own error, a product's
  rounding each: 24 u (|x| + |y|) + H(out) of the result."""
import ctypes as C
import math

import numpy as np
import pytest

import mkimage as M

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
H = {M.F32: u, M.BF16: 2.0 ** -8, M.F16: 2.0 ** -11}
GUARD = 0x5A
NP = {M.F32: np.float32, M.BF16: np.uint16, M.F16: np.uint16}
NAME = {M.F32: "f32", M.BF16: "bf16", M.F16: "f16"}


def stored(a, dt):
    """float64 -> (device bits, the float64 values they stand for)"""
    a = np.asarray(a, np.float32)
    if dt == M.F32:
        return a, a.astype(np.float64)
    bits = M.bf16_bits(a) if dt == M.BF16 else M.f16_bits(a)
    return bits, values(bits, dt)


def values(bits, dt):
    if dt == M.F32:
        return bits.astype(np.float64)
    return (M.bf16_to_f32(bits) if dt == M.BF16 else M.f16_to_f32(bits)).astype(np.float64)


class Rows:
    """Rows of width n inside rows of ld elements of a guarded buffer, from column col."""

    def __init__(self, rows, ld, dt, fill=None):
        self.shape, self.dt = (rows, ld), dt
        host = np.full(rows * ld * np.dtype(NP[dt]).itemsize, GUARD, np.uint8).view(NP[dt]).reshape(rows, ld) if fill is None else fill
        self.dev = M.Dev(host.nbytes)
        self.dev.write(host)
        self.before = host

    def at(self, col=0, row=0):
        return self.dev.p + (row * self.shape[1] + col) * np.dtype(NP[self.dt]).itemsize

    def read(self):
        return self.dev.to_array(NP[self.dt], self.shape)


def dev(a):
    return M.Dev.from_array(a)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------

def seen_of(doc, nk):
    q_row, q_rows, k_row, k_rows, q_pos, block, prefix = doc
    pos = q_pos + np.arange(q_rows)[:, None]
    key = np.arange(nk)[None]
    return (block == 0) | (pos >= block) | (key <= pos) | (key < prefix), np.abs(pos - key)


def attend(q, k, v, docs, scale, cap, slopes, dt, out_dt):
    """(out, tolerance) of every row of the documents in 64 bits; rows of none are NaN."""
    rows, heads, d = q.shape
    group = heads // k.shape[1]
    out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for doc in docs:
        q_row, q_rows, k_row, k_rows = doc[:4]
        if not q_rows:
            continue
        see, dist = seen_of(doc, k_rows)
        for h in range(heads):
            qq, kk, vv = q[q_row:q_row + q_rows, h], k[k_row:k_row + k_rows, h // group], v[k_row:k_row + k_rows, h // group]
            o, t = np.zeros((q_rows, d)), np.zeros((q_rows, d))
            for i in range(q_rows):
                on = see[i] if k_rows else np.zeros(0, bool)
                if not on.any():
                    continue
                with np.errstate(all="ignore"):
                    s = kk[on] @ qq[i] * scale
                    ds = (d + 8) * u * scale * (np.abs(kk[on]) @ np.abs(qq[i])) + 4 * u * np.abs(s)
                    if cap:
                        s, ds = cap * np.tanh(s / cap), ds + 16 * u * cap
                    if slopes is not None:
                        bias = float(slopes[h]) * dist[i][on]
                        s, ds = s - bias, ds + 8 * u * np.abs(bias)
                    m = s.max()
                    if m == -np.inf:
                        continue
                    p = np.exp(s - m)
                    l = p.sum()
                    pv = np.where(p[:, None] > 0, p[:, None] * vv[on], np.where(np.isfinite(vv[on]), 0.0, np.nan))
                    o[i] = pv.sum(0) / l
                    # (keys that weigh nothing move nothing: their scores may be -inf)
                    e = 2 * np.max(np.where(p > 1e-30, ds + 8 * u * (np.abs(s) + abs(m)), 0)) + 8 * u + on.sum() * u
                    t[i] = H[out_dt] * np.abs(o[i]) + (H[dt] + e) * (np.abs(pv)).sum(0) / l + (
                        2.0 ** -25 * np.abs(vv[on]).sum(0) / l if dt == M.F16 else 0.0) + (2.0 ** -25 if out_dt == M.F16 else 1e-38)
            out[q_row:q_row + q_rows, h], tol[q_row:q_row + q_rows, h] = o, t
    return out, tol


class Attn:
    """A packed batch on the device: q|k|v in one buffer's rows when `fused`, of nq query and nk key rows."""

    def __init__(self, docs, nq, nk, heads, kv, d, dt, out_dt=None, scale=None, cap=0.0, slopes=None, seed=0, pad=0, gain=1.0, edit=None):
        rng = np.random.default_rng(seed)
        self.docs, self.dt, self.out_dt = docs, dt, out_dt or dt
        self.scale = d ** -0.5 if scale is None else scale
        self.cap, self.slopes = cap, slopes
        raw = {"q": rng.standard_normal((nq, heads, d)) * gain, "k": rng.standard_normal((nk, kv, d)), "v": rng.standard_normal((nk, kv, d))}
        if edit:
            edit(raw)
        self.val, self.buf = {}, {}
        for n, x in raw.items():
            width = x.shape[1] * d
            host = np.full((max(len(x), 1), width + pad), np.nan, np.float32)
            host[:len(x), :width] = x.reshape(len(x), -1)
            bits, v = stored(host, dt)
            self.buf[n] = Rows(*host.shape, dt, fill=bits)
            self.val[n] = v[:len(x), :width].reshape(x.shape)
        self.out = Rows(max(nq, 1), heads * d + pad, self.out_dt)
        self.heads, self.kv, self.d, self.pad = heads, kv, d, pad
        self.keep = [dev(np.asarray(slopes, np.float32))] if slopes is not None else []

    def args(self):
        g = M.AttnPackedArgs()
        g.q, g.k, g.v, g.out = (b.at() for b in (self.buf["q"], self.buf["k"], self.buf["v"], self.out))
        g.ldq, g.ldk, g.ldv, g.ldo = (b.shape[1] for b in (self.buf["q"], self.buf["k"], self.buf["v"], self.out))
        g.dtype, g.out_dtype, g.heads, g.kv_heads, g.d = self.dt, self.out_dt, self.heads, self.kv, self.d
        g.scale, g.cap = self.scale, self.cap
        g.slopes = self.keep[0].p if self.slopes is not None else None
        self.table = (M.AttnDoc * max(len(self.docs), 1))(*[M.AttnDoc(*v) for v in self.docs])
        g.docs, g.n_docs = self.table, len(self.docs)
        return g

    def run(self, workspace=True, stream=None):
        g = self.args()
        if workspace:
            need = C.c_uint64()
            M.call("mk_attention_packed_workspace", C.byref(g), C.byref(need))
            self.space = M.Dev(need.value)
            M.call("mk_memset", self.space.p, 0xFF, max(need.value, 16))
            g.workspace, g.workspace_bytes = self.space.p, need.value
        self.g = g
        M.call("mk_attention_packed", C.byref(g), stream)
        return self

    def result(self):
        M.sync()
        got = self.out.read()
        n = self.heads * self.d
        rest = got[:, n:].tobytes()
        assert rest == self.out.before[:, n:].tobytes(), "columns behind the heads were written"
        mine = np.zeros(len(got), bool)
        for doc in self.docs:
            mine[doc[0]:doc[0] + doc[1]] = True
        assert (got[~mine] == self.out.before[~mine]).all(), "rows of no document were written"
        return got[:, :n].reshape(len(got), self.heads, self.d), mine

    def check(self, workspace=True):
        got, mine = self.run(workspace).result()
        want, tol = attend(self.val["q"], self.val["k"], self.val["v"], self.docs, self.scale, self.cap, self.slopes, self.dt, self.out_dt)
        got = values(got, self.out_dt)[mine]
        want, tol = want[mine], tol[mine]
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan), np.argwhere(np.isnan(got) != nan)[:5]
        ok = (np.abs(got - want) <= tol) | nan | (got == want)
        worst = np.nanmax(np.where(nan, 0, np.abs(got - want) / np.maximum(tol, 1e-300)), initial=0)
        assert ok.all(), (worst, np.argwhere(~ok)[:5])
        return worst


def packed(lens_q, lens_k=None, mask="full", s=None, gap=0, same=True):
    """Documents one after the other, `gap` rows between them."""
    lens_k = lens_k or lens_q
    s = s or [0] * len(lens_q)
    docs, q, k = [], 0, 0
    for a, b, t in zip(lens_q, lens_k, s):
        block = {"full": 0, "causal": 0xFFFFFFFF, "text": t, "prefix": 0xFFFFFFFF}[mask]
        docs.append((q, a, k, b, b - a, block, t if mask == "prefix" else 0))
        q, k = q + a + gap, k + b + gap
    return docs, q + 1, k + 1


MASKS = ["full", "causal", "text", "prefix"]


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", MASKS)
def test_attention_documents(gpu, mask, d, dt):
    lens = [1, 2, 31, 64, 65, 130, 0, 33]
    docs, nq, nk = packed(lens, mask=mask, s=[0, 1, 7, 64, 3, 100, 0, 33], gap=3)
    Attn(docs, nq, nk, 4, 2, d, dt, pad=8, seed=d).check()


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("mask", MASKS)
def test_attention_cap_and_bias(gpu, mask, dt):
    docs, nq, nk = packed([97, 5, 200], mask=mask, s=[20, 5, 64])
    slopes = np.float32([0.5, 0.03125, 0.0, 2.0])
    for cap, sl in ((20.0, None), (0.0, slopes), (7.5, slopes)):
        Attn(docs, nq, nk, 4, 4, 64, dt, cap=cap, slopes=sl, gain=3.0).check()
        Attn(docs, nq, nk, 4, 1, 128, dt, cap=cap, slopes=sl, gain=3.0).check()


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("heads, kv, d", [(8, 1, 128), (8, 8, 64), (6, 2, 128), (5, 1, 64), (40, 2, 64)])
@pytest.mark.parametrize("mask", ["full", "causal"])
def test_attention_few_rows_over_many_keys(gpu, mask, heads, kv, d, workspace):
    docs, nq, nk = packed([1, 3, 1, 7], [4099, 777, 1, 1500], mask=mask)
    slopes = np.float32(2.0 ** -np.arange(1, heads + 1) / 16)
    Attn(docs, nq, nk, heads, kv, d, M.BF16).check(workspace)
    Attn(docs, nq, nk, heads, kv, d, M.F16, slopes=slopes, cap=30.0, gain=2.0).check(workspace)


@pytest.mark.parametrize("lens_q, lens_k", [([5], [0]), ([5, 3], [0, 4]), ([40], [9]), ([300, 4], [64, 200]), ([1], [1]), ([129], [1]),
                                            ([1, 1, 1], [63, 64, 65]), ([127, 128, 129], [127, 128, 129])])
@pytest.mark.parametrize("mask", ["full", "causal", "prefix"])
def test_attention_rows_that_see_nothing_and_edges(gpu, mask, lens_q, lens_k):
    # more query rows than keys under a causal mask: the first have negative positions
    docs, nq, nk = packed(lens_q, lens_k, mask=mask, s=[min(2, n) if mask == "prefix" and i else 0 for i, n in enumerate(lens_k)])
    for dt in (M.BF16, M.F16):
        a = Attn(docs, nq, nk, 3, 3, 128, dt, pad=16)
        a.check()


def test_attention_empty_rows_are_zero(gpu):
    docs, nq, nk = packed([70], [6], mask="causal")
    a = Attn(docs, nq, nk, 2, 2, 64, M.BF16)
    got, mine = a.run().result()
    assert (got[:64] == 0).all() and (values(got[64:70], M.BF16) != 0).any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("mask", ["full", "causal", "text"])
def test_attention_unseen_rows_reach_nothing(gpu, mask, where, bad):
    # the rows between the documents, and under causal masks the last keys of each
    docs, nq, nk = packed([100, 33, 65], mask=mask, s=[50, 33, 2], gap=5)

    def edit(raw):
        x = raw[where]
        for doc in docs:
            x[doc[2] + doc[3]:doc[2] + doc[3] + 5] = bad
            if mask == "causal":
                x[doc[2] + doc[3] - 1] = bad
                x[doc[2] + doc[3] // 2, 0, 3] = bad
        x[-1] = bad

    for d in (64, 128):
        a = Attn(docs, nq, nk, 2, 2, d, M.BF16, edit=edit)
        got, mine = a.run().result()
        got = values(got, M.BF16)
        want, tol = attend(a.val["q"], a.val["k"], a.val["v"], docs, a.scale, 0.0, None, M.BF16, M.BF16)
        with np.errstate(all="ignore"):
            fine = np.isfinite(want)
            assert np.isfinite(got[fine & mine[:, None, None]]).all()
            assert (np.abs(got - want)[fine] <= tol[fine]).all()
            if where == "v":  # a seen infinity or NaN shows
                assert not np.isfinite(got[~fine & mine[:, None, None]]).any()


def test_attention_scores_far_apart_and_large(gpu):
    # scores to +-1e4 in log units, ascending so that the running maximum moves in every tile; equal scores; tiny ones
    n = 333

    def edit(raw):
        raw["q"][:] = 1.0
        raw["k"][:, 0] = np.linspace(-30, 30, len(raw["k"]))[:, None]
        raw["k"][:, 1] = 0.125
        raw["k"][:, 2] = np.linspace(30, -30, len(raw["k"]))[:, None]

    for dt in (M.BF16, M.F16):
        for scale in (1.0, 1e-3, 0.0, 8.0):
            docs, nq, nk = packed([n, 64])
            Attn(docs, nq, nk, 3, 3, 128, dt, scale=scale, edit=edit).check()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("level", [23, 24, 26, 28, 31, 34, 60, 100, 120])
@pytest.mark.parametrize("dt", [M.BF16, M.F16])
def test_attention_scores_of_any_size(gpu, dt, level, sign):
    """Scores of 1, 2 or 3 times 1 to 2 x 2^level: the largest ones' keys share the weight, however far the scores are from fp32's
    integers (half a step of a score passes a weight's exponent range from 2^31 on)."""
    for d, heads, kv, rows, nk, workspace, by in ((128, 4, 1, 3, 300, True, 1.1), (64, 2, 2, 40, 130, False, 1.3), (128, 2, 2, 140, 70, True, 1.7), (64, 4, 2, 40, 130, True, 1.9)):
        def edit(raw):
            raw["q"][:] = 0.0
            raw["q"][:, :, 5] = 1.0
            raw["k"][:] = 0.0
            raw["k"][:, :, 5] = sign * (1 + np.random.default_rng(level).integers(0, 3, raw["k"].shape[:2]))
        a = Attn([(0, rows, 0, nk, nk - rows, 0xFFFFFFFF, 0)], rows, nk, heads, kv, d, dt, scale=float(np.float32(by * 2.0 ** level)), edit=edit)
        # the score's rounding moves all equal scores alike: the tolerance counts that of the weights and sums alone
        want, _ = attend(a.val["q"], a.val["k"], a.val["v"], a.docs, a.scale, 0.0, None, dt, dt)
        got = values(a.run(workspace).result()[0], dt)
        v = np.abs(a.val["v"]).max()
        np.testing.assert_allclose(got, want, rtol=0, atol=(2 * H[dt] + nk * u) * v)


def test_attention_minus_infinity_scores(gpu):
    # keys whose score is -inf weigh nothing; a row of only such keys is zero
    docs, nq, nk = packed([4, 4], [80, 3])

    def edit(raw):
        raw["q"][:] = np.abs(raw["q"]) + 0.1
        raw["k"][::2, 0, 0] = -np.inf
        raw["k"][80:83, 0, 0] = -np.inf

    a = Attn(docs, nq, nk, 1, 1, 64, M.BF16, edit=edit)
    got, _ = a.run().result()
    want, tol = attend(a.val["q"], a.val["k"], a.val["v"], docs, a.scale, 0.0, None, M.BF16, M.BF16)
    got = values(got, M.BF16)
    assert (np.abs(got - want)[:8] <= tol[:8]).all() and (got[4:8] == 0).all()


def test_attention_shared_keys_and_order(gpu):
    # two documents over one prompt's keys, documents in any order, one empty
    docs = [(50, 20, 0, 90, 70, 0, 0), (0, 33, 0, 90, 57, 0xFFFFFFFF, 0), (33, 0, 5, 0, 0, 0, 0), (40, 10, 10, 64, 0, 0xFFFFFFFF, 20)]
    Attn(docs, 75, 90, 4, 2, 128, M.BF16).check()


def test_attention_more_documents_than_a_launch(gpu):
    lens = [1 + i % 5 for i in range(230)]
    docs, nq, nk = packed(lens, mask="causal")
    Attn(docs, nq, nk, 2, 1, 64, M.F16).check()


def test_attention_output_type_and_same_bits_again(gpu):
    docs, nq, nk = packed([200, 9], mask="causal")
    for dt, out in ((M.BF16, M.F16), (M.F16, M.BF16)):
        a = Attn(docs, nq, nk, 4, 4, 128, dt, out_dt=out)
        a.check()
        one = a.run().result()[0].copy()
        assert np.array_equal(one, a.run().result()[0])


# ---------------------------------------------------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------------------------------------------------

class Lora:
    def __init__(self, rows, K, N, rank, parts, adapters, ids, dt, c_dt, seed=0, pad=0, base=True, scale=True, in_place=False, edit=None, grouped=0):
        rng = np.random.default_rng(seed)
        self.grouped = grouped
        self.sizes, self.dt, self.c_dt, self.pad = (rows, K, N, rank, parts, adapters), dt, c_dt, pad
        raw = {"x": rng.standard_normal((rows, K)) * np.exp(rng.standard_normal(K) * 0.5), "a": rng.standard_normal((adapters, parts * rank, K)) * K ** -0.5,
               "b": rng.standard_normal((adapters, N, rank)) * rank ** -0.5, "base": rng.standard_normal((rows, N))}
        if edit:
            edit(raw)
        self.val, self.buf = {}, {}
        for n, x in raw.items():
            t = c_dt if n == "base" else dt
            ld = x.shape[-1] + (pad if n in ("x", "base") else 0)
            host = np.full((int(np.prod(x.shape[:-1])), ld), np.nan, np.float32)
            host[:, :x.shape[-1]] = x.reshape(-1, x.shape[-1])
            bits, v = stored(host, t)
            self.buf[n], self.val[n] = Rows(*host.shape, t, fill=bits), v[:, :x.shape[-1]].reshape(x.shape)
        self.ids = None if ids is None else np.asarray(ids, np.int32)
        self.scale = np.exp(rng.standard_normal(adapters) * 0.5).astype(np.float32) if scale else None
        self.c = self.buf["base"] if in_place else Rows(rows, N + pad, c_dt)
        self.base = base
        self.keep = [dev(self.ids) if self.ids is not None else None, dev(self.scale) if scale else None]

    def args(self):
        g = M.LoraRowsArgs()
        g.x, g.a, g.b = (self.buf[n].at() for n in ("x", "a", "b"))
        g.base = self.buf["base"].at() if self.base else None
        g.c = self.c.at()
        g.ids, g.scale = (k.p if k else None for k in self.keep)
        g.ldx, g.ldbase, g.ldc = self.buf["x"].shape[1], self.buf["base"].shape[1], self.c.shape[1]
        g.rows, g.K, g.N, g.rank, g.parts, g.adapters = self.sizes
        g.dtype, g.c_dtype, g.grouped = self.dt, self.c_dt, self.grouped
        need = C.c_uint64()
        M.call("mk_lora_rows_workspace", C.byref(g), C.byref(need))
        self.space = M.Dev(need.value)
        M.call("mk_memset", self.space.p, 0xFF, max(need.value, 16))
        g.workspace, g.workspace_bytes = self.space.p, need.value
        return g

    def run(self, stream=None):
        self.g = self.args()
        M.call("mk_lora_rows", C.byref(self.g), stream)
        return self

    def result(self):
        M.sync()
        got, N = self.c.read(), self.sizes[2]
        assert got[:, N:].tobytes() == self.c.before[:, N:].tobytes(), "columns behind N were written"
        return values(got[:, :N], self.c_dt)

    def want(self):
        rows, K, N, rank, parts, adapters = self.sizes
        x, c = self.val["x"], (self.val["base"].copy() if self.base else np.zeros((rows, N)))
        tol = np.zeros((rows, N))
        ids = self.ids if self.ids is not None else np.zeros(rows, int)
        w = N // parts
        with np.errstate(all="ignore"):
            for a in range(adapters):
                r = np.flatnonzero(ids == a)
                if not len(r):
                    continue
                s = float(self.scale[a]) if self.scale is not None else 1.0
                t, ta = x[r] @ self.val["a"][a].T, np.abs(x[r]) @ np.abs(self.val["a"][a]).T
                dt = (K / 8 + 16) * u * ta
                for p in range(parts):
                    b = self.val["b"][a, p * w:(p + 1) * w]
                    j = slice(p * rank, (p + 1) * rank)
                    c[r, p * w:(p + 1) * w] += s * (t[:, j] @ b.T)
                    # (the row's largest t scales half values: its smallest ones keep 2^-22 of that)
                    big = np.abs(t[:, j]).max(1, keepdims=True) + np.zeros_like(t[:, j])
                    e = dt[:, j] + H[self.dt] ** 2 * np.maximum(np.abs(t[:, j]), big * 2.0 ** -6) + (rank + 8) * u * np.abs(t[:, j])
                    tol[r, p * w:(p + 1) * w] = s * (e @ np.abs(b).T)
            tol += (H[self.c_dt] + 2 * u) * np.abs(c) + 2 * u * np.abs(self.val["base"]) + (2.0 ** -25 if self.c_dt == M.F16 else 1e-38)
        return c, tol

    def check(self):
        got = self.run().result()
        want, tol = self.want()
        nan = ~np.isfinite(want)
        assert np.array_equal(~np.isfinite(got), nan)
        err = np.where(nan, 0, np.abs(np.where(nan, 0, got) - np.where(nan, 0, want)))
        assert (err[~nan] <= tol[~nan]).all(), (np.nanmax(err / tol), np.argwhere(err > tol)[:5])


LORA_SIZES = [(1, 8, 8, 8, 1, 1), (1, 4096, 264, 16, 1, 3), (5, 72, 24, 8, 3, 2), (17, 520, 144, 24, 2, 5), (33, 64, 512, 40, 1, 4), (64, 256, 256, 16, 4, 64),
              (65, 1000, 1032, 64, 1, 3), (130, 128, 96, 128, 3, 2), (200, 136, 128, 256, 1, 2), (300, 2056, 776, 8, 1, 7), (513, 64, 48, 32, 3, 3)]


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("rows, K, N, rank, parts, adapters", LORA_SIZES)
def test_lora_rows(gpu, rows, K, N, rank, parts, adapters, dt):
    rng = np.random.default_rng(rows + K)
    mixed = rng.integers(-1, adapters, rows)
    runs = np.sort(rng.integers(0, adapters, rows))
    runs[rows // 2:rows // 2 + 3] = -1
    for c_dt, ids, pad in ((dt, mixed, 8), (M.F32, runs, 0)):
        Lora(rows, K, N, rank, parts, adapters, ids, dt, c_dt, pad=pad).check()


@pytest.mark.parametrize("c_dt", [M.F32, M.F16], ids=NAME.get)
@pytest.mark.parametrize("adapters, seen", [(2, 2), (7, 5), (1024, 1024), (1025, 300), (64, 1)])
def test_lora_many_rows_in_no_order(gpu, adapters, seen, c_dt):
    # sizes whose products go by tiles: 2^26 of them and more in both
    rows, K, N, rank = 4500, 512, 512, 32
    rng = np.random.default_rng(adapters)
    ids = rng.integers(-1, seen, rows) * (adapters // seen)
    for kw in (dict(), dict(in_place=True), dict(grouped=1)):
        Lora(rows, K, N, rank, 1, adapters, ids, M.F16, c_dt, pad=8, **kw).check()


@pytest.mark.parametrize("rows", [3, 150])
def test_lora_without_base_scale_or_ids_and_in_place(gpu, rows):
    for kw in (dict(base=False), dict(scale=False), dict(ids=None), dict(in_place=True), dict(base=False, ids=[-1] * rows),
               dict(ids=[-1] * rows), dict(ids=[2 ** 31 - 1, -2 ** 31, 3] * (rows // 3))):
        kw = dict(dict(ids=np.arange(rows) % 3), **kw)
        Lora(rows, 136, 72, 16, 3, 3, kw.pop("ids"), M.BF16, M.BF16, pad=16, **kw).check()


@pytest.mark.parametrize("rows", [6, 130])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_lora_infinities_stay_with_their_rows(gpu, rows, bad):
    def edit(raw):
        raw["x"][1, 3] = bad
        raw["a"][2, 5, 7] = bad
        raw["b"][3, 9, 1] = bad

    for dt in (M.BF16, M.F16):
        Lora(rows, 72, 64, 8, 1, 5, np.arange(rows) % 5, dt, M.F32, edit=edit).check()


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("c_dt", [M.F32, M.BF16], ids=NAME.get)
@pytest.mark.parametrize("rank", [32, 64, 128])
def test_lora_the_same_bits_on_every_run_of_many_tiles(gpu, rank, c_dt, dt):
    # (fp32 rows once came out with a few values of other registers, in some tiles of a large launch)
    rows, K, N = 4100, 256, 2048
    a = Lora(rows, K, N, rank, 1, 3, np.arange(rows) * 3 // rows, dt, c_dt)
    first = a.run().result()
    want, tol = a.want()
    assert (np.abs(first - want) <= tol).all()
    for _ in range(5):
        assert np.array_equal(a.run().result(), first)


def test_lora_half_values_of_any_size(gpu):
    # t beyond the half range, and far below it
    def edit(raw):
        raw["x"][0] *= 1e3
        raw["a"][0] = np.abs(raw["a"][0]) * 1e2
        raw["x"][0] = np.abs(raw["x"][0])
        raw["x"][1] *= 1e-3
        raw["b"][:] *= 1e-2

    for rows in (4, 100):
        Lora(rows, 2048, 64, 16, 1, 2, np.arange(rows) % 2, M.F16, M.F32, edit=edit).check()


# ---------------------------------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------------------------------

class Rope:
    def __init__(self, rows, heads, kv, d, dims, dt, out_dt, mode=1, series=0, norm=True, pos=None, pos_dt=None, pad=0, in_place=False, theta=10000.0,
                 k_scale=0.0, seed=0, far=100):
        rng = np.random.default_rng(seed)
        self.rows, self.heads, self.kv, self.d, self.dims = rows, heads, kv, d, dims
        self.dt, self.out_dt, self.mode, self.series, self.theta, self.k_scale, self.pad = dt, out_dt, mode, series, theta, k_scale, pad
        self.pos_dt = M.I32 if pos_dt is None else pos_dt
        pos = rng.integers(-far, far, (rows, len(dims))) if pos is None else np.asarray(pos)
        self.pos = pos.astype(np.int32 if self.pos_dt == M.I32 else np.float32)
        self.val, self.buf, self.out = {}, {}, {}
        for n, h in (("q", heads), ("k", kv)):
            host = np.full((rows, h * d + pad), np.nan, np.float32)
            host[:, :h * d] = rng.standard_normal((rows, h * d)) * 2
            bits, v = stored(host, dt)
            self.buf[n], self.val[n] = Rows(*host.shape, dt, fill=bits), v[:, :h * d].reshape(rows, h, d)
            self.out[n] = self.buf[n] if in_place else Rows(rows, h * d + pad, out_dt)
        self.w = {n: (1 + 0.1 * rng.standard_normal(d)).astype(np.float32) if norm else None for n in "qk"}
        self.keep = [dev(self.w["q"]), dev(self.w["k"])] if norm else []
        self.dpos = dev(self.pos)

    def args(self):
        g = M.RopeRowsArgs()
        g.q, g.q_out, g.ldq, g.ldqo = self.buf["q"].at(), self.out["q"].at(), self.buf["q"].shape[1], self.out["q"].shape[1]
        if self.kv:
            g.k, g.k_out, g.ldk, g.ldko = self.buf["k"].at(), self.out["k"].at(), self.buf["k"].shape[1], self.out["k"].shape[1]
        g.rows, g.heads, g.kv_heads, g.d, g.dtype, g.out_dtype = self.rows, self.heads, self.kv, self.d, self.dt, self.out_dt
        if self.keep:
            g.norm_q, g.norm_k, g.eps = self.keep[0].p, self.keep[1].p, 1e-6
        g.k_scale = self.k_scale
        g.pos, g.pos_ld, g.pos_dtype = self.dpos.p, self.pos.shape[1] if len(self.pos) > 1 or self.rows == 1 else 0, self.pos_dt
        g.axes = len(self.dims)
        g.axis_dims = (C.c_uint32 * 4)(*self.dims)
        g.theta, g.series, g.rope_mode = self.theta, self.series, self.mode
        return g

    def run(self, stream=None):
        self.g = self.args()
        M.call("mk_rope_rows", C.byref(self.g), stream)
        return self

    def want(self, n):
        R = sum(self.dims)
        x = self.val[n].copy()
        if self.w[n] is not None:
            x = x / np.sqrt((x * x).mean(2, keepdims=True) + float(np.float32(1e-6))) * self.w[n].astype(np.float64)
        if n == "k" and self.k_scale:
            x = x * float(np.float32(self.k_scale))
        y, size = x.copy(), np.abs(x)
        pair = 0
        for a, dim in enumerate(self.dims):
            for j in range(dim // 2):
                f = np.longdouble(self.theta) ** (np.longdouble(-2) * (j if self.series == 0 else pair) / (dim if self.series == 0 else R))
                pos = np.broadcast_to(self.pos[:, a], self.rows).astype(np.longdouble)
                with np.errstate(invalid="ignore"):
                    c, s = np.cos(pos * f)[:, None].astype(np.float64), np.sin(pos * f)[:, None].astype(np.float64)
                e = 2 * math.pi * 2.0 ** -31 * (1 + (np.abs(np.where(np.isfinite(pos), pos, 0)) * 2.0 ** -20 if self.pos_dt == M.F32 else 0 * pos))[:, None].astype(np.float64)
                i, k = (pair, pair + R // 2) if self.mode == 1 else (2 * pair, 2 * pair + 1)
                y[..., i], y[..., k] = x[..., i] * c - x[..., k] * s, x[..., i] * s + x[..., k] * c
                both = np.abs(x[..., i]) + np.abs(x[..., k])
                size[..., i] = size[..., k] = both * (1 + e / (24 * u))
                pair += 1
        return y, 24 * u * size + H[self.out_dt] * np.abs(y) + (2.0 ** -25 if self.out_dt == M.F16 else 0)

    def check(self):
        self.run()
        M.sync()
        for n, h in (("q", self.heads), ("k", self.kv)):
            got = self.out[n].read()
            assert got[:, h * self.d:].tobytes() == self.out[n].before[:, h * self.d:].tobytes()
            if not h:
                continue
            got = values(got[:, :h * self.d], self.out_dt).reshape(self.rows, h, self.d)
            want, tol = self.want(n)
            nan = np.isnan(want)
            assert np.array_equal(np.isnan(got), nan)
            ok = (np.abs(got - want) <= tol) | nan
            assert ok.all(), (n, np.nanmax(np.abs(got - want) / tol), np.argwhere(~ok)[:5])


DIMS = {128: [[128], [16, 56, 56], [32, 48, 48], [40, 24], [2, 2, 2, 2]], 64: [[64], [16, 24, 24], [8], [10, 6, 20, 4]]}


@pytest.mark.parametrize("d, dims", [(d, v) for d in DIMS for v in DIMS[d]])
@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("series", [0, 1])
def test_rope_axes(gpu, d, dims, mode, series):
    Rope(37, 5, 3, d, dims, M.F32, M.F32, mode, series, pad=4).check()
    Rope(6, 3, 0, d, dims, M.BF16, M.F16, mode, series, norm=False, pos_dt=M.F32, pos=np.random.default_rng(1).uniform(-50, 50, (6, len(dims)))).check()


@pytest.mark.parametrize("dt", [M.F32, M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("out", [M.F32, M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("rows, heads, kv", [(1, 32, 8), (3, 1, 1), (2050, 7, 2)])
def test_rope_types_and_rows(gpu, rows, heads, kv, dt, out):
    Rope(rows, heads, kv, 128, [16, 56, 56], dt, out, k_scale=0.125).check()
    Rope(rows, heads, kv, 64, [16, 24, 16], dt, out, mode=2, norm=False).check()


@pytest.mark.parametrize("dt", [M.F32, M.BF16, M.F16], ids=NAME.get)
def test_rope_in_place(gpu, dt):
    for mode in (1, 2):
        for rows in (5, 2100):
            Rope(rows, 6, 6, 64, [16, 24, 16], dt, dt, mode, in_place=True, pad=8).check()


@pytest.mark.parametrize("pos_dt", [M.I32, M.F32])
def test_rope_far_positions(gpu, pos_dt):
    far = [0, 1, -1, 2 ** 20, -2 ** 20 - 1, 2 ** 24 - 1, -(2 ** 31), 2 ** 31 - 128, 10 ** 9]
    pos = np.array([[a, b] for a, b in zip(far, reversed(far))])
    for theta in (1.0, 10000.0, 1e6):
        Rope(len(far), 2, 2, 128, [64, 64], M.F32, M.F32, pos=pos, pos_dt=pos_dt, theta=theta, norm=False).check()


def test_rope_one_row_of_positions_for_all_and_not_numbers(gpu):
    Rope(9, 2, 1, 64, [32, 32], M.F32, M.F32, pos=np.array([[3, 77]])).check()
    Rope(4, 2, 1, 64, [32, 16], M.F32, M.F32, pos=np.array([[1, np.nan], [np.inf, 2], [0.25, -3.75], [-np.inf, 0]]), pos_dt=M.F32).check()
