"""mk_gemm_i8, mk_gate_norm and mk_quantize_i8_rows against their definitions in 64 bits.

Tolerances. u = 2^-24 is half a step of fp32. A stored 16-bit value adds half its step, relative 2^-8 (bf16) or 2^-11
(half, absolute 2^-25 below its normal range). The int8 product's sum is exact, so its value carries the roundings of the
scaled sum: float(sum), two products and an addition, 4 u (|p| + |b|) with p the scaled sum. The activations add those of
their own instructions: exp2 and rcp, 1 ulp (2 u) each, on an argument that the roundings of t before it move by
2 u |t| absolutely each, so a sigmoid is off by at most (8 + 4 |t|) u of itself, and its slope times |t| stays below 1."""
import ctypes as C

import numpy as np
import pytest
from scipy.special import erf

import mkimage as M

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
HALF = {M.F32: 0.0, M.BF16: 2.0 ** -8, M.F16: 2.0 ** -11}
GUARD = 0x5A


def dev_bytes(n):
    d = M.Dev(n)
    M.call("mk_memset", d.p, GUARD, n)
    return d


def stored(a, dt):
    """float64 -> (device array bits, the float64 values they stand for)"""
    a = np.asarray(a, np.float32)
    if dt == M.F32:
        return a, a.astype(np.float64)
    bits = M.bf16_bits(a) if dt == M.BF16 else M.f16_bits(a)
    return bits, (M.bf16_to_f32(bits) if dt == M.BF16 else M.f16_to_f32(bits)).astype(np.float64)


NP = {M.F32: np.float32, M.BF16: np.uint16, M.F16: np.uint16, M.I8: np.int8}
BYTES = {M.F32: 4, M.BF16: 2, M.F16: 2, M.I8: 1}


def values(bits, dt):
    if dt == M.BF16:
        return M.bf16_to_f32(bits).astype(np.float64)
    if dt == M.F16:
        return M.f16_to_f32(bits).astype(np.float64)
    return bits.astype(np.float64)


def codes_of(v):
    """int8 codes and fp32 scales of float64 rows. In 64 bits 127 v / a is exact half way between two codes and on the
    right side of it elsewhere: v and a have 24 bits, so it is 2^-33 or more away."""
    a = np.abs(v).max(1, keepdims=True)
    zero = a < 2.0 ** -100
    q = np.rint(np.where(zero, 0.0, 127.0 * v / np.where(zero, 1.0, a)))
    s = np.where(zero, np.float32(1), a.astype(np.float32) / np.float32(127))
    return q.astype(np.int8), s[:, 0].astype(np.float32)


# ---------------------------------------------------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------------------------------------------------

def quantize(bits, dt, rows, cols, ld, stream=None, offset=0):
    """offset: elements from the start of the allocation to the first row (alignment)"""
    src = M.Dev(offset * BYTES[dt] + bits.nbytes)
    src.write(bits, offset * BYTES[dt])
    q, s = dev_bytes(rows * cols + 64), dev_bytes(rows * 4 + 64)
    M.call("mk_quantize_i8_rows", src.p + offset * BYTES[dt], dt, rows, cols, ld, q.p, s.p, stream)
    M.sync()
    out = q.to_array(np.int8, rows * cols + 64)
    sc = s.to_array(np.uint8, rows * 4 + 64)
    assert (out[rows * cols:] == GUARD).all() and (sc[rows * 4:] == GUARD).all()
    return out[:rows * cols].reshape(rows, cols), sc[:rows * 4].view(np.float32)


@pytest.mark.parametrize("dt", [M.F32, M.BF16, M.F16])
@pytest.mark.parametrize("rows, cols, pad, offset", [
    (1, 1, 0, 0), (1, 16, 0, 0), (3, 5, 2, 0), (2, 64, 0, 0), (7, 1000, 0, 0), (5, 4096, 0, 0), (300, 272, 16, 0),
    (4, 12288, 0, 0), (3, 16400, 0, 0), (5, 1536, 0, 0), (3, 1552, 16, 0), (3, 3056, 0, 0),
    (2, 8192, 0, 0), (2, 24576, 0, 0), (1, 65536, 0, 0), (1, 65552, 0, 0), (2, 40000, 0, 0),
    (2, 33333, 3, 0), (9, 256, 0, 1), (2, 1024, 8, 4), (1100, 80, 0, 0)])
def test_quantize_rows_equal_the_definition(gpu, dt, rows, cols, pad, offset):
    rng = np.random.default_rng(rows * 7 + cols)
    x = rng.standard_normal((rows, cols + pad)) * np.exp(rng.standard_normal((rows, 1)) * 3)
    x[:, cols:] = 1e4  # what lies between the rows is not theirs
    bits, v = stored(x, dt)
    q, s = quantize(bits, dt, rows, cols, cols + pad, offset=offset)
    wq, ws = codes_of(v[:, :cols])
    assert np.array_equal(s.view(np.uint32), ws.view(np.uint32))
    assert np.array_equal(q, wq)


@pytest.mark.parametrize("cols", [64, 77, 20000])
def test_quantize_ties_go_to_even(gpu, cols):
    # every middle between two codes: a = 254 m, v = +-(2 k + 1) m, for powers m, and their neighbours
    rows = []
    for m in (1.0, 2.0 ** -60, 2.0 ** 90, 0.7):
        m = float(np.float32(m))
        mid = np.float32((2 * np.arange(0, 32) + 1) * m)
        for v in (mid, -mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(np.inf))):
            r = np.zeros(cols, np.float32)
            r[:32] = v
            r[-1] = np.float32(254 * m)
            rows.append(r)
    x = np.array(rows)
    q, s = quantize(x, M.F32, len(x), cols, cols)
    wq, ws = codes_of(x.astype(np.float64))
    assert np.array_equal(s, ws) and np.array_equal(q, wq)
    # m = 1: (2 k + 1) / 2 to even
    assert list(q[0, :4]) == [0, 2, 2, 4] and list(q[1, :4]) == [0, -2, -2, -4]


@pytest.mark.parametrize("cols", [48, 50, 17000])
@pytest.mark.parametrize("dt", [M.F32, M.BF16])
def test_quantize_zero_tiny_and_nonfinite_rows(gpu, dt, cols):
    x = np.random.default_rng(1).standard_normal((9, cols)).astype(np.float32)
    x[1] = 0
    x[2] = x[2] * 2.0 ** -120
    x[3, cols // 2] = np.inf
    x[4, cols - 1] = -np.inf
    x[5, 0] = np.nan
    x[6, 1:3] = np.nan, np.inf
    x[7, 5] = 3.3e38
    bits, v = stored(x, dt)
    q, s = quantize(bits, dt, 9, cols, cols)
    for r in (3, 4, 5, 6):
        assert np.isnan(s[r]) and not q[r].any()
    for r in (1, 2):
        assert s[r] == 1 and not q[r].any()
    for r in (0, 7, 8):
        wq, ws = codes_of(v[r:r + 1])
        assert s[r] == ws[0] and np.array_equal(q[r], wq[0])


# ---------------------------------------------------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------------------------------------------------

class Product:
    def __init__(self, m, n, k, epi=M.EPI_STORE, c=M.F32, batch=1, lda=None, ldc=None, bias=True, split=0, seg=0,
                 extremes=False, seed=0, offset=0):
        rng = np.random.default_rng(seed + m + 3 * n + 5 * k)
        self.m, self.n, self.k, self.epi, self.c, self.batch = m, n, k, epi, c, batch
        self.glu = epi in (M.EPI_SWIGLU, M.EPI_GEGLU)
        self.rmw = epi in (M.EPI_GATE_ADD, M.EPI_GATE_TANH, M.EPI_ADD)
        self.cols = n // 2 if self.glu else n
        self.lda, self.ldc = lda or k, ldc or self.cols
        self.sa, self.sc = self.lda * m + 32, self.ldc * m + 8
        self.A = np.full((batch * self.sa), 99, np.int8)
        lo = -128 if extremes else -127
        a = np.full((batch, m, k), lo, np.int8) if extremes else rng.integers(lo, 128, (batch, m, k), dtype=np.int8)
        for b in range(batch):
            for r in range(m):
                self.A[b * self.sa + r * self.lda: b * self.sa + r * self.lda + k] = a[b, r]
        self.W = np.full((n, k), lo, np.int8) if extremes else rng.integers(lo, 128, (n, k), dtype=np.int8)
        spread = 127.0 * 127.0 * np.sqrt(k) / 3 if not extremes else 128.0 * 128.0 * k
        self.asc = (np.exp(rng.standard_normal((batch, m)) * 0.5) / spread).astype(np.float32)
        self.wsc = np.exp(rng.standard_normal(n) * 0.5).astype(np.float32)
        self.bias = rng.standard_normal(n).astype(np.float32) if bias else None
        self.gate = rng.standard_normal(3 * n).astype(np.float32)
        self.split, self.seg, self.offset = split, seg, offset
        self.x = rng.standard_normal((batch, m, self.cols)).astype(np.float32)
        p = np.einsum("bmk,nk->bmn", a.astype(np.float64), self.W.astype(np.float64), optimize=True)
        p = p * self.asc[..., None].astype(np.float64) * self.wsc.astype(np.float64)
        self.pre = p + (self.bias if bias else 0.0)
        self.mag = np.abs(p) + (np.abs(self.bias) if bias else 0.0)

    def want(self):
        """The definition's values and how far the kernel's may be off."""
        v, e = self.pre, 4 * u * self.mag
        if self.epi == M.EPI_GELU_TANH:
            t = np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
            y = v / (1 + np.exp(-2 * t))
            # slope of GELU below 1.13; the fit's argument 2 t in log2 units has 4 roundings
            return y, 1.13 * e + np.abs(y) * (8 + 8 * np.abs(2 * t)) * u + 1e-30
        if self.epi == M.EPI_SILU:
            y = v / (1 + np.exp(-v))
            return y, 1.1 * e + np.abs(y) * (8 + 4 * np.abs(v)) * u
        if self.glu:
            f = self.cols
            a, b, ea, eb = v[..., :f], v[..., f:], e[..., :f], e[..., f:]
            if self.epi == M.EPI_SWIGLU:
                s = a / (1 + np.exp(-a))
                return s * b, np.abs(b) * (1.1 * ea + np.abs(s) * (8 + 4 * np.abs(a)) * u) + np.abs(s) * eb + 4 * u * np.abs(s * b)
            g = 0.5 * b * (1 + erf(b * np.sqrt(0.5)))
            # z Phi(-z) is fitted within 8.5e-8; exp2 and the polynomial's roundings add less than 16 u of values below z / 2
            return a * g, np.abs(g) * ea + np.abs(a) * (1.13 * eb + 0.5 * np.abs(b) * (2e-7 + 32 * u)) + 4 * u * np.abs(a * g)
        if self.rmw:
            row = np.arange(self.m) % (self.seg or 1 << 32)
            at = np.where(row < self.split, 2 * self.n, 0)[:, None] + np.arange(self.n)
            g = np.ones((self.m, self.n)) if self.epi == M.EPI_ADD else self.gate[at].astype(np.float64)
            eg = 0
            if self.epi == M.EPI_GATE_TANH:
                eg = (16 + 8 * np.abs(g)) * u  # 2 sigmoid(2 g) - 1: twice a sigmoid's error
                g = np.tanh(g)
            return self.x + g * v, np.abs(g) * e + np.abs(v) * eg + 2 * u * (np.abs(self.x) + 2 * np.abs(g * v))
        return v, e

    def run(self, stream=None, rows=None):
        """C as float64 [batch][m][cols]; what lies around it is checked to be left alone."""
        size = BYTES[self.c]
        self.dA = M.Dev(self.offset + self.A.nbytes)
        self.dA.write(self.A, self.offset)
        self.dW, self.dS, self.dWs = (M.Dev.from_array(t) for t in (self.W, self.asc, self.wsc))
        self.dB = M.Dev.from_array(self.bias) if self.bias is not None else None
        self.dG = M.Dev.from_array(self.gate)
        self.dC = dev_bytes(self.batch * self.sc * size + 64)
        if self.rmw:
            c = np.frombuffer(bytes([GUARD]) * self.dC.nbytes, np.uint8).copy()
            f = c[:self.batch * self.sc * 4].view(np.float32)
            for b in range(self.batch):
                for r in range(self.m):
                    f[b * self.sc + r * self.ldc: b * self.sc + r * self.ldc + self.cols] = self.x[b, r]
            self.dC.write(c)
        g = self.args(self.dC)
        if rows:
            g.M = rows
        M.call("mk_gemm_i8", C.byref(g), self.dS.p, stream)
        M.sync()
        return self.read(self.dC, rows)

    def args(self, c):
        g = M.GemmArgs()
        g.a, g.w, g.wscale, g.c = self.dA.p + self.offset, self.dW.p, self.dWs.p, c.p
        g.bias = self.dB.p if self.dB else None
        g.gate, g.gate_alt, g.split, g.seg_rows = self.dG.p, 2 * self.n, self.split, self.seg
        g.M, g.N, g.K, g.lda, g.ldc, g.stride_a, g.stride_c = self.m, self.n, self.k, self.lda, self.ldc, self.sa, self.sc
        g.batch, g.w_dtype, g.c_dtype, g.epilogue = self.batch, M.I8, self.c, self.epi
        return g

    def read(self, c, rows=None):
        raw = c.to_array(np.uint8, c.nbytes)
        size, seen = BYTES[self.c], np.zeros(c.nbytes, bool)
        out = np.empty((self.batch, rows or self.m, self.cols), NP[self.c])
        for b in range(self.batch):
            for r in range(rows or self.m):
                lo = (b * self.sc + r * self.ldc) * size
                out[b, r] = raw[lo:lo + self.cols * size].view(NP[self.c])
                seen[lo:lo + self.cols * size] = True
        if not (self.rmw and rows):
            assert (raw[~seen] == GUARD).all()
        self.bits = out
        return values(out, self.c)

    def check(self, **kw):
        got = self.run(**kw)
        w, e = self.want()
        tol = e + HALF[self.c] * (np.abs(w) + e) + (2.0 ** -25 if self.c == M.F16 else 0)
        bad = np.abs(got - w) > tol
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], (np.abs(got - w) / tol).max())


SHAPES = [(1, 4, 16), (1, 64, 64), (1, 516, 4112), (2, 60, 48), (5, 132, 80), (15, 64, 1040), (16, 128, 128), (17, 260, 272),
          (23, 4096, 256), (33, 68, 144), (64, 256, 512), (65, 12, 400), (77, 640, 2048), (129, 132, 1168), (255, 516, 128),
          (257, 260, 144), (300, 1028, 336), (700, 388, 208), (2050, 136, 64)]


@pytest.mark.parametrize("m, n, k", SHAPES)
def test_product_shapes(gpu, m, n, k):
    Product(m, n, k).check()


@pytest.mark.parametrize("c", [M.BF16, M.F16, M.F32])
@pytest.mark.parametrize("epi", [M.EPI_STORE, M.EPI_GELU_TANH, M.EPI_SILU, M.EPI_SWIGLU, M.EPI_GEGLU])
@pytest.mark.parametrize("m, n, k", [(1, 264, 1296), (13, 520, 128), (70, 264, 208), (300, 520, 336)])
def test_product_epilogues(gpu, m, n, k, epi, c):
    Product(m, n, k, epi, c).check()


@pytest.mark.parametrize("epi", [M.EPI_GATE_ADD, M.EPI_GATE_TANH, M.EPI_ADD])
@pytest.mark.parametrize("m, n, k", [(1, 264, 1296), (13, 132, 128), (70, 260, 208), (300, 516, 336)])
def test_product_residual(gpu, m, n, k, epi):
    Product(m, n, k, epi, split=3, seg=7).check()
    Product(m, n, k, epi, ldc=n + 4, bias=False).check()


@pytest.mark.parametrize("m, n, k", [(1, 68, 2064), (7, 132, 80), (40, 260, 144), (150, 260, 272), (280, 516, 144)])
def test_product_batches_and_strides(gpu, m, n, k):
    Product(m, n, k, batch=3, lda=k + 48, ldc=n + 12, c=M.BF16, offset=16).check()
    Product(m, n, k, epi=M.EPI_GATE_ADD, batch=2, lda=k + 16, ldc=n + 4, split=2, seg=5).check()
    Product(m, 2 * n, k, epi=M.EPI_SWIGLU, batch=2, lda=k + 16, ldc=n + 20, c=M.F16, bias=False).check()


@pytest.mark.parametrize("epi, c", [(M.EPI_STORE, M.F16), (M.EPI_GELU_TANH, M.BF16), (M.EPI_SWIGLU, M.BF16), (M.EPI_GEGLU, M.F32),
                                    (M.EPI_GATE_TANH, M.F32), (M.EPI_ADD, M.F32)])
@pytest.mark.parametrize("m, n, k", [(1, 72, 8208), (17, 72, 8208), (61, 136, 6160)])
def test_product_small_with_long_k(gpu, m, n, k, epi, c):
    Product(m, n, k, epi, c, batch=2, lda=k + 16, ldc=n + 4, split=5, seg=16).check()


# On 256 compute units: 32 x 32 (GEGLU: 32 x 64), 64 x 32 and 64 x 64 tiles, 64 x 128 in 4 stages and in 2, 128 x 128; the mixed
# kernel's 128 x 128 tiles in one and two rounds, 256 x 256 ones in a partial round; a whole round and one and two rounds of 128 x
# 128 parts, 64 x 64 parts; chains and a partial round, 128 x 128 parts, 64 x 64 parts; two whole rounds of an odd number of k steps.
@pytest.mark.parametrize("m, n, k", [(257, 516, 336), (150, 3076, 176), (150, 6000, 1040), (150, 6000, 176), (2048, 2304, 176),
                                     (1030, 6000, 176), (8300, 4100, 336), (2040, 1028, 1040), (1537, 8200, 176), (2818, 6000, 592),
                                     (4300, 5124, 2064), (2040, 8200, 176), (6200, 4100, 720), (8300, 4100, 720), (6200, 5124, 2192),
                                     (8300, 4100, 592), (50, 1028, 720), (200, 1040, 4112), (50, 4100, 176), (50, 8200, 176),
                                     (100, 8200, 1040), (515, 8200, 720)])
@pytest.mark.parametrize("epi, c", [(M.EPI_STORE, M.BF16), (M.EPI_GELU_TANH, M.F16), (M.EPI_GEGLU, M.F16), (M.EPI_GATE_TANH, M.F32)])
def test_product_many_tiles(gpu, m, n, k, epi, c):
    n -= n % 8 if epi == M.EPI_GEGLU else 0
    Product(m, n, k, epi, c, split=100, seg=m).check()


@pytest.mark.parametrize("m", [1, 20, 130])
def test_product_sums_are_exact_at_the_largest_k(gpu, m):
    # -128 x -128 131056 times: 2147221504, and the same with one row's sign turned
    k = 131056
    p = Product(m, 8, k, extremes=True, bias=False)
    p.W[3] = 127
    p.asc[:], p.wsc[:] = 1.0, 1.0
    s = np.full(8, 128.0 * 128.0 * k)
    s[3] = -128.0 * 127.0 * k
    got = p.run()
    assert np.array_equal(got, np.broadcast_to(s.astype(np.float32).astype(np.float64), (1, m, 8)))


@pytest.mark.parametrize("epi, c, n", [(M.EPI_STORE, M.F32, 268), (M.EPI_GELU_TANH, M.BF16, 268), (M.EPI_SWIGLU, M.BF16, 520),
                                       (M.EPI_GATE_TANH, M.F32, 268)])
def test_product_row_bits_do_not_depend_on_the_launch(gpu, epi, c, n):
    # the first rows of a large launch alone, in launches of every size class
    p = Product(1100, n, 1040, epi, c)
    p.run()
    whole = p.bits.copy()
    for rows in (1, 2, 16, 17, 40, 64, 65, 128, 200, 300, 600, 1099):
        p.run(rows=rows)
        assert np.array_equal(p.bits[0], whole[0, :rows]), rows


@pytest.mark.parametrize("m, n, k", [(9, 68, 272), (300, 260, 144)])
def test_product_nonfinite_scales_stay_in_their_row(gpu, m, n, k):
    p = Product(m, n, k, c=M.BF16)
    p.asc[0, 3], p.asc[0, m - 1] = np.nan, np.inf
    got = p.run()[0]
    assert np.isnan(got[3]).all() and not np.isfinite(got[m - 1]).any()
    keep = [r for r in range(m) if r not in (3, m - 1)]
    w, e = p.want()
    assert (np.abs(got[keep] - w[0, keep]) <= e[0, keep] + HALF[M.BF16] * (np.abs(w[0, keep]) + e[0, keep])).all()


@pytest.mark.parametrize("m, n, k", [(3, 24, 48), (70, 264, 208), (300, 1032, 336)])
def test_geglu_of_infinite_gates(gpu, m, n, k):
    # b Phi(b) is b at +inf and 0 at -inf; a NaN stays in its column
    p = Product(m, n, k, M.EPI_GEGLU)
    f = n // 2
    p.bias[f + 1], p.bias[f + 2], p.bias[f + 3] = np.inf, -np.inf, np.nan
    got, a = p.run()[0], p.pre[0, :, 1]
    assert (np.abs(a) > p.mag[0, :, 1] * 4 * u).all()
    assert np.array_equal(got[:, 1], np.copysign(np.inf, a)) and (got[:, 2] == 0).all() and np.isnan(got[:, 3]).all()
    assert np.isfinite(np.delete(got, [1, 2, 3], 1)).all()


def test_product_empty(gpu):
    g = M.GemmArgs()
    d = dev_bytes(4096)
    g.a = g.w = g.wscale = g.c = d.p
    g.N, g.K, g.lda, g.ldc, g.w_dtype, g.c_dtype = 64, 64, 64, 64, M.I8, M.BF16
    for rows, batch in ((0, 1), (3, 0)):
        g.M, g.batch = rows, batch
        M.call("mk_gemm_i8", C.byref(g), d.p, None)
    M.sync()
    assert (d.to_array(np.uint8, 4096) == GUARD).all()


# ---------------------------------------------------------------------------------------------------------------------
# the fused residual and norms
# ---------------------------------------------------------------------------------------------------------------------

def norm64(v, kind, w, b, eps, depth):
    """The norm in 64 bits and its error beyond the input's own, `e` relative to the parts."""
    if kind == M.NORM_NONE:
        return v, np.zeros_like(v), np.ones(v.shape[0])
    mean = v.mean(1, keepdims=True) if kind == M.NORM_LAYER else np.zeros((v.shape[0], 1))
    d = v - mean
    rs = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    w = 1.0 if w is None else w.astype(np.float64)
    b = 0.0 if b is None else b.astype(np.float64)
    h = d * rs
    # the mean's sum: depth additions; the variance's: depth + 2 relative, half of it in rs; rsqrt and division 2 ulp;
    # then the subtraction, two products and an addition
    em = (depth + 2) * u * np.abs(v).mean(1, keepdims=True) if kind == M.NORM_LAYER else 0.0
    e = np.abs(w) * (rs * (em + u * (np.abs(v) + np.abs(mean))) + np.abs(h) * ((depth + 2) / 2 + 8) * u) + 2 * u * (np.abs(h * w) + np.abs(b))
    return h * w + b, e, (rs * np.abs(w)).max(1) if np.ndim(w) else rs[:, 0]


class GateNorm:
    def __init__(self, rows, n, y=M.BF16, out=M.BF16, norm1=0, norm2=M.NORM_LAYER, vectors=True, gate=True, tanh=False,
                 scale=True, shift=True, split=0, seg=0, alpha=0.0, in_place=False, store_x=True, pad=0, seed=0,
                 samples=1, spread=1.0):
        rng = np.random.default_rng(seed + rows + 3 * n)
        self.__dict__.update(rows=rows, n=n, y=y, out=out, norm1=norm1, norm2=norm2, tanh=tanh, split=split, seg=seg,
                             alpha=alpha, in_place=in_place, store_x=store_x)
        self.ldx, self.ldy, self.ldo = n + pad, n + 2 * pad, n + 3 * pad
        col = np.exp(rng.standard_normal(n) * spread)
        self.x = (rng.standard_normal((rows, n)) * col * 2).astype(np.float32)
        self.ybits, self.yv = stored(rng.standard_normal((rows, n)) * col, y) if y is not None else (None, None)
        vec = lambda on, mean: (mean + 0.2 * rng.standard_normal(n)).astype(np.float32) if on else None  # noqa: E731
        self.w1 = vec(norm1 and vectors, 1.0)
        self.b1 = vec(norm1 == M.NORM_LAYER and vectors, 0.0)
        self.w2 = vec(norm2 and vectors, 1.0)
        self.b2 = vec(norm2 == M.NORM_LAYER and vectors, 0.0)
        self.stride = 7 * n
        self.mod = (rng.standard_normal((samples, 7 * n)) * 0.5).astype(np.float32)
        self.parts = {"gate": 0 if gate and y is not None else None, "scale": n if scale and out is not None else None,
                      "shift": 2 * n if shift and out is not None else None}

    def part(self, name, none):
        at = self.parts[name]
        r = np.arange(self.rows)
        seg = self.seg or 1 << 40
        if at is None:
            return np.full((self.rows, self.n), none)
        at = (r // seg)[:, None] * self.stride + np.where(r % seg < self.split, 4 * self.n, 0)[:, None] + at
        return self.mod.ravel()[at + np.arange(self.n)].astype(np.float64)

    def want(self):
        depth = self.n / 64 + 10  # more than any thread adds in a row, and the steps that join the threads
        x = self.x.astype(np.float64)
        if self.y is not None:
            v, ev, _ = norm64(self.yv, self.norm1, self.w1, self.b1, 1e-5, depth)
            g = self.part("gate", 1.0)
            eg = 0.0
            if self.tanh:
                eg = (16 + 8 * np.abs(g)) * u
                g = np.tanh(g)
            al = np.float64(np.float32(self.alpha or 1.0))
            ex = np.abs(g) * ev + eg * np.abs(v) + 2 * u * (np.abs(al * x) + np.abs(g * v))
            x = al * x + g * v
        else:
            ex = np.zeros_like(x)
        h, eh, k = norm64(x, self.norm2, self.w2, self.b2, 1e-6, depth)
        # x' off by ex moves h by at most rs w (ex + mean ex) and, through the statistics, as much again of |h| / rms
        eh = eh + k[:, None] * (ex + ex.mean(1, keepdims=True)) + (
            np.abs(h) * k[:, None] * np.sqrt((ex * ex).mean(1, keepdims=True)) if self.norm2 else 0.0)
        sc, sh = self.part("scale", 0.0), self.part("shift", 0.0)
        return x, ex, h * (1 + sc) + sh, eh * np.abs(1 + sc) + 3 * u * (np.abs(h * (1 + sc)) + np.abs(sh))

    def run(self, stream=None):
        self.upload()
        M.call("mk_gate_norm", C.byref(self.args()), stream)
        M.sync()
        return self.read()

    def upload(self):
        rows, n = self.rows, self.n

        def strided(a, ld):
            size = a.dtype.itemsize
            host = np.full(((rows - 1) * ld + n) * size + 64, GUARD, np.uint8)
            h = host[:-64].view(a.dtype)
            for r in range(rows):
                h[r * ld:r * ld + n] = a[r]
            return M.Dev.from_array(host)

        self.dx = strided(self.x, self.ldx)
        self.dy = strided(self.ybits, self.ldy) if self.y is not None else None
        self.dxo = self.dx if self.in_place else dev_bytes(self.dx.nbytes)
        self.do = dev_bytes(((rows - 1) * self.ldo + n) * BYTES[self.out] + 64) if self.out is not None else None
        self.ds = dev_bytes(rows * 4 + 64)
        self.dm = M.Dev.from_array(self.mod)
        self.dv = {k: M.Dev.from_array(getattr(self, k)) for k in ("w1", "b1", "w2", "b2") if getattr(self, k) is not None}

    def args(self):
        g = M.GateNormArgs()
        g.x = self.dx.p
        if self.y is not None:
            g.y, g.y_dtype, g.ldy = self.dy.p, self.y, self.ldy
            g.x_out = self.dxo.p if self.store_x else None
        if self.out is not None:
            g.out, g.out_dtype, g.ldo = self.do.p, self.out, self.ldo
            g.out_scale = self.ds.p if self.out == M.I8 else None
        for k, d in self.dv.items():
            setattr(g, k, d.p)
        for k, at in self.parts.items():
            if at is not None:
                setattr(g, k, self.dm.p + 4 * at)
        g.rows, g.n, g.ldx, g.alt, g.mod_stride, g.split, g.seg_rows = (self.rows, self.n, self.ldx, 4 * self.n, self.stride,
                                                                        self.split, self.seg)
        g.norm1, g.norm2, g.tanh_gate, g.residual_scale, g.eps1, g.eps2 = (self.norm1, self.norm2, int(self.tanh), self.alpha,
                                                                           1e-5, 1e-6)
        return g

    def rows_of(self, dev, ld, dt):
        raw = dev.to_array(np.uint8, dev.nbytes)
        size, seen = BYTES[dt], np.zeros(dev.nbytes, bool)
        out = np.empty((self.rows, self.n), NP[dt])
        for r in range(self.rows):
            out[r] = raw[r * ld * size:(r * ld + self.n) * size].view(NP[dt])
            seen[r * ld * size:(r * ld + self.n) * size] = True
        assert (raw[~seen] == GUARD).all()
        return out

    def read(self):
        x = h = s = None
        if self.y is not None and self.store_x:
            x = self.rows_of(self.dxo, self.ldx, M.F32)
        elif self.y is not None and not self.in_place:
            assert (self.dxo.to_array(np.uint8, self.dxo.nbytes) == GUARD).all()
        if self.out is not None:
            h = self.rows_of(self.do, self.ldo, self.out)
        sc = self.ds.to_array(np.uint8, self.ds.nbytes)
        used = self.rows * 4 if self.out == M.I8 else 0
        assert (sc[used:] == GUARD).all()
        if used:
            s = sc[:used].view(np.float32)
        return x, h, s

    def check(self, **kw):
        x, h, s = self.run(**kw)
        wx, ex, wh, eh = self.want()
        if x is not None:
            assert (np.abs(x - wx) <= ex).all(), (np.abs(x - wx) / ex).max()
        if self.out is None:
            return
        if self.out == M.I8:
            top, et = np.abs(wh).max(1), eh.max(1)
            assert (np.abs(s * 127.0 - top) <= et + 2 * u * top).all()
            # a code is half a step from the h it was made of, which is within eh of the definition's
            tol = 0.5 * s[:, None] * (1 + 1e-6) + eh
            assert (np.abs(h * s[:, None].astype(np.float64) - wh) <= tol).all()
            assert (np.abs(h.astype(int)).max(1) == 127).all()
            return
        got = values(h, self.out)
        tol = eh + HALF[self.out] * (np.abs(wh) + eh) + (2.0 ** -25 if self.out == M.F16 else 0)
        assert (np.abs(got - wh) <= tol).all(), (np.abs(got - wh) / tol).max()


WIDTHS = [4, 8, 64, 252, 256, 260, 516, 1024, 1280, 2048, 4096, 4100, 5120, 8192, 12288, 16384]


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_gate_norm_widths(gpu, n, rows):
    GateNorm(rows, n).check()
    GateNorm(rows, n, out=M.I8, norm1=M.NORM_RMS, norm2=M.NORM_RMS, alpha=0.5).check()


@pytest.mark.parametrize("n", [512, 1024, 1280, 1540, 2048, 3332, 4096, 6144, 8192, 8196, 16384])
def test_gate_norm_many_rows(gpu, n):
    g = GateNorm(517, n, out=M.I8, norm1=M.NORM_RMS, split=20, seg=260, samples=2)
    g.check()
    x, h, s = g.read()
    for rows in (300, 5, 1):  # the first rows alone: the same bits
        g.rows, g.x, g.ybits = rows, g.x[:rows], g.ybits[:rows]
        x1, h1, s1 = g.run()
        assert np.array_equal(x1, x[:rows]) and np.array_equal(h1, h[:rows]) and np.array_equal(s1, s[:rows])


@pytest.mark.parametrize("y", [M.F32, M.BF16, M.F16])
@pytest.mark.parametrize("out", [M.F32, M.BF16, M.F16, M.I8])
@pytest.mark.parametrize("n", [516, 4096])
def test_gate_norm_types(gpu, y, out, n):
    GateNorm(33, n, y, out, tanh=True).check()
    GateNorm(5, n, y, out, norm1=M.NORM_LAYER, norm2=M.NORM_RMS, gate=False, alpha=-1.5, pad=4).check()


@pytest.mark.parametrize("norm1", [0, 1, 2])
@pytest.mark.parametrize("norm2", [0, 1, 2])
@pytest.mark.parametrize("vectors", [False, True])
def test_gate_norm_kinds(gpu, norm1, norm2, vectors):
    GateNorm(9, 772, norm1=norm1, norm2=norm2, vectors=vectors).check()
    GateNorm(9, 772, norm1=norm1, norm2=norm2, vectors=vectors, gate=False, scale=False, shift=False, out=M.I8).check()


@pytest.mark.parametrize("rows, n, seg, split, samples", [(10, 256, 5, 2, 2), (77, 1280, 26, 26, 3), (300, 516, 0, 40, 1),
                                                          (2300, 260, 1000, 300, 3), (6, 4096, 1, 0, 6), (5000, 128, 2500, 0, 2)])
def test_gate_norm_modulation_rows(gpu, rows, n, seg, split, samples):
    GateNorm(rows, n, seg=seg, split=split, samples=samples).check()
    GateNorm(rows, n, seg=seg, split=split, samples=samples, tanh=True, shift=False, out=M.I8).check()


@pytest.mark.parametrize("n", [260, 4096])
def test_gate_norm_parts(gpu, n):
    GateNorm(40, n, in_place=True, pad=4).check()
    GateNorm(40, n, in_place=True, out=M.I8, norm1=1, norm2=1, alpha=0.25).check()
    GateNorm(40, n, y=None).check()                        # the norm alone
    GateNorm(40, n, y=None, out=M.I8, pad=8).check()       # into int8 rows
    GateNorm(40, n, y=None, out=M.I8, norm2=0, scale=False, shift=False).check()  # quantised as it is
    GateNorm(40, n, out=None, norm2=0).check()             # the residual alone
    GateNorm(40, n, out=None, norm2=0, norm1=2, in_place=True).check()
    GateNorm(40, n, store_x=False).check()
    GateNorm(40, n, scale=False).check()
    GateNorm(40, n, shift=False, gate=False).check()


@pytest.mark.parametrize("out", [M.F32, M.I8])
@pytest.mark.parametrize("n", [512, 4096, 12288])
def test_gate_norm_constant_and_offset_rows(gpu, out, n):
    # a variance far below the mean's square: the two-pass form keeps it. x' = x exactly (y = 0)
    g = GateNorm(6, n, y=M.F32, out=out, gate=False, scale=False, shift=False, vectors=False)
    g.ybits[:] = 0
    g.yv[:] = 0
    g.x[:] = 1000.0 + np.random.default_rng(3).standard_normal((6, n)).astype(np.float32)
    g.x[2] = 5.0   # no variance at all: h is the rounding of x - mean, over sqrt(eps)
    x, h, s = g.run()
    assert np.array_equal(x, g.x)
    wx, ex, wh, eh = g.want()
    rows = [0, 1, 3, 4, 5]
    got = h.astype(np.float64) * (s[:, None] if out == M.I8 else 1)
    tol = eh + (0.5 * s[:, None] * (1 + 1e-6) if out == M.I8 else 0)
    assert (np.abs(got - wh)[rows] <= tol[rows]).all()
    assert np.abs(got[2]).max() <= (n / 64 + 12) * u * 5.0 / np.sqrt(1e-6)


@pytest.mark.parametrize("out", [M.BF16, M.I8])
@pytest.mark.parametrize("n", [516, 4096, 8192])
def test_gate_norm_nonfinite_rows_stay_alone(gpu, out, n):
    g = GateNorm(300, n, out=out)
    x, h, s = g.run()
    h0, x0 = h.copy(), x.copy()
    g.x[3, 7] = np.nan
    g.x[4, n - 1] = np.inf
    g.ybits[5, 0] = 0x7F80  # bf16 infinity
    g.x[298, 1] = -np.inf
    x, h, s = g.run()
    bad = [3, 4, 5, 298]
    keep = [r for r in range(300) if r not in bad]
    assert np.array_equal(x[keep], x0[keep]) and np.array_equal(h[keep], h0[keep])
    for r in bad:
        if out == M.I8:
            assert np.isnan(s[r]) and not h[r].any()
        else:
            assert np.isnan(values(h[r], out)).any()


def test_gate_norm_zero_rows(gpu):
    # norms of zeros are zeros: a row of zeros in every stage, int8 scale 1
    g = GateNorm(4, 1024, norm1=1, norm2=1, gate=False, scale=False, shift=False, out=M.I8)
    g.x[1] = 0
    g.ybits[1] = 0
    x, h, s = g.run()
    assert not x[1].any() and not h[1].any() and s[1] == 1
    g = GateNorm(0x1000, 4, out=None, norm2=0)  # many short rows
    g.check()


def test_gate_norm_empty(gpu):
    d = dev_bytes(4096)
    g = M.GateNormArgs()
    g.x = g.x_out = g.y = g.out = d.p
    g.n, g.ldx, g.ldy, g.ldo, g.y_dtype, g.out_dtype = 64, 64, 64, 64, M.F32, M.F32
    M.call("mk_gate_norm", C.byref(g), None)
    M.sync()
    assert (d.to_array(np.uint8, 4096) == GUARD).all()


# ---------------------------------------------------------------------------------------------------------------------
# a run of them: norm -> int8 rows -> gated product -> int8 rows -> product -> the next block's norm
# ---------------------------------------------------------------------------------------------------------------------

class Ffn:
    """A feed-forward block in int8 between two fused norms, on buffers of its own; n wide, f hidden."""

    def __init__(self, rows, n, f, seed=0):
        rng = np.random.default_rng(seed)
        self.rows, self.n, self.f = rows, n, f
        col = np.exp(rng.standard_normal(n) * 0.5)
        self.x = (rng.standard_normal((rows, n)) * col).astype(np.float32)
        self.y, self.yv = stored(rng.standard_normal((rows, n)) * col, M.BF16)
        self.mod = (rng.standard_normal(6 * n) * 0.3).astype(np.float32)
        self.up, self.ups = codes_of(rng.standard_normal((2 * f, n)) * 0.05)
        self.down, self.downs = codes_of(rng.standard_normal((n, f)) * 0.05)
        D = M.Dev.from_array
        self.dx, self.dy, self.dmod, self.dup, self.dups, self.ddown, self.ddowns = map(
            D, (self.x, self.y, self.mod, self.up, self.ups, self.down, self.downs))
        self.bufs = {k: M.Dev(b) for k, b in dict(x1=rows * n * 4, h=rows * n, hs=rows * 4, u=rows * f * 2, uq=rows * f,
                                                  us=rows * 4, y1=rows * n * 2, x2=rows * n * 4, h2=rows * n * 2).items()}
        b, mod = self.bufs, self.dmod.p
        self.n1, self.n2 = M.GateNormArgs(), M.GateNormArgs()
        for g, x, y, xo, out, dt, at in ((self.n1, self.dx, self.dy, b["x1"], b["h"], M.I8, 0),
                                         (self.n2, b["x1"], b["y1"], b["x2"], b["h2"], M.BF16, 3 * n)):
            g.x, g.y, g.x_out, g.out = x.p, y.p, xo.p, out.p
            g.rows, g.n, g.ldx, g.ldy, g.ldo, g.y_dtype, g.out_dtype = rows, n, n, n, n, M.BF16, dt
            g.gate, g.scale, g.shift = mod + 4 * at, mod + 4 * (at + n), mod + 4 * (at + 2 * n)
            g.tanh_gate, g.norm2, g.eps1, g.eps2 = 1, M.NORM_LAYER, 1e-6, 1e-6
        self.n1.out_scale = b["hs"].p
        self.g1, self.g2 = M.GemmArgs(), M.GemmArgs()
        for g, a, w, ws, c, nn, kk, epi, ldc in ((self.g1, b["h"], self.dup, self.dups, b["u"], 2 * f, n, M.EPI_SWIGLU, f),
                                                 (self.g2, b["uq"], self.ddown, self.ddowns, b["y1"], n, f, M.EPI_STORE, n)):
            g.a, g.w, g.wscale, g.c, g.M, g.N, g.K, g.lda, g.ldc = a.p, w.p, ws.p, c.p, rows, nn, kk, kk, ldc
            g.batch, g.w_dtype, g.c_dtype, g.epilogue = 1, M.I8, M.BF16, epi

    def launch(self, stream):
        b = self.bufs
        M.call("mk_gate_norm", C.byref(self.n1), stream)
        M.call("mk_gemm_i8", C.byref(self.g1), b["hs"].p, stream)
        M.call("mk_quantize_i8_rows", b["u"].p, M.BF16, self.rows, self.f, self.f, b["uq"].p, b["us"].p, stream)
        M.call("mk_gemm_i8", C.byref(self.g2), b["us"].p, stream)
        M.call("mk_gate_norm", C.byref(self.n2), stream)

    def read(self):
        b, r, n, f = self.bufs, self.rows, self.n, self.f
        shape = dict(x1=(r, n), h=(r, n), hs=(r,), u=(r, f), uq=(r, f), us=(r,), y1=(r, n), x2=(r, n), h2=(r, n))
        types = dict(x1=np.float32, h=np.int8, hs=np.float32, u=np.uint16, uq=np.int8, us=np.float32, y1=np.uint16,
                     x2=np.float32, h2=np.uint16)
        return {k: b[k].to_array(types[k], shape[k]) for k in shape}

    def clear(self):
        for d in self.bufs.values():
            M.call("mk_memset", d.p, 0xFF, d.nbytes)


def same(a, b):
    return all(np.array_equal(a[k].view(np.uint8), b[k].view(np.uint8)) for k in a)


@pytest.mark.parametrize("rows, n, f", [(1, 256, 512), (5, 640, 1296), (77, 512, 1024), (300, 1280, 656)])
def test_ffn_run_matches_64_bits(gpu, rows, n, f):
    w = Ffn(rows, n, f)
    w.launch(None)
    M.sync()
    r = w.read()
    mod = w.mod.astype(np.float64).reshape(6, n)

    def norm(x, sc, sh):
        d = x - x.mean(1, keepdims=True)
        return d / np.sqrt((d * d).mean(1, keepdims=True) + 1e-6) * (1 + sc) + sh

    # stage by stage on what the stage before it wrote, each rounding counted
    x1 = w.x + np.tanh(mod[0]) * w.yv
    assert np.abs(r["x1"] - x1).max() <= 1e-6 * np.abs(x1).max()
    h = norm(r["x1"].astype(np.float64), mod[1], mod[2])
    assert (np.abs(r["h"] * r["hs"][:, None].astype(np.float64) - h) <= r["hs"][:, None] * 0.5 * (1 + 1e-6) + 1e-5 * (1 + np.abs(h))).all()
    a = (r["h"].astype(np.float64) @ w.up.T.astype(np.float64)) * r["hs"][:, None] * w.ups.astype(np.float64)
    g = a[:, :f] / (1 + np.exp(-a[:, :f])) * a[:, f:]
    assert (np.abs(values(r["u"], M.BF16) - g) <= HALF[M.BF16] * np.abs(g) * (1 + 2 ** -10) + 1e-5 * np.abs(a).max() ** 2 * 0.01).all()
    uq, us = codes_of(values(r["u"], M.BF16))
    assert np.array_equal(uq, r["uq"]) and np.array_equal(us, r["us"])
    y = (uq.astype(np.float64) @ w.down.T.astype(np.float64)) * us[:, None] * w.downs.astype(np.float64)
    assert (np.abs(values(r["y1"], M.BF16) - y) <= HALF[M.BF16] * np.abs(y) * (1 + 2 ** -10) + 1e-30).all()
    x2 = r["x1"] + np.tanh(mod[3]) * values(r["y1"], M.BF16)
    assert np.abs(r["x2"] - x2).max() <= 1e-6 * np.abs(x2).max()
    h2 = norm(r["x2"].astype(np.float64), mod[4], mod[5])
    assert (np.abs(values(r["h2"], M.BF16) - h2) <= HALF[M.BF16] * np.abs(h2) * (1 + 2 ** -10) + 1e-5 * (1 + np.abs(h2))).all()
    # and the whole against real arithmetic: three 8-bit roundings (a step is 1/127 of a row's largest value, about 4 of
    # its rms: 4 / 127 / sqrt(12) = 0.9% of the rms each, which a sum over many terms keeps) and the two of bf16
    hr = norm(x1, mod[1], mod[2])
    ar = hr @ (w.up * w.ups[:, None].astype(np.float64)).T
    yr = (ar[:, :f] / (1 + np.exp(-ar[:, :f])) * ar[:, f:]) @ (w.down * w.downs[:, None].astype(np.float64)).T
    got = values(r["y1"], M.BF16)
    assert np.linalg.norm(got - yr) <= 0.06 * np.linalg.norm(yr)


def test_two_streams_at_once_and_a_captured_run(gpu):
    hip = C.CDLL("libamdhip64.so.7")
    works = [Ffn(300, 640, 1296, 1), Ffn(7, 640, 1296, 2)]
    handles = [C.c_void_p() for _ in works]
    for h in handles:
        M.call("mk_stream_create", C.byref(h))
    alone = []
    for w in works:
        w.launch(None)
        M.sync()
        alone.append(w.read())
        w.clear()
    M.sync()
    for _ in range(3):
        for w, h in zip(works, handles):
            w.launch(h.value)
    M.sync()
    for w, a in zip(works, alone):
        assert same(w.read(), a)
    graphs = []
    for w, h in zip(works, handles):  # two graphs, replayed side by side
        graph, run = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(h, 0) == 0
        w.launch(h.value)
        assert hip.hipStreamEndCapture(h, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
        graphs.append((graph, run))
    for _ in range(3):
        for w in works:
            w.clear()
        M.sync()
        for (_, run), h in zip(graphs, handles):
            assert hip.hipGraphLaunch(run, h) == 0
        M.sync()
        for w, a in zip(works, alone):
            assert same(w.read(), a)
        works[0].launch(None)  # the program's own work between the replays
        M.sync()
        assert same(works[0].read(), alone[0])
    for graph, run in graphs:
        assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    for h in handles:
        M.call("mk_stream_destroy", h.value)


def test_fused_norm_equals_the_two_passes_it_replaces(gpu):
    # mk_gate_add then mk_ln_modulate on the same rows: the same formulas in fp32, so within their roundings
    rows, n = 300, 2048
    g = GateNorm(rows, n, tanh=True, vectors=False, split=40, samples=1)
    x, h, _ = g.run()
    dx, y = M.Dev.from_array(g.x), M.Dev(rows * n * 2)
    M.call("mk_gate_add", dx.p, M.Dev.from_array(g.ybits).p, M.BF16, rows, n, g.dm.p, 4 * n, 40, rows, 1, None)
    M.call("mk_ln_modulate", dx.p, rows, n, g.dm.p + 4 * n, g.dm.p + 8 * n, 4 * n, 40, rows, 1e-6, y.p, None)
    M.sync()
    x2, h2 = dx.to_array(np.float32, (rows, n)), values(y.to_array(np.uint16, (rows, n)), M.BF16)
    wx, ex, wh, eh = g.want()
    assert (np.abs(x - x2) <= 2 * ex).all()
    assert (np.abs(values(h, M.BF16) - h2) <= 2 * (eh + HALF[M.BF16] * (np.abs(wh) + eh))).all()
