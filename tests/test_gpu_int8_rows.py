"""The int8 operators over more rows than one grid dimension takes workgroups for (2^21), and over rows whose offsets pass 32
bits, in elements and in bytes."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_int8_ops import BYTES, GateNorm, Product, codes_of, dev_bytes, quantize
from test_int8_kernels import kind

pytestmark = pytest.mark.gpu


# 5 columns: a workgroup a row; 16: four rows a workgroup, a wave each
@pytest.mark.parametrize("rows, cols", [((1 << 21) + 5, 5), ((1 << 23) + 5, 16)])
def test_quantize_rows_beyond_a_grid_dimension(gpu, rows, cols):
    x = np.random.default_rng(1).standard_normal((rows, cols), dtype=np.float32)
    q, s = quantize(x, M.F32, rows, cols, cols)
    for lo in range(0, rows, 1 << 20):
        at = slice(lo, min(lo + (1 << 20), rows))
        wq, ws = codes_of(x[at].astype(np.float64))
        assert np.array_equal(s[at], ws) and np.array_equal(q[at], wq)


def test_gate_norm_rows_beyond_a_grid_dimension(gpu):
    # x' = x + y alone: one rounding, so numpy's bits
    rows, n = (1 << 23) + 5, 4
    rng = np.random.default_rng(2)
    x, y = (rng.standard_normal((rows, n), dtype=np.float32) for _ in range(2))
    dx, dy, out = M.Dev.from_array(x), M.Dev.from_array(y), dev_bytes(rows * n * 4 + 64)
    g = M.GateNormArgs()
    g.x, g.y, g.x_out = dx.p, dy.p, out.p
    g.rows, g.n, g.ldx, g.ldy, g.y_dtype = rows, n, n, n, M.F32
    M.call("mk_gate_norm", C.byref(g), None)
    M.sync()
    raw = out.to_array(np.uint8, rows * n * 4 + 64)
    assert np.array_equal(raw[:-64].view(np.float32).reshape(rows, n), x + y)
    assert np.array_equal(raw[-64:], dev_bytes(64).to_array(np.uint8, 64))


def read(d, at, dtype, count):
    out = np.empty(count, dtype)
    M.call("mk_memcpy_d2h", out.ctypes.data, d.p + at, out.nbytes)
    return out


def scatter(rows, ld):
    """The rows of a host array, `ld` elements apart on the device."""
    d = M.Dev(((len(rows) - 1) * ld + rows.shape[1]) * rows.itemsize)
    for r, row in enumerate(rows):
        d.write(row, r * ld * rows.itemsize)
    return d


@pytest.mark.parametrize("tile, m, n, k", [((64, 128, 2), 600, 2056, 336), ((16, 16, 0), 600, 8, 2064)])
@pytest.mark.parametrize("epi, c", [(M.EPI_STORE, M.BF16), (M.EPI_GATE_ADD, M.F32)])
def test_product_rows_far_apart(gpu, tile, m, n, k, epi, c):
    # the longest lda: 5 GB of A; C over 2^32 elements
    lda, ldc, size = (1 << 23) - 16, 1 << 23, BYTES[c]
    assert kind(m, n, k, epi, lda=lda) == tile
    p = Product(m, n, k, epi, c, split=2, seg=5)
    p.run()
    want = p.bits[0]
    a = scatter(p.A[:m * k].reshape(m, k), lda)
    out = scatter(p.x[0], ldc) if p.rmw else M.Dev(((m - 1) * ldc + n) * size)
    g = p.args(out)
    g.a, g.lda, g.ldc = a.p, lda, ldc
    M.call("mk_gemm_i8", C.byref(g), p.dS.p, None)
    M.sync()
    for r in range(m):
        assert np.array_equal(read(out, r * ldc * size, want.dtype, n), want[r]), r


def test_product_batch_items_far_apart(gpu):
    m, n, k, far = 37, 136, 336, (1 << 32) + 16
    p = Product(m, n, k, batch=2)
    p.run()
    a = scatter(np.stack([p.A[b * p.sa:b * p.sa + m * k] for b in range(2)]), far)
    out = M.Dev((far + m * n) * 4)
    g = p.args(out)
    g.a, g.stride_a, g.stride_c = a.p, far, far
    M.call("mk_gemm_i8", C.byref(g), p.dS.p, None)
    M.sync()
    for b in range(2):
        assert np.array_equal(read(out, b * far * 4, np.float32, m * n).reshape(m, n), p.bits[b])


@pytest.mark.parametrize("out", [M.I8, M.BF16])
def test_gate_norm_rows_far_apart(gpu, out):
    rows, n, ld = 5, 512, 1 << 30
    g = GateNorm(rows, n, out=out, norm1=M.NORM_RMS, split=2, seg=3, samples=2)
    x, h, s = g.run()
    dx, dy, do = scatter(g.x, ld), scatter(g.ybits, ld), M.Dev(((rows - 1) * ld + n) * BYTES[out])
    a = g.args()
    a.x, a.x_out, a.y, a.out, a.ldx, a.ldy, a.ldo = dx.p, dx.p, dy.p, do.p, ld, ld, ld
    M.call("mk_gate_norm", C.byref(a), None)
    M.sync()
    for r in range(rows):
        assert np.array_equal(read(dx, r * ld * 4, np.float32, n), x[r])
        assert np.array_equal(read(do, r * ld * BYTES[out], h.dtype, n), h[r])


@pytest.mark.parametrize("cols", [512, 500])
@pytest.mark.parametrize("dt, ld", [(M.F32, 1 << 30), (M.BF16, 1 << 31)])
def test_quantize_rows_far_apart(gpu, dt, ld, cols):
    rows = 5
    x = np.random.default_rng(3).standard_normal((rows, cols)).astype(np.float32)
    bits = x if dt == M.F32 else M.bf16_bits(x)
    wq, ws = codes_of((x if dt == M.F32 else M.bf16_to_f32(bits)).astype(np.float64))
    src, q, s = scatter(bits, ld), M.Dev(rows * cols), M.Dev(rows * 4)
    M.call("mk_quantize_i8_rows", src.p, dt, rows, cols, ld, q.p, s.p, None)
    M.sync()
    assert np.array_equal(q.to_array(np.int8, (rows, cols)), wq) and np.array_equal(s.to_array(np.float32, rows), ws)


@pytest.mark.parametrize("cols", [65536, 65535])
def test_quantize_codes_past_32_bits(gpu, cols):
    rows = (1 << 32) // cols + 3
    src, q, s = M.Dev(rows * cols * 2), M.Dev(rows * cols), M.Dev(rows * 4)
    last = M.bf16_bits(np.random.default_rng(4).standard_normal((2, cols)).astype(np.float32))
    src.write(last, (rows - 2) * cols * 2)
    M.call("mk_quantize_i8_rows", src.p, M.BF16, rows, cols, cols, q.p, s.p, None)
    M.sync()
    wq, ws = codes_of(M.bf16_to_f32(last).astype(np.float64))
    assert np.array_equal(read(q, (rows - 2) * cols, np.int8, 2 * cols).reshape(2, cols), wq)
    sc = s.to_array(np.float32, rows)
    assert np.array_equal(sc[-2:], ws) and (sc[:-2] == 1).all()
    assert not read(q, 0, np.int8, 1 << 20).any() and not read(q, (rows - 18) * cols, np.int8, 16 * cols).any()
