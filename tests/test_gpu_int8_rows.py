"""mk_quantize_i8_rows and mk_gate_norm over more rows than one grid dimension takes workgroups for (2^21)."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_int8_ops import codes_of, dev_bytes, quantize

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
