"""mk_rope_rows from 2^22 values on, where a wave turns four groups of heads with one row's cosines and sines (below: one): heads that
end inside a group, both modes and series, types, in place. Tolerances as in test_gpu_packed_ops.py."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_packed_ops import NAME, Rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode, series", [(1, 0), (2, 0), (1, 1), (2, 1)])
@pytest.mark.parametrize("rows, heads, kv, d, dims", [(3700, 7, 2, 128, [16, 56, 56]), (2731, 9, 3, 128, [40, 24]), (2979, 17, 5, 64, [16, 24, 16]),
                                                      (33001, 2, 0, 64, [8]), (1023, 33, 0, 128, [2, 2, 2, 2])])
def test_rope_heads_that_end_inside_a_group(gpu, rows, heads, kv, d, dims, mode, series):
    assert rows * (heads + kv) * d >= 1 << 22
    Rope(rows, heads, kv, d, dims, M.BF16, M.BF16, mode, series, pad=4, k_scale=0.5 if kv else 0.0).check()


@pytest.mark.parametrize("dt", [M.F32, M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("out", [M.F32, M.BF16, M.F16], ids=NAME.get)
def test_rope_types_of_many_rows(gpu, dt, out):
    rng = np.random.default_rng(1)
    Rope(2300, 10, 5, 128, [32, 48, 48], dt, out, pos_dt=M.F32, pos=rng.uniform(-4096, 4096, (2300, 3))).check()
    Rope(3700, 14, 5, 64, [16, 24, 16], dt, out, mode=2, norm=False).check()
    if dt == out:
        Rope(2300, 10, 5, 128, [128], dt, dt, in_place=True, pad=8).check()


def test_rope_either_side_of_the_border_is_the_same(gpu):
    """Rows' values do not depend on how many rows there are."""
    a = Rope(4096, 6, 2, 128, [16, 56, 56], M.BF16, M.BF16, pos=np.arange(4096)[:, None] * [1, 3, -7])
    a.run()
    M.sync()
    whole = {n: a.out[n].read().copy() for n in "qk"}
    g = a.g
    g.rows = 4095  # 2^22 values less a row
    for n in "qk":
        M.call("mk_memset", a.out[n].dev.p, 0x5A, a.out[n].dev.nbytes)
    M.call("mk_rope_rows", C.byref(g), None)
    M.sync()
    for n in "qk":
        assert np.array_equal(a.out[n].read()[:4095], whole[n][:4095])
