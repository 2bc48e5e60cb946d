"""mk_attention_packed where its variants meet: infinities under masks that cut a tile and in whole tiles, half weights far below the
largest, workspaces of any size, one wave a workgroup and split keys. Tolerances as in test_gpu_packed_ops.py."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_packed_ops import H, NAME, Attn, attend, packed, u, values

pytestmark = pytest.mark.gpu

CAUSAL = 0xFFFFFFFF


def one_dim(raw):
    """Scores that are k's dim 5 alone."""
    raw["q"][:], raw["k"][:] = 0.0, 0.0
    raw["q"][:, :, 5] = 1.0


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("rows, heads, kv, d, workspace", [(100, 2, 2, 64, True), (100, 2, 1, 128, True), (7, 2, 2, 64, False), (5, 2, 1, 128, True)])
@pytest.mark.parametrize("block", [0, CAUSAL])
def test_infinite_values_without_weight(gpu, block, rows, heads, kv, d, workspace, dt):
    """A seen key of weight zero (3000 below the others in natural units, in any precision) with an infinite value: 0 x inf is NaN,
    whether a mask cuts its tile (causal: 100 rows' tiles are all cut for some row) or not. With weight: the infinity."""
    nk = 300

    def edit(raw):
        one_dim(raw)
        raw["k"][nk - rows + rows // 2, :, 5] = -30.0
        raw["v"][nk - rows + rows // 2, 0, 3] = np.inf
        raw["v"][nk - 1, 0, 7] = -np.inf
        raw["v"][10, 0, 9] = np.inf
        raw["k"][20, :, 5] = -30.0
        raw["v"][20, 0, 40] = -np.inf

    a = Attn([(0, rows, 0, nk, nk - rows, block, 0)], rows, nk, heads, kv, d, dt, scale=100.0, edit=edit)
    a.check(workspace)
    got = values(a.result()[0], dt)
    assert (got[:, 0, 9] == np.inf).all() and np.isnan(got[:, 0, 40]).all() and np.isnan(got[-1, 0, 3]) and got[-1, 0, 7] == -np.inf
    assert block == 0 or np.isfinite(got[0, 0, 3])
