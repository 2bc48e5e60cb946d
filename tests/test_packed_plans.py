"""Which kernels a mk_lora_rows call takes, by its sizes alone, on 256 compute units (no GPU)."""
import ctypes as C

import pytest

import mkimage as M
import test_gpu_lora_tiles
import test_gpu_packed_ops

P = 1 << 20  # an aligned address that no call may touch
ONE, A_TILE, COLUMNS, SPLITS, ORDER, FUSE = range(6)


def args(rows, K, N, rank, parts=1, adapters=4, **kw):
    g = M.LoraRowsArgs()
    g.x = g.a = g.b = g.base = g.c = g.ids = P
    g.ldx, g.ldbase, g.ldc = K, N, N
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters, g.dtype, g.c_dtype = rows, K, N, rank, parts, adapters, M.BF16, M.BF16
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def plan(*a, cus=256, **kw):
    out = (C.c_uint32 * 6)(*[99] * 6)
    M.call("mk_lora_rows_plan", C.byref(args(*a, **kw)), cus, out)
    return list(out)


def test_plan_refusals():
    f, out = M.lib().mk_lora_rows_plan, (C.c_uint32 * 6)()
    assert f(None, 256, out) == 1 and f(C.byref(args(5, 64, 64, 8)), 256, None) == 1
    assert f(C.byref(args(5, 64, 64, 8)), 0, out) == 1
    assert f(C.byref(args(0, 64, 64, 8)), 256, out) == 1 and b"no rows" in M.lib().mk_last_error()
    assert f(C.byref(args(5, 64, 64, 12)), 256, out) == 1 and b"rank" in M.lib().mk_last_error()


@pytest.mark.parametrize("size, takes", test_gpu_lora_tiles.TILES)
def test_the_tests_of_tiles_take_tiles(size, takes):
    got = plan(*size)
    assert got[ONE] == 0 and tuple(got[i] for i in (A_TILE, COLUMNS, SPLITS, FUSE)) == takes


def test_the_tests_of_few_rows_take_the_other_kernels():
    kinds = {(p[ONE], p[A_TILE] > 0, p[COLUMNS] > 0) for p in (plan(*size) for size in test_gpu_packed_ops.LORA_SIZES)}
    assert kinds == {(1, False, False), (0, False, False)}


def test_rows_in_no_order_are_sorted_where_a_product_takes_tiles():
    assert plan(4352, 4096, 12288, 32, 3)[ORDER] == 1
    for kw in (dict(ids=None), dict(grouped=1), dict(adapters=1), dict(adapters=1025)):
        assert plan(4352, 4096, 12288, 32, 3, **kw)[ORDER] == 0
    # one of the products by rows
    for size, tiles in (((2000, 1280, 5120, 16), (0, 512)), ((600, 12288, 640, 16), (32, 0)), ((300, 4096, 24576, 16, 2), (0, 512))):
        got = plan(*size)
        assert (got[A_TILE], got[COLUMNS]) == tiles and got[ORDER] == 1
        assert plan(*size, grouped=1)[ORDER] == 0
    # (only what goes by tiles has to be in reach)
    assert plan(600, 12288, 640, 16, ldc=(1 << 23) - 8, c_dtype=M.F32)[ORDER] == 1
    assert plan(600, 12288, 640, 16, ldx=(1 << 23) - 8)[ORDER] == 0
    assert plan(24, 4096, 12288, 16, 3)[ORDER] == 0 and plan(1000, 1280, 1280, 16)[ORDER] == 0


def test_k_is_split_as_far_as_the_workspace_reaches():
    size = (2048, 12288, 4096, 64)
    full = plan(*size)[SPLITS]
    one = 2048 * (4 * 64 + 8)
    assert full >= 8
    for splits in range(1, full + 2):
        room = one + (splits - 1) * 2048 * 4 * 64
        a, b = plan(*size, workspace=P, workspace_bytes=room)[SPLITS], plan(*size, workspace=P, workspace_bytes=room - 16)[SPLITS]
        assert 1 <= b <= a <= splits and b < max(splits, 2)
    assert a == full
    # the workspace of many rows (one split) serves fewer, which would have taken more of it
    many = 16384 * (4 * 64 + 8)
    assert plan(16384, 12288, 4096, 64, workspace=P, workspace_bytes=many)[SPLITS] == 1
    assert 1 < plan(13056, 12288, 4096, 64, workspace=P, workspace_bytes=4 * many)[SPLITS]
    assert plan(13056, 12288, 4096, 64, workspace=P, workspace_bytes=many)[SPLITS] == 1


def test_rows_are_sorted_as_far_as_byte_offsets_reach():
    # below 2^31 bytes from the first row on, of x (16 bits), base and c (their type's)
    for rows, kw, sorted_ in ((87000, dict(), 1), (87500, dict(), 0), (43600, dict(c_dtype=M.F32), 1), (43800, dict(c_dtype=M.F32), 0),
                              (43600, dict(ldx=24576), 1), (43800, dict(ldx=24576), 0), (43800, dict(ldbase=24576), 0), (43800, dict(ldbase=24576, base=None), 1),
                              (1 << 18, dict(ldx=4096, ldc=4088, ldbase=4088), 0), (1 << 18, dict(ldx=4088, ldc=4088, ldbase=4088), 1),
                              ((1 << 18) + 1, dict(ldx=8, ldc=8, ldbase=8), 0)):
        kw = dict(dict(ldx=4096, ldc=12288, ldbase=12288), **kw)
        assert plan(rows, 8, 8, 8, **kw)[ORDER] == sorted_, (rows, kw)


def test_a_product_of_2_to_26_and_more_goes_by_tiles():
    assert plan(1024, 4096, 4088, 16)[A_TILE:COLUMNS + 1] == [32, 0]
    assert plan(1024, 4088, 4096, 16)[A_TILE:COLUMNS + 1] == [0, 512]
    assert plan(1024, 4096, 4096, 16)[A_TILE:COLUMNS + 1] == [32, 512]
    assert plan(1023, 4096, 4096, 16)[:3] == [0, 0, 0]
