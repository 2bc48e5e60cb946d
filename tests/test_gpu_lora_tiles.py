"""mk_lora_rows on the kernels of many rows: their edges, parts, ranks, tails, infinities and half range, and either product by
tiles beside the other by rows. Which kernels a size takes is asked of mk_lora_rows_plan (256 compute units). Tolerances as in
test_gpu_packed_ops.py."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_packed_ops import H, NAME, Lora, Rows, dev, stored, u, values

pytestmark = pytest.mark.gpu

ONE, A_TILE, COLUMNS, SPLITS, ORDER, FUSE = range(6)


def plan(lora, **kw):
    g = lora.args() if isinstance(lora, Lora) else lora
    for k, v in kw.items():
        setattr(g, k, v)
    out = (C.c_uint32 * 6)()
    M.call("mk_lora_rows_plan", C.byref(g), 256, out)
    return list(out)


def ids_of(kind, rows, adapters, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "none":
        return None
    mixed = rng.integers(-1, adapters, rows)
    if kind == "mixed":
        return mixed
    runs = np.sort(rng.integers(0, adapters, rows))
    runs[rows // 2:rows // 2 + 70] = -1
    return runs


# rows, K, N, rank, parts, adapters, and what the plan has to say: A's rows a tile, columns a workgroup, splits of K, shared B
TILES = [((4161, 72, 24, 8, 3, 3), (32, 512, 1, 0)), ((4097, 8, 8, 8, 1, 2), (32, 512, 1, 0)), ((4161, 136, 1032, 40, 1, 4), (64, 512, 2, 0)),
         ((4200, 200, 528, 24, 2, 5), (64, 512, 2, 0)), ((4161, 128, 96, 128, 3, 2), (128, 512, 1, 1)), ((4161, 136, 128, 256, 1, 2), (128, 512, 1, 1)),
         ((4161, 520, 776, 96, 1, 3), (96, 512, 3, 1)), ((4161, 1160, 72, 16, 1, 9), (32, 512, 3, 0)), ((4127, 264, 416, 72, 4, 2), (96, 512, 1, 1)),
         ((5000, 3080, 136, 160, 1, 2), (96, 512, 3, 1)), ((130, 12296, 2072, 256, 1, 2), (128, 512, 14, 1)), ((130, 8200, 4112, 136, 2, 3), (96, 512, 13, 1))]


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("size, takes", TILES, ids=lambda v: "x".join(map(str, v)))
def test_lora_tiles(gpu, size, takes, dt):
    rows, adapters = size[0], size[5]
    for c_dt, ids, pad, kw in ((dt, "mixed", 8, dict()), (M.F32, "runs", 0, dict(in_place=True)), (M.BF16 if dt == M.F16 else M.F16, "runs", 16, dict(grouped=1))):
        a = Lora(*size[:5], adapters, ids_of(ids, rows, adapters), dt, c_dt, pad=pad, **kw)
        got = plan(a)
        assert got[ONE] == 0 and tuple(got[i] for i in (A_TILE, COLUMNS, SPLITS, FUSE)) == takes, got
        assert got[ORDER] == (not kw.get("grouped"))
        a.check()


@pytest.mark.parametrize("size, rows_first", [((3000, 8, 2816, 8, 1, 5), True), ((2100, 256, 3080, 16, 1, 4), True), ((300, 1032, 24616, 16, 1, 3), True),
                                              ((600, 8200, 64, 16, 1, 4), False), ((77, 20000, 40, 48, 1, 3), False), ((400, 4104, 72, 24, 3, 2), False)])
@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
def test_lora_one_product_by_rows_the_other_by_tiles(gpu, size, rows_first, dt):
    for c_dt, ids, kw in ((dt, "mixed", dict(pad=8)), (M.F32, "runs", dict(in_place=True)), (dt, "mixed", dict(base=False, grouped=1))):
        a = Lora(*size, ids_of(ids, size[0], size[5]), dt, c_dt, **kw)
        got = plan(a)
        assert got[ONE] == 0 and (got[A_TILE] == 0) == rows_first and (got[COLUMNS] == 0) != rows_first, got
        a.check()


@pytest.mark.parametrize("rank", [8, 72])
@pytest.mark.parametrize("c_dt", [M.BF16, M.F32], ids=NAME.get)
def test_lora_tiles_without_base_scale_or_ids_and_in_place(gpu, c_dt, rank):
    rows = 4131
    for kw in (dict(base=False), dict(scale=False), dict(ids=None), dict(in_place=True), dict(base=False, ids=[-1] * rows), dict(ids=[-1] * rows),
               dict(ids=[-1] * rows, in_place=True), dict(ids=[2 ** 31 - 1, -2 ** 31, 3] * (rows // 3)), dict(base=False, scale=False, ids=None)):
        kw = dict(dict(ids=np.arange(rows) % 3), **kw)
        a = Lora(rows, 40, 72, rank, 3, 3, kw.pop("ids"), M.BF16, c_dt, pad=16, **kw)
        assert plan(a)[:3] == [0, 32 if rank == 8 else 128, 512]
        a.check()


@pytest.mark.parametrize("rank", [8, 64])
@pytest.mark.parametrize("c_dt", [M.BF16, M.F32], ids=NAME.get)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("ids", ["in order", "grouped", "mixed"])
def test_lora_tiles_infinities_stay_with_their_rows(gpu, ids, bad, c_dt, rank):
    """Of rows with and without adapters in x, and of adapters in A and B; five adapters in every tile where the rows are said to be grouped."""
    rows = 4160

    def edit(raw):
        raw["x"][1, 3] = raw["x"][70, 0] = raw["x"][4159, 71] = bad
        raw["a"][2, 5, 7] = raw["a"][3, 7, 71] = bad
        raw["b"][3, 9, 1] = bad
        raw["base"][5, 4] = bad

    which = np.arange(rows) % 5
    which[70] = -1
    which = which if ids != "in order" else np.sort(which)
    for dt in (M.BF16, M.F16):
        a = Lora(rows, 72, 64, rank, 1, 5, which, dt, c_dt, edit=edit, grouped=int(ids == "grouped"))
        assert plan(a)[:5] == [0, 32 if rank == 8 else 64, 512, 1, int(ids != "grouped")]
        a.check()


@pytest.mark.parametrize("parts", [1, 3])
def test_lora_tiles_half_values_of_any_size(gpu, parts):
    # t beyond the half range, and far below it, rows of either next to each other
    def edit(raw):
        big = np.arange(rows) % 4 == 0
        raw["x"][big] = np.abs(raw["x"][big]) * 1e3
        raw["x"][np.arange(rows) % 4 == 1] *= 1e-3
        raw["a"][0] = np.abs(raw["a"][0]) * 1e2
        raw["a"][1] *= 1e-3
        raw["b"][:] *= 1e-2

    rows = 4100
    for ids, kw in ((np.arange(rows) // 2 % 2, dict()), (np.arange(rows) // 2 % 2, dict(grouped=1)), (np.arange(rows) // 2050, dict())):
        a = Lora(rows, 2048, 24 * parts, 16, parts, 2, ids, M.F16, M.F32, edit=edit, **kw)
        assert plan(a)[COLUMNS] == 512 and plan(a)[A_TILE] > 0
        a.check()


@pytest.mark.parametrize("rows, per, parts, blocks", [(5500, 2056, 4, 2), (16384, 1032, 4, 4), (24001, 1288, 2, 2)])
@pytest.mark.parametrize("c_dt", [M.BF16, M.F32], ids=NAME.get)
def test_lora_several_blocks_of_columns_a_wave(gpu, rows, per, parts, blocks, c_dt):
    """Enough tiles and columns for 2 and 4 blocks: 300 rows of c against the definition, all of them between two calls."""
    K, N, rank, adapters = 64, per * parts, 8, 3
    rng = np.random.default_rng(rows)
    (xb, x), (ab, a), (bb, b) = (stored(rng.standard_normal(s), M.BF16) for s in ((rows, K), (adapters, parts * rank, K), (adapters, N, rank)))
    ids = ids_of("runs", rows, adapters).astype(np.int32)
    keep = [dev(v) for v in (xb, ab, bb, ids)]
    c = Rows(rows, N + 8, c_dt)
    g = M.LoraRowsArgs()
    g.x, g.a, g.b, g.ids, g.c, g.ldx, g.ldc = *(k.p for k in keep), c.at(), K, N + 8
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters, g.dtype, g.c_dtype = rows, K, N, rank, parts, adapters, M.BF16, c_dt
    assert plan(g)[COLUMNS] == 512 * blocks
    need = C.c_uint64()
    M.call("mk_lora_rows_workspace", C.byref(g), C.byref(need))
    space = M.Dev(need.value)
    g.workspace, g.workspace_bytes = space.p, need.value
    M.call("mk_lora_rows", C.byref(g), None)
    M.sync()
    first = c.read()
    assert first[:, N:].tobytes() == c.before[:, N:].tobytes()
    M.call("mk_lora_rows", C.byref(g), None)
    M.sync()
    assert c.read().tobytes() == first.tobytes()
    r = np.concatenate([np.arange(70), rng.integers(0, rows, 160), np.arange(rows - 70, rows)])
    on = (ids[r] >= 0)[:, None]
    t, ta = (np.einsum("rk,rik->ri", p, q) for p, q in ((x[r], a[ids[r]]), (np.abs(x[r]), np.abs(a[ids[r]]))))
    want, tol = np.zeros((len(r), N)), np.zeros((len(r), N))
    for p in range(parts):
        j, w = slice(p * rank, (p + 1) * rank), slice(p * per, (p + 1) * per)
        bp = b[ids[r], w]
        want[:, w] = np.einsum("rj,rnj->rn", t[:, j], bp) * on
        e = (K / 8 + 16) * u * ta[:, j] + (H[M.BF16] ** 2 + (rank + 8) * u) * np.abs(t[:, j])
        tol[:, w] = np.einsum("rj,rnj->rn", e, np.abs(bp))
    got = values(first[r, :N], c_dt)
    assert (np.abs(got - want) <= tol + (H[c_dt] + 2 * u) * np.abs(want)).all()


@pytest.mark.parametrize("c_dt", [M.BF16, M.F32], ids=NAME.get)
def test_lora_tiles_of_rows_past_32_bits(gpu, c_dt):
    # rows of 8388600 elements, the most there may be: a tile's 64 of them in fp32 end just below 2^31 bytes
    ld, rows, K, N, rank = (1 << 23) - 8, 300, 1024, 1032, 256
    rng = np.random.default_rng(7)
    (xb, x), (ab, a), (bb, b) = (stored(rng.standard_normal(s) * std, M.BF16) for s, std in
                                 (((rows, K), 1.0), ((2, rank, K), K ** -0.5), ((2, N, rank), rank ** -0.5)))
    cb, base = stored(rng.standard_normal((rows, N)), c_dt)
    size = cb.dtype.itemsize
    ids = (np.arange(rows) % 2).astype(np.int32)
    keep = [dev(v) for v in (ab, bb, ids)]
    xs, cs = M.Dev(((rows - 1) * ld + K) * 2), M.Dev(((rows - 1) * ld + N) * size)
    for r in range(rows):
        xs.write(xb[r], r * ld * 2)
        cs.write(cb[r], r * ld * size)
    g = M.LoraRowsArgs()
    g.x, g.a, g.b, g.ids, g.base, g.c = xs.p, keep[0].p, keep[1].p, keep[2].p, cs.p, cs.p
    g.ldx = g.ldbase = g.ldc = ld
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters, g.dtype, g.c_dtype = rows, K, N, rank, 1, 2, M.BF16, c_dt
    assert plan(g)[:3] == [0, 128, 512]
    need = C.c_uint64()
    M.call("mk_lora_rows_workspace", C.byref(g), C.byref(need))
    space = M.Dev(need.value)
    g.workspace, g.workspace_bytes = space.p, need.value
    M.call("mk_lora_rows", C.byref(g), None)
    M.sync()
    got = np.empty((rows, N), cb.dtype)
    for r in range(rows):
        M.call("mk_memcpy_d2h", got[r].ctypes.data, cs.p + r * ld * size, N * size)
    want, tol = base.copy(), np.zeros((rows, N))
    for i in range(2):
        r = ids == i
        t, ta = x[r] @ a[i].T, np.abs(x[r]) @ np.abs(a[i]).T
        want[r] += t @ b[i].T
        tol[r] = ((K / 8 + 16) * u * ta + (H[M.BF16] ** 2 + (rank + 8) * u) * np.abs(t)) @ np.abs(b[i]).T
    tol += (H[c_dt] + 2 * u) * np.abs(want) + 2 * u * np.abs(base)
    assert (np.abs(values(got, c_dt) - want) <= tol).all()


@pytest.mark.parametrize("size", [(4161, 1160, 72, 16, 1, 9), (130, 12296, 2072, 256, 1, 2), (77, 20000, 40, 48, 1, 3)])
def test_lora_takes_the_workspace_that_it_is_given(gpu, size):
    """From one split of K, the least that is taken, to all of them: the same rows, nothing behind the workspace, 16 bytes less refused."""
    rows, K, N, rank, parts, adapters = size
    least = -(-rows * (4 * parts * rank + 8) // 16) * 16
    a = Lora(*size, ids_of("mixed", rows, adapters), M.BF16, M.BF16)
    full = plan(a)[SPLITS]
    want, tol = a.want()
    for splits in (1, 2, full):
        g = a.args()
        size = least + (splits - 1) * rows * 4 * parts * rank
        space, guard = M.Dev(size + 4096), np.full(4096, 0x5A, np.uint8)
        M.call("mk_memset", space.p, 0xFF, size)
        space.write(guard, size)
        g.workspace, g.workspace_bytes = space.p, size
        assert plan(g)[SPLITS] <= splits and (splits < full or plan(g)[SPLITS] == full)
        M.call("mk_lora_rows", C.byref(g), None)
        assert (np.abs(a.result() - want) <= tol).all()
        assert np.array_equal(space.to_array(np.uint8, (size + 4096,))[size:], guard)
    g.workspace_bytes = least - 16
    with pytest.raises(M.MkError, match="workspace"):
        M.call("mk_lora_rows", C.byref(g), None)


def test_lora_rows_in_no_order_up_to_the_sort_s_reach(gpu):
    # 40000 rows of 26840 bf16 elements: 2147200000 bytes, the last row's offset just below 2^31
    rows, ld, K, N, rank = 40000, 26840, 16, 8, 8
    rng = np.random.default_rng(3)
    (xb, x), (ab, a), (bb, b) = (stored(rng.standard_normal(s), M.BF16) for s in ((rows, K), (3, rank, K), (3, N, rank)))
    ids = rng.integers(-1, 3, rows).astype(np.int32)
    keep = [dev(v) for v in (ab, bb, ids)]
    xs, cs = M.Dev(((rows - 1) * ld + K) * 2), M.Dev(((rows - 1) * ld + N) * 2)
    for r in range(rows):
        xs.write(xb[r], r * ld * 2)
    g = M.LoraRowsArgs()
    g.x, g.a, g.b, g.ids, g.c, g.ldx, g.ldc = xs.p, keep[0].p, keep[1].p, keep[2].p, cs.p, ld, ld
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters, g.dtype, g.c_dtype = rows, K, N, rank, 1, 3, M.BF16, M.BF16
    assert plan(g)[ORDER] == 1 and plan(g, ldc=ld + 8)[ORDER] == 0
    g.ldc = ld
    need = C.c_uint64()
    M.call("mk_lora_rows_workspace", C.byref(g), C.byref(need))
    space = M.Dev(need.value)
    g.workspace, g.workspace_bytes = space.p, need.value
    M.call("mk_lora_rows", C.byref(g), None)
    M.sync()
    got = np.empty((rows, N), np.uint16)
    for r in range(rows):
        M.call("mk_memcpy_d2h", got[r].ctypes.data, cs.p + r * ld * 2, N * 2)
    want, tol = np.zeros((rows, N)), np.zeros((rows, N))
    for i in range(3):
        r = ids == i
        t, ta = x[r] @ a[i].T, np.abs(x[r]) @ np.abs(a[i]).T
        want[r] = t @ b[i].T
        tol[r] = ((K / 8 + 16) * u * ta + (H[M.BF16] ** 2 + (rank + 8) * u) * np.abs(t)) @ np.abs(b[i]).T
    assert (np.abs(values(got, M.BF16) - want) <= tol + (H[M.BF16] + 2 * u) * np.abs(want)).all()


@pytest.mark.parametrize("seed", range(30))
def test_lora_random_sizes(gpu, seed):
    """Any sizes, on whichever kernels they take; tens of thousands of rows with short rows, few rows with long ones."""
    rng = np.random.default_rng(2000 + seed)
    parts, rank = int(rng.integers(1, 5)), 8 * int(rng.choice([1, 2, 3, 4, 5, 8, 9, 16, 20, 32]))
    rows = int(np.exp(rng.uniform(0, np.log(12000))))
    most = int(min(4096, 6e6 // rows, 3e8 // (rows * parts * rank)))
    K = 8 * int(rng.integers(1, max(most // 8, 1) + 1))
    N = 8 * parts * int(rng.integers(1, max(min(most, 3e8 / (rows * rank)) // (8 * parts), 1) + 1))
    adapters = int(rng.choice([1, 2, 3, 9, 40]))
    dt = int(rng.choice([M.BF16, M.F16]))
    in_place = bool(rng.random() < 0.3)
    a = Lora(rows, K, N, rank, parts, adapters, ids_of(str(rng.choice(["mixed", "runs", "none"])), rows, adapters, seed), dt, int(rng.choice([dt, M.F32])), seed=seed,
             pad=8 * int(rng.integers(0, 3)), base=in_place or bool(rng.random() < 0.8), scale=bool(rng.random() < 0.7), in_place=in_place, grouped=int(rng.random() < 0.3))
    print(a.sizes, plan(a), flush=True)
    a.check()


@pytest.mark.parametrize("size", [(4161, 520, 264, 24, 3, 5), (300, 1032, 24616, 16, 1, 3), (600, 8200, 64, 16, 1, 4)])
def test_lora_said_to_be_grouped_or_not_the_same_bits(gpu, size):
    for ids in ("mixed", "runs"):
        got = []
        for grouped in (0, 1):
            a = Lora(*size, ids_of(ids, size[0], size[5]), M.BF16, M.F32, grouped=grouped)
            assert plan(a)[ORDER] == 1 - grouped
            got.append(a.run().result())
        assert np.array_equal(*got)
