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


@pytest.mark.parametrize("rows, heads, kv, d, workspace", [(1, 1, 1, 128, False), (3, 4, 1, 64, True), (40, 1, 1, 64, False)])
def test_half_weights_far_below_the_largest(gpu, rows, heads, kv, d, workspace):
    """2^17 keys that each weigh about 2^-25.5 of one: together 0.3% of it. A weight loses 2^-31 of the largest at most."""
    n = (1 << 17) + 1

    def edit(raw):
        one_dim(raw)
        raw["k"][:, :, 5] = -17.675
        raw["v"][:] = 1.0
        # (the last key's tile is the first one taken)
        raw["k"][-1, :, 5] = raw["v"][-1] = 0.0

    a = Attn([(0, rows, 0, n, n - 1, 0, 0)], rows, n, heads, kv, d, M.F16, scale=1.0, edit=edit)
    got = values(a.run(workspace).result()[0], M.F16)
    p = np.exp(a.val["k"][0, 0, 5]) * (n - 1)
    want = p / (1 + p)
    assert 2.0 ** -9 < want < 2.0 ** -8
    assert np.abs(got - want).max() <= (2 * H[M.F16] + (n + 2 * d) * u) * want + n * 2.0 ** -31


@pytest.mark.parametrize("part", [0.0, 0.3, 0.9])
def test_attention_takes_the_workspace_that_it_is_given(gpu, part):
    """A workspace of a part of what the keys' best split needs, none of it among them: fewer splits, the same rows."""
    docs, nq, nk = packed([1, 3, 7], [4099, 777, 1500], mask="causal")
    for heads, kv, d in ((8, 1, 128), (8, 8, 64), (40, 2, 64)):
        a = Attn(docs, nq, nk, heads, kv, d, M.BF16)
        g, need = a.args(), C.c_uint64()
        M.call("mk_attention_packed_workspace", C.byref(g), C.byref(need))
        assert need.value > 4096
        size = int(need.value * part) // 16 * 16
        space, guard = M.Dev(need.value), np.full(need.value - size, 0x5A, np.uint8)
        M.call("mk_memset", space.p, 0xFF, need.value)
        space.write(guard, size)
        g.workspace, g.workspace_bytes = space.p, size
        M.call("mk_attention_packed", C.byref(g), None)
        got, mine = a.result()
        assert np.array_equal(space.to_array(np.uint8, (need.value,))[size:], guard)
        want, tol = attend(a.val["q"], a.val["k"], a.val["v"], docs, a.scale, 0.0, None, M.BF16, M.BF16)
        assert (np.abs(values(got, M.BF16) - want)[mine] <= tol[mine]).all()


def test_attention_one_workspace_for_a_large_batch_and_small_ones(gpu):
    # the rows of four images fill the chip without splits, so they need none
    big, need = Attn(packed([2176, 1101, 2377, 1801])[0], 1, 1, 32, 32, 64, M.BF16), C.c_uint64(7)
    M.call("mk_attention_packed_workspace", C.byref(big.args()), C.byref(need))
    space = M.Dev(max(need.value, 16))
    for lens_q, lens_k in (([1], [16411]), ([1, 1, 1], [5000, 77, 900]), ([40], [3000])):
        docs, nq, nk = packed(lens_q, lens_k, mask="causal")
        a = Attn(docs, nq, nk, 8, 2, 64, M.BF16)
        g = a.args()
        g.workspace, g.workspace_bytes = space.p, need.value
        M.call("mk_attention_packed", C.byref(g), None)
        got, mine = a.result()
        want, tol = attend(a.val["q"], a.val["k"], a.val["v"], docs, a.scale, 0.0, None, M.BF16, M.BF16)
        assert (np.abs(values(got, M.BF16) - want)[mine] <= tol[mine]).all()


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("form", ["one wave", "four waves", "split, one wave", "split, four waves"])
def test_unseen_values_reach_nothing_on_any_variant(gpu, form, where, bad, dt):
    """As test_attention_unseen_rows_reach_nothing, in half too, with up to 16 rows a key head (one wave a workgroup) and with keys
    split over workgroups, capped and with a bias; every row behind a document is bad for 70 rows, more than a tile."""
    one, split = "one" in form, "split" in form
    lens_q = [3, 7, 1, 5] if one else [3, 40, 100, 33]
    lens_k = [1500, 1200, 17, 2050] if split else [65, 33, 1, 130] if one else [65, 100, 101, 33]
    docs, nq, nk = packed(lens_q, lens_k, mask="causal", gap=70)
    nq, nk = nq + 70, nk + 70

    def edit(raw):
        x = raw[where]
        for doc in docs:
            end = doc[2] + doc[3]
            x[end:end + 70] = bad
            if doc[3] > 1:
                x[end - 1, 0] = bad
                x[end - 1 - doc[1] // 2, 1, 3] = bad

    for heads, kv, d, cap, slopes in ((2, 2, 64, 0.0, None), (4, 2, 128, 0.0, np.float32([0.5, 0.25, 0.0, 0.01])), (2, 2, 64, 9.0, None)):
        a = Attn(docs, nq, nk, heads, kv, d, dt, cap=cap, slopes=slopes, edit=edit, seed=len(form))
        g, need = a.args(), C.c_uint64()
        M.call("mk_attention_packed_workspace", C.byref(g), C.byref(need))
        assert (need.value > 0) == split, need.value
        got, mine = a.run().result()
        got = values(got, dt)
        want, tol = attend(a.val["q"], a.val["k"], a.val["v"], docs, a.scale, cap, slopes, dt, dt)
        with np.errstate(all="ignore"):
            fine = np.isfinite(want) & mine[:, None, None]
            assert (np.abs(got - want)[fine] <= tol[fine]).all()
            rest = ~np.isfinite(want) & mine[:, None, None]
            assert not np.isfinite(got[rest]).any()
            # a seen NaN makes its row NaN: all dims of it in K, its own in V
            assert rest.any() and (not np.isnan(bad) or np.isnan(got[rest]).all())


def test_seen_scores_of_infinity_make_the_row_nan(gpu):
    for dt in (M.BF16, M.F16):
        for rows, nk in ((5, 90), (40, 300)):
            def edit(raw):
                one_dim(raw)
                raw["k"][nk - rows + 2, :, 5] = np.inf

            docs = [(0, rows, 0, nk, nk - rows, CAUSAL, 0)]
            a = Attn(docs, rows, nk, 2, 2, 64, dt, edit=edit)
            got = values(a.run().result()[0], dt)
            assert np.isnan(got[2:]).all() and np.isfinite(got[:2]).all()


def test_no_keys_and_null_k_and_v(gpu):
    a = Attn([(0, 5, 0, 0, 0, 0, 0), (7, 140, 3, 0, 4, CAUSAL, 0)], 150, 1, 2, 2, 64, M.BF16)
    g = a.args()
    g.k = g.v = None
    M.call("mk_attention_packed", C.byref(g), None)
    got, mine = a.result()
    assert (got[mine] == 0).all() and mine.sum() == 145


@pytest.mark.parametrize("dt", [M.BF16, M.F16], ids=NAME.get)
@pytest.mark.parametrize("rows, nk, workspace", [(1, 1, False), (3, 130, True), (3, 2000, True), (70, 300, False)])
def test_a_row_with_one_key_of_weight_is_its_value(gpu, rows, nk, workspace, dt):
    """The largest score's own weight is a power of two, with no rounding: scores up to 1000, off by 2^-14 at most (2^-25 of them in log2
    units), move the weight and the sum alike by far less than half a step of the output's type."""
    for d, heads, kv, slopes in ((64, 3, 3, None), (128, 4, 1, None), (64, 2, 2, np.float32([0.25, 0.0]))):
        def edit(raw):
            one_dim(raw)
            raw["k"][:, :, 5] = -900.0
            for g in range(kv):
                raw["k"][(7 * g + 5) % nk, g, 5] = 0.37 * 2 ** (4 * g)

        a = Attn([(0, rows, 0, nk, nk - rows, 0, 0)], rows, nk, heads, kv, d, dt, scale=1.0, slopes=slopes, edit=edit)
        got = a.run(workspace).result()[0]
        bits = M.bf16_bits if dt == M.BF16 else M.f16_bits
        for h in range(heads):
            g = h // (heads // kv)
            want = bits(a.val["v"][(7 * g + 5) % nk, g].astype(np.float32))
            assert (got[:, h] == want).all(), (d, h)
