"""Which kernels of the int8 path the library holds, and which ones a launch can take (no GPU)."""
import ctypes as C
import re

import pytest

import mkimage as M
import test_gpu_int8_ops


def built(name, args):
    """The template arguments of the library's kernels of that name: whole numbers, in order."""
    pat = re.compile(rb"%d%s%sE" % (len(name), name.encode(), b"I" + rb"L[a-z](\d+)E" * args))
    return {tuple(map(int, m if args > 1 else (m,))) for m in pat.findall(M.LIB_PATH.read_bytes())}


def cdiv(a, b):
    return -(-a // b)


def test_gate_norm_kernels_are_those_that_a_width_takes():
    # waves a row by its width, then the float4s a thread that hold it
    def kernel(n):
        w = next((w for w, most in ((1, 512), (2, 1536), (4, 3328), (8, 8192)) if n <= most), 16)
        return w, cdiv(n, 256 * w)

    assert built("gate_norm_kernel", 2) == {kernel(n) for n in range(4, 16385, 4)}


def test_quantize_kernels_are_those_that_a_width_takes():
    # the fewest waves that hold the row in 24 elements a thread, 16 beyond; then 8 elements at a time
    def kernel(n):
        w = next((w for w in (1, 2, 4, 8) if n <= 1536 * w), 16)
        return w, cdiv(n, 512 * w)

    used = {kernel(n) for n in range(16, 65537, 16)}
    assert built("quantize_i8_kernel", 3) == {(t,) + k for t in (M.F32, M.BF16, M.F16) for k in used}
    assert built("quantize_i8_any_kernel", 1) == {(t,) for t in (M.F32, M.BF16, M.F16)}


# ---------------------------------------------------------------------------------------------------------------------
# the product: which kernel a launch takes on 256 compute units
# ---------------------------------------------------------------------------------------------------------------------

GLU = (M.EPI_SWIGLU, M.EPI_GEGLU)


def args(m, n, k, epi=M.EPI_STORE, batch=1, lda=None):
    g = M.GemmArgs()
    g.a = g.w = g.c = g.gate = g.wscale = 4096  # (not read)
    g.M, g.N, g.K, g.lda, g.ldc, g.batch = m, n, k, lda or k, n, batch
    g.w_dtype, g.c_dtype, g.epilogue = M.I8, M.F32, epi
    return g


def plan(m, n, k, epi=M.EPI_STORE, batch=1, lda=None, cus=256):
    """(rows, channels, k steps in LDS, workgroups in chains, side of the last round's parts, workgroups) of a launch"""
    out = (C.c_uint32 * 6)()
    M.call("mk_gemm_i8_plan", C.byref(args(m, n, k, epi, batch, lda)), cus, out)
    return tuple(out)


def kind(*a, **kw):
    """The plan without its numbers of workgroups: one of KINDS, or of KINDS_GLU for a gated unit."""
    bm, bn, stages, chains, side, _ = plan(*a, **kw)
    return (bm, bn, stages) if bm < 256 else (256, "chain" if chains else "one", side)


MIXED = {(128, 128, 4), (256, "one", 0), (256, "one", 64), (256, "one", 128)}
TILES = {(64, 64, 4), (64, 128, 4), (64, 128, 2), (128, 128, 2)}
KINDS_GLU = {(16, 32, 0), (32, 64, 6)} | TILES | MIXED
KINDS = {(16, 16, 0), (32, 32, 8), (64, 32, 6)} | TILES | MIXED | {(256, "chain", 0), (256, "chain", 64), (256, "chain", 128)}

# A shape for each: m, n, k of a batch of 3 whose rows are padded by 16 (gated: 2 n / 2 channels of both parts), with more k
# steps than a workgroup keeps in LDS.
SHAPES = {(16, 16, 0): (37, 136, 336), (16, 32, 0): (37, 136, 336), (32, 32, 8): (37, 520, 1040), (32, 64, 6): (37, 1032, 848),
          (64, 32, 6): (37, 1544, 848), (64, 64, 4): (37, 3080, 592), (64, 128, 2): (37, 6152, 336), (64, 128, 4): (37, 6152, 848),
          (128, 128, 2): (130, 8200, 592), (128, 128, 4): (130, 4104, 592), (256, "one", 0): (257, 8200, 592),
          (256, "one", 64): (1537, 6152, 592), (256, "one", 128): (1030, 5128, 336), (256, "chain", 0): (900, 8200, 400),
          (256, "chain", 64): (1537, 6152, 400), (256, "chain", 128): (2600, 4104, 400)}


def kinds(epi):
    return sorted(KINDS_GLU if epi in GLU else KINDS, key=str)


@pytest.mark.parametrize("epi", [M.EPI_STORE, M.EPI_GATE_ADD, M.EPI_SWIGLU])
def test_every_kernel_has_a_shape_that_takes_it(epi):
    for want in kinds(epi):
        m, n, k = SHAPES[want]
        assert kind(m, n, k, epi, batch=3, lda=k + 16) == want
        assert want[0] == 16 or -(-k // 128) > (2 if want[0] == 256 else want[2])


def test_the_library_holds_the_kernels_that_a_launch_takes():
    plain, gated = range(3), (3,)  # epilogue classes: store, activation, residual; gated unit
    assert built("gemm_i8_kernel", 4) == {t + (e,) for ks, es in ((KINDS, plain), (KINDS_GLU, gated)) for e in es
                                          for t in ks - MIXED if t[0] not in (16, 256)}
    assert built("gemm_i8_mixed_kernel", 2) == {(e, chain) for e in plain for chain in (0, 1)} | {(3, 0)}
    assert built("gemm_i8_16_kernel", 1) == {(e,) for e in range(4)}


@pytest.mark.parametrize("epi", [M.EPI_STORE, M.EPI_SWIGLU])
def test_no_launch_takes_another_kernel(epi):
    known = KINDS_GLU if epi in GLU else KINDS
    seen = {kind(m, n, k, epi, batch) for m in (1, 17, 50, 100, 200, 500, 1000, 2000, 5000, 33333)
            for n in (8, 72, 520, 1032, 2568, 4104, 8200, 30000) for k in (16, 176, 400, 1168, 4112, 131056) for batch in (1, 3)}
    assert seen <= known


@pytest.mark.parametrize("epi, want", [(M.EPI_STORE, KINDS - {(16, 16, 0)}), (M.EPI_GEGLU, KINDS_GLU)])
def test_many_tiles_shapes_reach_every_kernel(epi, want):
    marks = test_gpu_int8_ops.test_product_many_tiles.pytestmark
    shapes = next(m.args[1] for m in marks if m.name == "parametrize" and m.args[0] == "m, n, k")
    assert {kind(m, n - n % 8 if epi in GLU else n, k, epi) for m, n, k in shapes} == want


def test_plan_follows_the_device():
    # half the rows on half the compute units: the same tiles
    for m, n, k in ((2048, 8192, 4096), (4096, 4096, 4096), (16384, 4096, 4096)):
        whole, half = plan(m, n, k, cus=256), plan(m // 2, n, k, cus=128)
        assert whole[:3] == half[:3] and whole[4] == half[4]
    assert plan(16384, 4096, 4096)[3] == 256 and plan(16384, 4096, 4096, cus=64)[3] == 64


def test_plan_refusals():
    f, out = M.lib().mk_gemm_i8_plan, (C.c_uint32 * 6)()
    g = args(5, 64, 64)
    assert f(None, 256, out) == 1 and f(C.byref(g), 0, out) == 1 and f(C.byref(g), 256, None) == 1
    for kw, word in ((dict(M=0), b"empty"), (dict(batch=0), b"empty"), (dict(K=24), b"K must"), (dict(w_dtype=M.BF16), b"MK_I8"),
                     (dict(lda=48), b"lda"), (dict(wscale=None), b"null"), (dict(M=0x7FFFFFFF), b"2^31")):
        g = args(5, 64, 64)
        for k, v in kw.items():
            setattr(g, k, v)
        assert f(C.byref(g), 256, out) == 1 and word in M.lib().mk_last_error()
    # more workgroups than a grid holds, on any of the tiles
    g = args(0x7FFFFF00, 64, 16, batch=65535)
    assert f(C.byref(g), 256, out) == 1 and b"2^32" in M.lib().mk_last_error()
