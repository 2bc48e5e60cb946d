"""mk_gemm_i8, mk_gate_norm and mk_quantize_i8_rows without a GPU: what they refuse, before any device work, and the
binding's extent checks of their operands."""
import ctypes as C

import pytest

import mkimage as M
from test_binding_extents import stub  # noqa: F401

PTR = 0x7F0000000000  # an address that nothing here reads


def gemm(**kw):
    g = M.GemmArgs()
    g.a = g.w = g.c = g.wscale = g.bias = PTR
    g.M, g.N, g.K, g.lda, g.ldc, g.batch = 0, 64, 64, 64, 64, 1
    g.w_dtype, g.c_dtype, g.epilogue = M.I8, M.BF16, M.EPI_STORE
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def gemm_status(ascale=PTR, **kw):
    return M.lib().mk_gemm_i8(C.byref(gemm(**kw)), ascale, None)


def test_gemm_i8_takes_what_it_documents():
    # M = 0: every check runs and nothing is launched
    for kw in (dict(), dict(K=16, lda=16), dict(N=4, ldc=4), dict(K=131056, lda=131056), dict(bias=None),
               dict(N=8, ldc=4, epilogue=M.EPI_SWIGLU), dict(epilogue=M.EPI_ADD, c_dtype=M.F32),
               dict(epilogue=M.EPI_GATE_TANH, c_dtype=M.F32, gate=PTR, gate_alt=-8, split=3, seg_rows=7),
               dict(lda=80, ldc=68), dict(batch=0, M=5), dict(c=PTR + 8), dict(batch=3, stride_a=16, stride_c=4)):
        assert gemm_status(**kw) == 0, (kw, M.lib().mk_last_error())


@pytest.mark.parametrize("kw, status, word", [
    (dict(a=None), 1, b"null"), (dict(w=None), 1, b"null"), (dict(c=None), 1, b"null"), (dict(wscale=None), 1, b"null"),
    (dict(ascale=None), 1, b"null"), (dict(w_dtype=M.BF16), 1, b"MK_I8"), (dict(w_dtype=M.FP8), 1, b"MK_I8"),
    (dict(epilogue=M.EPI_HEADS), 5, b"HEADS"), (dict(epilogue=M.EPI_PAIR_SUM), 5, b"PAIR_SUM"),
    (dict(epilogue=10), 1, b"epilogue"), (dict(K=0), 1, b"K must"), (dict(K=24), 1, b"K must"), (dict(N=0), 1, b"K must"),
    (dict(N=6), 1, b"K must"), (dict(N=12, epilogue=M.EPI_GEGLU), 1, b"K must"),
    (dict(K=131072, lda=131072), 1, b"K must"), (dict(c_dtype=M.I8), 1, b"C must"), (dict(c_dtype=M.FP8), 1, b"C must"),
    (dict(epilogue=M.EPI_ADD), 1, b"f32 C"), (dict(epilogue=M.EPI_GATE_ADD, gate=PTR), 1, b"f32 C"),
    (dict(epilogue=M.EPI_GATE_ADD, c_dtype=M.F32), 1, b"without a gate"), (dict(lda=48), 1, b"lda"),
    (dict(lda=72), 1, b"lda"), (dict(lda=1 << 23), 1, b"lda"), (dict(ldc=60), 1, b"lda"), (dict(ldc=66), 1, b"lda"),
    (dict(batch=2, stride_a=8), 1, b"lda"), (dict(batch=2, stride_c=2), 1, b"lda"), (dict(a=PTR + 8), 1, b"aligned"),
    (dict(w=PTR + 1), 1, b"aligned"), (dict(wscale=PTR + 4), 1, b"aligned"), (dict(bias=PTR + 8), 1, b"aligned"),
    (dict(ascale=PTR + 2), 1, b"aligned"), (dict(c=PTR + 4), 1, b"aligned"), (dict(c=PTR + 8, c_dtype=M.F32), 1, b"aligned"),
    (dict(epilogue=M.EPI_GATE_ADD, c_dtype=M.F32, gate=PTR + 4), 1, b"aligned"),
    (dict(epilogue=M.EPI_GATE_ADD, c_dtype=M.F32, gate=PTR, gate_alt=2), 1, b"aligned"),
    (dict(M=0x7FFFFFFF), 1, b"2^31"), (dict(M=1, batch=65536), 1, b"65535"),
])
def test_gemm_i8_refusals(kw, status, word):
    assert gemm_status(**kw) == status
    assert word in M.lib().mk_last_error()


def test_gemm_i8_null_arguments():
    assert M.lib().mk_gemm_i8(None, PTR, None) == 1


def test_mk_gemm_still_refuses_int8_weights():
    g = gemm(M=4)
    assert M.lib().mk_gemm(C.byref(g), None) == 1 and b"weights must be" in M.lib().mk_last_error()


def gate_norm(**kw):
    g = M.GateNormArgs()
    g.x = g.x_out = g.y = g.out = PTR
    g.n, g.ldx, g.ldy, g.ldo = 64, 64, 64, 64
    g.y_dtype, g.out_dtype, g.norm2, g.eps1, g.eps2 = M.BF16, M.BF16, M.NORM_LAYER, 1e-6, 1e-6
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def gate_norm_status(**kw):
    return M.lib().mk_gate_norm(C.byref(gate_norm(**kw)), None)


def test_gate_norm_takes_what_it_documents():
    for kw in (dict(), dict(n=4, ldx=4, ldy=4, ldo=4), dict(n=16384, ldx=16384, ldy=16384, ldo=16384),
               dict(y=None, x_out=None), dict(out=None, norm2=0), dict(x_out=None), dict(norm2=0),
               dict(out_dtype=M.I8, out_scale=PTR), dict(norm1=M.NORM_RMS, w1=PTR, norm2=M.NORM_RMS, w2=PTR),
               dict(norm1=M.NORM_LAYER, w1=PTR, b1=PTR, b2=PTR), dict(gate=PTR, scale=PTR, shift=PTR, alt=-4, mod_stride=8),
               dict(y=PTR + 8, out=PTR + 4, out_dtype=M.I8, out_scale=PTR + 4), dict(y_dtype=M.F32, out_dtype=M.F32)):
        assert gate_norm_status(**kw) == 0, (kw, M.lib().mk_last_error())


@pytest.mark.parametrize("kw, word", [
    (dict(x=None), b"null"), (dict(y=None, out=None, x_out=None, norm2=0), b"null"), (dict(n=0), b"multiple of 4"),
    (dict(n=62), b"multiple of 4"), (dict(n=16388, ldx=16388, ldy=16388, ldo=16388), b"multiple of 4"),
    (dict(norm1=3), b"NONE"), (dict(norm2=3), b"NONE"), (dict(norm1=M.NORM_RMS, b1=PTR), b"NONE"),
    (dict(norm2=M.NORM_RMS, b2=PTR), b"NONE"), (dict(w1=PTR), b"NONE"), (dict(norm2=0, w2=PTR), b"NONE"),
    (dict(y=None), b"need y"), (dict(y=None, x_out=None, gate=PTR), b"need y"),
    (dict(y=None, x_out=None, norm1=1), b"need y"), (dict(y=None, x_out=None, residual_scale=0.5), b"need y"),
    (dict(out=None), b"need out"), (dict(out=None, norm2=0, scale=PTR), b"need out"),
    (dict(out=None, norm2=0, shift=PTR), b"need out"), (dict(out=None, norm2=0, x_out=None), b"no output"),
    (dict(y_dtype=M.FP8), b"y must"), (dict(y_dtype=M.I8), b"y must"), (dict(out_dtype=M.FP8), b"y must"),
    (dict(out_dtype=M.I8), b"out_scale"), (dict(ldx=60), b"ldx"), (dict(ldy=66), b"ldx"), (dict(ldo=-64), b"ldx"),
    (dict(gate=PTR, alt=2), b"alt"), (dict(scale=PTR, mod_stride=1), b"alt"), (dict(x=PTR + 8), b"aligned"),
    (dict(x_out=PTR + 4), b"aligned"), (dict(y=PTR + 4), b"aligned"), (dict(out=PTR + 2), b"aligned"),
    (dict(out=PTR + 8, out_dtype=M.F32), b"aligned"), (dict(gate=PTR + 4), b"aligned"), (dict(scale=PTR + 8), b"aligned"),
    (dict(shift=PTR + 8), b"aligned"), (dict(w2=PTR + 4), b"aligned"), (dict(b2=PTR + 4), b"aligned"),
    (dict(norm1=1, w1=PTR + 4), b"aligned"), (dict(norm1=2, b1=PTR + 4), b"aligned"),
    (dict(out_dtype=M.I8, out_scale=PTR + 2), b"aligned"), (dict(rows=0x80000000), b"2^31"),
])
def test_gate_norm_refusals(kw, word):
    assert gate_norm_status(**kw) == 1
    assert word in M.lib().mk_last_error()


def test_gate_norm_null_arguments():
    assert M.lib().mk_gate_norm(None, None) == 1


def test_quantize_i8_refusals():
    f = M.lib().mk_quantize_i8_rows
    assert f(PTR, M.BF16, 0, 64, 64, PTR, PTR, None) == 0
    for args in ((None, M.BF16, 0, 64, 64, PTR, PTR), (PTR, M.BF16, 0, 64, 64, None, PTR),
                 (PTR, M.BF16, 0, 64, 64, PTR, None), (PTR, M.FP8, 0, 64, 64, PTR, PTR), (PTR, M.I8, 0, 64, 64, PTR, PTR),
                 (PTR, M.BF16, 0, 0, 64, PTR, PTR), (PTR, M.BF16, 0, 64, 63, PTR, PTR), (PTR, M.BF16, 0, 64, -64, PTR, PTR),
                 (PTR, M.BF16, 1 << 31, 64, 64, PTR, PTR), (PTR + 1, M.BF16, 0, 64, 64, PTR, PTR),
                 (PTR + 2, M.F32, 0, 64, 64, PTR, PTR), (PTR, M.BF16, 0, 64, 64, PTR, PTR + 2)):
        assert f(*args, None) == 1, args
        assert b"quantize_i8_rows" in M.lib().mk_last_error()


def test_extents(stub):  # noqa: F811
    lib, alloc = stub
    rows, n, k = 5, 64, 96

    def call(short):
        need = dict(a=rows * k, w=n * k, c=rows * n * 2, wscale=n * 4, bias=n * 4, ascale=rows * 4)
        p = {q: alloc(b - (4 if q == short else 0)) for q, b in need.items()}
        s = p.pop("ascale")
        M.call("mk_gemm_i8", C.byref(gemm(M=rows, K=k, lda=k, **p)), s, None)

    call(None)
    for short in ("a", "w", "c", "wscale", "bias", "ascale"):
        with pytest.raises(M.MkError, match="mk_gemm_i8: %s:" % (short.upper() if len(short) == 1 else short)):
            call(short)
    g = gemm(M=rows, K=k, lda=k, a=alloc(rows * k), w=alloc(n * k), c=alloc(rows * n * 4), wscale=alloc(n * 4), bias=None,
             epilogue=M.EPI_GATE_ADD, c_dtype=M.F32, gate=alloc((n + 64) * 4 - 4), gate_alt=64, split=2, seg_rows=5)
    with pytest.raises(M.MkError, match="gate"):
        M.call("mk_gemm_i8", C.byref(g), alloc(rows * 4), None)

    def norm(short):
        need = dict(x=rows * n * 4, x_out=rows * n * 4, y=rows * n * 2, out=rows * n, out_scale=rows * 4, w2=n * 4,
                    gate=(2 * 200 + 100 + n) * 4, shift=(2 * 200 + 100 + n) * 4)
        p = {q: alloc(b - (4 if q == short else 0)) for q, b in need.items()}
        M.call("mk_gate_norm", C.byref(gate_norm(rows=rows, out_dtype=M.I8, seg_rows=2, split=1, alt=100, mod_stride=200, **p)),
               None)

    norm(None)
    for short in ("x", "x_out", "y", "out", "out_scale", "w2", "gate", "shift"):
        with pytest.raises(M.MkError, match="mk_gate_norm: %s:" % short):
            norm(short)
    M.call("mk_quantize_i8_rows", alloc((4 * 80 + 64) * 4), M.F32, rows, 64, 80, alloc(rows * 64), alloc(rows * 4), None)
    for src, dst, sc in ((4, 0, 0), (0, 1, 0), (0, 0, 4)):
        with pytest.raises(M.MkError, match="mk_quantize_i8_rows"):
            M.call("mk_quantize_i8_rows", alloc((4 * 80 + 64) * 4 - src), M.F32, rows, 64, 80, alloc(rows * 64 - dst),
                   alloc(rows * 4 - sc), None)
    assert lib.calls == ["mk_gemm_i8", "mk_gate_norm", "mk_quantize_i8_rows"]
