"""Calls whose sizes leave nothing to do: MK_OK, with null operands too (an empty array's address is often null). No GPU."""
import ctypes as C

import pytest

import mkimage as M


def ok(name, g):
    status = getattr(M.lib(), name)(C.byref(g), None)
    assert status == 0, M.lib().mk_last_error().decode()


@pytest.mark.parametrize("docs", [[], [(0, 0, 0, 8, 0, 0, 0), (0, 0, 5, 5, 0, 0, 0)], [(0, 0, 0, 0, 0, 0, 0)]])
def test_attention_of_no_rows(docs):
    g = M.AttnPackedArgs()
    g.ldq = g.ldo = g.ldk = g.ldv = 256
    g.heads = g.kv_heads = 2
    g.d, g.dtype, g.out_dtype = 128, M.BF16, M.BF16
    table = (M.AttnDoc * max(len(docs), 1))(*[M.AttnDoc(*v) for v in docs])
    g.docs, g.n_docs = table if docs else None, len(docs)
    ok("mk_attention_packed", g)
    need = C.c_uint64(7)
    assert M.lib().mk_attention_packed_workspace(C.byref(g), C.byref(need)) == 0 and need.value == 0
    g.d = 96  # sizes are checked all the same
    assert M.lib().mk_attention_packed(C.byref(g), None) == 1


def test_attention_with_rows_and_null_operands_is_refused():
    for lost, k_rows in (("q", 8), ("out", 8), ("k", 8), ("v", 8), ("q", 0), ("out", 0)):
        g = M.AttnPackedArgs()
        g.q = g.k = g.v = g.out = 1 << 20
        g.ldq = g.ldo = g.ldk = g.ldv = 256
        g.heads = g.kv_heads = 2
        g.d, g.dtype, g.out_dtype = 128, M.BF16, M.BF16
        table = (M.AttnDoc * 2)(M.AttnDoc(0, 0, 0, 8, 0, 0, 0), M.AttnDoc(0, 4, 0, k_rows, 0, 0, 0))
        g.docs, g.n_docs = table, 2
        setattr(g, lost, None)
        assert M.lib().mk_attention_packed(C.byref(g), None) == 1 and b"null" in M.lib().mk_last_error()


def test_adapters_of_no_rows():
    g = M.LoraRowsArgs()
    g.ldx, g.ldbase, g.ldc = 256, 96, 96
    g.K, g.N, g.rank, g.parts, g.adapters = 256, 96, 16, 3, 2
    g.dtype, g.c_dtype = M.BF16, M.F32
    ok("mk_lora_rows", g)
    g.ldbase = 104  # (no base and no c: nothing is in place)
    ok("mk_lora_rows", g)
    g.rank = 12
    assert M.lib().mk_lora_rows(C.byref(g), None) == 1


@pytest.mark.parametrize("kv", [0, 2])
def test_rotary_of_no_rows(kv):
    g = M.RopeRowsArgs()
    g.ldq = g.ldqo = g.ldk = g.ldko = 512
    g.heads, g.kv_heads, g.d = 4, kv, 128
    g.dtype, g.out_dtype, g.pos_dtype = M.F32, M.BF16, M.I32
    g.pos_ld, g.axes, g.axis_dims = 1, 1, (C.c_uint32 * 4)(128)
    g.theta, g.rope_mode = 10000.0, 1
    ok("mk_rope_rows", g)
    g.d = 96
    assert M.lib().mk_rope_rows(C.byref(g), None) == 1
