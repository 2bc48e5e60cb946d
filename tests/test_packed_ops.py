"""Refusals of the packed batch's entry points, host only: every one comes before a launch, so no device is needed."""
import ctypes as C

import pytest

import mkimage as M

P = 1 << 20  # an aligned address that no call may touch


def refused(name, args, *rest, match=""):
    L = M.lib()
    status = getattr(L, name)(C.byref(args), *rest)
    assert status == 1, status
    assert match in L.mk_last_error().decode()


def attn(**kw):
    g = M.AttnPackedArgs()
    g.q = g.k = g.v = P
    g.out = 4 * P
    g.ldq = g.ldo = 512
    g.ldk = g.ldv = 256
    g.dtype = g.out_dtype = M.BF16
    g.heads, g.kv_heads, g.d, g.scale = 4, 2, 128, 0.1
    docs = kw.pop("docs", [(0, 8, 0, 8, 0, 0, 0)])
    g.table = (M.AttnDoc * max(len(docs), 1))(*[M.AttnDoc(*v) for v in docs])
    g.docs, g.n_docs = g.table, len(docs)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize("kw, match", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(dtype=M.F32), "bf16 or f16"), (dict(out_dtype=M.I8), "output"),
    (dict(heads=0), "kv_heads"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=3), "kv_heads"), (dict(heads=65536), "kv_heads"),
    (dict(d=96), "head dim"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(cap=-2.0), "cap"), (dict(cap=float("inf")), "cap"), (dict(cap=4097.0), "cap"), (dict(scale=1.2e38, cap=1e-3), "cap"), (dict(scale=3e38), "scale"), (dict(ldq=504), "rows must"), (dict(ldq=516), "rows must"), (dict(ldk=-256), "rows must"),
    (dict(ldv=1 << 24), "rows must"), (dict(ldo=500), "rows must"), (dict(docs=None), "null"), (dict(q=P + 8), "aligned"), (dict(out=P + 2), "aligned"),
    (dict(workspace=P + 4), "aligned"), (dict(slopes=P + 2), "aligned"),
    (dict(docs=[(0, 8, 0, 8, 0, 0, 0), (7, 2, 0, 8, 0, 0, 0)]), "share"), (dict(docs=[(10, 8, 0, 8, 0, 0, 0), (0, 11, 0, 8, 0, 0, 0)]), "share"),
    (dict(docs=[(0xFFFFFFF0, 100, 0, 8, 0, 0, 0)]), "2^31"), (dict(docs=[(0, 8, 0x7FFFFFFF, 1, 0, 0, 0)]), "2^31"),
    (dict(docs=[(0, 8, 0, 8, 0x7FFFFFFF, 0, 0)]), "positions"), (dict(docs=[(0, (1 << 27) + 1, 0, 8, 0, 0, 0)]), "2^29")])
def test_attention_packed_refusals(kw, match):
    if kw.get("docs", 0) is None:
        g = attn()
        g.docs = None
    else:
        g = attn(**kw)
    refused("mk_attention_packed", g, None, match=match)


def test_attention_packed_nothing_to_do():
    for docs in ([], [(0, 0, 0, 8, 0, 0, 0), (0, 0, 5, 5, 0, 0, 0)]):
        g = attn(docs=docs)
        assert M.lib().mk_attention_packed(C.byref(g), None) == 0
        need = C.c_uint64(7)
        assert M.lib().mk_attention_packed_workspace(C.byref(g), C.byref(need)) == 0 and need.value == 0
    assert M.lib().mk_attention_packed(None, None) == 1
    assert M.lib().mk_attention_packed_workspace(C.byref(attn()), None) == 1


def lora(**kw):
    g = M.LoraRowsArgs()
    g.x = g.a = g.b = g.base = P
    g.c, g.workspace, g.workspace_bytes = 4 * P, 8 * P, 1 << 30
    g.ldx, g.ldbase, g.ldc = 256, 96, 96
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters = 5, 256, 96, 16, 3, 2
    g.dtype, g.c_dtype = M.BF16, M.F32
    for k, v in kw.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize("kw, match", [
    (dict(x=None), "null"), (dict(c=None), "null"), (dict(dtype=M.F32), "bf16 or f16"), (dict(c_dtype=M.I8), "base and c"), (dict(parts=0), "parts"),
    (dict(parts=5), "parts"), (dict(rank=0), "parts"), (dict(rank=12), "parts"), (dict(rank=264), "parts"), (dict(adapters=0), "adapter"), (dict(K=0), "K must"),
    (dict(K=252), "K must"), (dict(N=88), "K must"), (dict(N=0), "K must"), (dict(rows=(1 << 28) + 1), "rows"), (dict(grouped=2), "grouped"), (dict(ldx=248), "ldx"), (dict(ldx=1 << 23), "ldx"), (dict(ldc=1 << 23), "ldx"), (dict(ldbase=1 << 24), "ldx"), (dict(K=(1 << 22) + 8), "K must"), (dict(ldx=260), "ldx"),
    (dict(ldc=88), "ldx"), (dict(ldbase=100), "ldx"), (dict(base=4 * P, ldbase=104), "in place"), (dict(x=P + 8), "aligned"), (dict(c=P + 4), "aligned"),
    (dict(ids=P + 1), "aligned"), (dict(workspace=P + 8), "aligned"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=16), "workspace")])
def test_lora_rows_refusals(kw, match):
    refused("mk_lora_rows", lora(**kw), None, match=match)


def test_lora_rows_nothing_to_do():
    assert M.lib().mk_lora_rows(C.byref(lora(rows=0, workspace=None)), None) == 0
    need = C.c_uint64(7)
    assert M.lib().mk_lora_rows_workspace(C.byref(lora(rows=0)), C.byref(need)) == 0 and need.value == 0
    assert M.lib().mk_lora_rows_workspace(C.byref(lora(rank=3)), C.byref(need)) == 1


def rope(**kw):
    g = M.RopeRowsArgs()
    g.q = g.k = P
    g.q_out, g.k_out, g.pos = 2 * P, 4 * P, 8 * P
    g.ldq = g.ldqo = 512
    g.ldk = g.ldko = 256
    g.rows, g.heads, g.kv_heads, g.d = 4, 4, 2, 128
    g.dtype = g.out_dtype = M.BF16
    g.pos_ld, g.pos_dtype, g.axes = 2, M.I32, 2
    g.axis_dims = (C.c_uint32 * 4)(*kw.pop("dims", (32, 96)))
    g.theta, g.rope_mode = 10000.0, 1
    for k, v in kw.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize("kw, match", [
    (dict(q=None), "null"), (dict(pos=None), "null"), (dict(k=None), "together"), (dict(kv_heads=0), "together"), (dict(heads=0), "heads"), (dict(d=96), "heads"),
    (dict(dtype=M.I8), "dtype"), (dict(out_dtype=M.I32), "dtype"), (dict(pos_dtype=M.BF16), "positions"), (dict(axes=0), "axes"), (dict(axes=5), "axes"),
    (dict(dims=(31, 97)), "multiples of 2"), (dict(dims=(0, 64)), "multiples of 2"), (dict(dims=(32, 98)), "sum"), (dict(dims=(32, 104)), "sum"),
    (dict(dims=(0xFFFFFFFE, 10)), "sum"), (dict(theta=0.5), "theta"), (dict(theta=float("nan")), "theta"), (dict(theta=float("inf")), "theta"),
    (dict(series=2), "series"), (dict(rope_mode=0), "rope_mode"), (dict(rope_mode=3), "rope_mode"), (dict(ldq=508), "rows must"), (dict(ldk=258), "rows must"),
    (dict(pos_ld=1), "pos_ld"), (dict(pos_ld=-2), "pos_ld"), (dict(q=P + 4), "aligned"), (dict(dtype=M.F32, q=P + 8), "aligned"), (dict(norm_q=P + 2), "aligned"),
    (dict(q_out=P, dtype=M.F32), "in place"), (dict(q_out=P, ldqo=520), "in place"), (dict(rows=1 << 31), "rows")])
def test_rope_rows_refusals(kw, match):
    refused("mk_rope_rows", rope(**kw), None, match=match)


def test_rope_rows_nothing_to_do():
    assert M.lib().mk_rope_rows(C.byref(rope(rows=0)), None) == 0
    assert M.lib().mk_rope_rows(None, None) == 1
