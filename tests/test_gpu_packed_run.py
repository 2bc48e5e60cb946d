"""The packed batch's operators together, as a block uses them between mk_gemm's projections, captured and on two streams;
random batches; rows further apart than 32 bits reach. Tolerances as in test_gpu_packed_ops.py."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_packed_ops import Attn, H, Lora, Rope, attend, packed, stored, u, values

pytestmark = pytest.mark.gpu


class Block:
    """qkv = x W^T + adapters; rotary positions in place; attention of the documents; out = attention O^T + adapters."""

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.lens, self.s = [130, 33, 1, 200], [17, 33, 0, 40]
        self.docs, _, _ = packed(self.lens, mask="text", s=self.s)
        rows, D, self.heads, self.kv, d = sum(self.lens), 512, 4, 2, 128
        self.rows, self.D, self.d = rows, D, d
        self.N = (self.heads + 2 * self.kv) * d
        bf = lambda *s, std=1.0: stored(rng.standard_normal(s) * std, M.BF16)  # noqa: E731
        self.x, self.w, self.o = bf(rows, D), bf(self.N, D, std=D ** -0.5), bf(D, self.heads * d, std=(self.heads * d) ** -0.5)
        self.a1, self.b1 = bf(3, 16, D, std=D ** -0.5), bf(3, self.N, 16, std=0.25)
        self.a2, self.b2 = bf(3, 24, self.heads * d, std=(self.heads * d) ** -0.5), bf(3, D, 24, std=0.2)
        self.ids = np.repeat([0, -1, 2, 1], self.lens).astype(np.int32)
        self.scale = np.float32([0.5, 1.0, 2.0])
        self.pos = rng.integers(0, 64, (rows, 3)).astype(np.int32)
        self.nq, self.nk = (1 + 0.1 * rng.standard_normal((2, d))).astype(np.float32)
        self.dev = {n: M.Dev.from_array(v) for n, v in dict(
            x=self.x[0], w=self.w[0], o=self.o[0], a1=self.a1[0], b1=self.b1[0], a2=self.a2[0], b2=self.b2[0], ids=self.ids, scale=self.scale,
            pos=self.pos, nq=self.nq, nk=self.nk).items()}
        self.qkv, self.att, self.out = M.Dev(rows * self.N * 2), M.Dev(rows * self.heads * d * 2), M.Dev(rows * D * 4)
        self.calls()

    def gemm(self, a, w, c, M_, N, K, c_dtype):
        g = M.GemmArgs()
        g.a, g.w, g.c, g.M, g.N, g.K, g.lda, g.ldc, g.batch = a.p, w.p, c.p, M_, N, K, K, N, 1
        g.w_dtype, g.c_dtype, g.epilogue = M.BF16, c_dtype, M.EPI_STORE
        return "mk_gemm", g

    def space(self, g, name):
        need = C.c_uint64()
        M.call(name, C.byref(g), C.byref(need))
        keep = M.Dev(need.value)
        g.workspace, g.workspace_bytes = keep.p, need.value
        return keep

    def lora(self, x, a, b, c, K, N, rank, c_dtype):
        g = M.LoraRowsArgs()
        g.x, g.a, g.b, g.scale, g.ids, g.base, g.c = x.p, a.p, b.p, self.dev["scale"].p, self.dev["ids"].p, c.p, c.p
        g.ldx, g.ldbase, g.ldc = K, N, N
        g.rows, g.K, g.N, g.rank, g.parts, g.adapters, g.dtype, g.c_dtype = self.rows, K, N, rank, 1, 3, M.BF16, c_dtype
        return ("mk_lora_rows", g), self.space(g, "mk_lora_rows_workspace")

    def calls(self):
        v, hd, kd = self.dev, self.heads * self.d, self.kv * self.d
        r = M.RopeRowsArgs()
        r.q = r.q_out = self.qkv.p
        r.k = r.k_out = self.qkv.p + hd * 2
        r.ldq = r.ldk = r.ldqo = r.ldko = self.N
        r.rows, r.heads, r.kv_heads, r.d, r.dtype, r.out_dtype = self.rows, self.heads, self.kv, self.d, M.BF16, M.BF16
        r.norm_q, r.norm_k, r.eps = v["nq"].p, v["nk"].p, 1e-6
        r.pos, r.pos_ld, r.pos_dtype, r.axes, r.axis_dims = v["pos"].p, 3, M.I32, 3, (C.c_uint32 * 4)(16, 56, 56)
        r.theta, r.series, r.rope_mode = 10000.0, M.ROPE_OWN, 2
        t = M.AttnPackedArgs()
        t.q, t.k, t.v, t.out = self.qkv.p, self.qkv.p + hd * 2, self.qkv.p + (hd + kd) * 2, self.att.p
        t.ldq = t.ldk = t.ldv = self.N
        t.ldo, t.dtype, t.out_dtype, t.heads, t.kv_heads, t.d, t.scale = hd, M.BF16, M.BF16, self.heads, self.kv, self.d, self.d ** -0.5
        self.table = (M.AttnDoc * len(self.docs))(*[M.AttnDoc(*w) for w in self.docs])
        t.docs, t.n_docs = self.table, len(self.docs)
        l1, s1 = self.lora(v["x"], v["a1"], v["b1"], self.qkv, self.D, self.N, 16, M.BF16)
        l2, s2 = self.lora(self.att, v["a2"], v["b2"], self.out, hd, self.D, 24, M.F32)
        self.keep = [s1, s2, self.space(t, "mk_attention_packed_workspace")]
        self.run_calls = [self.gemm(v["x"], v["w"], self.qkv, self.rows, self.N, self.D, M.BF16), l1, ("mk_rope_rows", r), ("mk_attention_packed", t),
                          self.gemm(self.att, v["o"], self.out, self.rows, self.D, hd, M.F32), l2]

    def run(self, stream=None, upto=None):
        for name, g in self.run_calls[:upto]:
            M.call(name, C.byref(g), stream)

    def read(self, dev, width, dt=M.BF16):
        M.sync()
        return values(dev.to_array(np.float32 if dt == M.F32 else np.uint16, (self.rows, width)), dt)


def adapters(x, a, b, ids, scale, base, c_dt, K, rank):
    want, tol = base.copy(), np.zeros_like(base)
    for i in range(len(scale)):
        r = ids == i
        t, ta = x[r] @ a[i].T, np.abs(x[r]) @ np.abs(a[i]).T
        want[r] += scale[i] * (t @ b[i].T)
        tol[r] = scale[i] * (((K / 8 + 16) * u * ta + (H[M.BF16] ** 2 + (rank + 8) * u) * np.abs(t)) @ np.abs(b[i]).T)
    return want, tol + (H[c_dt] + 2 * u) * np.abs(want) + 2 * u * np.abs(base)


def test_a_packed_block(gpu):
    b = Block(5)
    hd, kd, d = b.heads * b.d, b.kv * b.d, b.d
    b.run(upto=1)
    base = b.read(b.qkv, b.N)
    b.run(upto=2)
    qkv = b.read(b.qkv, b.N)
    want, tol = adapters(b.x[1], b.a1[1], b.b1[1], b.ids, b.scale, base, M.BF16, b.D, 16)
    assert (np.abs(qkv - want) <= tol).all()
    b.run(upto=3)
    turned = b.read(b.qkv, b.N)
    assert np.array_equal(turned[:, hd + kd:], qkv[:, hd + kd:])  # the values stay
    ref = Rope.__new__(Rope)
    ref.rows, ref.dims, ref.theta, ref.series, ref.mode, ref.k_scale, ref.out_dt, ref.pos_dt, ref.pos = b.rows, [16, 56, 56], 10000.0, 0, 2, 0.0, M.BF16, M.I32, b.pos
    ref.w = {"q": b.nq, "k": b.nk}
    ref.val = {"q": qkv[:, :hd].reshape(b.rows, b.heads, d), "k": qkv[:, hd:hd + kd].reshape(b.rows, b.kv, d)}
    for n, cols in (("q", slice(0, hd)), ("k", slice(hd, hd + kd))):
        want, tol = ref.want(n)
        assert (np.abs(turned[:, cols] - want.reshape(b.rows, -1)) <= tol.reshape(b.rows, -1)).all()
    b.run(upto=4)
    q, k, v = (turned[:, c].reshape(b.rows, -1, d) for c in (slice(0, hd), slice(hd, hd + kd), slice(hd + kd, b.N)))
    want, tol = attend(q, k, v, b.docs, d ** -0.5, 0.0, None, M.BF16, M.BF16)
    att = b.read(b.att, hd)
    assert (np.abs(att - want.reshape(b.rows, -1)) <= tol.reshape(b.rows, -1)).all()
    b.run(upto=5)
    base = b.read(b.out, b.D, M.F32)
    b.run()
    want, tol = adapters(att, b.a2[1], b.b2[1], b.ids, b.scale, base, M.F32, hd, 24)
    assert (np.abs(b.read(b.out, b.D, M.F32) - want) <= tol).all()


def hip():
    h = C.CDLL("libamdhip64.so")
    for f in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphExecDestroy", "hipGraphDestroy"):
        getattr(h, f).restype = C.c_int
    return h


def test_captured_and_on_two_streams(gpu):
    blocks = [Block(1), Block(2)]
    solo = []
    for b in blocks:
        b.run()
        solo.append(b.read(b.out, b.D, M.F32))
    h = hip()
    streams, execs = [], []
    for b in blocks:
        s = C.c_void_p()
        M.call("mk_stream_create", C.byref(s))
        streams.append(s)
        # (mk_gemm runs whole tiles under capture, with its own rounding: the operators behind the projections are captured)
        b.run()
        M.sync()
        graph, run = C.c_void_p(), C.c_void_p()
        assert h.hipStreamBeginCapture(s, 0) == 0
        for name, g in b.run_calls[1:4]:
            M.call(name, C.byref(g), s)
        assert h.hipStreamEndCapture(s, C.byref(graph)) == 0
        assert h.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
        execs.append((graph, run))
    for rep in range(4):
        for b in blocks:
            M.call("mk_memset", b.att.p, 0, b.att.nbytes)
            M.call("mk_memset", b.keep[2].p, 0x7F, max(b.keep[2].nbytes, 16))
        for (graph, run), b, s in zip(execs, blocks, streams):
            for name, g in b.run_calls[:1]:
                M.call(name, C.byref(g), s)
            assert h.hipGraphLaunch(run, s) == 0
            for name, g in b.run_calls[4:]:
                M.call(name, C.byref(g), s)
        if rep % 2:
            # eager work of the program's own between two replays
            Attn([(0, 70, 0, 70, 0, 0xFFFFFFFF, 0)], 70, 70, 2, 2, 64, M.BF16).run()
        for b, s, want in zip(blocks, streams, solo):
            M.call("mk_stream_synchronize", s)
            assert np.array_equal(b.read(b.out, b.D, M.F32), want), rep
    for (graph, run), s in zip(execs, streams):
        assert h.hipGraphExecDestroy(run) == 0 and h.hipGraphDestroy(graph) == 0
        M.call("mk_stream_destroy", s)


@pytest.mark.parametrize("seed", range(40))
def test_random_batches(gpu, seed):
    rng = np.random.default_rng(1000 + seed)
    docs = int(rng.integers(1, 7))
    kv = int(rng.choice([1, 2, 3]))
    heads, d = kv * int(rng.choice([1, 2, 4, 7])), int(rng.choice([64, 128]))
    k = [int(v) for v in rng.integers(0, int(rng.choice([5, 70, 300])), docs)]
    q = [int(v) for v in rng.integers(0, int(rng.choice([3, 40, 90])), docs)]
    mask = str(rng.choice(["full", "causal", "text", "prefix"]))
    table, nq, nk = packed(q, k, mask=mask, s=[int(rng.integers(0, n + 1)) for n in k], gap=int(rng.integers(0, 3)))
    dt = int(rng.choice([M.BF16, M.F16]))
    order = rng.permutation(docs)
    slopes = np.float32(rng.uniform(0, 0.5, heads)) if rng.random() < 0.4 else None
    a = Attn([table[i] for i in order], nq, nk, heads, kv, d, dt, out_dt=int(rng.choice([M.BF16, M.F16])), cap=float(rng.choice([0.0, 0.0, 8.0])),
             slopes=slopes, seed=seed, pad=8 * int(rng.integers(0, 3)), gain=float(rng.choice([0.2, 1.0, 5.0])))
    a.check(bool(rng.random() < 0.7))


@pytest.mark.parametrize("heads, kv, d", [(4, 1, 128), (6, 6, 64)])
def test_attention_long_cache(gpu, heads, kv, d):
    docs, nq, nk = packed([1, 2], [70001, 20000], mask="causal")
    Attn(docs, nq, nk, heads, kv, d, M.BF16).check()
    Attn(docs, nq, nk, heads, kv, d, M.F16, slopes=np.float32(2.0 ** -np.arange(1, heads + 1) / 256)).check()


def far_rows(rows, ld, bits, col, dev):
    for r in range(rows):
        dev.write(bits[r], (r * ld + col) * bits.dtype.itemsize)


def test_attention_rows_past_32_bits(gpu):
    # rows of 2^23 elements: 530 of them are 8.9 GB, the last one's first element is past 2^32
    ld, nq, nk, d = 1 << 23, 70, 530, 64
    rng = np.random.default_rng(0)
    (qb, q), (kb, k), (vb, v) = (stored(rng.standard_normal((n, d)), M.BF16) for n in (nq, nk, nk))
    big = M.Dev(((nk - 1) * ld + 4 * d) * 2)
    far_rows(nk, ld, kb, 0, big)
    far_rows(nk, ld, vb, d, big)
    g = M.AttnPackedArgs()
    shift = (nk - nq) * ld * 2
    far_rows(nq, ld, qb, (nk - nq) * ld + 2 * d, big)
    g.q, g.k, g.v, g.out = big.p + 2 * d * 2 + shift, big.p, big.p + d * 2, big.p + 3 * d * 2 + shift
    g.ldq = g.ldk = g.ldv = g.ldo = ld
    g.dtype = g.out_dtype = M.BF16
    g.heads, g.kv_heads, g.d, g.scale = 1, 1, d, 0.125
    doc = (0, nq, 0, nk, nk - nq, 0xFFFFFFFF, 0)
    table = (M.AttnDoc * 1)(M.AttnDoc(*doc))
    g.docs, g.n_docs = table, 1
    M.call("mk_attention_packed", C.byref(g), None)
    M.sync()
    got = np.stack([np.empty(d, np.uint16) for _ in range(nq)])
    for r in range(nq):
        M.call("mk_memcpy_d2h", got[r].ctypes.data, g.out + r * ld * 2, d * 2)
    want, tol = attend(q[:, None], k[:, None], v[:, None], [doc], 0.125, 0.0, None, M.BF16, M.BF16)
    assert (np.abs(values(got, M.BF16) - want[:, 0]) <= tol[:, 0]).all()


@pytest.mark.parametrize("rows", [300, 700])
def test_lora_and_rope_rows_past_32_bits(gpu, rows):
    # rows of 8388600 elements: x, base and c (bf16), and heads to be turned, all in one buffer
    ld, K, N, rank = (1 << 23) - 8, 64, 64, 8
    rng = np.random.default_rng(rows)
    xb, x = stored(rng.standard_normal((rows, K)), M.BF16)
    cb, c = stored(rng.standard_normal((rows, N)), M.BF16)
    big = M.Dev(((rows - 1) * ld + 256) * 2)
    far_rows(rows, ld, xb, 0, big)
    far_rows(rows, ld, cb, 64, big)
    far_rows(rows, ld, xb, 128, big)
    ab, a = stored(rng.standard_normal((2, rank, K)) * 0.2, M.BF16)
    bb, b = stored(rng.standard_normal((2, N, rank)), M.BF16)
    ids = (np.arange(rows) % 2).astype(np.int32)
    keep = [M.Dev.from_array(v) for v in (ab, bb, ids, np.full((rows, 1), 3, np.int32))]
    g = M.LoraRowsArgs()
    g.x, g.a, g.b, g.ids, g.base, g.c = big.p, keep[0].p, keep[1].p, keep[2].p, big.p + 128, big.p + 128
    g.ldx = g.ldbase = g.ldc = ld
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters, g.dtype, g.c_dtype = rows, K, N, rank, 1, 2, M.BF16, M.BF16
    need = C.c_uint64()
    M.call("mk_lora_rows_workspace", C.byref(g), C.byref(need))
    space = M.Dev(need.value)
    g.workspace, g.workspace_bytes = space.p, need.value
    M.call("mk_lora_rows", C.byref(g), None)
    r = M.RopeRowsArgs()
    r.q = r.q_out = big.p + 256
    r.ldq = r.ldqo = ld
    r.rows, r.heads, r.d, r.dtype, r.out_dtype = rows, 1, 64, M.BF16, M.BF16
    r.pos, r.pos_ld, r.pos_dtype, r.axes, r.axis_dims = keep[3].p, 1, M.I32, 1, (C.c_uint32 * 4)(64)
    r.theta, r.rope_mode = 100.0, 1
    M.call("mk_rope_rows", C.byref(r), None)
    M.sync()
    got, turned = np.empty((rows, N), np.uint16), np.empty((rows, 64), np.uint16)
    for i in range(rows):
        M.call("mk_memcpy_d2h", got[i].ctypes.data, big.p + (i * ld + 64) * 2, N * 2)
        M.call("mk_memcpy_d2h", turned[i].ctypes.data, big.p + (i * ld + 128) * 2, 128)
    want, tol = adapters(x, a, b, ids, np.float32([1, 1]), c, M.BF16, K, rank)
    assert (np.abs(values(got, M.BF16) - want) <= tol).all()
    f = 100.0 ** (-2.0 * np.arange(32) / 64) * 3
    y = np.concatenate([x[:, :32] * np.cos(f) - x[:, 32:] * np.sin(f), x[:, :32] * np.sin(f) + x[:, 32:] * np.cos(f)], 1)
    both = np.abs(x[:, :32]) + np.abs(x[:, 32:])
    assert (np.abs(values(turned, M.BF16) - y) <= 24 * u * np.concatenate([both, both], 1) + H[M.BF16] * np.abs(y)).all()


def test_the_binding_refuses_short_buffers(gpu):
    a = Attn([(0, 8, 0, 8, 0, 0, 0)], 8, 8, 2, 2, 64, M.BF16)
    for docs in ([(0, 9, 0, 8, 0, 0, 0)], [(0, 8, 1, 8, 0, 0, 0)]):
        a.docs = docs
        with pytest.raises(M.MkError, match="its allocation holds"):
            a.run(workspace=False)
    lo = Lora(4, 64, 64, 8, 1, 2, [0, 1, 0, 1], M.BF16, M.F32)
    g = lo.args()
    g.adapters = 3
    with pytest.raises(M.MkError, match="its allocation holds"):
        M.call("mk_lora_rows", C.byref(g), None)
    r = Rope(4, 2, 1, 64, [64], M.BF16, M.F32)
    g = r.args()
    g.rows = 5
    with pytest.raises(M.MkError, match="its allocation holds"):
        M.call("mk_rope_rows", C.byref(g), None)
