"""The int8 path of a transformer block, operator by operator and as a run: what is timed, and its plain form.

Kinds (case["kind"]):
- "norm":    mk_gate_norm: a block's output (optionally normed) times its gate added to the scaled fp32 residual, and the
             next block's modulated norm of the sum, in one pass. `mode` says which model's: "mmdit" (gate, layer norm,
             scale and shift, a modulation row for each sample), "q21" (tanh gate, layer norm, scale only, the text rows
             modulated apart) or "sandwich" (RMS norms with weights before and after the block, a residual scale);
- "product": mk_gemm_i8 over int8 rows that the previous operator left;
- "linear":  mk_quantize_i8_rows and mk_gemm_i8: a linear layer on 16- or 32-bit activations;
- "ffn":     the run of them: mk_gate_norm to int8 rows, the gated up-projection, mk_quantize_i8_rows of the hidden rows
             and the down-projection, whose output the next block's mk_gate_norm would take.

Widths are the 2.1 graph's (4096, FFN 12288), SDXL's (1280, GEGLU 2 x 5120, context 2048) and generic ones; rows are token
grids of 512 x 512 to 2048 x 2048 images with their prompts, a context's 77 rows, and single rows.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
ALPHA = 0.875        # the sandwich mode's residual scale
TINY = 2.0 ** -100   # rows below it count as zero


def listed():
    return [
        # one token's residual between two sandwich-normed blocks: latency
        dict(name="norm_1_row", kind="norm", mode="sandwich", segs=1, rows=1, n=4096, split=0, y="bf16", out="bf16"),
        # SDXL-wide rows of a portrait image, half activations
        dict(name="norm_1333x1280_f16", kind="norm", mode="sandwich", segs=1, rows=1333, n=1280, split=0, y="f16", out="f16"),
        # the 2.1 graph at 1024 x 1024: 256 text rows modulated at t = 0, 4096 image rows
        dict(name="norm_1024px_q21", kind="norm", mode="q21", segs=1, rows=4352, n=4096, split=256, y="bf16", out="bf16"),
        # a guided batch of 2 at 2048 x 2048, each sample with a modulation row of its own
        dict(name="norm_2048px_batch2", kind="norm", mode="mmdit", segs=2, rows=16384, n=4096, split=0, y="bf16", out="bf16"),
        # one row through the widest projection: all of the weights for one token
        dict(name="product_1_row", kind="product", m=1, n=12288, k=4096, epi="store", c="bf16"),
        # the keys and values of a 77-row context
        dict(name="product_77_context", kind="product", m=77, n=2560, k=2048, epi="store", c="f16"),
        # SDXL's GEGLU projection for both samples of a portrait image: rows that no tile divides
        dict(name="product_geglu_portrait", kind="product", m=3952, n=10240, k=1280, epi="geglu", c="bf16"),
        # the up-projection at 1024 x 1024
        dict(name="product_1024px_gelu", kind="product", m=4352, n=12288, k=4096, epi="gelu", c="bf16"),
        # a handful of prompt tokens
        dict(name="linear_23_rows", kind="linear", m=23, n=4096, k=4096, epi="store", c="bf16", x="bf16"),
        # the down-projection at 1024 x 1024, into fp32
        dict(name="linear_1024px_down", kind="linear", m=4352, n=4096, k=12288, epi="store", c="f32", x="bf16"),
        # the largest: both samples' up-projection at 2048 x 2048
        dict(name="linear_2048px_up", kind="linear", m=32768, n=12288, k=4096, epi="silu", c="bf16", x="bf16"),
        # the 2.1 graph's FFN at 1024 x 1024, norm to down-projection
        dict(name="ffn_1024px", kind="ffn", mode="q21", segs=1, rows=4352, n=4096, f=12288, split=256, epi="swiglu"),
    ]


MOST_ELEMENTS, MOST_MACS = 32768 * 4096, 32768 * 12288 * 4096


def _log(rng, lo, hi, of=1):
    return max(of, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / of)) * of)


def draw(rng):
    kind = rng.choice(["norm", "norm", "product", "product", "linear", "linear", "ffn"])
    mode = rng.choice(["mmdit", "q21", "sandwich"])
    if kind == "norm":
        n = _log(rng, 64, 12288, 4)
        segs = rng.choice([1, 1, 2, 3])
        rows = min(_log(rng, 1, 32768), MOST_ELEMENTS // (n * segs))
        return dict(kind=kind, mode=mode, segs=segs, rows=rows, n=n, split=rng.randint(0, rows),
                    y=rng.choice(["bf16", "f16", "f32"]), out=rng.choice(["bf16", "f16"]))
    if kind == "ffn":
        n, f = _log(rng, 128, 5120, 16), _log(rng, 256, 12288, 16)
        rows = min(_log(rng, 1, 8192), MOST_MACS // (4 * n * f))
        return dict(kind=kind, mode=mode, segs=1, rows=rows, n=n, f=f, split=rng.randint(0, rows),
                    epi=rng.choice(["swiglu", "geglu"]))
    epi = rng.choice(["store", "store", "gelu", "silu", "swiglu", "geglu"])
    n, k = _log(rng, 64, 12288, 8), _log(rng, 64, 12288, 16)
    m = min(_log(rng, 1, 32768), MOST_MACS // (n * k))
    case = dict(kind=kind, m=m, n=n, k=k, epi=epi, c=rng.choice(["bf16", "f16", "f32"] if epi == "store" else ["bf16", "f16"]))
    if kind == "linear":
        case["x"] = rng.choice(["bf16", "f16", "f32"])
    return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------------------------------------

class Rng:
    """Normal draws on the device: call number i of a seed is the same tensor everywhere."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std).add_(mean)


def _channels(rng, n):
    """Channel magnitudes of a transformer's activations: log-normal, so that a few channels are many times the rest."""
    return torch.exp(rng.normal(n, std=0.7))


def _codes(x):
    """int8 rows of x and their scales, as stored weights and rows have them (input data, not a timed step)."""
    s = x.abs().amax(1).clamp_(min=TINY) / 127.0
    return torch.round(x / s[:, None]).to(torch.int8), s


def _weight(rng, n, k):
    return _codes(rng.normal(n, k, std=0.02))


def _norm_inputs(case, rng):
    """x, y and the norm's vectors: mod [segs][6 n] holds gate, scale, shift and the same for the rows below split."""
    rows, n = case["segs"] * case["rows"], case["n"]
    d = {"x": rng.normal(rows, n) * _channels(rng, n) * 3.0,
         "y": (rng.normal(rows, n) * _channels(rng, n)).to(DTYPES[case.get("y", "bf16")])}
    if case["mode"] == "sandwich":
        d.update(w1=rng.normal(n, std=0.1, mean=1.0), w2=rng.normal(n, std=0.1, mean=1.0))
    else:
        d.update(mod=rng.normal(case["segs"], 6 * n, std=0.3))
    return d


def inputs(case, seed):
    rng, kind = Rng(seed), case["kind"]
    if kind == "norm":
        return _norm_inputs(case, rng)
    if kind == "ffn":
        d = _norm_inputs(case, rng)
        n, f = case["n"], case["f"]
        d["up"], d["up_s"] = _weight(rng, 2 * f, n)
        d["down"], d["down_s"] = _weight(rng, n, f)
        d["up_b"], d["down_b"] = rng.normal(2 * f, std=0.02), rng.normal(n, std=0.02)
        return d
    x = rng.normal(case["m"], case["k"]) * _channels(rng, case["k"])
    d = {"x": x.to(DTYPES[case["x"]])} if kind == "linear" else dict(zip(("q", "q_s"), _codes(x)))
    d["w"], d["w_s"] = _weight(rng, case["n"], case["k"])
    d["b"] = rng.normal(case["n"], std=0.02)
    return d


# ---------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------

def _quantize(x):
    """int8 rows (as floats) and fp32 scales: s = max|x| / 127, q = 127 x / max|x| rounded to nearest, ties to even. In 64
    bits: a value half way between two codes is one, whatever the type."""
    a = x.abs().amax(1, keepdim=True).double()
    zero = a < TINY
    q = torch.round(torch.where(zero, torch.zeros((), dtype=F64, device=x.device), 127.0 * x.double() / a))
    return q.float(), torch.where(zero, torch.ones_like(a), a / 127.0).float()


def _normed(v, mode, w):
    if mode == "rms":
        return v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * w
    d = v - v.mean(1, keepdim=True)
    return d * torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)


def _mod_rows(case, mod):
    """gate, scale and shift of every row: [segs rows][n] each."""
    n, rows = case["n"], case["rows"]
    first = torch.arange(rows, device=mod.device) < case["split"]
    m = mod.view(case["segs"], 2, 3, n)
    m = torch.where(first[None, :, None, None], m[:, 1, None], m[:, 0, None]).reshape(case["segs"] * rows, 3, n)
    return m[:, 0], m[:, 1], m[:, 2]


def _gate_norm(case, d):
    """x' and h, in 32 bits."""
    y = d["y"].float()
    if case["mode"] == "sandwich":
        x = ALPHA * d["x"] + _normed(y, "rms", d["w1"])
        return x, _normed(x, "rms", d["w2"])
    gate, scale, shift = _mod_rows(case, d["mod"])
    if case["mode"] == "q21":
        x = d["x"] + torch.tanh(gate) * y
        return x, _normed(x, "layer", None) * (1.0 + scale)
    x = d["x"] + gate * y
    return x, _normed(x, "layer", None) * (1.0 + scale) + shift


def _epilogue(v, epi):
    """GELU in its tanh form, SiLU, and the gated units: silu(a) b, and a times the erf GELU of b."""
    if epi == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if epi == "silu":
        return v / (1.0 + torch.exp(-v))
    if epi in ("swiglu", "geglu"):
        a, b = v.chunk(2, 1)
        return a / (1.0 + torch.exp(-a)) * b if epi == "swiglu" else a * (0.5 * b * (1.0 + torch.erf(b * math.sqrt(0.5))))
    return v


def _product(q, q_s, w, w_s, bias, epi):
    return _epilogue(torch.mm(q, w.float().t()) * q_s * w_s + bias, epi)


def _plain(case, d):
    kind = case["kind"]
    if kind == "norm":
        x, h = _gate_norm(case, d)
        return {"x": x, "h": h.to(DTYPES[case["out"]])}
    if kind == "ffn":
        x, h = _gate_norm(case, d)
        u = _product(*_quantize(h), d["up"], d["up_s"], d["up_b"], case["epi"]).bfloat16()
        return {"x": x, "y": _product(*_quantize(u), d["down"], d["down_s"], d["down_b"], "store").bfloat16()}
    q, s = _quantize(d["x"]) if kind == "linear" else (d["q"].float(), d["q_s"][:, None])
    return {"c": _product(q, s, d["w"], d["w_s"], d["b"], case["epi"]).to(DTYPES[case["c"]])}


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------

def _binding():
    path = os.path.join(os.getcwd(), "mako-image_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mkimage
    return mkimage


def _empty(dt, *shape):
    return torch.empty(*shape, dtype=DTYPES.get(dt, torch.int8), device="cuda")


def _norm_call(M, case, d, out, out_scale):
    rows, n = case["segs"] * case["rows"], case["n"]
    codes = {torch.float32: M.F32, torch.bfloat16: M.BF16, torch.float16: M.F16, torch.int8: M.I8}
    g = M.GateNormArgs()
    x = torch.empty_like(d["x"])
    g.x, g.x_out, g.y, g.out = d["x"].data_ptr(), x.data_ptr(), d["y"].data_ptr(), out.data_ptr()
    g.out_scale = out_scale.data_ptr() if out_scale is not None else None
    g.rows, g.n, g.ldx, g.ldy, g.ldo = rows, n, n, n, n
    g.y_dtype, g.out_dtype = codes[d["y"].dtype], codes[out.dtype]
    g.eps1 = g.eps2 = EPS
    if case["mode"] == "sandwich":
        g.norm1, g.w1, g.norm2, g.w2, g.residual_scale = M.NORM_RMS, d["w1"].data_ptr(), M.NORM_RMS, d["w2"].data_ptr(), ALPHA
    else:
        mod = d["mod"].data_ptr()
        g.norm2, g.gate, g.scale, g.tanh_gate = M.NORM_LAYER, mod, mod + 4 * n, int(case["mode"] == "q21")
        g.shift = mod + 8 * n if case["mode"] == "mmdit" else None
        g.alt, g.split, g.seg_rows, g.mod_stride = 3 * n, case["split"], case["rows"], 6 * n
    return x, ("mk_gate_norm", C.byref(g))


def _gemm_call(M, q, q_s, w, w_s, bias, out, epi):
    g = M.GemmArgs()
    g.a, g.w, g.wscale, g.bias, g.c = q.data_ptr(), w.data_ptr(), w_s.data_ptr(), bias.data_ptr(), out.data_ptr()
    g.M, g.N, g.K, g.lda, g.ldc, g.batch = q.shape[0], w.shape[0], w.shape[1], w.shape[1], out.shape[1], 1
    g.w_dtype, g.c_dtype = M.I8, {torch.float32: M.F32, torch.bfloat16: M.BF16, torch.float16: M.F16}[out.dtype]
    g.epilogue = {"store": M.EPI_STORE, "gelu": M.EPI_GELU_TANH, "silu": M.EPI_SILU, "swiglu": M.EPI_SWIGLU,
                  "geglu": M.EPI_GEGLU}[epi]
    return "mk_gemm_i8", C.byref(g), q_s.data_ptr()


def _quantize_call(M, x, q, q_s):
    dt = {torch.float32: M.F32, torch.bfloat16: M.BF16, torch.float16: M.F16}[x.dtype]
    return "mk_quantize_i8_rows", x.data_ptr(), dt, x.shape[0], x.shape[1], x.shape[1], q.data_ptr(), q_s.data_ptr()


def _calls(M, case, d):
    """The calls of a pass (all but the stream), what they return, and the buffers that they use."""
    kind = case["kind"]
    if kind == "norm":
        h = _empty(case["out"], case["segs"] * case["rows"], case["n"])
        x, call = _norm_call(M, case, d, h, None)
        return [call], {"x": x, "h": h}, ()
    if kind == "ffn":
        rows, n, f = case["rows"], case["n"], case["f"]
        h, hs, u = _empty("i8", rows, n), _empty("f32", rows), _empty("bf16", rows, f)
        uq, us, y = _empty("i8", rows, f), _empty("f32", rows), _empty("bf16", rows, n)
        x, call = _norm_call(M, case, d, h, hs)
        return [call, _gemm_call(M, h, hs, d["up"], d["up_s"], d["up_b"], u, case["epi"]), _quantize_call(M, u, uq, us),
                _gemm_call(M, uq, us, d["down"], d["down_s"], d["down_b"], y, "store")], {"x": x, "y": y}, (h, hs, u, uq, us)
    m, n, k = case["m"], case["n"], case["k"]
    c = _empty(case["c"], m, n // 2 if case["epi"] in ("swiglu", "geglu") else n)
    if kind == "product":
        return [_gemm_call(M, d["q"], d["q_s"], d["w"], d["w_s"], d["b"], c, case["epi"])], {"c": c}, ()
    q, qs = _empty("i8", m, k), _empty("f32", m)
    return [_quantize_call(M, d["x"], q, qs), _gemm_call(M, q, qs, d["w"], d["w_s"], d["b"], c, case["epi"])], {"c": c}, (q, qs)


def prepare(case, seed):
    s = {"case": case, "data": inputs(case, seed)}
    if own:
        # argument blocks and buffers, as a program sets them up once for its layers
        s["M"] = _binding()
        s["calls"], s["out"], s["keep"] = _calls(s["M"], case, s["data"])
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        stream = torch.cuda.current_stream().cuda_stream or None
        call = s["M"].call
        for c in s["calls"]:
            call(*c, stream)
        return s["out"]
    return _plain(s["case"], s["data"])


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _norm_work(case, out_bytes):
    rows, n = case["segs"] * case["rows"], case["n"]
    vectors = 2 * n if case["mode"] == "sandwich" else case["segs"] * (2 if case["split"] else 1) * n * (
        3 if case["mode"] == "mmdit" else 2)
    return rows * n * (8 + SIZE[case.get("y", "bf16")] + out_bytes) + 4 * vectors, 16 * rows * n


def work(case):
    kind = case["kind"]
    if kind == "norm":
        b, f = _norm_work(case, SIZE[case["out"]])
    elif kind == "ffn":
        rows, n, ff = case["rows"], case["n"], case["f"]
        b, f = _norm_work(case, 0)
        b += 3 * n * ff + 4 * (4 * ff + 2 * n) + 2 * rows * n
        f += 6 * rows * n * ff
    else:
        m, n, k = case["m"], case["n"], case["k"]
        cols = n // 2 if case["epi"] in ("swiglu", "geglu") else n
        b = m * (k * SIZE[case["x"]] if kind == "linear" else k + 4) + n * (k + 8) + m * cols * SIZE[case["c"]]
        f = 2 * m * n * k
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    d = inputs(case, seed)
    kind = case["kind"]

    def rounded_codes(v):
        top = v.abs().max(1).values[:, None]
        unit = torch.where(top < TINY, torch.full_like(top, math.inf), top / 127.0)
        codes = torch.where(torch.isinf(unit), torch.zeros_like(v), v * 127.0 / torch.where(top < TINY, torch.ones_like(top), top))
        return torch.round(codes), torch.where(torch.isinf(unit), torch.ones_like(unit), unit)

    def linear(codes, unit, w, w_s, bias):
        return (codes @ w.to(F64).T) * unit * w_s.to(F64)[None, :] + bias.to(F64)[None, :]

    def act(v, epi):
        half = v.shape[1] // 2
        if epi == "gelu":
            return 0.5 * v * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3)))
        if epi == "silu":
            return v * torch.sigmoid(v)
        if epi == "swiglu":
            return v[:, :half] * torch.sigmoid(v[:, :half]) * v[:, half:]
        if epi == "geglu":
            return v[:, :half] * v[:, half:] * 0.5 * torch.erfc(-v[:, half:] / 2.0 ** 0.5)
        return v

    def by_row():
        """x' and h, segment by segment and its two spans of rows."""
        xs, hs = [], []
        for b in range(case["segs"]):
            for lo, hi, alt in ((0, case["split"], 1), (case["split"], case["rows"], 0)):
                if lo == hi:
                    continue
                at = slice(b * case["rows"] + lo, b * case["rows"] + hi)
                x, y = d["x"][at].to(F64), d["y"][at].to(F64)
                if case["mode"] == "sandwich":
                    x = ALPHA * x + y / (y.pow(2).mean(1, True) + EPS).sqrt() * d["w1"].to(F64)
                    h = x / (x.pow(2).mean(1, True) + EPS).sqrt() * d["w2"].to(F64)
                else:
                    gate, scale, shift = d["mod"][b].to(F64).reshape(2, 3, -1)[alt]
                    x = x + (gate.tanh() if case["mode"] == "q21" else gate) * y
                    h = (x - x.mean(1, True)) / (x.var(1, unbiased=False, keepdim=True) + EPS).sqrt() * (1.0 + scale)
                    h = h + shift if case["mode"] == "mmdit" else h
                xs.append(x)
                hs.append(h)
        return torch.cat(xs), torch.cat(hs)

    if kind == "norm":
        x, h = by_row()
        return {"x": x, "h": h}
    if kind == "ffn":
        x, h = by_row()
        u = act(linear(*rounded_codes(h), d["up"], d["up_s"], d["up_b"]), case["epi"])
        u = u.to(torch.bfloat16).to(F64)  # the hidden rows are stored in bf16
        return {"x": x, "y": linear(*rounded_codes(u), d["down"], d["down_s"], d["down_b"])}
    codes, unit = rounded_codes(d["x"].to(F64)) if kind == "linear" else (d["q"].to(F64), d["q_s"].to(F64)[:, None])
    return {"c": act(linear(codes, unit, d["w"], d["w_s"], d["b"]), case["epi"])}
