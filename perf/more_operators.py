"""A packed batch of requests, operator by operator: what is timed, and its plain form.

Rows of several requests (images of different sizes, prompts of different lengths, each with a LoRA of its own or none) lie one
after the other and go through shared projections. Kinds (case["kind"]):
- "attn": mk_attention_packed: softmax attention of each document's query rows over its own keys, masks "full", "causal",
          "text" (the first `s` positions causal, the rest see every key) or "prefix" (causal, the first `s` keys seen by
          every row), scores optionally capped by a tanh or lowered by a slope times the distance;
- "lora": mk_lora_rows: base + scale (x A^T) B^T with the adapter of each row, one A for each of `parts` column blocks;
- "rope": mk_rope_rows: per-head RMS norm (optional) and rotary positions of several axes on query and key rows.

Widths are the 2.1 graph's (4096, 32 x 128, FFN 12288), SDXL's (20 x 64, 1280) and generic ones; rows are token grids of 512 x
512 to 2048 x 1024 images with their prompts, prompts alone, and single rows.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # one new query row over a long cache, eight query heads a key head: latency
        dict(name="attn_1_token", kind="attn", q="1", k="16411", s="0", mask="causal", heads=32, kv=8, d=128, dt="bf16", cap=0.0, bias=False),
        # a text encoder's prompts of eight requests, packed, causal, scores capped
        dict(name="attn_8_prompts_capped", kind="attn", q="77,13,512,256,1,340,129,64", k="77,13,512,256,1,340,129,64", s="0",
             mask="causal", heads=32, kv=8, d=128, dt="bf16", cap=30.0, bias=False),
        # image rows of three sizes over their own prompts' keys, half heads of 64, a bias by distance
        dict(name="attn_cross_bias_f16", kind="attn", q="4096,1024,1333", k="77,154,231", s="0", mask="full", heads=20, kv=20, d=64,
             dt="f16", cap=0.0, bias=True),
        # joint text and image rows of four requests, 512 x 512 to 1024 x 1024, causal text
        dict(name="attn_4_images", kind="attn", q="4352,1101,2377,1801", k="4352,1101,2377,1801", s="256,77,73,201", mask="text",
             heads=32, kv=32, d=128, dt="bf16", cap=0.0, bias=False),
        # the largest: two 2048 x 1024 images
        dict(name="attn_2_large_images", kind="attn", q="8448,8301", k="8448,8301", s="256,109", mask="text", heads=32, kv=32, d=128,
             dt="bf16", cap=0.0, bias=False),
        # one row and its adapter through a square projection: latency
        dict(name="lora_1_row", kind="lora", rows=1, k=4096, n=4096, rank=16, parts=1, adapters=4, runs=1, dt="bf16", c="bf16"),
        # 24 rows of as many requests, sixteen adapters, in no order, through q|k|v
        dict(name="lora_24_rows_mixed", kind="lora", rows=24, k=4096, n=12288, rank=16, parts=3, adapters=16, runs=0, dt="bf16", c="bf16"),
        # four requests' images through q|k|v, one without an adapter
        dict(name="lora_4_images_qkv", kind="lora", rows=4352, k=4096, n=12288, rank=32, parts=3, adapters=4, runs=4, dt="bf16", c="bf16"),
        # the down-projection of eight requests at 1024 x 1024, into fp32 rows, half activations
        dict(name="lora_8_images_down", kind="lora", rows=16401, k=12288, n=4096, rank=64, parts=1, adapters=6, runs=8, dt="f16", c="f32"),
        # one row's queries and keys: latency
        dict(name="rope_1_row", kind="rope", rows=1, heads=32, kv=8, d=128, axes="128", shared=False, mode=1, norm=True, x="bf16", out="bf16", pos="i32", far=1 << 20),
        # SDXL-sized heads of an image, half, no norm
        dict(name="rope_1333_f16", kind="rope", rows=1333, heads=20, kv=20, d=64, axes="16,24,24", shared=False, mode=2, norm=False, x="f16", out="f16", pos="i32", far=64),
        # a video's rows, fp32 out of the projection, three axes that share one series of frequencies
        dict(name="rope_video", kind="rope", rows=32760, heads=32, kv=32, d=128, axes="32,48,48", shared=True, mode=1, norm=True, x="f32", out="bf16", pos="f32", far=4096),
    ]


def _log(rng, lo, hi, of=1):
    return max(of, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / of)) * of)


MOST_SCORES, MOST_MACS, MOST_VALUES = 2 * 32 * 8448 * 8448, 16401 * 12288 * 64, 32760 * 64 * 128


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "lora", "lora", "rope"])
    dt = rng.choice(["bf16", "bf16", "f16"])
    if kind == "attn":
        docs, d = rng.choice([1, 1, 2, 3, 5, 8]), rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8, 10, 16])
        heads = kv * rng.choice([1, 1, 2, 4, 5])
        mask = rng.choice(["full", "causal", "text", "prefix"])
        most = min(int(math.sqrt(MOST_SCORES / (docs * heads))), 16384)
        k = [_log(rng, 1, most) for _ in range(docs)]
        # all rows, one new row over a cache, or any number of rows over other keys
        form = rng.choice(["self", "self", "token", "cross"])
        q = k if form == "self" else [1] * docs if form == "token" else [min(_log(rng, 1, most), most) for _ in k]
        s = [rng.randint(0, n) if mask in ("text", "prefix") else 0 for n in k]
        text = [",".join(map(str, v)) for v in (q, k, s)]
        return dict(kind=kind, q=text[0], k=text[1], s=text[2], mask=mask, heads=heads, kv=kv, d=d, dt=dt,
                    cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.choice([False, False, True]))
    if kind == "lora":
        parts, rank = rng.choice([1, 2, 3]), rng.choice([8, 16, 24, 32, 64, 128])
        k, n = _log(rng, 256, 12288, 8), _log(rng, 256, 12288, 8 * parts)
        rows = min(_log(rng, 1, 16384), 16384 * 12288 // max(k, n), MOST_MACS // (max(k * parts, n) * rank))
        runs = rng.choice([0, 1, 2, 5, 9])
        return dict(kind=kind, rows=rows, k=k, n=n, rank=rank, parts=parts, adapters=rng.randint(1, 8), runs=runs, dt=dt,
                    c=rng.choice([dt, "f32"]))
    d = rng.choice([64, 128])
    axes, shared = rng.choice([([d], False), ([16, 56, 56], False), ([32, 48, 48], True), ([64, 64], False), ([40, 24], True)]
                              if d == 128 else [([64], False), ([16, 24, 24], False), ([16, 24, 24], True), ([16, 16], False)])
    kv = rng.choice([1, 4, 8, 20])
    heads = kv * rng.choice([1, 1, 2, 4])
    rows = min(_log(rng, 1, 32760), MOST_VALUES // ((heads + kv) * d))
    x = rng.choice(["f32", "bf16", "f16"])
    return dict(kind=kind, rows=rows, heads=heads, kv=kv, d=d, axes=",".join(map(str, axes)), shared=shared, mode=rng.choice([1, 2]),
                norm=rng.choice([True, False]), x=x, out=rng.choice(["bf16", "f16"] if x == "f32" else [x]),
                pos=rng.choice(["i32", "i32", "f32"]), far=_log(rng, 16, 1 << 20))


# ---------------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------------------------------------

class Rng:
    """Draws on the device: call number i of a seed is the same tensor everywhere."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std).add_(mean)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)


def _lens(text):
    return [int(v) for v in text.split(",")]


def _documents(case):
    """(first query row, query rows, first key row, key rows, position of the first query row, block, prefix) of each: the query
    rows are the last of the keys' positions."""
    q, k, s = (_lens(case[n]) for n in ("q", "k", "s"))
    s = s if len(s) == len(q) else s * len(q)
    block = {"full": lambda p: 0, "causal": lambda p: 0xFFFFFFFF, "text": lambda p: p, "prefix": lambda p: 0xFFFFFFFF}[case["mask"]]
    return [(sum(q[:i]), q[i], sum(k[:i]), k[i], k[i] - q[i], block(s[i]), s[i] if case["mask"] == "prefix" else 0)
            for i in range(len(q))]


def inputs(case, seed):
    rng, kind = Rng(seed), case["kind"]
    if kind == "attn":
        dt, d = DTYPES[case["dt"]], case["d"]
        nq, nk = sum(_lens(case["q"])), sum(_lens(case["k"]))
        # normed heads with their channels' weights: scores of a few units, larger where they are capped
        spread = torch.exp(rng.normal(d, std=0.4)) * (3.0 if case["cap"] else 1.0)
        t = {"q": (rng.normal(nq, case["heads"], d) * spread).to(dt), "k": rng.normal(nk, case["kv"], d).to(dt),
             "v": rng.normal(nk, case["kv"], d).to(dt)}
        t["docs"] = torch.tensor(_documents(case), dtype=torch.int64, device="cuda")
        if case["bias"]:
            t["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, dtype=F32, device="cuda") / case["heads"])
        return t
    if kind == "lora":
        dt, n, k, r = DTYPES[case["dt"]], case["n"], case["k"], case["rank"]
        t = {"x": rng.normal(case["rows"], k).mul_(torch.exp(rng.normal(k, std=0.5))).to(dt),
             "a": rng.normal(case["adapters"], case["parts"] * r, k, std=k ** -0.5).to(dt),
             "b": rng.normal(case["adapters"], n, r, std=0.3 * r ** -0.5).to(dt),
             "scale": torch.exp(rng.normal(case["adapters"], std=0.3)),
             "base": rng.normal(case["rows"], n).to(DTYPES[case["c"]])}
        if case["runs"]:
            # requests one after the other, the last of several without an adapter
            cuts = rng.ints(0, case["rows"], case["runs"] - 1).sort().values
            run = torch.bucketize(torch.arange(case["rows"], dtype=torch.int32, device="cuda"), cuts, right=True).int()
            t["ids"] = torch.where((run == case["runs"] - 1) & (run > 0), -1, run % case["adapters"]).int()
        else:
            t["ids"] = rng.ints(-1, case["adapters"], case["rows"])
        return t
    dt, d = DTYPES[case["x"]], case["d"]
    axes = len(_lens(case["axes"]))
    t = {"q": rng.normal(case["rows"], case["heads"], d, std=2.0).to(dt), "k": rng.normal(case["rows"], case["kv"], d, std=2.0).to(dt),
         "pos": rng.ints(-(case["far"] // 2), case["far"], case["rows"], axes)}
    if case["pos"] == "f32":
        t["pos"] = t["pos"].float() / 4.0  # frames at a rate of their own
    if case["norm"]:
        t.update(wq=rng.normal(d, std=0.1, mean=1.0), wk=rng.normal(d, std=0.1, mean=1.0))
    return t


# ---------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------

def _padded(x, start, rows, most):
    """Rows start .. start + rows of x [rows][heads][d] for each document, as [documents][heads][most][d] in 32 bits."""
    at = torch.arange(most, device=x.device)[None] + start[:, None]
    at = torch.where(torch.arange(most, device=x.device)[None] < rows[:, None], at, start[:, None].clamp(max=x.shape[0] - 1))
    return x[at].float().transpose(1, 2).contiguous()


def _plain_attn(case, t):
    docs, group = t["docs"], case["heads"] // case["kv"]
    q0, nq, k0, nk, pos0, block, prefix = docs.unbind(1)
    mq, mk = max(_lens(case["q"])), max(_lens(case["k"]))
    q, k, v = _padded(t["q"], q0, nq, mq), _padded(t["k"], k0, nk, mk), _padded(t["v"], k0, nk, mk)
    n, d = len(docs), case["d"]
    q = q.reshape(n, case["kv"], group * mq, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(n, case["heads"], mq, mk).mul_(d ** -0.5)
    if case["cap"]:
        s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
    pos = pos0[:, None, None] + torch.arange(mq, device=q.device)[None, :, None]
    key = torch.arange(mk, device=q.device)[None, None, :]
    if case["bias"]:
        s = s - t["slopes"][None, :, None, None] * (pos - key).abs().float()[:, None]
    b = block[:, None, None]
    seen = ((b == 0) | (pos >= b) | (key <= pos) | (key < prefix[:, None, None])) & (key < nk[:, None, None])
    s = s.masked_fill_(~seen[:, None], -math.inf)
    top = s.amax(3, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p.reshape(n, case["kv"], group * mq, mk), v).reshape(n, case["heads"], mq, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).transpose(1, 2)
    return {"out": o[torch.arange(mq, device=q.device)[None] < nq[:, None]].to(DTYPES[case["dt"]])}


def _plain_lora(case, t):
    rows, adapters, parts, rank = case["rows"], case["adapters"], case["parts"], case["rank"]
    # every adapter's first product, the rows' own kept (those without an adapter keep none)
    h = torch.mm(t["x"].float(), t["a"].float().reshape(adapters * parts * rank, -1).t()).reshape(rows, adapters, parts, rank)
    mine = t["ids"][:, None] == torch.arange(adapters, device=h.device)[None]
    h = torch.where(mine[:, :, None, None], h * t["scale"][None, :, None, None], torch.zeros((), device=h.device))
    b = t["b"].float().reshape(adapters, parts, -1, rank)
    delta = torch.bmm(h.permute(2, 0, 1, 3).reshape(parts, rows, adapters * rank),
                      b.permute(1, 0, 3, 2).reshape(parts, adapters * rank, -1)).permute(1, 0, 2).reshape(rows, -1)
    return {"c": (t["base"].float() + delta).to(DTYPES[case["c"]])}


def _series(case):
    """The angle's step a position (64 bits) and the axis, of every pair."""
    dims = torch.tensor(_lens(case["axes"]), device="cuda")
    pairs = sum(_lens(case["axes"])) // 2
    i = torch.arange(pairs, device="cuda")
    ends = torch.cumsum(dims // 2, 0)
    axis = torch.bucketize(i, ends, right=True)
    j, dim = (i, torch.full_like(i, 2 * pairs)) if case["shared"] else (i - (ends - dims // 2)[axis], dims[axis])
    return THETA ** (-2.0 * j.to(F64) / dim.to(F64)), axis


def _plain_rope(case, t):
    step, axis = _series(case)
    angle = t["pos"][:, axis].to(F64) * step
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    pairs = cos.shape[2]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * w
        r, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
        u, v = (r[..., :pairs], r[..., pairs:]) if case["mode"] == 1 else (r[..., 0::2], r[..., 1::2])
        u, v = u * cos - v * sin, u * sin + v * cos
        r = torch.cat((u, v), 2) if case["mode"] == 1 else torch.stack((u, v), 3).flatten(2)
        return torch.cat((r, rest), 2).to(DTYPES[case["out"]])

    return {"q": turned(t["q"], t.get("wq")), "k": turned(t["k"], t.get("wk"))}


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------

def _binding():
    path = os.path.join(os.getcwd(), "mako-image_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mkimage
    return mkimage


def _code(M, dt):
    return {"f32": M.F32, "bf16": M.BF16, "f16": M.F16}[dt]


def _empty(dt, *shape):
    return torch.empty(*shape, dtype=DTYPES[dt], device="cuda")


def _workspace(M, name, args):
    """The bytes that the call asks for, from torch's allocator, as a program that keeps its workspace has it."""
    need = C.c_uint64()
    M.call(name, C.byref(args), C.byref(need))
    args.workspace_bytes = need.value
    space = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    args.workspace = space.data_ptr()
    return space


def _attn_call(M, case, t):
    d, docs = case["d"], _documents(case)
    g = M.AttnPackedArgs()
    out = _empty(case["dt"], t["q"].shape[0], case["heads"], d)
    g.q, g.k, g.v, g.out = (x.data_ptr() for x in (t["q"], t["k"], t["v"], out))
    g.ldq = g.ldo = case["heads"] * d
    g.ldk = g.ldv = case["kv"] * d
    g.dtype = g.out_dtype = _code(M, case["dt"])
    g.heads, g.kv_heads, g.d = case["heads"], case["kv"], d
    g.scale, g.cap = d ** -0.5, case["cap"]
    g.slopes = t["slopes"].data_ptr() if case["bias"] else None
    table = (M.AttnDoc * len(docs))(*[M.AttnDoc(*v) for v in docs])
    g.docs, g.n_docs = table, len(docs)
    return ("mk_attention_packed", g), {"out": out}, (table, _workspace(M, "mk_attention_packed_workspace", g))


def _lora_call(M, case, t):
    g = M.LoraRowsArgs()
    c = _empty(case["c"], case["rows"], case["n"])
    g.x, g.a, g.b, g.scale, g.ids, g.base, g.c = (x.data_ptr() for x in (t["x"], t["a"], t["b"], t["scale"], t["ids"], t["base"], c))
    g.ldx, g.ldbase, g.ldc = case["k"], case["n"], case["n"]
    g.rows, g.K, g.N, g.rank, g.parts, g.adapters = (case[n] for n in ("rows", "k", "n", "rank", "parts", "adapters"))
    g.dtype, g.c_dtype = _code(M, case["dt"]), _code(M, case["c"])
    return ("mk_lora_rows", g), {"c": c}, (_workspace(M, "mk_lora_rows_workspace", g),)


def _rope_call(M, case, t):
    g, d = M.RopeRowsArgs(), case["d"]
    q, k = _empty(case["out"], case["rows"], case["heads"], d), _empty(case["out"], case["rows"], case["kv"], d)
    g.q, g.k, g.q_out, g.k_out, g.pos = (x.data_ptr() for x in (t["q"], t["k"], q, k, t["pos"]))
    g.ldq = g.ldqo = case["heads"] * d
    g.ldk = g.ldko = case["kv"] * d
    g.rows, g.heads, g.kv_heads, g.d = case["rows"], case["heads"], case["kv"], d
    g.dtype, g.out_dtype = _code(M, case["x"]), _code(M, case["out"])
    if case["norm"]:
        g.norm_q, g.norm_k, g.eps = t["wq"].data_ptr(), t["wk"].data_ptr(), EPS
    dims = _lens(case["axes"])
    g.axes, g.pos_ld, g.pos_dtype = len(dims), len(dims), M.I32 if case["pos"] == "i32" else M.F32
    g.axis_dims = (C.c_uint32 * 4)(*dims)
    g.theta, g.series, g.rope_mode = THETA, M.ROPE_SHARED if case["shared"] else M.ROPE_OWN, case["mode"]
    return ("mk_rope_rows", g), {"q": q, "k": k}, ()


def prepare(case, seed):
    s = {"case": case, "data": inputs(case, seed)}
    if own:
        # argument blocks, outputs and workspaces, as a program sets them up once for its layers
        s["M"] = M = _binding()
        (name, g), s["out"], s["keep"] = {"attn": _attn_call, "lora": _lora_call, "rope": _rope_call}[case["kind"]](M, case, s["data"])
        s["call"], s["args"] = (name, C.byref(g)), g
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        s["M"].call(*s["call"], torch.cuda.current_stream().cuda_stream or None)
        return s["out"]
    return {"attn": _plain_attn, "lora": _plain_lora, "rope": _plain_rope}[s["case"]["kind"]](s["case"], s["data"])


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def _pairs_seen(nq, nk, pos0, block, prefix):
    """(row, key) pairs of a document that its masks leave."""
    rows = torch.arange(nq, dtype=torch.int64) + pos0
    own_keys = (rows + 1).clamp(0, nk).maximum(torch.tensor(min(prefix, nk)))
    return int(torch.where((torch.tensor(block) == 0) | (rows >= block), torch.tensor(nk), own_keys).sum())


def work(case):
    kind = case["kind"]
    if kind == "attn":
        docs, d, size = _documents(case), case["d"], SIZE[case["dt"]]
        seen = sum(_pairs_seen(nq, nk, pos0, block, prefix) for _, nq, _, nk, pos0, block, prefix in docs)
        return {"bytes": size * d * sum(2 * v[1] * case["heads"] + 2 * v[3] * case["kv"] for v in docs), "flops": 4 * d * case["heads"] * seen}
    if kind == "lora":
        rows, k, n, r, parts = (case[v] for v in ("rows", "k", "n", "rank", "parts"))
        runs = case["runs"]
        used = min(case["adapters"], rows, rows if runs == 0 else max(runs - 1, 1))
        return {"bytes": SIZE[case["dt"]] * (rows * k + used * r * (parts * k + n)) + rows * (2 * n * SIZE[case["c"]] + 4),
                "flops": 2 * rows * r * (parts * k + n)}
    values = case["rows"] * (case["heads"] + case["kv"]) * case["d"]
    return {"bytes": values * (SIZE[case["x"]] + SIZE[case["out"]]) + 4 * case["rows"] * len(_lens(case["axes"])), "flops": 8 * values}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    t = inputs(case, seed)

    def attention():
        out = torch.zeros(t["q"].shape, dtype=F64, device="cuda")
        group = case["heads"] // case["kv"]
        for q0, nq, k0, nk, pos0, block, prefix in _documents(case):
            if not nk:
                continue
            j = torch.arange(nk, device="cuda")
            for h in range(case["heads"]):
                k, v = t["k"][k0:k0 + nk, h // group].to(F64), t["v"][k0:k0 + nk, h // group].to(F64)
                at = pos0 + torch.arange(nq, device="cuda")
                hidden = (j[None] > at[:, None]) & (j >= prefix)[None] & (at < block)[:, None] if block else None
                score = (t["q"][q0:q0 + nq, h].to(F64) / math.sqrt(case["d"])) @ k.T
                if case["cap"]:
                    score = case["cap"] * torch.tanh(score / case["cap"])
                if case["bias"]:
                    score = score - t["slopes"][h].to(F64) * (j[None] - at[:, None]).abs()
                if hidden is not None:
                    score[hidden] = -math.inf
                weight = torch.nan_to_num(torch.softmax(score, 1), nan=0.0)  # a row that sees nothing
                out[q0:q0 + nq, h] = weight @ v
        return {"out": out}

    def adapters():
        c = t["base"].to(F64)
        width = case["n"] // case["parts"]
        for a in range(case["adapters"]):
            rows = (t["ids"] == a).nonzero()[:, 0]
            if not len(rows):
                continue
            h = t["x"][rows].to(F64) @ t["a"][a].to(F64).T
            for p in range(case["parts"]):
                cols = slice(p * width, (p + 1) * width)
                c[rows, cols] += t["scale"][a].to(F64) * (h[:, p * case["rank"]:(p + 1) * case["rank"]] @ t["b"][a, cols].to(F64).T)
        return {"c": c}

    def rotary():
        dims, found = _lens(case["axes"]), {}
        total = sum(dims)
        for name, w in (("q", t.get("wq")), ("k", t.get("wk"))):
            x = t[name].to(F64)
            if w is not None:
                x = x / (x.pow(2).mean(2, True) + EPS).sqrt() * w.to(F64)
            y, first = x.clone(), 0
            for a, dim in enumerate(dims):
                for j in range(dim // 2):
                    i = first + j
                    angle = t["pos"][:, a].to(F64) * THETA ** (-2.0 * (i / total if case["shared"] else j / dim))
                    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
                    lo, hi = (i, i + total // 2) if case["mode"] == 1 else (2 * i, 2 * i + 1)
                    z = torch.complex(x[..., lo], x[..., hi]) * turn
                    y[..., lo], y[..., hi] = z.real, z.imag
                first += dim // 2
            found[name] = y
        return found

    return {"attn": attention, "lora": adapters, "rope": rotary}[case["kind"]]()
