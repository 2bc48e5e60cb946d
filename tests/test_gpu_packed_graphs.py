"""Captured calls of the packed operators on the kernels of many rows and of split keys: replayed with other inputs, adapters' numbers and
positions in the same buffers, and with whatever is left in the workspace, each replay against an eager call."""
import ctypes as C

import numpy as np
import pytest

import mkimage as M
from test_gpu_lora_tiles import ORDER, SPLITS, plan
from test_gpu_packed_ops import Attn, Lora, Rope, packed
from test_gpu_packed_run import hip

pytestmark = pytest.mark.gpu


class Captured:
    def __init__(self, *calls):
        self.h, self.s, graph, self.run = hip(), C.c_void_p(), C.c_void_p(), C.c_void_p()
        M.call("mk_stream_create", C.byref(self.s))
        assert self.h.hipStreamBeginCapture(self.s, 0) == 0
        for name, g in calls:
            M.call(name, C.byref(g), self.s)
        assert self.h.hipStreamEndCapture(self.s, C.byref(graph)) == 0
        assert self.h.hipGraphInstantiate(C.byref(self.run), graph, None, None, 0) == 0
        self.graph = graph

    def replay(self):
        assert self.h.hipGraphLaunch(self.run, self.s) == 0

    def wait(self):
        M.call("mk_stream_synchronize", self.s)

    def close(self):
        assert self.h.hipGraphExecDestroy(self.run) == 0 and self.h.hipGraphDestroy(self.graph) == 0
        M.call("mk_stream_destroy", self.s)


def test_adapters_of_many_rows_replayed_with_other_rows_and_numbers(gpu):
    rng = np.random.default_rng(0)
    many, wide = Lora(4161, 520, 264, 24, 3, 5, rng.integers(-1, 5, 4161), M.BF16, M.BF16, pad=8), Lora(300, 1032, 24616, 16, 1, 3, rng.integers(-1, 3, 300), M.F16, M.F32)
    graphs = []
    for a in (many, wide):
        g = a.args()
        p = plan(g)
        assert p[ORDER] == 1 and (a is wide or p[SPLITS] > 1)
        graphs.append(Captured(("mk_lora_rows", g)))
        a.g = g
    for rep in range(4):
        for a in (many, wide):
            adapters = a.sizes[5]
            ids = [rng.integers(-1, adapters, a.sizes[0]), np.sort(rng.integers(0, adapters, a.sizes[0])), np.full(a.sizes[0], -1), rng.integers(-1, adapters + 1, a.sizes[0])][rep]
            a.ids = ids.astype(np.int32)
            a.keep[0].write(a.ids)
            x = np.roll(a.buf["x"].before, rep, 0)
            a.buf["x"].dev.write(x)
            a.val["x"] = np.roll(a.val["x"], 1 if rep else 0, 0)
            M.call("mk_memset", a.space.p, 0xFF, a.g.workspace_bytes)
        M.sync()
        for c in graphs:
            c.replay()
        if rep % 2:
            Rope(300, 4, 4, 64, [64], M.F16, M.F16).check()  # eager work of the program's own, with the replays on their streams
        for c, a in zip(graphs, (many, wide)):
            c.wait()
            want, tol = a.want()
            got = a.result()
            assert (np.abs(got - want) <= tol).all(), rep
            M.call("mk_lora_rows", C.byref(a.g), None)
            assert np.array_equal(a.result(), got), rep
    for c in graphs:
        c.close()


def test_attention_over_split_keys_replayed_with_other_rows(gpu):
    docs, nq, nk = packed([1, 3, 1, 7], [4099, 777, 1, 1500], mask="causal")
    jobs = [Attn(docs, nq, nk, 8, 1, 128, M.BF16), Attn([(0, 40, 0, 3000, 2960, 0, 0)], 40, 3000, 4, 4, 64, M.F16, cap=20.0, slopes=np.float32([0.1, 0.0, 0.01, 1.0]))]
    for a in jobs:
        a.check()  # (its arguments and workspace are what is captured)
        assert a.g.workspace_bytes > 0
    graphs = [Captured(("mk_attention_packed", a.g)) for a in jobs]
    for rep in range(4):
        for a in jobs:
            for n in "qkv":
                x = np.roll(a.buf[n].before, rep, 0)
                a.buf[n].dev.write(x)
            M.call("mk_memset", a.space.p, 0xFF, a.g.workspace_bytes)
            M.call("mk_memset", a.out.dev.p, 0x33, a.out.dev.nbytes)
        M.sync()
        for c in graphs:
            c.replay()
        if rep % 2:
            Rope(300, 4, 4, 64, [64], M.F16, M.F16).check()
        for c, a in zip(graphs, jobs):
            c.wait()
            got = a.out.read()
            M.call("mk_memset", a.out.dev.p, 0x33, a.out.dev.nbytes)
            M.call("mk_attention_packed", C.byref(a.g), None)
            M.sync()
            assert np.array_equal(a.out.read(), got), rep
    for c in graphs:
        c.close()
