"""Every kernel of mk_gemm_i8 where its loops, batches and rows can go wrong, each shape checked to take the kernel it is
meant for; tolerances are test_gpu_int8_ops.py's."""
import numpy as np
import pytest

import mkimage as M
from test_gpu_int8_ops import Product
from test_int8_kernels import GLU, SHAPES, kind, kinds

pytestmark = pytest.mark.gpu

# tile: (m, n, k steps). The steps pass what a workgroup keeps in LDS and leave every remainder of it to the loop's end, so
# that loads made inside the loop are used and each stage is loaded again.
STEPS = {(32, 32, 8): (50, 1032, range(9, 17)), (64, 32, 6): (37, 4104, range(7, 13)), (32, 64, 6): (50, 2056, range(7, 13)),
         (64, 64, 4): (37, 8200, range(5, 9)), (64, 128, 4): (100, 8200, range(7, 11)), (64, 128, 2): (100, 8200, range(3, 7)),
         (128, 128, 2): (1537, 4104, range(3, 6)), (128, 128, 4): (200, 8200, range(5, 9)),
         (256, "one", 0): (900, 8200, range(5, 7)), (256, "one", 128): (3100, 5128, (4, 5)),
         (256, "chain", 0): (3100, 8200, (4,)), (256, "chain", 128): (4300, 8200, (4,))}


@pytest.mark.parametrize("epi, tile, m, n, ke", [
    (epi, t, m, n, ke) for epi in (M.EPI_STORE, M.EPI_SWIGLU) for t, (m, n, kes) in STEPS.items() for ke in kes if t in kinds(epi)])
def test_product_loops_past_the_stages(gpu, epi, tile, m, n, ke):
    k = 128 * ke - 48  # the last step is partial
    assert kind(m, n, k, epi) == tile
    Product(m, n, k, epi).check()


# Every epilogue on every kernel, three batch items in padded rows of A and C, a split inside each item's segments: chains go
# on from one item to the next, and so do the parts of the last round.
EPILOGUES = [(M.EPI_STORE, M.BF16), (M.EPI_GELU_TANH, M.F32), (M.EPI_SILU, M.F16), (M.EPI_ADD, M.F32), (M.EPI_GATE_ADD, M.F32),
             (M.EPI_GATE_TANH, M.F32), (M.EPI_SWIGLU, M.BF16), (M.EPI_GEGLU, M.F32)]


@pytest.mark.parametrize("epi, c, tile", [(epi, c, tile) for epi, c in EPILOGUES for tile in kinds(epi)])
def test_product_batches_on_every_kernel(gpu, epi, c, tile):
    m, n, k = SHAPES[tile]
    assert kind(m, n, k, epi, batch=3, lda=k + 16) == tile
    cols = n // 2 if epi in GLU else n
    Product(m, n, k, epi, c, batch=3, lda=k + 16, ldc=cols + 4, split=m // 3, seg=m // 2 + 1).check()


# (m, n, k) of a whole launch and row counts whose launches take the other kernels
LAUNCHES = [(5400, 6152, 400, (9, 22, 40, 80, 200, 1000, 1300, 2600, 4000, 5200)), (2000, 4104, 848, (7, 15, 40, 120, 300, 600, 920))]


@pytest.mark.parametrize("epi, c", [(M.EPI_STORE, M.F32), (M.EPI_GELU_TANH, M.F16), (M.EPI_SILU, M.BF16), (M.EPI_GATE_TANH, M.F32),
                                    (M.EPI_SWIGLU, M.F32), (M.EPI_GEGLU, M.BF16)])
def test_product_row_bits_are_the_same_on_every_kernel(gpu, epi, c):
    seen = set()
    for m, n, k, prefixes in LAUNCHES:
        p = Product(m, n, k, epi, c, split=50, seg=300)
        p.run()
        whole = p.bits.copy()
        seen.add(kind(m, n, k, epi))
        for rows in prefixes:
            p.run(rows=rows)
            assert np.array_equal(p.bits[0].view(np.uint8), whole[0, :rows].view(np.uint8)), (rows, kind(rows, n, k, epi))
            seen.add(kind(rows, n, k, epi))
    assert seen >= set(kinds(epi)) - {(256, "one", 64)}


@pytest.mark.parametrize("tile, m, n, epi", [((32, 32, 8), 50, 1032, M.EPI_STORE), ((64, 32, 6), 37, 4104, M.EPI_STORE),
                                             ((64, 64, 4), 37, 8200, M.EPI_STORE), ((32, 64, 6), 50, 2056, M.EPI_GEGLU),
                                             ((64, 64, 4), 37, 8200, M.EPI_GEGLU)])
def test_product_sums_are_exact_at_the_largest_k_in_tiles(gpu, tile, m, n, epi):
    k = 131056
    assert kind(m, n, k, epi) == tile
    p = Product(m, n, 16, epi, bias=False)
    p.k = p.lda = k
    p.sa = m * k
    p.A, p.W = np.full(m * k, -128, np.int8), np.full((n, k), -128, np.int8)
    p.W[3] = 127
    p.asc[:], p.wsc[:] = 1.0, 1.0
    s = np.full(p.cols, 128.0 * 128.0 * k, np.float32)  # 2147221504: to fp32 once
    s[3] = -128.0 * 127.0 * k
    if epi == M.EPI_GEGLU:
        s = s * np.float32(128.0 * 128.0 * k)  # the gate's GELU is the gate itself: one more product
    assert np.array_equal(p.run(), np.broadcast_to(s.astype(np.float64), (1, m, p.cols)))


# One and two k steps, no more than any kernel keeps in LDS, whole ones and parts.
@pytest.mark.parametrize("epi", [M.EPI_STORE, M.EPI_GEGLU])
@pytest.mark.parametrize("k", [16, 112, 128, 176, 256])
def test_product_of_one_or_two_steps(gpu, k, epi):
    seen = set()
    for m, n in ((1, 8), (17, 6152), (17, 8200), (50, 4104), (50, 6152), (50, 8200), (100, 8200), (1537, 4104), (1537, 8200),
                 (4300, 136), (4300, 8200)):
        Product(m, n, k, epi).check()
        seen.add(kind(m, n, k, epi))
    assert seen >= {(64, 128, 2), (128, 128, 2), (256, "one", 0)} and len(seen) >= 5
