"""Which kernels of the int8 path the library holds, and which ones a launch can take (no GPU)."""
import re

import mkimage as M


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
