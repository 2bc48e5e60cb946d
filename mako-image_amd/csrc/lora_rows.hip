// mk_lora_rows: low-rank adapters of many requests beside a shared projection.
#include "common.hpp"

#include <type_traits>

namespace mk {

namespace {

struct LoraP {
    const uint16_t *x, *a, *b;
    const float* scale;
    const int32_t* ids;
    const void* base;
    void* c;
    float* t; // workspace: [rows][parts rank]
    int64_t ldx, ldbase, ldc;
    uint32_t rows, K, N, rank, parts, adapters;
};

template <bool F16> __device__ inline float widen(uint16_t h) { return F16 ? h2f_bits(h) : bf2f_bits(h); }
// the adapter of a row, or -1
__device__ inline int adapter_of(const LoraP& p, uint32_t row)
{
    const int id = p.ids ? p.ids[row] : 0;
    return id >= 0 && uint32_t(id) < p.adapters ? id : -1;
}

// t[row][i] = x[row] . A[a][i], a wave for each
template <bool F16> __global__ __launch_bounds__(256) void shrink_kernel(LoraP p)
{
    const uint32_t width = p.parts * p.rank, row = blockIdx.y, i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= width)
        return;
    const int a = adapter_of(p, row);
    if (a < 0)
        return;
    const uint16_t* x = p.x + int64_t(row) * p.ldx;
    const uint16_t* w = p.a + (int64_t(a) * width + i) * p.K;
    float s = 0.0f;
    for (uint32_t k = lane; k < p.K; k += 64)
        s += widen<F16>(x[k]) * widen<F16>(w[k]);
    s = wave_sum(s);
    if (lane == 0)
        p.t[int64_t(row) * width + i] = s;
}

// c[row][n] = base[row][n] + scale t[row] . B[a][n], a thread for each
template <bool F16, uint32_t CT> __global__ __launch_bounds__(256) void expand_kernel(LoraP p)
{
    const uint32_t row = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
    if (n >= p.N)
        return;
    const int a = adapter_of(p, row);
    float v = 0.0f;
    if (a >= 0) {
        const uint32_t part = n / (p.N / p.parts);
        const float* t = p.t + int64_t(row) * p.parts * p.rank + part * p.rank;
        const uint16_t* w = p.b + (int64_t(a) * p.N + n) * p.rank;
        for (uint32_t j = 0; j < p.rank; ++j)
            v += t[j] * widen<F16>(w[j]);
        if (p.scale)
            v *= p.scale[a];
    }
    const int64_t ci = int64_t(row) * p.ldc + n, bi = int64_t(row) * p.ldbase + n;
    if constexpr (CT == MK_F32) {
        static_cast<float*>(p.c)[ci] = (p.base ? static_cast<const float*>(p.base)[bi] : 0.0f) + v;
    } else {
        const float o = p.base ? widen<CT == MK_F16>(static_cast<const uint16_t*>(p.base)[bi]) : 0.0f;
        static_cast<uint16_t*>(p.c)[ci] = CT == MK_F16 ? f2h_bits(o + v) : f2bf_bits(o + v);
    }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// sizes and types, for the call and for its workspace's size
mk_status check_sizes(const mk_lora_rows_args* a)
{
    if (a->dtype != MK_BF16 && a->dtype != MK_F16)
        return fail(MK_ERR_ARG, "lora_rows: x, a and b must be bf16 or f16");
    if (a->c_dtype != MK_F32 && a->c_dtype != MK_BF16 && a->c_dtype != MK_F16)
        return fail(MK_ERR_ARG, "lora_rows: base and c must be f32, bf16 or f16");
    if (!a->parts || a->parts > 4 || !a->rank || a->rank % 8 || a->rank > 256 || !a->adapters || a->adapters > 0x7fffffffu)
        return fail(MK_ERR_ARG, "lora_rows: 1 to 4 parts of rank a multiple of 8 up to 256, 1 adapter or more");
    if (!a->K || a->K % 8 || a->K > (1u << 24) || !a->N || a->N % (8 * a->parts) || a->N > (1u << 24))
        return fail(MK_ERR_ARG, "lora_rows: K must be a multiple of 8, N of 8 parts, up to 2^24");
    if (a->rows > 0x7fffffffu)
        return fail(MK_ERR_ARG, "lora_rows: more than 2^31 - 1 rows");
    return MK_OK;
}
uint64_t workspace_of(const mk_lora_rows_args* a) { return round_up(uint64_t(a->rows) * a->parts * a->rank * 4, 16); }

} // namespace

} // namespace mk

using namespace mk;

extern "C" {

mk_status mk_lora_rows_workspace(const mk_lora_rows_args* a, uint64_t* bytes)
{
    if (!a || !bytes)
        return fail(MK_ERR_ARG, "lora_rows_workspace: null argument");
    MK_TRY(check_sizes(a));
    *bytes = workspace_of(a);
    return MK_OK;
}

mk_status mk_lora_rows(const mk_lora_rows_args* a, void* stream)
{
    if (!a || !a->x || !a->a || !a->b || !a->c)
        return fail(MK_ERR_ARG, "lora_rows: null argument (x, a, b and c are required)");
    MK_TRY(check_sizes(a));
    if (a->ldx < int64_t(a->K) || a->ldx % 8 || a->ldc < int64_t(a->N) || a->ldc % 8 ||
        (a->base && (a->ldbase < int64_t(a->N) || a->ldbase % 8)))
        return fail(MK_ERR_ARG, "lora_rows: ldx, ldbase and ldc must be multiples of 8, at least the row");
    if (a->base == a->c && a->ldbase != a->ldc)
        return fail(MK_ERR_ARG, "lora_rows: in place needs ldbase == ldc");
    if (!aligned(a->x, 16) || !aligned(a->a, 16) || !aligned(a->b, 16) || !aligned(a->base, 16) || !aligned(a->c, 16) ||
        !aligned(a->workspace, 16) || !aligned(a->scale, 4) || !aligned(a->ids, 4))
        return fail(MK_ERR_ARG, "lora_rows: operands and workspace must be 16-byte aligned (scale and ids 4)");
    if (!a->rows)
        return MK_OK;
    if (!a->workspace || a->workspace_bytes < workspace_of(a))
        return fail(MK_ERR_ARG, "lora_rows: the workspace is smaller than mk_lora_rows_workspace says");
    LoraP p{static_cast<const uint16_t*>(a->x), static_cast<const uint16_t*>(a->a), static_cast<const uint16_t*>(a->b), a->scale,
            a->ids, a->base, a->c, static_cast<float*>(a->workspace), a->ldx, a->ldbase, a->ldc, a->rows, a->K, a->N, a->rank,
            a->parts, a->adapters};
    hipStream_t s = static_cast<hipStream_t>(stream);
    // rows in the grid's second dimension, at most 65535 a launch
    const uint32_t width = a->parts * a->rank, csize = a->c_dtype == MK_F32 ? 4 : 2;
    for (uint32_t r0 = 0; r0 < a->rows; r0 += 65535) {
        LoraP c = p;
        c.rows = a->rows - r0 < 65535 ? a->rows - r0 : 65535;
        c.x += int64_t(r0) * p.ldx;
        c.t += int64_t(r0) * width;
        c.ids = p.ids ? p.ids + r0 : nullptr;
        c.base = p.base ? static_cast<const char*>(p.base) + int64_t(r0) * p.ldbase * csize : nullptr;
        c.c = static_cast<char*>(p.c) + int64_t(r0) * p.ldc * csize;
        const dim3 g1(cdiv(width, 4), c.rows), g2(cdiv(p.N, 256), c.rows);
        const bool f16 = a->dtype == MK_F16;
        f16 ? shrink_kernel<true><<<g1, 256, 0, s>>>(c) : shrink_kernel<false><<<g1, 256, 0, s>>>(c);
        if (a->c_dtype == MK_F32)
            f16 ? expand_kernel<true, MK_F32><<<g2, 256, 0, s>>>(c) : expand_kernel<false, MK_F32><<<g2, 256, 0, s>>>(c);
        else if (a->c_dtype == MK_BF16)
            f16 ? expand_kernel<true, MK_BF16><<<g2, 256, 0, s>>>(c) : expand_kernel<false, MK_BF16><<<g2, 256, 0, s>>>(c);
        else
            f16 ? expand_kernel<true, MK_F16><<<g2, 256, 0, s>>>(c) : expand_kernel<false, MK_F16><<<g2, 256, 0, s>>>(c);
    }
    MK_LAUNCH_CHECK("lora_rows");
    return MK_OK;
}

} // extern "C"
