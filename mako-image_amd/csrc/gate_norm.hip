// The residual update, the norms around it and int8 row quantisation: mk_gate_norm, mk_quantize_i8_rows.
#include "common.hpp"

#include <cmath>
#include <string>
#include <type_traits>

namespace mk {

namespace {

constexpr uint32_t kMaxCols = 16384;

// ------------------------------------------------------------------------------------------------------------
// int8 codes: scale = a / 127 with a the row's largest magnitude, code = 127 v / a to the nearest integer, ties to even.
// ------------------------------------------------------------------------------------------------------------
struct Quant {
    float a, inv, scale; // inv = 127 / a; 0 for a row that counts as zero or holds an infinity or a NaN
};

// bits: the largest magnitude as its fp32 bits (an integer maximum, so that a NaN wins over an infinity over a number)
__device__ inline Quant quant_of(uint32_t bits)
{
    const float a = __builtin_bit_cast(float, bits);
    if (bits >= 0x7f800000u)
        return {0.0f, 0.0f, __builtin_nanf("")};
    if (a < 0x1p-100f)
        return {0.0f, 0.0f, 1.0f};
    return {a, 127.0f / a, a / 127.0f};
}

// 127 v / a rounded. The fp32 product is off by less than 2e-5 (|t| <= 127, two roundings), so it decides every value
// that is further than that from the middle between two codes; in the middle 254 v is compared with (2 lo + 1) a, both
// exact in 64 bits (24 and 8 bit factors).
__device__ inline int quant_code(float v, const Quant& q)
{
    const float t = v * q.inv;
    float r = rintf(t);
    if (fabsf(t - r) > 0.4999f) {
        const float lo = floorf(t);
        const double x = 254.0 * double(v), m = double(q.a) * (2.0 * double(lo) + 1.0);
        r = x < m ? lo : x > m ? lo + 1.0f : 2.0f * rintf(0.5f * lo + 0.25f);
    }
    return int(r);
}
__device__ inline uint32_t quant_pack(const f32x4& v, const Quant& q)
{
    if (q.inv == 0.0f)
        return 0;
    uint32_t o = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        o |= (uint32_t(quant_code(v[e], q)) & 255u) << (8 * e);
    return o;
}
__device__ inline uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

__device__ inline f32x4 load_row4(const void* p, uint64_t at, uint32_t dtype)
{
    if (dtype == MK_F32)
        return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + at);
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint16_t h = uint16_t(v[e >> 1] >> (16 * (e & 1)));
        o[e] = dtype == MK_BF16 ? bf2f_bits(h) : h2f_bits(h);
    }
    return o;
}

// Sum over a workgroup of 256, every thread gets it.
__device__ inline float block_sum(float v, float* red)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}
__device__ inline uint32_t block_max(uint32_t v, float* red)
{
    for (int m = 32; m; m >>= 1)
        v = max(v, uint32_t(__shfl_xor(int(v), m)));
    uint32_t* r = reinterpret_cast<uint32_t*>(red);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        r[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(r[0], r[1]), max(r[2], r[3]));
}

__device__ inline f32x4 vec4(const float* p, uint64_t at, float none)
{
    return p ? *reinterpret_cast<const f32x4*>(p + at) : f32x4{none, none, none, none};
}

// The row in LDS, normed in place: each thread owns the float4s threadIdx.x + 256 i.
__device__ inline void norm_row(f32x4* row, uint32_t nv, uint32_t n, uint32_t kind, const float* w, const float* b,
                                float eps, float* red)
{
    if (kind == MK_NORM_NONE)
        return;
    float mean = 0.0f, s = 0.0f;
    if (kind == MK_NORM_LAYER) {
        for (uint32_t c = threadIdx.x; c < nv; c += 256)
            s += row[c][0] + row[c][1] + row[c][2] + row[c][3];
        mean = block_sum(s, red) / float(n);
    }
    s = 0.0f;
    for (uint32_t c = threadIdx.x; c < nv; c += 256)
        for (int e = 0; e < 4; ++e)
            s += (row[c][e] - mean) * (row[c][e] - mean);
    const float inv = rsqrtf(block_sum(s, red) / float(n) + eps);
    for (uint32_t c = threadIdx.x; c < nv; c += 256) {
        const f32x4 ww = vec4(w, 4 * c, 1.0f), bb = vec4(b, 4 * c, 0.0f);
        for (int e = 0; e < 4; ++e)
            row[c][e] = (row[c][e] - mean) * inv * ww[e] + bb[e];
    }
}

__global__ __launch_bounds__(256) void gate_norm_kernel(mk_gate_norm_args g)
{
    extern __shared__ f32x4 row[];
    __shared__ float red[4];
    const uint32_t r = blockIdx.x, nv = g.n / 4;
    const uint32_t seg = r / g.seg_rows, i = r - seg * g.seg_rows;
    const int64_t mod = int64_t(seg) * g.mod_stride + (i < g.split ? g.alt : 0);
    const f32x4* x = reinterpret_cast<const f32x4*>(g.x + uint64_t(r) * g.ldx);
    if (g.y) {
        for (uint32_t c = threadIdx.x; c < nv; c += 256)
            row[c] = load_row4(g.y, uint64_t(r) * g.ldy + 4 * c, g.y_dtype);
        norm_row(row, nv, g.n, g.norm1, g.w1, g.b1, g.eps1, red);
        for (uint32_t c = threadIdx.x; c < nv; c += 256) {
            const f32x4 gt = vec4(g.gate, mod + 4 * c, 1.0f), xv = x[c];
            f32x4 o;
            for (int e = 0; e < 4; ++e)
                o[e] = fmaf(g.gate && g.tanh_gate ? tanh_f(gt[e]) : gt[e], row[c][e], g.residual_scale * xv[e]);
            row[c] = o;
            if (g.x_out)
                reinterpret_cast<f32x4*>(g.x_out + uint64_t(r) * g.ldx)[c] = o;
        }
    } else {
        for (uint32_t c = threadIdx.x; c < nv; c += 256)
            row[c] = x[c];
    }
    if (!g.out)
        return;
    norm_row(row, nv, g.n, g.norm2, g.w2, g.b2, g.eps2, red);
    uint32_t m = 0;
    for (uint32_t c = threadIdx.x; c < nv; c += 256) {
        const f32x4 sc = vec4(g.scale, mod + 4 * c, 0.0f), sh = vec4(g.shift, mod + 4 * c, 0.0f);
        f32x4 h = row[c];
        for (int e = 0; e < 4; ++e) {
            h[e] = fmaf(h[e], 1.0f + sc[e], sh[e]);
            m = max(m, abs_bits(h[e]));
        }
        const uint64_t at = uint64_t(r) * g.ldo + 4 * c;
        row[c] = h;
        if (g.out_dtype == MK_F32)
            *reinterpret_cast<f32x4*>(static_cast<float*>(g.out) + at) = h;
        else if (g.out_dtype != MK_I8)
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(g.out) + at) =
                u32x2{pack_x2(h[0], h[1], g.out_dtype == MK_F16), pack_x2(h[2], h[3], g.out_dtype == MK_F16)};
    }
    if (g.out_dtype != MK_I8)
        return;
    const Quant q = quant_of(block_max(m, red));
    for (uint32_t c = threadIdx.x; c < nv; c += 256)
        *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(g.out) + uint64_t(r) * g.ldo + 4 * c) = quant_pack(row[c], q);
    if (threadIdx.x == 0)
        g.out_scale[r] = q.scale;
}

__device__ inline float load1(const void* p, uint64_t at, uint32_t dtype)
{
    if (dtype == MK_F32)
        return static_cast<const float*>(p)[at];
    const uint16_t h = static_cast<const uint16_t*>(p)[at];
    return dtype == MK_BF16 ? bf2f_bits(h) : h2f_bits(h);
}

__global__ __launch_bounds__(256) void quantize_i8_kernel(const void* src, uint32_t dtype, uint64_t cols, int64_t ld,
                                                          int8_t* dst, float* scale)
{
    __shared__ float red[4];
    const uint64_t r = blockIdx.x;
    uint32_t m = 0;
    for (uint64_t c = threadIdx.x; c < cols; c += 256)
        m = max(m, abs_bits(load1(src, r * ld + c, dtype)));
    const Quant q = quant_of(block_max(m, red));
    for (uint64_t c = threadIdx.x; c < cols; c += 256)
        dst[r * cols + c] = q.inv == 0.0f ? int8_t(0) : int8_t(quant_code(load1(src, r * ld + c, dtype), q));
    if (threadIdx.x == 0)
        scale[r] = q.scale;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool float_type(uint32_t t) { return t == MK_F32 || t == MK_BF16 || t == MK_F16; }

} // namespace

} // namespace mk

using namespace mk;

extern "C" {

mk_status mk_gate_norm(const mk_gate_norm_args* a, void* stream)
{
    if (!a || !a->x || (!a->y && !a->out))
        return fail(MK_ERR_ARG, "gate_norm: null argument (x and y or out are required)");
    if (!a->n || a->n % 4 || a->n > kMaxCols)
        return fail(MK_ERR_ARG, "gate_norm: n must be a multiple of 4 up to 16384");
    if (a->norm1 > MK_NORM_LAYER || a->norm2 > MK_NORM_LAYER || (a->b1 && a->norm1 != MK_NORM_LAYER) ||
        (a->b2 && a->norm2 != MK_NORM_LAYER) || (a->w1 && !a->norm1) || (a->w2 && !a->norm2))
        return fail(MK_ERR_ARG, "gate_norm: norms are NONE, RMS (w) or LAYER (w, b)");
    if (!a->y && (a->norm1 || a->gate || a->x_out || (a->residual_scale != 0.0f && a->residual_scale != 1.0f)))
        return fail(MK_ERR_ARG, "gate_norm: norm1, gate, residual_scale and x_out need y");
    if (!a->out && (a->norm2 || a->scale || a->shift))
        return fail(MK_ERR_ARG, "gate_norm: norm2, scale and shift need out");
    if (!a->out && !a->x_out)
        return fail(MK_ERR_ARG, "gate_norm: no output");
    if ((a->y && !float_type(a->y_dtype)) || (a->out && !float_type(a->out_dtype) && a->out_dtype != MK_I8))
        return fail(MK_ERR_ARG, "gate_norm: y must be f32, bf16 or f16, out one of them or int8");
    if (a->out && a->out_dtype == MK_I8 && !a->out_scale)
        return fail(MK_ERR_ARG, "gate_norm: int8 rows need out_scale");
    const int64_t n = a->n;
    if (a->ldx < n || a->ldx % 4 || (a->y && (a->ldy < n || a->ldy % 4)) || (a->out && (a->ldo < n || a->ldo % 4)))
        return fail(MK_ERR_ARG, "gate_norm: ldx, ldy and ldo must be multiples of 4, at least n");
    const bool mod = a->gate || a->scale || a->shift;
    if (mod && (a->alt % 4 || a->mod_stride % 4))
        return fail(MK_ERR_ARG, "gate_norm: alt and mod_stride must be multiples of 4");
    auto size = [](uint32_t t) -> uintptr_t { return t == MK_F32 ? 16 : t == MK_I8 ? 4 : 8; };
    if (!aligned(a->x, 16) || !aligned(a->x_out, 16) || !aligned(a->w1, 16) || !aligned(a->b1, 16) ||
        !aligned(a->w2, 16) || !aligned(a->b2, 16) || !aligned(a->gate, 16) || !aligned(a->scale, 16) ||
        !aligned(a->shift, 16) || (a->y && !aligned(a->y, size(a->y_dtype))) ||
        (a->out && !aligned(a->out, size(a->out_dtype))) || !aligned(a->out_scale, 4))
        return fail(MK_ERR_ARG, "gate_norm: x, x_out and the vectors must be 16-byte aligned, y and out for 4 elements");
    if (!a->rows)
        return MK_OK;
    if (a->rows > 0x7fffffffu)
        return fail(MK_ERR_ARG, "gate_norm: more than 2^31 - 1 rows");
    mk_gate_norm_args g = *a;
    if (!g.seg_rows)
        g.seg_rows = 0xffffffffu;
    if (g.residual_scale == 0.0f)
        g.residual_scale = 1.0f;
    gate_norm_kernel<<<g.rows, 256, g.n * sizeof(float), static_cast<hipStream_t>(stream)>>>(g);
    MK_LAUNCH_CHECK("gate_norm");
    return MK_OK;
}

mk_status mk_quantize_i8_rows(const void* src, uint32_t src_dtype, uint64_t rows, uint64_t cols, int64_t ld, void* dst,
                              float* scale, void* stream)
{
    if (!src || !dst || !scale)
        return fail(MK_ERR_ARG, "quantize_i8_rows: null pointer");
    if (!float_type(src_dtype))
        return fail(MK_ERR_ARG, "quantize_i8_rows: src must be f32, bf16 or f16");
    if (!cols || ld < 0 || uint64_t(ld) < cols || rows > 0x7fffffffu)
        return fail(MK_ERR_ARG, "quantize_i8_rows: cols must be at least 1, ld at least cols, rows below 2^31");
    if (!aligned(src, src_dtype == MK_F32 ? 4 : 2) || !aligned(scale, 4))
        return fail(MK_ERR_ARG, "quantize_i8_rows: src and scale must be aligned for an element");
    if (!rows)
        return MK_OK;
    quantize_i8_kernel<<<uint32_t(rows), 256, 0, static_cast<hipStream_t>(stream)>>>(src, src_dtype, cols, ld,
                                                                                    static_cast<int8_t*>(dst), scale);
    MK_LAUNCH_CHECK("quantize_i8_rows");
    return MK_OK;
}

} // extern "C"
