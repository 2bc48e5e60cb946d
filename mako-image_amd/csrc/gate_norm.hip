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

// f(std::integral_constant<uint32_t, t>{}) for the float type t: one branch around code specialised for each
template <class F> __device__ inline void with_type(uint32_t t, F&& f)
{
    if (t == MK_BF16)
        f(std::integral_constant<uint32_t, MK_BF16>{});
    else if (t == MK_F16)
        f(std::integral_constant<uint32_t, MK_F16>{});
    else
        f(std::integral_constant<uint32_t, MK_F32>{});
}
template <uint32_t T> __device__ inline float widen(uint16_t h) { return T == MK_BF16 ? bf2f_bits(h) : h2f_bits(h); }
// 4 elements of type T as floats
template <uint32_t T> __device__ inline f32x4 load4(const void* p, uint64_t at)
{
    if constexpr (T == MK_F32) {
        return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + at);
        return f32x4{widen<T>(uint16_t(v[0])), widen<T>(uint16_t(v[0] >> 16)), widen<T>(uint16_t(v[1])),
                     widen<T>(uint16_t(v[1] >> 16))};
    }
}
template <uint32_t T> __device__ inline float load1(const void* p, uint64_t at)
{
    if constexpr (T == MK_F32)
        return static_cast<const float*>(p)[at];
    else
        return widen<T>(static_cast<const uint16_t*>(p)[at]);
}

__device__ inline uint32_t wave_max_bits(uint32_t v)
{
#if defined(__HIP_DEVICE_COMPILE__)
    // the VALU ladder of wave_reduce, on the bits
    return __builtin_bit_cast(uint32_t, wave_reduce(__builtin_bit_cast(float, v), [](float a, float b) {
                                  return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, a),
                                                                       __builtin_bit_cast(uint32_t, b)));
                              }));
#else
    return v;
#endif
}

// Workgroups in two grid dimensions: one holds fewer than 2^32 threads.
dim3 grid_of(uint32_t groups)
{
    constexpr uint32_t kMost = 1u << 21; // of up to 1024 threads
    return groups <= kMost ? dim3(groups) : dim3(kMost, cdiv(groups, kMost));
}
// The row of a wave (W = 1: four rows a workgroup) or of a workgroup; past the last one in the last workgroups. (At most
// 2^31 - 1 rows: no overflow.)
template <int W> __device__ inline uint32_t row_of()
{
    const uint32_t group = blockIdx.y * gridDim.x + blockIdx.x;
    return W == 1 ? group * 4 + (threadIdx.x >> 6) : group;
}

// Reductions over the W waves of a row, every thread gets the result. Each reduction of a kernel has a slot of its own in
// LDS, so it takes one barrier; the waves' sums are added in their order.
template <int W> struct RowRed {
    float* slots; // W floats a reduction
    __device__ float sum(float v, int i)
    {
        v = wave_sum(v);
        if constexpr (W > 1) {
            float* s = slots + i * W;
            if ((threadIdx.x & 63) == 0)
                s[threadIdx.x >> 6] = v;
            __syncthreads();
            v = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w)
                v += s[w];
        }
        return v;
    }
    __device__ uint32_t max_bits(uint32_t v, int i)
    {
        v = wave_max_bits(v);
        if constexpr (W > 1) {
            uint32_t* s = reinterpret_cast<uint32_t*>(slots + i * W);
            if ((threadIdx.x & 63) == 0)
                s[threadIdx.x >> 6] = v;
            __syncthreads();
            v = 0;
#pragma unroll
            for (int w = 0; w < W; ++w)
                v = max(v, s[w]);
        }
        return v;
    }
};

__device__ inline f32x4 vec4(const float* p, int64_t at, float none)
{
    return p ? *reinterpret_cast<const f32x4*>(p + at) : f32x4{none, none, none, none};
}

// The thread's NV float4s of a vector (`none` without one, zeros past its end)
template <int W, int NV>
__device__ inline void load_vec(f32x4 (&o)[NV], const float* p, int64_t at, uint32_t c0, uint32_t nv, float none)
{
    if (p) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            o[i] = c0 + 64 * W * i < nv ? *reinterpret_cast<const f32x4*>(p + at + 4 * (c0 + 64 * W * i)) : f32x4{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            o[i] = f32x4{none, none, none, none};
    }
}

// A row's norm in registers: each thread holds NV float4s, c = first + 64 W i of the row's nv (zeros past its end).
template <int W, int NV>
__device__ inline void norm_row(f32x4 (&v)[NV], uint32_t c0, uint32_t nv, uint32_t n, uint32_t kind, const float* w,
                                const float* b, float eps, RowRed<W>& red, int slot)
{
    if (kind == MK_NORM_NONE)
        return;
    float mean = 0.0f, s = 0.0f;
    if (kind == MK_NORM_LAYER) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            s += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        mean = red.sum(s, slot) / float(n);
    }
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (c0 + 64 * W * i < nv) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[i][e] -= mean;
                s = fmaf(v[i][e], v[i][e], s);
            }
        }
    const float inv = rsqrtf(red.sum(s, slot + 1) / float(n) + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = c0 + 64 * W * i;
        if (c < nv) {
            const f32x4 ww = vec4(w, 4 * int64_t(c), 1.0f), bb = vec4(b, 4 * int64_t(c), 0.0f);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[i][e] = fmaf(v[i][e] * inv, ww[e], bb[e]);
        }
    }
}

// mk_gate_norm, one pass: the row of x and y in registers (W waves a row, NV float4s a thread; W = 1: four rows a workgroup),
// the statistics two-pass over them (the mean first, then the squares about it: a variance far below the mean's square keeps
// its digits). Bound by HBM: 8 bytes of residual, 2 of y and 2 (int8: 1) of out an element. Measured with three sets of
// buffers in turn: 4352 x 4096 38.3 us (5.6 TB/s), 32768 x 4096 294 us (5.5), 32768 x 1280 88 us (5.7), to int8 4352 x
// 4096 37.5 us; a copy runs at 5.0. The residual's nontemporal loads and stores are worth 47 -> 38 us of the first; y is the
// last product's output and out the next one's input, which the caches may hold. Loading the vectors (w, scale, shift) with
// the row costs the registers of half the waves: 47 -> 53 us.
template <int W, int NV>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void gate_norm_kernel(mk_gate_norm_args g)
{
    __shared__ float slots[5 * W];
    RowRed<W> red{slots};
    const uint32_t r = row_of<W>();
    if (r >= g.rows)
        return;
    const uint32_t nv = g.n / 4, c0 = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const uint32_t seg = r / g.seg_rows, at = r - seg * g.seg_rows;
    const int64_t mod = int64_t(seg) * g.mod_stride + (at < g.split ? g.alt : 0);
    const float* x = g.x + uint64_t(r) * g.ldx;
    f32x4 v[NV], xv[NV], gt[NV];
    if (g.y)
        with_type(g.y_dtype, [&](auto t) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t c = c0 + 64 * W * i;
                v[i] = c < nv ? load4<decltype(t)::value>(g.y, uint64_t(r) * g.ldy + 4 * c) : f32x4{0, 0, 0, 0};
            }
        });
    // the residual is not used again before the next block's end: its loads and stores pass the caches by
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = c0 + 64 * W * i;
        xv[i] = c < nv ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(x + 4 * c)) : f32x4{0, 0, 0, 0};
    }
    if (g.y) {
        load_vec<W, NV>(gt, g.gate, mod, c0, nv, 1.0f);
        norm_row<W, NV>(v, c0, nv, g.n, g.norm1, g.w1, g.b1, g.eps1, red, 0);
        if (g.gate && g.tanh_gate)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    gt[i][e] = tanh_f(gt[i][e]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = c0 + 64 * W * i;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[i][e] = fmaf(gt[i][e], v[i][e], g.residual_scale * xv[i][e]);
            if (g.x_out && c < nv)
                __builtin_nontemporal_store(v[i], reinterpret_cast<f32x4*>(g.x_out + uint64_t(r) * g.ldx + 4 * c));
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            v[i] = xv[i];
    }
    if (!g.out)
        return;
    norm_row<W, NV>(v, c0, nv, g.n, g.norm2, g.w2, g.b2, g.eps2, red, 2);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = c0 + 64 * W * i;
        const f32x4 s = c < nv ? vec4(g.scale, mod + 4 * c, 0.0f) : f32x4{0, 0, 0, 0};
        const f32x4 h = c < nv ? vec4(g.shift, mod + 4 * c, 0.0f) : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[i][e] = fmaf(v[i][e], 1.0f + s[e], h[e]);
    }
    if (g.out_dtype == MK_I8) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (c0 + 64 * W * i < nv)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    m = max(m, abs_bits(v[i][e]));
        const Quant q = quant_of(red.max_bits(m, 4));
        int8_t* o = static_cast<int8_t*>(g.out) + uint64_t(r) * g.ldo;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (c0 + 64 * W * i < nv)
                *reinterpret_cast<uint32_t*>(o + 4 * (c0 + 64 * W * i)) = quant_pack(v[i], q);
        if (c0 == 0)
            g.out_scale[r] = q.scale;
        return;
    }
    with_type(g.out_dtype, [&](auto t) {
        constexpr uint32_t T = decltype(t)::value;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = c0 + 64 * W * i;
            if (c < nv) {
                const uint64_t o = uint64_t(r) * g.ldo + 4 * c;
                if constexpr (T == MK_F32)
                    *reinterpret_cast<f32x4*>(static_cast<float*>(g.out) + o) = v[i];
                else
                    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(g.out) + o) =
                        u32x2{pack_x2(v[i][0], v[i][1], T == MK_F16), pack_x2(v[i][2], v[i][3], T == MK_F16)};
            }
        }
    });
}

// NV .. MOST: the float4s a thread that the rows of W waves need
template <int W, int NV, int MOST> void launch_gate_norm(const mk_gate_norm_args& g, hipStream_t s)
{
    if constexpr (NV < MOST) {
        if (g.n > uint32_t(NV) * 256 * W)
            return launch_gate_norm<W, NV + 1, MOST>(g, s);
    }
    gate_norm_kernel<W, NV><<<grid_of(W == 1 ? cdiv(g.rows, 4) : g.rows), W == 1 ? 256 : 64 * W, 0, s>>>(g);
}

// mk_quantize_i8_rows: W waves a row, NV times 8 elements a thread, which stay in registers between the row's maximum and its
// codes. Bound by HBM: the source once, a byte an element back. Measured: 32768 x 4096 bf16 69 us (5.8 TB/s), f32 119 us
// (5.6), 4352 x 12288 bf16 30 us (5.3).
// 8 elements of T, as loaded
template <uint32_t T> struct Raw8 {
    u32x4 w[T == MK_F32 ? 2 : 1];
    __device__ f32x4 half(int h) const
    {
        if constexpr (T == MK_F32) {
            return __builtin_bit_cast(f32x4, w[h]);
        } else {
            const uint32_t a = w[0][2 * h], b = w[0][2 * h + 1];
            return f32x4{widen<T>(uint16_t(a)), widen<T>(uint16_t(a >> 16)), widen<T>(uint16_t(b)), widen<T>(uint16_t(b >> 16))};
        }
    }
};

template <uint32_t T, int W, int NV>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void quantize_i8_kernel(const void* src, uint32_t rows, uint32_t nv,
                                                                             int64_t ld, int8_t* dst, float* scale)
{
    __shared__ float slots[W];
    RowRed<W> red{slots};
    const uint32_t r = row_of<W>();
    if (r >= rows)
        return;
    const uint32_t c0 = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const char* s = static_cast<const char*>(src) + uint64_t(r) * ld * (T == MK_F32 ? 4 : 2);
    Raw8<T> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = c0 + 64 * W * i;
        v[i] = c < nv ? *reinterpret_cast<const Raw8<T>*>(s + uint64_t(c) * sizeof(Raw8<T>)) : Raw8<T>{};
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 f = v[i].half(h);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                m = max(m, abs_bits(f[e]));
        }
    const Quant q = quant_of(red.max_bits(m, 0));
    u32x2* d = reinterpret_cast<u32x2*>(dst + uint64_t(r) * nv * 8);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = c0 + 64 * W * i;
        if (c < nv)
            d[c] = u32x2{quant_pack(v[i].half(0), q), quant_pack(v[i].half(1), q)};
    }
    if (c0 == 0)
        scale[r] = q.scale;
}

// Rows of any width and alignment, read twice.
template <uint32_t T>
__global__ __launch_bounds__(256) void quantize_i8_any_kernel(const void* src, uint32_t rows, uint64_t cols,
                                                              int64_t ld, int8_t* dst, float* scale)
{
    __shared__ float slots[4];
    RowRed<4> red{slots};
    const uint64_t r = row_of<4>();
    if (r >= rows)
        return;
    uint32_t m = 0;
    for (uint64_t c = threadIdx.x; c < cols; c += 256)
        m = max(m, abs_bits(load1<T>(src, r * ld + c)));
    const Quant q = quant_of(red.max_bits(m, 0));
    for (uint64_t c = threadIdx.x; c < cols; c += 256)
        dst[r * cols + c] = q.inv == 0.0f ? int8_t(0) : int8_t(quant_code(load1<T>(src, r * ld + c), q));
    if (threadIdx.x == 0)
        scale[r] = q.scale;
}

// NV .. MOST: the turns of 8 elements a thread that the rows of W waves need
template <uint32_t T, int W, int NV, int MOST>
void launch_quantize(const void* src, uint32_t rows, uint32_t cols, int64_t ld, int8_t* dst, float* scale, hipStream_t s)
{
    if constexpr (NV < MOST) {
        if (cols > uint32_t(NV) * 512 * W)
            return launch_quantize<T, W, NV + 1, MOST>(src, rows, cols, ld, dst, scale, s);
    }
    quantize_i8_kernel<T, W, NV><<<grid_of(W == 1 ? cdiv(rows, 4) : rows), W == 1 ? 256 : 64 * W, 0, s>>>(
        src, rows, cols / 8, ld, dst, scale);
}
template <uint32_t T>
void quantize_rows(const void* src, uint32_t rows, uint64_t cols, int64_t ld, int8_t* dst, float* scale, bool vector,
                   hipStream_t s)
{
    if (!vector || cols > 65536) {
        quantize_i8_any_kernel<T><<<grid_of(rows), 256, 0, s>>>(src, rows, cols, ld, dst, scale);
        return;
    }
    // the fewest waves that hold the row in 24 elements a thread (4352 x 4096, 1 / 2 / 4 / 8 waves: 15.3 / 11.6 / 10.4 / 14.8
    // us; 4352 x 1280: 6.1 / 5.8 / 7.6 / 9.1; 4352 x 12288, 4 / 8 / 16: 32.9 / 30.7 / 30.0)
    const uint32_t n = uint32_t(cols), waves = cdiv(n, 1536);
    if (waves <= 1)
        launch_quantize<T, 1, 1, 3>(src, rows, n, ld, dst, scale, s);
    else if (waves <= 2)
        launch_quantize<T, 2, 2, 3>(src, rows, n, ld, dst, scale, s);
    else if (waves <= 4)
        launch_quantize<T, 4, 2, 3>(src, rows, n, ld, dst, scale, s);
    else if (waves <= 8)
        launch_quantize<T, 8, 2, 3>(src, rows, n, ld, dst, scale, s);
    else
        launch_quantize<T, 16, 2, 8>(src, rows, n, ld, dst, scale, s);
}

void launch_rows(const mk_gate_norm_args& g, hipStream_t s)
{
    // waves a row by its width alone, so that a row's sums, and its bits, do not depend on the rows beside it. More waves than
    // that wait at barriers (us on 1 / 2 / 4 / 8 / 16 waves: 32768 x 512 46 / 44 / 66, 32768 x 1280 - / 95 / 108 / 155, 10000 x
    // 2560 - / 65 / 62 / 69), fewer hold too few rows' loads in flight (32768 x 4096 - / - / 303 / 298 / 355, 9000 x 8192 - / - / - /
    // 171 / 179) and take longer over a single one (1 x 4096 - / - / 5.1 / 3.9 / 3.4).
    if (g.n <= 512)
        launch_gate_norm<1, 1, 2>(g, s);
    else if (g.n <= 1536)
        launch_gate_norm<2, 2, 3>(g, s);
    else if (g.n <= 3328)
        launch_gate_norm<4, 2, 4>(g, s);
    else if (g.n <= 8192)
        launch_gate_norm<8, 2, 4>(g, s);
    else
        launch_gate_norm<16, 3, 4>(g, s);
}

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
    hipStream_t s = static_cast<hipStream_t>(stream);
    launch_rows(g, s);
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
    // 16-byte loads and 8-byte stores: rows of a multiple of 16 elements, 16-byte aligned
    const bool vector = cols % 16 == 0 && aligned(src, 16) && aligned(dst, 8) && ld % (src_dtype == MK_F32 ? 4 : 8) == 0;
    int8_t* d = static_cast<int8_t*>(dst);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (src_dtype == MK_F32)
        quantize_rows<MK_F32>(src, uint32_t(rows), cols, ld, d, scale, vector, s);
    else if (src_dtype == MK_BF16)
        quantize_rows<MK_BF16>(src, uint32_t(rows), cols, ld, d, scale, vector, s);
    else
        quantize_rows<MK_F16>(src, uint32_t(rows), cols, ld, d, scale, vector, s);
    MK_LAUNCH_CHECK("quantize_i8_rows");
    return MK_OK;
}

} // extern "C"
