// mk_rope_rows: per-head RMS norm and rotary positions of several axes on the query and key heads of packed rows.
#include "common.hpp"

#include <cmath>

namespace mk {

namespace {

constexpr uint32_t kMaxPairs = 64;

// What the kernel knows of a pair: the turns that a position adds, as a fraction of 2^64, and its axis.
struct RopeP {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t ldq, ldk, ldqo, ldko, pos_ld;
    const float *norm_q, *norm_k;
    const void* pos;
    uint32_t rows, heads, kv_heads, d, pairs;
    float eps, k_scale;
    uint64_t turn[kMaxPairs];
    uint8_t axis[kMaxPairs];
};

template <uint32_t T> __device__ inline f32x4 load4(const void* p, int64_t at)
{
    if constexpr (T == MK_F32) {
        return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + at);
        f32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t h = uint16_t(v[i / 2] >> (16 * (i % 2)));
            r[i] = T == MK_BF16 ? bf2f_bits(h) : h2f_bits(h);
        }
        return r;
    }
}
template <uint32_t T> __device__ inline void store4(void* p, int64_t at, const f32x4& v)
{
    if constexpr (T == MK_F32)
        __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(static_cast<float*>(p) + at));
    else
        __builtin_nontemporal_store(u32x2{pack_x2(v[0], v[1], T == MK_F16), pack_x2(v[2], v[3], T == MK_F16)}, reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + at));
}

// The fraction of a turn, in 2^-32: an int32 position times the pair's fraction modulo 2^64 is exact; an fp32 one goes through
// a double, whose 53 bits hold the product's turns.
__device__ inline uint32_t turns_of(int32_t pos, uint64_t turn) { return uint32_t((uint64_t(int64_t(pos)) * turn) >> 32); }
__device__ inline uint32_t turns_of(float pos, uint64_t turn)
{
    const double t = double(pos) * (double(turn) * 0x1p-64);
    return uint32_t(int64_t(rint((t - rint(t)) * 0x1p32)));
}
// cos and sin of that fraction: the nearest quarter turn off in integers, Taylor series up to an eighth of a turn either way
// (|x| <= pi / 4: the first terms left out are x^11 / 11! < 1.8e-9 and x^12 / 12! < 1.2e-10, below fp32's rounding).
__device__ inline void cos_sin(uint32_t turns, float& c, float& s)
{
    const uint32_t quarter = (turns + 0x20000000u) >> 30;
    const float x = float(int32_t(turns - (quarter << 30))) * 1.4629180792671596e-9f, z = x * x; // 2 pi / 2^32
    const float sx = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float cx = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const float a = quarter & 1 ? sx : cx, b = quarter & 1 ? cx : sx;
    c = (quarter + 1) & 2 ? -a : a;
    s = quarter & 2 ? -b : b;
}

// A lane holds 8 values of a head as two groups of 4: pairs 4 l .. 4 l + 3, with their partners R / 2 further (mode 1) or next
// to them (mode 2), or 8 values that are not turned. So d / 8 lanes share a head, a wave holds 64 / (d / 8) heads of one row,
// IT times: the row's cosines and sines are made once a lane for all of them. Bound by memory: every value is read and
// written once (32760 rows of 64 heads of 128 from fp32 to bf16 290 us, 5.6 TB/s; 1333 of 40 of 64 in half 5.9 on the device).
// Stored non-temporally, which leaves the projection's rows, still to be read, their place in the caches (16384 bf16 rows of 64 heads
// 136 -> 110 us, 4352 38 -> 33; attention behind it takes the same time).
template <uint32_t IN, uint32_t OUT, typename POS, int MODE, int IT> __global__ __launch_bounds__(256) void rope_kernel(RopeP p)
{
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= p.rows)
        return;
    const uint32_t per = p.d / 8, l = lane & (per - 1), turned = p.pairs / 4; // lanes of a head that turn pairs
    const uint32_t wave_heads = 64 / per, h0 = blockIdx.y * wave_heads * IT + lane / per, all = p.heads + p.kv_heads;
    const uint32_t o0 = l < turned ? (MODE == 1 ? 4 * l : 8 * l) : 8 * l;
    const uint32_t o1 = l < turned && MODE == 1 ? o0 + p.pairs : o0 + 4;

    f32x4 a[IT], b[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const uint32_t h = h0 + i * wave_heads;
        if (h < all) {
            const bool is_k = h >= p.heads;
            const void* x = is_k ? p.k : p.q;
            const int64_t at = int64_t(row) * (is_k ? p.ldk : p.ldq) + int64_t(is_k ? h - p.heads : h) * p.d;
            a[i] = load4<IN>(x, at + o0);
            b[i] = load4<IN>(x, at + o1);
        } else {
            a[i] = b[i] = f32x4{};
        }
    }
    float c[4], s[4];
    if (l < turned) {
        const POS* pos = static_cast<const POS*>(p.pos) + int64_t(row) * p.pos_ld;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const POS v = pos[p.axis[4 * l + j]];
            cos_sin(turns_of(v, p.turn[4 * l + j]), c[j], s[j]);
            if (__builtin_isinf(float(v)) || __builtin_isnan(float(v)))
                c[j] = s[j] = __builtin_nanf("");
        }
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const uint32_t h = h0 + i * wave_heads;
        const bool is_k = h >= p.heads;
        const float* w = is_k ? p.norm_k : p.norm_q;
        f32x4 u = a[i], v = b[i];
        // (all lanes add, those past the last head too: the sums cross lanes)
        float sq = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sq += u[j] * u[j] + v[j] * v[j];
        sq = oct_sum(sq);
#if defined(__HIP_DEVICE_COMPILE__)
        if (p.d == 128)
            sq += dpp_f<0x140>(sq); // row_mirror: the other 8 lanes of the head's 16
#endif
        if (h >= all)
            continue;
        if (w) {
            const float inv = rsqrtf(sq / float(p.d) + p.eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] *= inv * w[o0 + j];
                v[j] *= inv * w[o1 + j];
            }
        }
        if (l < turned) {
            if constexpr (MODE == 1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = u[j], y = v[j];
                    u[j] = x * c[j] - y * s[j];
                    v[j] = x * s[j] + y * c[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = u[2 * j], y = u[2 * j + 1];
                    u[2 * j] = x * c[j] - y * s[j];
                    u[2 * j + 1] = x * s[j] + y * c[j];
                    x = v[2 * j], y = v[2 * j + 1];
                    v[2 * j] = x * c[2 + j] - y * s[2 + j];
                    v[2 * j + 1] = x * s[2 + j] + y * c[2 + j];
                }
            }
        }
        if (is_k) {
            u *= p.k_scale;
            v *= p.k_scale;
        }
        void* out = is_k ? p.k_out : p.q_out;
        const int64_t at = int64_t(row) * (is_k ? p.ldko : p.ldqo) + int64_t(is_k ? h - p.heads : h) * p.d;
        store4<OUT>(out, at + o0, u);
        store4<OUT>(out, at + o1, v);
    }
}

template <uint32_t IN, uint32_t OUT, typename POS, int MODE> void launch_it(const RopeP& p, hipStream_t s)
{
    const uint32_t wave_heads = 64 / (p.d / 8), steps = cdiv(p.heads + p.kv_heads, wave_heads);
    // us with 4 steps a wave / with 1, heads of 128: 64 rows of 40 heads 5.2 / 3.7, 512 of 40 5.7 / 5.5; 1024 of 64 9.2 / 11.0, 4352 of
    // 10 8.1 / 8.8, 16384 of 64 109 / 132 (a wave's sines serve four times the heads)
    if (uint64_t(p.rows) * (p.heads + p.kv_heads) * p.d >= 1u << 22)
        rope_kernel<IN, OUT, POS, MODE, 4><<<dim3(cdiv(p.rows, 4), cdiv(steps, 4)), 256, 0, s>>>(p);
    else
        rope_kernel<IN, OUT, POS, MODE, 1><<<dim3(cdiv(p.rows, 4), steps), 256, 0, s>>>(p);
}
template <uint32_t IN, uint32_t OUT> void launch_mode(const RopeP& p, bool f32_pos, uint32_t mode, hipStream_t s)
{
    if (mode == 1)
        f32_pos ? launch_it<IN, OUT, float, 1>(p, s) : launch_it<IN, OUT, int32_t, 1>(p, s);
    else
        f32_pos ? launch_it<IN, OUT, float, 2>(p, s) : launch_it<IN, OUT, int32_t, 2>(p, s);
}
template <uint32_t IN> void launch_out(const RopeP& p, uint32_t out, bool f32_pos, uint32_t mode, hipStream_t s)
{
    if (out == MK_F32)
        launch_mode<IN, MK_F32>(p, f32_pos, mode, s);
    else if (out == MK_BF16)
        launch_mode<IN, MK_BF16>(p, f32_pos, mode, s);
    else
        launch_mode<IN, MK_F16>(p, f32_pos, mode, s);
}

int64_t size_of(uint32_t t) { return t == MK_F32 ? 4 : 2; }
bool float_type(uint32_t t) { return t == MK_F32 || t == MK_BF16 || t == MK_F16; }

} // namespace

} // namespace mk

using namespace mk;

extern "C" mk_status mk_rope_rows(const mk_rope_rows_args* a, void* stream)
{
    if (!a)
        return fail(MK_ERR_ARG, "rope_rows: null argument");
    if (a->rows && (!a->q || !a->q_out || !a->pos))
        return fail(MK_ERR_ARG, "rope_rows: null argument (q, q_out and pos are required)");
    if (a->rows && (!!a->k != !!a->k_out || !!a->k != !!a->kv_heads))
        return fail(MK_ERR_ARG, "rope_rows: k, k_out and kv_heads come together");
    if (!a->heads || a->heads > 65535 || a->kv_heads > 65535 || (a->d != 64 && a->d != 128))
        return fail(MK_ERR_ARG, "rope_rows: 1 to 65535 heads of dim 64 or 128");
    if (!float_type(a->dtype) || !float_type(a->out_dtype))
        return fail(MK_ERR_ARG, "rope_rows: dtype and out_dtype must be f32, bf16 or f16");
    if (a->pos_dtype != MK_I32 && a->pos_dtype != MK_F32)
        return fail(MK_ERR_ARG, "rope_rows: positions must be i32 or f32");
    if (a->axes < 1 || a->axes > 4)
        return fail(MK_ERR_ARG, "rope_rows: 1 to 4 axes");
    uint64_t turned = 0;
    for (uint32_t i = 0; i < a->axes; ++i) {
        if (!a->axis_dims[i] || a->axis_dims[i] % 2)
            return fail(MK_ERR_ARG, "rope_rows: axis_dims must be multiples of 2");
        turned += a->axis_dims[i];
    }
    if (turned % 8 || turned > a->d)
        return fail(MK_ERR_ARG, "rope_rows: the sum of axis_dims must be a multiple of 8, at most d");
    if (!(a->theta >= 1.0) || std::isinf(a->theta))
        return fail(MK_ERR_ARG, "rope_rows: theta must be finite, at least 1");
    if (a->series > MK_ROPE_SHARED || (a->rope_mode != 1 && a->rope_mode != 2))
        return fail(MK_ERR_ARG, "rope_rows: series OWN or SHARED, rope_mode 1 or 2");
    const int64_t nq = int64_t(a->heads) * a->d, nk = int64_t(a->kv_heads) * a->d;
    auto bad = [](int64_t ld, int64_t n) { return ld < n || ld % 4; };
    if (bad(a->ldq, nq) || bad(a->ldqo, nq) || (a->k && (bad(a->ldk, nk) || bad(a->ldko, nk))))
        return fail(MK_ERR_ARG, "rope_rows: rows must hold their heads and start at multiples of 4 elements");
    if (a->pos_ld && a->pos_ld < int64_t(a->axes))
        return fail(MK_ERR_ARG, "rope_rows: pos_ld must be 0 or at least axes");
    const uintptr_t in = a->dtype == MK_F32 ? 16 : 8, out = a->out_dtype == MK_F32 ? 16 : 8;
    if (!aligned(a->q, in) || !aligned(a->k, in) || !aligned(a->q_out, out) || !aligned(a->k_out, out) || !aligned(a->pos, 4) ||
        !aligned(a->norm_q, 4) || !aligned(a->norm_k, 4))
        return fail(MK_ERR_ARG, "rope_rows: q, k and their outputs must be aligned for 4 elements, the rest for one");
    if ((a->q && a->q == a->q_out && (a->dtype != a->out_dtype || a->ldq != a->ldqo)) ||
        (a->k && a->k == a->k_out && (a->dtype != a->out_dtype || a->ldk != a->ldko)))
        return fail(MK_ERR_ARG, "rope_rows: in place needs equal types and strides");
    if (!a->rows)
        return MK_OK;
    if (a->rows > 0x7fffffffu)
        return fail(MK_ERR_ARG, "rope_rows: more than 2^31 - 1 rows");
    RopeP p{a->q, a->k, a->q_out, a->k_out, a->ldq, a->ldk, a->ldqo, a->ldko, a->pos_ld, a->norm_q, a->norm_k, a->pos,
            a->rows, a->heads, a->kv_heads, a->d, uint32_t(turned / 2), a->eps, a->k_scale == 0.0f ? 1.0f : a->k_scale, {}, {}};
    // theta^(-2 j / dim) radians as turns of 2^64, in extended doubles: a power for every 16th pair (150 ns each), products
    // between them, so an error below 2^-59, 2^-30 of a turn at the largest positions
    const bool own = a->series == MK_ROPE_OWN;
    const long double theta = a->theta, unit = 18446744073709551616.0L / 6.283185307179586476925286766559L;
    long double f = 0.0L, ratio = 0.0L;
    uint32_t pair = 0;
    for (uint32_t i = 0; i < a->axes; ++i)
        for (uint32_t j = 0; j < a->axis_dims[i] / 2; ++j, ++pair) {
            const uint32_t at = own ? j : pair;
            const long double dim = own ? a->axis_dims[i] : uint32_t(turned);
            if (at == 0)
                ratio = powl(theta, -2.0L / dim);
            f = at % 16 ? f * ratio : powl(theta, -2.0L * at / dim) * unit;
            p.turn[pair] = uint64_t(f);
            p.axis[pair] = uint8_t(i);
        }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32_pos = a->pos_dtype == MK_F32;
    // a grid dimension holds fewer than 2^32 threads: at most 2^24 rows (2^30 threads) a launch
    constexpr uint32_t kMost = 1u << 24;
    auto rows_on = [](const void* x, int64_t bytes) { return x ? static_cast<const char*>(x) + bytes : nullptr; };
    for (uint32_t r0 = 0; r0 < a->rows; r0 += kMost) {
        p.rows = a->rows - r0 < kMost ? a->rows - r0 : kMost;
        p.q = rows_on(a->q, int64_t(r0) * a->ldq * size_of(a->dtype));
        p.k = rows_on(a->k, int64_t(r0) * a->ldk * size_of(a->dtype));
        p.q_out = const_cast<char*>(rows_on(a->q_out, int64_t(r0) * a->ldqo * size_of(a->out_dtype)));
        p.k_out = const_cast<char*>(rows_on(a->k_out, int64_t(r0) * a->ldko * size_of(a->out_dtype)));
        p.pos = rows_on(a->pos, int64_t(r0) * a->pos_ld * 4);
        if (a->dtype == MK_F32)
            launch_out<MK_F32>(p, a->out_dtype, f32_pos, a->rope_mode, s);
        else if (a->dtype == MK_BF16)
            launch_out<MK_BF16>(p, a->out_dtype, f32_pos, a->rope_mode, s);
        else
            launch_out<MK_F16>(p, a->out_dtype, f32_pos, a->rope_mode, s);
    }
    MK_LAUNCH_CHECK("rope_rows");
    return MK_OK;
}
