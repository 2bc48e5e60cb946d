// proj in 8-bit integers: C = epilogue(ascale[r] wscale[n] sum_k A[r][k] W[n][k] + bias[n]), int32 sums.
#include "common.hpp"

#include <string>
#include <type_traits>

namespace mk {

namespace {

struct I8P {
    const int8_t* a;
    const int8_t* w;
    const float* ascale;
    const float* wscale;
    const float* bias;
    const float* gate;
    void* c;
    int64_t lda, ldc, sa, sc, gate_alt;
    uint32_t M, N, K, batch;
    uint32_t split, seg_rows;
    uint32_t epi, c_dtype;
};

// The scaled sums of four channels: float(sum) ascale wscale + bias, the same expression everywhere, so a value does not
// depend on which kernel made it.
__device__ inline f32x4 i8_scaled(const int (&s)[4], float as, const f32x4& ws, const f32x4& b)
{
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[e] = fmaf(float(s[e]) * as, ws[e], b[e]);
    return v;
}

__device__ inline f32x4 load4(const float* p, uint32_t c, float none)
{
    return p ? *reinterpret_cast<const f32x4*>(p + c) : f32x4{none, none, none, none};
}

// A thread computes one token's four channels (with a gated unit, of both parts) straight from memory.
__global__ __launch_bounds__(256) void gemm_i8_plain_kernel(I8P p)
{
    const bool glu = p.epi == MK_EPI_SWIGLU || p.epi == MK_EPI_GEGLU;
    const uint32_t cols = glu ? p.N / 2 : p.N;
    const uint32_t r = blockIdx.x * 16 + threadIdx.x / 16, c = (blockIdx.y * 16 + threadIdx.x % 16) * 4, z = blockIdx.z;
    if (r >= p.M || c >= cols)
        return;
    const int8_t* a = p.a + int64_t(z) * p.sa + int64_t(r) * p.lda;
    const int8_t* w = p.w + uint64_t(c) * p.K;
    int s[2][4] = {};
    for (uint32_t k = 0; k < p.K; k += 16) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(a + k);
        for (int h = 0; h < (glu ? 2 : 1); ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u32x4 y = *reinterpret_cast<const u32x4*>(w + (uint64_t(h) * cols + e) * p.K + k);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[h][e] = __builtin_amdgcn_sdot4(int(x[i]), int(y[i]), s[h][e], false);
            }
    }
    const float as = p.ascale[uint64_t(z) * p.M + r];
    f32x4 v = i8_scaled(s[0], as, load4(p.wscale, c, 1.0f), load4(p.bias, c, 0.0f));
    if (glu) {
        const f32x4 g = i8_scaled(s[1], as, load4(p.wscale, cols + c, 1.0f), load4(p.bias, cols + c, 0.0f));
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = p.epi == MK_EPI_SWIGLU ? silu_f(v[e]) * g[e] : v[e] * (0.5f * g[e] * (1.0f + erf_fit(g[e] * 0.70710678f)));
    } else if (p.epi == MK_EPI_GELU_TANH || p.epi == MK_EPI_SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = p.epi == MK_EPI_SILU ? silu_f(v[e]) : gelu_tanh_f(v[e]);
    }
    const int64_t at = int64_t(z) * p.sc + int64_t(r) * p.ldc + c;
    if (p.epi == MK_EPI_GATE_ADD || p.epi == MK_EPI_GATE_TANH || p.epi == MK_EPI_ADD) {
        f32x4* x = reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + at);
        f32x4 o = *x;
        const f32x4 g = load4(p.gate, (r % p.seg_rows < p.split ? p.gate_alt : 0) + c, 1.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[e] = fmaf(p.epi == MK_EPI_ADD ? 1.0f : p.epi == MK_EPI_GATE_TANH ? tanh_f(g[e]) : g[e], v[e], o[e]);
        *x = o;
    } else if (p.c_dtype == MK_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + at) = v;
    } else {
        const bool h = p.c_dtype == MK_F16;
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.c) + at) = u32x2{pack_x2(v[0], v[1], h), pack_x2(v[2], v[3], h)};
    }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

} // namespace

} // namespace mk

using namespace mk;

extern "C" mk_status mk_gemm_i8(const mk_gemm_args* a, const float* ascale, void* stream)
{
    if (!a || !a->a || !a->w || !a->c || !a->wscale || !ascale)
        return fail(MK_ERR_ARG, "gemm_i8: null argument (A, W, C, ascale and wscale are required)");
    if (a->w_dtype != MK_I8)
        return fail(MK_ERR_ARG, "gemm_i8: w_dtype must be MK_I8");
    if (a->epilogue == MK_EPI_HEADS || a->epilogue == MK_EPI_PAIR_SUM)
        return fail(MK_ERR_UNSUPPORTED, "gemm_i8: no HEADS or PAIR_SUM epilogue");
    if (a->epilogue > MK_EPI_PAIR_SUM)
        return fail(MK_ERR_ARG, "gemm_i8: unknown epilogue");
    const bool glu = a->epilogue == MK_EPI_SWIGLU || a->epilogue == MK_EPI_GEGLU;
    const bool gated = a->epilogue == MK_EPI_GATE_ADD || a->epilogue == MK_EPI_GATE_TANH;
    const uint32_t nq = glu ? 8 : 4;
    if (!a->K || !a->N || a->K % 16 || a->N % nq || a->K > 131056)
        return fail(MK_ERR_ARG, "gemm_i8: K must be a multiple of 16 up to 131056 and N of " + std::to_string(nq) + " (K " +
                                    std::to_string(a->K) + ", N " + std::to_string(a->N) + ")");
    if (a->c_dtype != MK_F32 && a->c_dtype != MK_BF16 && a->c_dtype != MK_F16)
        return fail(MK_ERR_ARG, "gemm_i8: C must be f32, bf16 or f16");
    if ((gated || a->epilogue == MK_EPI_ADD) && a->c_dtype != MK_F32)
        return fail(MK_ERR_ARG, "gemm_i8: the residual epilogues take an f32 C");
    if (gated && !a->gate)
        return fail(MK_ERR_ARG, "gemm_i8: gated epilogue without a gate");
    const uint32_t cols = glu ? a->N / 2 : a->N;
    if (a->lda < a->K || a->lda % 16 || a->lda >= (1 << 23) || a->ldc < cols || a->ldc % 4 ||
        (a->batch > 1 && (a->stride_a % 16 || a->stride_c % 4)))
        return fail(MK_ERR_ARG, "gemm_i8: lda >= K and stride_a must be multiples of 16 (lda below 2^23), ldc >= the columns "
                                "of C and stride_c multiples of 4");
    if (!aligned(a->a, 16) || !aligned(a->w, 16) || !aligned(a->wscale, 16) || !aligned(a->bias, 16) ||
        !aligned(ascale, 4) || !aligned(a->c, a->c_dtype == MK_F32 ? 16 : 8) ||
        (gated && (!aligned(a->gate, 16) || a->gate_alt % 4)))
        return fail(MK_ERR_ARG, "gemm_i8: A, W, wscale, bias and gate must be 16-byte aligned, C for 4 elements, gate_alt a "
                                "multiple of 4");
    if (!a->M || !a->batch)
        return MK_OK;
    if (a->M > 0x7fffff00u || a->batch > 65535)
        return fail(MK_ERR_ARG, "gemm_i8: more than 2^31 - 256 rows or 65535 batch items");
    const I8P p{static_cast<const int8_t*>(a->a),
                static_cast<const int8_t*>(a->w),
                ascale,
                a->wscale,
                a->bias,
                gated ? a->gate : nullptr,
                a->c,
                a->lda,
                a->ldc,
                a->batch > 1 ? a->stride_a : 0,
                a->batch > 1 ? a->stride_c : 0,
                a->gate_alt,
                a->M,
                a->N,
                a->K,
                a->batch,
                a->split,
                a->seg_rows ? a->seg_rows : 0xffffffffu,
                a->epilogue,
                a->c_dtype};
    hipStream_t s = static_cast<hipStream_t>(stream);
    gemm_i8_plain_kernel<<<dim3(cdiv(p.M, 16), cdiv(cols, 64), p.batch), 256, 0, s>>>(p);
    MK_LAUNCH_CHECK("gemm_i8");
    return MK_OK;
}
