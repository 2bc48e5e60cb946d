// proj in 8-bit integers on gfx950: C = epilogue(ascale[r] wscale[n] sum_k A[r][k] W[n][k] + bias[n]), the sums exact in
// int32 (v_mfma_i32_16x16x64_i8), so their order, and with it the kernel that a launch takes, does not show in a result.
//
// What bounds it: up to 16 rows the weight's bytes (1 x 12288 x 4096: 9.5 us, 5.3 TB/s with a launch's own time); tens to
// hundreds of rows what a CU takes from its L2 (80 to 110 bytes a ns); over a short k the epilogue, and most of all the fp32
// residual's, 8 bytes an output with no product under them (4400 x 8192 x 2048 ADD 148 us, STORE 72); from about 2000 rows the
// matrix cores at the clock that lasting load leaves: 8192^3 415 us (2.65 POP/s) with them 69% busy at 1.83 GHz, some launches
// later 484 us (2.27), 75% at 1.44 GHz; 32768 x 12288 x 4096 1296 us (2.54), 64% at 1.89 GHz, and 1636 us (2.02), 73% at 1.32
// GHz (rocprofv3 counters, each time from the launch that was counted; no LDS bank conflicts in the 256 x 256 tiles). There
// neither the waves' priority nor fragments read further ahead changed the time, within 0.5%.
#include "common.hpp"

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>
#include <utility>

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

__device__ inline f32x4 load4(const float* p, uint32_t c, float none)
{
    return p ? *reinterpret_cast<const f32x4*>(p + c) : f32x4{none, none, none, none};
}

// Epilogue classes (template): a plain store, an activation, the fp32 residual, a gated unit.
enum { EC_STORE, EC_ACT, EC_RMW, EC_GLU };
constexpr int epi_class(uint32_t epi)
{
    return epi == MK_EPI_STORE                                 ? EC_STORE
           : epi == MK_EPI_GELU_TANH || epi == MK_EPI_SILU      ? EC_ACT
           : epi == MK_EPI_SWIGLU || epi == MK_EPI_GEGLU        ? EC_GLU
                                                                : EC_RMW;
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ inline i32x4 mfma_i8(const i32x4& w, const i32x4& a, const i32x4& c)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, a, c, 0, 0, 0);
#else
    return c;
#endif
}

// What a lane's four channels need: scales, bias, the gate rows (g1 for rows below the split; tanh applied).
struct Ch4 {
    f32x4 ws, b, g0, g1;
};
__device__ inline Ch4 channels4(const I8P& p, uint32_t c)
{
    Ch4 k;
    k.ws = *reinterpret_cast<const f32x4*>(p.wscale + c);
    k.b = load4(p.bias, c, 0.0f);
    k.g0 = load4(p.gate, c, 1.0f);
    k.g1 = p.gate && p.split ? *reinterpret_cast<const f32x4*>(p.gate + p.gate_alt + c) : k.g0;
    if (p.epi == MK_EPI_GATE_TANH)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k.g0[e] = tanh_f(k.g0[e]);
            k.g1[e] = tanh_f(k.g1[e]);
        }
    return k;
}
// sum * ascale (t) to the channel's value: one rounding for the product with wscale and the bias, everywhere
__device__ inline f32x4 scaled(const f32x4& t, const f32x4& ws, const f32x4& b)
{
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[e] = fmaf(t[e], ws[e], b[e]);
    return v;
}
template <bool GELU> __device__ inline f32x4 act4(const f32x4& v)
{
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        o[e] = GELU ? gelu_tanh_f(v[e]) : silu_f(v[e]);
    return o;
}
// g Phi(g), Phi the normal distribution: max(g, 0) - |g| Phi(-|g|). log2 Phi(-z) for z >= 0 is a polynomial of degree 8,
// fitted here by iterated least squares to Phi's own error on [0, 5.8] (Phi within 2.7e-7, z Phi(-z) within 8.5e-8, Phi(-z)
// to 8e-5 of itself up to z = 5.5); beyond, it falls faster than Phi does. In a tile's epilogue these instructions run
// alone: with erf_fit's longer series and its IEEE division 3952 x 10240 x 1280 GEGLU took 79 us, with a rational form (a
// reciprocal more) 68, so 66.
__device__ inline float gelu_erf_f(float g)
{
    const float z = fabsf(g);
    float q = fmaf(-5.577092e-07f, z, 9.50235062e-06f);
    q = fmaf(q, z, -3.01707514e-05f);
    q = fmaf(q, z, -0.0005522336f);
    q = fmaf(q, z, 0.0076639154f);
    q = fmaf(q, z, -0.052960813f);
    q = fmaf(q, z, -0.459032208f);
    q = fmaf(q, z, -1.15113127f);
    q = fmaf(q, z, -0.999999285f);
    // (the factor is bounded where Phi has long been 0: an infinite g gives g or 0, a NaN stays one by q)
    return fmaf(-fminf(z, 1e4f), __builtin_amdgcn_exp2f(q), fmaxf(g, 0.0f));
}
template <bool SWI> __device__ inline float glu1(float a, float g) { return SWI ? silu_f(a) * g : a * gelu_erf_f(g); }
__device__ inline f32x4 residual4(const I8P& p, uint32_t row, const f32x4& x, const f32x4& v, const Ch4& k)
{
    const f32x4 g = row % p.seg_rows < p.split ? k.g1 : k.g0;
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        o[e] = fmaf(g[e], v[e], x[e]);
    return o;
}
// f(std::bool_constant<flag>{}): one branch on a uniform flag around code specialised for each value
template <class F> __device__ inline void with_flag(bool flag, F&& f)
{
    if (flag)
        f(std::true_type{});
    else
        f(std::false_type{});
}

// ------------------------------------------------------------------------------------------------------------
// Tiles. The weight is the matrix cores' A operand (its rows are output channels), the activation the B operand, so a lane
// of v_mfma_i32_16x16x64_i8 holds 4 consecutive channels of one token. NW waves, 2 along the channels.
// ------------------------------------------------------------------------------------------------------------

// LDS rows are 128 bytes of k, 8 chunks of 16. A 16-byte read serves 16 lanes a cycle, here 16 consecutive rows at one
// chunk; rows r and r + 1 fall in opposite halves of the 64 banks, so the chunk is XOR-ed with (row >> 1) & 7.
__device__ inline int swz_chunk(int row, int kc) { return kc ^ ((row >> 1) & 7); }
__device__ inline int swz(int row, int kc) { return row * 128 + (swz_chunk(row, kc) << 4); }
// s_waitcnt immediate: vmcnt vm, lgkmcnt 0 (vmcnt's bits 3:0 and 15:14, expcnt not waited for)
constexpr int wait_vm(int vm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4); }

// Channels that a wave stages at a time in the epilogue, 16 tokens of them (64 at most, 4 KB; a gated unit writes half)
constexpr int epi_channels(int bn, bool glu)
{
    const int wo = glu ? bn / 4 : bn / 2;
    return wo < 64 ? wo : 64;
}
// LDS bytes of a tile: the stages; behind them, for a chain of tiles, the epilogue's staging, which else reuses them.
template <int BM, int BN, int NW, int NSTG, bool CHAIN> constexpr int tile_lds()
{
    return NSTG * (BM + BN) * 128 + (CHAIN ? NW * 16 * epi_channels(BN, false) * 4 : 0);
}

// f(std::integral_constant<int, 0>{}), f(1), ..
template <class F, int... I> __device__ __forceinline__ void for_each_int(F&& f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}

// Tiles of BM tokens x BN channels, `count` of them one after the other: at(i, z, m0, n0) gives the i-th's batch item, first
// token and first output channel. CHAIN: the last k steps of a tile load the first ones of the next, and the epilogue
// stages in LDS of its own, so that a workgroup's next tile starts where the last one ends.
template <int BM, int BN, int NW, int NSTG, int EC, bool CHAIN, class At>
__device__ __forceinline__ void i8_tiles(const I8P& p, int8_t* smem, uint32_t count, At at)
{
    constexpr bool GLU = EC == EC_GLU;
    constexpr int NT = 64 * NW, WM = BM / (NW / 2), WC = BN / 2, TB = WM / 16, CB = WC / 16;
    constexpr int RA = BM * 8 / NT, RW = BN * 8 / NT, ND = RA + RW; // direct loads a thread makes a k step
    static_assert((NSTG - 1) * ND <= 63 && (!CHAIN || NSTG == 2), "");
    int8_t(*sW)[BN * 128] = reinterpret_cast<int8_t(*)[BN * 128]>(smem);
    int8_t(*sA)[BM * 128] = reinterpret_cast<int8_t(*)[BM * 128]>(smem + NSTG * BN * 128);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave & 1, wm = wave >> 1;

    const int cols = int(GLU ? p.N / 2 : p.N);
    // GLU: the tile makes channels n0 .. n0 + BN / 2, a wave's rows are WC / 2 rows of the first part and the same
    // channels' rows of the second, so a lane's blocks cb and cb + CB / 2 are the two operands of one output.

    // The lane, as a value that the compiler does not know: what is derived from it is computed where it stands, not ahead of
    // the k loop, whose registers are all taken.
    auto here = [&]() __attribute__((always_inline)) {
        int l = lane;
        if (CHAIN)
            asm volatile("" : "+v"(l));
        return l;
    };
    // Direct loads: wave w's round i fills LDS chunks (i NW + w) 64 + lane; chunk P holds row P / 8 and k chunk
    // swz_chunk(row, P % 8). Buffer loads: the resource spans the tile's rows, the lane's byte offset selects row and
    // chunk, the k offset is a scalar; rows past the end read the last one. Chunks past K (in the last k steps) read out of
    // the resource's range, which gives zeros.
    static_assert(NW % 2 == 0, "a round's rows are a multiple of 16");
    const int kc = (lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7); // the lane's k chunk, the same in every round
    uint32_t z, oa[RA], ow[RW];
    int m0, n0;
    BufRes rsA, rsW0, rsW1;
    auto set = [&](uint32_t tile) __attribute__((always_inline)) {
        at(tile, z, m0, n0);
        const int lane = here();
        const int nr = min(cols - n0, GLU ? BN / 2 : BN), mr = min(int(p.M) - m0, BM);
        const int8_t* gW = p.w + uint64_t(n0) * p.K;
        rsA = buf_res(p.a + int64_t(z) * p.sa + int64_t(m0) * p.lda, uint32_t(int64_t(mr - 1) * p.lda + p.K));
        rsW0 = buf_res(gW, uint32_t(nr) * p.K);
        rsW1 = buf_res(GLU ? gW + uint64_t(cols) * p.K : gW, uint32_t(nr) * p.K);
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const int row = (i * NW + wave) * 8 + (lane >> 3);
            oa[i] = uint32_t(min(row, mr - 1)) * uint32_t(p.lda) + kc * 16;
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const int r = (i * NW + wave) * 8 + (lane >> 3);
            ow[i] = uint32_t(min(GLU ? (r / WC) * (WC / 2) + r % (WC / 2) : r, nr - 1)) * p.K + kc * 16;
        }
    };
    // direct load i (activation rounds first) of k step kt into stage buf; past: what leaves the range for the lanes whose
    // chunk lies past K
    auto dma1 = [&](int kt, uint32_t past, int buf, int i) __attribute__((always_inline)) {
        if (i < RA)
            buf_load_lds16(rsA, (lds_void*)&sA[buf][(i * NW + wave) * 1024], oa[i] + past, uint32_t(kt) * 128);
        else {
            const bool second = GLU && ((i - RA) * NW * 8 + wave * 8) % WC >= WC / 2;
            buf_load_lds16(second ? rsW1 : rsW0, (lds_void*)&sW[buf][((i - RA) * NW + wave) * 1024], ow[i - RA] + past,
                           uint32_t(kt) * 128);
        }
    };
    const int ke = int((p.K + 127) / 128); // a chain's is even: every tile starts in stage 0
    auto past = [&](int kt) { return kc * 16 >= int(p.K) - kt * 128 ? 0x80000000u : 0u; };

    i32x4 acc[CB][TB];
    // lane (r16, g4) supplies row r16 of a 16-row block and k bytes 16 g4 .. + 15 of a 64-deep substep, and holds channels
    // 4 g4 .. + 3 of token r16
    const int r16 = lane & 15, g4 = lane >> 4;
    // Two schedules. A small wave tile (at most 16 blocks) has too few products in a substep to cover the LDS's latency:
    // it reads a whole k step's fragments one step ahead (WIDE; two sets of registers). A large one reads a substep ahead.
    constexpr bool WIDE = CB * TB <= 16;
    static_assert(!WIDE || NSTG % 2 == 0, "a step's register set is its parity");
    i32x4 wf[CB], af0[TB], af1[TB];
    i32x4 fr[2][2][WIDE ? CB + TB : 1]; // [parity][substep][weight blocks, then token blocks]
    // (blocks are 16 rows apart, so the swizzle is the lane's: an address is one of two registers plus a constant)
    const int fw[2] = {swz(wn * WC + r16, g4), swz(wn * WC + r16, 4 + g4)};
    const int fa[2] = {swz(wm * WM + r16, g4), swz(wm * WM + r16, 4 + g4)};
    auto rdw = [&](int buf, int ks, int cb) { wf[cb] = *reinterpret_cast<const i32x4*>(&sW[buf][fw[ks] + cb * 2048]); };
    auto rda = [&](int buf, int ks, int tb, i32x4(&af)[TB]) {
        af[tb] = *reinterpret_cast<const i32x4*>(&sA[buf][fa[ks] + tb * 2048]);
    };
    // A substep: the weight fragments are single-buffered, each next one read into its registers after the last product that
    // uses it; the next token fragments go to the other buffer with the first channel block. The second substep (`load`) has
    // the step's barrier after its first TB products, whose fragments are there, and the direct loads of step gkt into
    // stage gbuf after every second product behind it. (The barrier behind four products, not before them, is 0.5% faster; a
    // load after every second product, not every one, 0.8%.) Every instruction is fenced: the order is this one.
    static_assert(WIDE || ND <= (CB - 1) * TB / 2, "a load after every second product");
    auto substep = [&](const i32x4(&af)[TB], int nbuf, int nks, i32x4(&naf)[TB], int gkt, int gbuf,
                       bool load) __attribute__((always_inline)) {
        const uint32_t gp = past(gkt);
        const int from = load ? TB : 0;
#pragma unroll
        for (int i = 0; i < CB * TB; ++i) {
            const int cb = i / TB, tb = i % TB;
            if (load && i == TB) {
                // step kt + 1 has landed (later ones may be in flight), and this stage is read
                __builtin_amdgcn_s_waitcnt(wait_vm((NSTG - 2) * ND));
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
            acc[cb][tb] = mfma_i8(wf[cb], af[tb], acc[cb][tb]);
            __builtin_amdgcn_sched_barrier(0);
            if (i < from)
                continue;
            if (i < from + TB) {
                rda(nbuf, nks, i - from, naf);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (load && i == TB) {
                rdw(nbuf, nks, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (tb == TB - 1) {
                rdw(nbuf, nks, cb);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (load && (i - TB) % 2 && (i - TB) / 2 < ND) {
                dma1(gkt, gp, gbuf, (i - TB) / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // fragment j of a step in the order of use: substep j / (CB + TB)
    auto frag = [&](int buf, int j, i32x4(&f)[2][WIDE ? CB + TB : 1]) {
        const int ks = j / (CB + TB), i = j % (CB + TB);
        f[ks][i] = *reinterpret_cast<const i32x4*>(i < CB ? &sW[buf][fw[ks] + i * 2048] : &sA[buf][fa[ks] + (i - CB) * 2048]);
    };
    // k step kt in stage `buf` (a constant: the loop is unrolled by NSTG): the first substep reads the second's fragments.
    // Where step kt + 1 has landed and, behind the barrier, in every wave, and every wave has read this stage, the second
    // one loads into it and reads step kt + 1's first fragments. The loads are those of k step kl: kt + NSTG, or the
    // next tile's.
    auto step = [&](int kl, auto buf_c) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value, nb = (buf + 1) % NSTG;
        if constexpr (WIDE) {
            // this step's fragments are in registers (read before the barrier), step kt + 1 has landed: its fragments
            // are read and step kt + NSTG goes into this stage while this step's products run
            constexpr int NM = 2 * CB * TB, NF = 2 * (CB + TB), RPM = (2 * NF + NM - 1) / NM, LPM = (2 * ND + NM - 1) / NM;
            __builtin_amdgcn_s_waitcnt(wait_vm((NSTG - 2) * ND));
            __builtin_amdgcn_s_barrier();
            const uint32_t gp = past(kl);
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                const int ks = i / (CB * TB), cb = i % (CB * TB) / TB, tb = i % TB;
                acc[cb][tb] = mfma_i8(fr[buf % 2][ks][cb], fr[buf % 2][ks][CB + tb], acc[cb][tb]);
                __builtin_amdgcn_sched_barrier(0);
                // the reads in the first half of the products, the loads behind them
#pragma unroll
                for (int j = i * RPM; j < (i + 1) * RPM && j < NF; ++j) {
                    frag(nb, j, fr[(buf + 1) % 2]);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int j = i * LPM; j < (i + 1) * LPM && j < ND; ++j) {
                    dma1(kl, gp, buf, j);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            return;
        }
        substep(af0, buf, 1, af1, 0, 0, false);
        substep(af1, nb, 0, af0, kl, buf, true);
    };

    // Epilogue: a wave stages ST tokens x up to 64 channels at a time (fp32, times the tokens' scales) in LDS of its own
    // and reads them back with its lanes along the channels, so that its stores are whole row segments. A wave's LDS
    // operations complete in order: no barrier. Rows of SC floats, their 16-byte chunks XOR-ed so that 16 rows at a chunk
    // cover all banks. (32 tokens keep more stores in flight; a chain has LDS for 16, the residual registers.)
    constexpr int WO = GLU ? WC / 2 : WC, SC = epi_channels(BN, GLU), NH = WO / SC; // channels a wave writes, stages at a time
    constexpr int ST = CHAIN || EC == EC_RMW || WM < 32 ? 16 : 32;
    constexpr int NCH = SC / 4, RPI = 64 / NCH, NI = ST / RPI; // chunks a row, rows an instruction, rows a lane
    auto epilogue = [&](uint32_t ez, int em0, int en0) __attribute__((always_inline)) {
        const int lane = here(), r16 = lane & 15, g4 = lane >> 4;
        float* st = reinterpret_cast<float*>(smem + (CHAIN ? NSTG * (BM + BN) * 128 : 0)) + wave * ST * SC;
        auto swap = [](int row) { return row / (64 / SC) % NCH; };
        const float* as = p.ascale + uint64_t(ez) * p.M;
        const int t0 = em0 + wm * WM, c0 = en0 + wn * WO;
        float sc[TB];
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
            sc[tb] = as[min(t0 + tb * 16 + r16, int(p.M) - 1)];
        const int lc = lane % NCH, lr = lane / NCH;
        Ch4 k[NH];
        if constexpr (!GLU)
#pragma unroll
            for (int h = 0; h < NH; ++h)
                k[h] = channels4(p, min(c0 + h * SC + 4 * lc, cols - 4)); // (cols is a multiple of 4)
        // slice s: tokens ST (s / NH) .. + ST - 1, channels SC (s % NH) .. + SC - 1
        constexpr int NSL = WM / ST * NH;
        auto token = [&](int s, int i) { return t0 + s / NH * ST + lr + RPI * i; };
        auto place = [&](int s) { return int64_t(ez) * p.sc + int64_t(token(s, 0)) * p.ldc + c0 + s % NH * SC + 4 * lc; };
        const int64_t next = int64_t(RPI) * p.ldc;
        // f(i) for the lane's rows of a slice that are C's; a whole slice has no guard between them
        auto rows = [&](int s, auto&& f) __attribute__((always_inline)) {
            if (c0 + s % NH * SC + 4 * lc >= cols)
                return;
            if (t0 + s / NH * ST + ST <= int(p.M)) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    f(i);
            } else {
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    if (token(s, i) < int(p.M))
                        f(i);
            }
        };
        // the residual's rows of a slice are loaded while the slice before it is added and stored
        f32x4 x[2][EC == EC_RMW ? NI : 1];
        auto residual = [&](int s) __attribute__((always_inline)) {
            const float* c = static_cast<const float*>(p.c) + place(s);
            rows(s, [&](int i) { x[s % 2][i] = *reinterpret_cast<const f32x4*>(c + i * next); });
        };
        if constexpr (EC == EC_RMW)
            residual(0);
        if constexpr (CHAIN)
            __builtin_amdgcn_s_waitcnt(wait_vm(0)); // the next tile's first steps have landed in this wave
        if constexpr (GLU) {
            with_flag(p.epi == MK_EPI_SWIGLU, [&](auto swi) __attribute__((always_inline)) {
#pragma unroll
                for (int cb = 0; cb < CB / 2; ++cb) {
                    const int c = min(c0 + cb * 16 + 4 * g4, cols - 4);
                    const f32x4 s1 = *reinterpret_cast<const f32x4*>(p.wscale + c);
                    const f32x4 s2 = *reinterpret_cast<const f32x4*>(p.wscale + cols + c);
                    const f32x4 b1 = load4(p.bias, c, 0.0f), b2 = load4(p.bias, cols + c, 0.0f);
#pragma unroll
                    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float a = fmaf(float(acc[cb][tb][e]) * sc[tb], s1[e], b1[e]);
                            const float g = fmaf(float(acc[cb + CB / 2][tb][e]) * sc[tb], s2[e], b2[e]);
                            acc[cb][tb][e] = __builtin_bit_cast(int, glu1<decltype(swi)::value>(a, g));
                        }
                }
            });
        }
#pragma unroll
        for (int s = 0; s < NSL; ++s) {
            const int h = s % NH;
#pragma unroll
            for (int cb = 0; cb < SC / 16; ++cb)
#pragma unroll
                for (int t = 0; t < ST / 16; ++t) {
                    const int tb = s / NH * (ST / 16) + t, row = 16 * t + r16;
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int a = acc[h * (SC / 16) + cb][tb][e];
                        v[e] = GLU ? __builtin_bit_cast(float, a) : float(a) * sc[tb];
                    }
                    *reinterpret_cast<f32x4*>(st + row * SC + 4 * ((cb * 4 + g4) ^ swap(row))) = v;
                }
            f32x4 v[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = lr + RPI * i;
                v[i] = *reinterpret_cast<const f32x4*>(st + row * SC + 4 * (lc ^ swap(row)));
                if constexpr (!GLU)
                    v[i] = scaled(v[i], k[h].ws, k[h].b);
            }
            if constexpr (EC == EC_ACT)
                with_flag(p.epi == MK_EPI_GELU_TANH, [&](auto gelu) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < NI; ++i)
                        v[i] = act4<decltype(gelu)::value>(v[i]);
                });
            if constexpr (EC == EC_RMW) {
                if (s + 1 < NSL)
                    residual(s + 1);
                float* c = static_cast<float*>(p.c) + place(s);
                rows(s, [&](int i) {
                    *reinterpret_cast<f32x4*>(c + i * next) = residual4(p, uint32_t(token(s, i)), x[s % 2][i], v[i], k[h]);
                });
            } else if (p.c_dtype == MK_F32) {
                float* c = static_cast<float*>(p.c) + place(s);
                rows(s, [&](int i) { *reinterpret_cast<f32x4*>(c + i * next) = v[i]; });
            } else {
                uint16_t* c = static_cast<uint16_t*>(p.c) + place(s);
                u32x2 o[NI];
                with_flag(p.c_dtype == MK_F16, [&](auto f16) {
#pragma unroll
                    for (int i = 0; i < NI; ++i)
                        o[i] = u32x2{pack_x2(v[i][0], v[i][1], decltype(f16)::value),
                                     pack_x2(v[i][2], v[i][3], decltype(f16)::value)};
                });
                rows(s, [&](int i) { *reinterpret_cast<u32x2*>(c + i * next) = o[i]; });
            }
        }
    };

    // k steps 0 .. NSTG - 1 of the first tile on their way
    set(0);
#pragma unroll
    for (int s = 0; s < NSTG; ++s) {
        const int kt = min(s, ke - 1);
#pragma unroll
        for (int i = 0; i < ND; ++i)
            dma1(kt, past(kt), s, i);
    }
    for (uint32_t tile = 0;;) {
        // step 0 in LDS: of the first tile, this wave's loads of it have landed; of later ones, all (before its stores)
        if (!CHAIN || !tile)
            __builtin_amdgcn_s_waitcnt(wait_vm((NSTG - 1) * ND));
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int i = 0; i < CB; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j)
                acc[i][j] = i32x4{0, 0, 0, 0};
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < 2 * (CB + TB); ++j)
                frag(0, j, fr[0]);
        } else {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
                rdw(0, 0, cb);
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
                rda(0, 0, tb, af0);
        }
        int kt = 0;
        uint32_t ez = z;
        int em0 = m0, en0 = n0;
        bool more = false;
        if constexpr (CHAIN) {
            using S0 = std::integral_constant<int, 0>;
            using S1 = std::integral_constant<int, 1>;
            for (; kt + 2 < ke; kt += 2) {
                step(kt + 2, S0{});
                step(kt + 3, S1{});
            }
            // the last two steps load the next tile's first two (the last tile's own, which nobody reads)
            more = ++tile < count;
            if (more)
                set(tile);
            step(0, S0{});
            step(1, S1{});
        } else {
            // past-the-end steps reload the last one (nobody reads them)
            for (; kt + NSTG - 1 < ke; kt += NSTG)
                for_each_int([&](auto i) __attribute__((always_inline)) { step(min(kt + decltype(i)::value + NSTG, ke - 1), i); },
                             std::make_integer_sequence<int, NSTG>{});
            for_each_int(
                [&](auto i) __attribute__((always_inline)) {
                    if (kt + decltype(i)::value < ke)
                        step(ke - 1, i);
                },
                std::make_integer_sequence<int, NSTG - 1>{});
            __builtin_amdgcn_s_waitcnt(0); // the last loads land before the LDS is reused
            __syncthreads();
        }
        epilogue(ez, em0, en0);
        if (!more)
            break;
    }
}

// Workgroup i runs on XCD i % 8 and each XCD has an L2 of its own: of n workgroups XCD x takes a run.
__device__ inline uint32_t xcd_run(uint32_t i, uint32_t n)
{
    const uint32_t x = i % 8;
    return x * (n / 8) + min(x, n % 8) + i / 8;
}
// Tile t of the launch, 8 token tiles at a time, so that a run of tiles shares weight panels
__device__ inline void locate(uint32_t t, uint32_t tiles_m, uint32_t tiles_n, uint32_t& z, uint32_t& tm, uint32_t& tn)
{
    const uint32_t per = tiles_m * tiles_n, in_group = 8 * tiles_n;
    z = t / per;
    t %= per;
    const uint32_t first = t / in_group * 8, g = min(tiles_m - first, 8u), i = t % in_group;
    tm = first + i % g;
    tn = i / g;
}

// A tile a workgroup of 4 waves (one a SIMD), as many workgroups on a CU as its 160 KB of LDS hold. Few rows or narrow
// outputs take small tiles (32 x 32; 32 x 64 for a gated unit), which spread over more CUs: 208 x 1040 x 10288 18 -> 11.6
// us, 16 x 4096 x 12288 12.8 -> 9.9, 77 x 2560 x 2048 4.3 -> 3.9. One with stages in flight (64 x 128 of 4) takes a long k
// fastest; with 2 stages and two or three workgroups on the CU, one's loads, epilogue and stores go on under the others'
// products, which is what counts over a short k (7431 x 768 x 96 GEGLU 9.7 -> 6.1 us, 896 x 4928 x 176 9.0 -> 6.5, 4400 x
// 1024 x 384 ADD 14.2 -> 11.2, 1700 x 2560 x 2560 24.4 -> 20.1 with 128 x 128).
template <int BM, int BN, int NSTG> constexpr int resident() { return 160 * 1024 / tile_lds<BM, BN, 4, NSTG, false>(); }

template <int BM, int BN, int NSTG, int EC>
__global__ __launch_bounds__(256, (resident<BM, BN, NSTG>())) __attribute__((amdgpu_waves_per_eu(
    resident<BM, BN, NSTG>(), resident<BM, BN, NSTG>()))) void gemm_i8_kernel(I8P p, uint32_t tiles_m, uint32_t tiles_n)
{
    __shared__ __attribute__((aligned(16))) int8_t smem[tile_lds<BM, BN, 4, NSTG, false>()];
    i8_tiles<BM, BN, 4, NSTG, EC, false>(p, smem, 1, [&](uint32_t, uint32_t& z, int& m0, int& n0) {
        uint32_t tm, tn;
        locate(xcd_run(blockIdx.x, gridDim.x), tiles_m, tiles_n, z, tm, tn);
        m0 = int(tm) * BM;
        n0 = int(tn) * (EC == EC_GLU ? BN / 2 : BN);
    });
}

// 256 x 256 tiles, the first `whole` of them in `chains` workgroups (CHAIN: one a compute unit, which go from tile to tile;
// else as many as tiles), the rest in parts of side x side (128 or 64) a workgroup: whole rounds of the chip take the large
// tile, the last, partial one spreads over all of it. A chain saves 1.8 us a tile (32768 x 12288 x 4096 1343 -> 1298 us)
// where the number of k steps is even; the gated epilogues have no registers for it (4352 x 24576 x 4096 SwiGLU 372 ->
// 398).
template <int EC, bool CHAIN>
__global__ __launch_bounds__(512, 2) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_i8_mixed_kernel(
    I8P p, uint32_t tiles_m, uint32_t tiles_n, uint32_t whole, uint32_t chains, uint32_t side)
{
    constexpr int BO = EC == EC_GLU ? 128 : 256; // output channels of a tile
    __shared__ __attribute__((aligned(16))) int8_t smem[tile_lds<256, 256, 8, 2, CHAIN>()];
    static_assert(tile_lds<128, 128, 8, 4, false>() <= sizeof(smem) && tile_lds<64, 64, 8, 8, false>() <= sizeof(smem), "");
    if (blockIdx.x < chains) {
        i8_tiles<256, 256, 8, 2, EC, CHAIN>(p, smem, CHAIN ? (whole - blockIdx.x - 1) / chains + 1 : 1,
                                            [&](uint32_t i, uint32_t& z, int& m0, int& n0) {
                                                uint32_t tm, tn;
                                                locate(xcd_run(blockIdx.x + i * chains, whole), tiles_m, tiles_n, z, tm, tn);
                                                m0 = int(tm) * 256;
                                                n0 = int(tn) * BO;
                                            });
        return;
    }
    const uint32_t i = xcd_run(blockIdx.x - chains, gridDim.x - chains);
    uint32_t bz, tm, tn, bm, bn;
    if (whole) {
        const uint32_t n = 256 / side, part = i % (n * n);
        locate(whole + i / (n * n), tiles_m, tiles_n, bz, tm, tn);
        bm = tm * 256 + part / n * side;
        bn = tn * BO + part % n * (side * BO / 256);
    } else { // less than a round: the launch's tiles are 128 x 128
        locate(i, tiles_m, tiles_n, bz, tm, tn);
        bm = tm * 128;
        bn = tn * (BO / 2);
    }
    if (bm >= p.M || bn >= (EC == EC_GLU ? p.N / 2 : p.N))
        return;
    auto at = [&](uint32_t, uint32_t& z, int& m0, int& n0) {
        z = bz;
        m0 = int(bm);
        n0 = int(bn);
    };
    if (side == 128)
        i8_tiles<128, 128, 8, 4, EC, false>(p, smem, 1, at);
    else
        i8_tiles<64, 64, 8, 8, EC, false>(p, smem, 1, at);
}

// ------------------------------------------------------------------------------------------------------------
// 16 rows x 16 channels a workgroup, its 8 waves every eighth 256 bytes of k each, straight from memory to registers: for
// few rows (up to 16 read the weight once) and for small products of long k, whose few larger tiles leave the chip idle.
// The rows of an operand lie in 64-byte pieces of 16 rows a load, which brings 40 to 60 bytes a ns and CU, half of what the
// direct loads of a tile do. The sums meet in LDS. Up to 16 rows bound by the weight's bytes: 1 x 4096 x 4096 5.0 us, 1 x
// 4096 x 12288 9.9 us, a launch alone 3; 98 x 176 x 11344 9.6 us, on 64 x 32 tiles 19.4. 4 or 16 waves, 128 or 512 bytes a
// turn: within 15%.
// ------------------------------------------------------------------------------------------------------------
constexpr int k16Waves = 8;

template <int EC> __global__ __launch_bounds__(64 * k16Waves) void gemm_i8_16_kernel(I8P p)
{
    constexpr bool GLU = EC == EC_GLU;
    constexpr int CB = GLU ? 2 : 1, NS = 4;
    constexpr uint32_t kUnit = 64 * NS, kStep = k16Waves * kUnit;
    __shared__ i32x4 red[k16Waves][CB][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g4 = lane >> 4, cols = int(GLU ? p.N / 2 : p.N), n0 = int(blockIdx.x) * 16;
    const uint32_t z = blockIdx.y;
    const int m0 = int(blockIdx.z) * 16, nr = min(cols - n0, 16), M = min(int(p.M) - m0, 16);
    const int8_t* gA = p.a + int64_t(z) * p.sa + int64_t(m0) * p.lda;
    const int8_t* gW = p.w + uint64_t(n0) * p.K;
    const BufRes rsA = buf_res(gA, uint32_t(int64_t(M - 1) * p.lda + p.K));
    const BufRes rsW[2] = {buf_res(gW, uint32_t(nr) * p.K), buf_res(GLU ? gW + uint64_t(cols) * p.K : gW, uint32_t(nr) * p.K)};
    const uint32_t ow = uint32_t(min(r16, nr - 1)) * p.K + g4 * 16, oa = uint32_t(min(r16, M - 1)) * uint32_t(p.lda) + g4 * 16;
    i32x4 acc[CB] = {};
    struct Unit {
        i32x4 w[NS][CB], a[NS];
    };
    auto load = [&](uint32_t k, Unit& f) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            // chunks past K: out of range, zeros (k itself stays in a scalar register)
            const bool in = k + s * 64 + g4 * 16 < p.K;
#pragma unroll
            for (int c = 0; c < CB; ++c)
                f.w[s][c] = __builtin_bit_cast(i32x4, buf_load16(rsW[c], in ? ow + s * 64 : 0x80000000u, k));
            f.a[s] = __builtin_bit_cast(i32x4, buf_load16(rsA, in ? oa + s * 64 : 0x80000000u, k));
        }
    };
    auto mul = [&](const Unit& f) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int c = 0; c < CB; ++c)
                acc[c] = mfma_i8(f.w[s][c], f.a[s], acc[c]);
    };
    // two units in turn, each loaded while the other one is multiplied
    Unit f0, f1;
    uint32_t k = uint32_t(wave) * kUnit;
    if (k < p.K)
        load(k, f0);
    for (; k < p.K; k += 2 * kStep) {
        if (k + kStep < p.K)
            load(k + kStep, f1);
        mul(f0);
        if (k + kStep >= p.K)
            break;
        if (k + 2 * kStep < p.K)
            load(k + 2 * kStep, f0);
        mul(f1);
    }
#pragma unroll
    for (int c = 0; c < CB; ++c)
        red[wave][c][lane] = acc[c];
    __syncthreads();
    const int tok = r16, ch = n0 + 4 * g4;
    if (wave || tok >= M || ch >= cols)
        return;
    i32x4 s[CB] = {};
#pragma unroll
    for (int w = 0; w < k16Waves; ++w)
#pragma unroll
        for (int c = 0; c < CB; ++c)
            s[c] += red[w][c][lane];
    const float as = p.ascale[uint64_t(z) * p.M + m0 + tok];
    const Ch4 kc = channels4(p, ch);
    f32x4 t;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        t[e] = float(s[0][e]) * as;
    f32x4 v = scaled(t, kc.ws, kc.b);
    if constexpr (GLU) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            t[e] = float(s[CB - 1][e]) * as;
        const f32x4 g = scaled(t, *reinterpret_cast<const f32x4*>(p.wscale + cols + ch), load4(p.bias, cols + ch, 0.0f));
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = p.epi == MK_EPI_SWIGLU ? glu1<true>(v[e], g[e]) : glu1<false>(v[e], g[e]);
    } else if constexpr (EC == EC_ACT) {
        v = p.epi == MK_EPI_GELU_TANH ? act4<true>(v) : act4<false>(v);
    }
    const int64_t at = int64_t(z) * p.sc + int64_t(m0 + tok) * p.ldc + ch;
    if constexpr (EC == EC_RMW) {
        f32x4* x = reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + at);
        *x = residual4(p, uint32_t(m0 + tok), *x, v, kc);
    } else if (p.c_dtype == MK_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + at) = v;
    } else {
        const bool h = p.c_dtype == MK_F16;
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.c) + at) = u32x2{pack_x2(v[0], v[1], h), pack_x2(v[2], v[3], h)};
    }
}

template <int BM, int BN, int NSTG, int EC> mk_status launch_tile(const I8P& p, hipStream_t s)
{
    const uint32_t cols = EC == EC_GLU ? p.N / 2 : p.N, tm = cdiv(p.M, BM), tn = cdiv(cols, EC == EC_GLU ? BN / 2 : BN);
    gemm_i8_kernel<BM, BN, NSTG, EC><<<tm * tn * p.batch, 256, 0, s>>>(p, tm, tn);
    MK_LAUNCH_CHECK("gemm_i8");
    return MK_OK;
}

// The kernel of a launch: the one with the least estimated time in us, beside a launch's own. A round of tiles, a workgroup
// of the kernel in every place that a CU has for one, takes so much a k step of 128 and so much beside (a start, an
// epilogue); the last round has 1, 2 or 3 workgroups on a CU. 16 x 16 rows come at 48 bytes a ns and CU, or all weights at
// 6.3 TB/s. A round of 256 x 256 tiles is bound by the matrix cores (1.5 a step; 0.95 where it is not full and the clock
// higher). Fitted to the kernels' times at 1500 shapes and epilogues (rows 1 .. 16000, N from 64, K from 96): on those the
// choice is within 0.7% of the best in the mean, 33% at worst (4000 x 1040 x 10288: 100 us, 76 in 128 x 128 tiles). The
// epilogue's bytes have no term (4400 x 8192 x 256 ADD: 74 us, 57 in 64 x 128 tiles of 2 stages). Measured, us:
//                             16x16  32x32  64x32  64x64  64x128  64x128, 2 stages  128x128  mixed
//   1 x 4096 x 4096             5.0           6.1    7.6      11                                14
//   77 x 2560 x 2048            9.3    3.9    4.3    4.8     7.1                               9.0
//   208 x 1040 x 10288           33     12     18     26      36
//   130 x 2560 x 2560            16    6.0    5.2    6.1     9.1
//   300 x 4096 x 12288                  47     38     35      28                51       56     36
//   1700 x 2560 x 2560                                24      26                23       21     25
//   1024 x 4096 x 4096                         36     28      24                23       24     19
//   896 x 4928 x 176 GEGLU                           9.0      11               6.4      7.4     10
//   300 x 1024 x 4096 GEGLU      18    7.1 (32x64)   8.4      12
// The mixed kernel's last, partial round takes 128 x 128 parts up to two rounds of them (4352 x 5120 x 4096, 84 tiles left:
// 91 us against 95 in whole tiles; 1024 x 8192 x 4096, 128: 40 and 44), then whole tiles (1024 x 9216 x 4096, 144: 54 and
// 44; 4352 x 7168 x 4096, 220: 131 and 112); 64 x 64 parts where they fit one round (4352 x 4096 x 12288, 16 left: 185 us,
// 210 in 128 x 128, 259 whole).
enum { K_NONE = -1, K_16X16, K_32X32, K_32X64, K_64X32, K_64X64, K_64X128, K_64X128_2, K_128X128_2, K_MIXED };
struct TileCost {
    int kernel;
    uint32_t bm, bn, stages, resident;
    double step[3], end[3]; // of a round with 1, 2, 3 workgroups on a CU
};
constexpr TileCost kTiles[] = {
    {K_128X128_2, 128, 128, 2, resident<128, 128, 2>(), {0.5, 0.81, 0}, {1.8, 4.4, 0}},
    {K_64X128_2, 64, 128, 2, resident<64, 128, 2>(), {0.44, 0.53, 0.97}, {0.7, 1.5, 3.4}},
    {K_64X128, 64, 128, 4, resident<64, 128, 4>(), {0.26, 0, 0}, {2.4, 0, 0}},
    {K_64X64, 64, 64, 4, resident<64, 64, 4>(), {0.15, 0.35, 0}, {0.66, 2.0, 0}},
    {K_64X32, 64, 32, 6, resident<64, 32, 6>(), {0.077, 0.25, 0}, {0.64, 1.5, 0}},
    {K_32X64, 32, 64, 6, resident<32, 64, 6>(), {0.11, 0.25, 0}, {0.48, 1.3, 0}},
    {K_32X32, 32, 32, 8, resident<32, 32, 8>(), {0.069, 0.115, 0}, {0.65, 0.77, 0}},
};
struct Plan {
    int kernel;
    bool chain; // these of the mixed kernel
    uint32_t tiles_m, tiles_n, whole, chains, side, grid;
};

Plan plan_of(const I8P& p, bool glu, uint32_t cus)
{
    // rows that start inside a cache line (inside a 64-byte half of one) cost the loads 1.2 (1.4) times as much
    const uint32_t inside = uint32_t(p.K | p.lda) % 128;
    const double slow = !inside ? 1.0 : inside == 64 ? 1.2 : 1.4, steps = slow * cdiv(p.K, 128);
    auto tiles = [&](uint32_t bm, uint32_t bn) { return uint64_t(cdiv(p.M, bm)) * cdiv(p.N, bn) * p.batch; };
    auto rounds = [&](uint64_t n) { return double((n + cus - 1) / cus); };
    Plan best{K_NONE, false, 0, 0, 0, 0, 0, 0};
    double least = 1e30;
    // a grid dimension holds fewer than 2^32 threads
    auto consider = [&](int k, double t, uint64_t threads) {
        if (t < least && threads < (uint64_t(1) << 32)) {
            least = t;
            best.kernel = k;
        }
    };
    // its bytes from the large cache, whatever the kernel; of kernels that wait for them the largest tile (1 x 12288 x 4096
    // 9.5 us on 64 x 64 tiles, 9.9 on 32 x 32)
    const double weights = double(p.N) * p.K * p.batch * 0.13e-6;
    const uint32_t parts = glu ? 2 : 1; // of the weight
    if (p.M <= 16 * 65535)
        consider(K_16X16,
                 std::max(rounds(tiles(16, 16 * parts)) * (p.K * (16.0 * parts + std::min(p.M, 16u)) * 2.1e-5 + 0.15),
                          1.25 * weights),
                 uint64_t(cdiv(p.N, 16 * parts)) * 512);
    for (const TileCost& c : kTiles) {
        // (a gated unit's two parts are blocks of 16 channels of a wave: 64 a tile at least)
        if (glu ? c.bn < 64 : c.kernel == K_32X64)
            continue;
        const uint64_t n = tiles(c.bm, c.bn), round = uint64_t(c.resident) * cus, last = (n % round + cus - 1) / cus;
        auto time = [&](uint64_t w) { return steps * c.step[w - 1] + c.end[w - 1]; };
        consider(c.kernel, std::max(double(n / round) * time(c.resident) + (last ? time(last) : 0.0), weights), n * 256);
    }
    // whole rounds of 256 x 256 tiles and the rest: as it is, in 128 x 128 parts up to two rounds of them, or in 64 x 64 ones
    // up to one
    const uint64_t big = tiles(256, 256), whole = big / cus * cus, rest = big - whole;
    const double msteps = (0.6 + 0.4 / slow) * steps;
    double last = msteps * 0.95 + 7.9;
    uint64_t tail = 0;
    best.side = 128;
    if (rest) {
        const uint64_t n128 = whole ? rest * 4 : tiles(128, 128);
        const double t128 = rounds(n128) * (msteps * 0.43 + 2.4), t64 = msteps * 0.13 + 0.7;
        if (n128 <= 2 * uint64_t(cus) && t128 < last) {
            last = t128;
            tail = n128;
        }
        if (whole && rest * 16 <= cus && t64 < last) {
            last = t64;
            tail = rest * 16;
            best.side = 64;
        }
    } else {
        last = 0.0;
    }
    const uint64_t tiled = tail ? whole : big;
    best.chain = !glu && tiled > cus && cdiv(p.K, 128) % 2 == 0;
    const uint64_t chains = best.chain ? cus : tiled;
    const uint64_t groups = chains + tail;
    consider(K_MIXED, double(whole / cus) * (msteps * 1.5 + 9.5) + last, groups * 512);
    const uint32_t tile = tail && !whole ? 128 : 256;
    best.tiles_m = cdiv(p.M, tile);
    best.tiles_n = cdiv(p.N, tile);
    best.whole = uint32_t(tiled);
    best.chains = uint32_t(chains);
    best.grid = uint32_t(groups);
    return best;
}

template <int EC> mk_status launch(const I8P& p, uint32_t cus, hipStream_t s)
{
    const Plan plan = plan_of(p, EC == EC_GLU, cus);
    switch (plan.kernel) {
    case K_16X16:
        gemm_i8_16_kernel<EC><<<dim3(cdiv(EC == EC_GLU ? p.N / 2 : p.N, 16), p.batch, cdiv(p.M, 16)), 64 * k16Waves, 0,
                                 s>>>(p);
        break;
    case K_32X32:
    case K_64X32:
        if constexpr (EC != EC_GLU)
            return plan.kernel == K_32X32 ? launch_tile<32, 32, 8, EC>(p, s) : launch_tile<64, 32, 6, EC>(p, s);
        return fail(MK_ERR_UNSUPPORTED, "gemm_i8: no gated tiles of 32 channels");
    case K_32X64:
        if constexpr (EC == EC_GLU)
            return launch_tile<32, 64, 6, EC>(p, s);
        return fail(MK_ERR_UNSUPPORTED, "gemm_i8: 32 x 64 tiles are the gated units'");
    case K_64X64:
        return launch_tile<64, 64, 4, EC>(p, s);
    case K_64X128:
        return launch_tile<64, 128, 4, EC>(p, s);
    case K_64X128_2:
        return launch_tile<64, 128, 2, EC>(p, s);
    case K_128X128_2:
        return launch_tile<128, 128, 2, EC>(p, s);
    case K_NONE:
        return fail(MK_ERR_ARG, "gemm_i8: a launch of more than 2^32 threads");
    default:
        if constexpr (EC != EC_GLU)
            if (plan.chain) {
                gemm_i8_mixed_kernel<EC, true><<<plan.grid, 512, 0, s>>>(p, plan.tiles_m, plan.tiles_n, plan.whole, plan.chains,
                                                                   plan.side);
                break;
            }
        gemm_i8_mixed_kernel<EC, false><<<plan.grid, 512, 0, s>>>(p, plan.tiles_m, plan.tiles_n, plan.whole, plan.chains,
                                                                   plan.side);
    }
    MK_LAUNCH_CHECK("gemm_i8");
    return MK_OK;
}

// Compute units of the current device, asked once a device (the question costs as much as a launch).
mk_status compute_units(uint32_t& n)
{
    static std::atomic<int> known[64];
    int dev = 0, cus = 0;
    MK_HIP(hipGetDevice(&dev));
    if (dev >= 0 && dev < 64)
        cus = known[dev].load(std::memory_order_relaxed);
    if (!cus) {
        MK_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
        cus = std::max(cus, 1);
        if (dev >= 0 && dev < 64)
            known[dev].store(cus, std::memory_order_relaxed);
    }
    n = uint32_t(cus);
    return MK_OK;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The checks of a call's arguments, and the kernels' (an empty product's, M or batch 0, too).
mk_status prepare(const mk_gemm_args* a, const float* ascale, I8P& p)
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
    if (!a->M || !a->batch) {
        p = {};
        return MK_OK;
    }
    if (a->M > 0x7fffff00u || a->N > 0x7fffff00u || a->batch > 65535)
        return fail(MK_ERR_ARG, "gemm_i8: more than 2^31 - 256 rows or channels or 65535 batch items");
    p = {static_cast<const int8_t*>(a->a),
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
    return MK_OK;
}

} // namespace

} // namespace mk

using namespace mk;

extern "C" {

mk_status mk_gemm_i8(const mk_gemm_args* a, const float* ascale, void* stream)
{
    I8P p;
    MK_TRY(prepare(a, ascale, p));
    if (!p.M)
        return MK_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint32_t n = 0;
    MK_TRY(compute_units(n));
    switch (epi_class(p.epi)) {
    case EC_STORE: return launch<EC_STORE>(p, n, s);
    case EC_ACT: return launch<EC_ACT>(p, n, s);
    case EC_GLU: return launch<EC_GLU>(p, n, s);
    default: return launch<EC_RMW>(p, n, s);
    }
}

mk_status mk_gemm_i8_plan(const mk_gemm_args* a, uint32_t cus, uint32_t* out)
{
    if (!a || !out || !cus)
        return fail(MK_ERR_ARG, "gemm_i8_plan: null argument or no compute units");
    I8P p;
    MK_TRY(prepare(a, a->wscale, p));
    if (!p.M)
        return fail(MK_ERR_ARG, "gemm_i8_plan: empty product");
    const bool glu = epi_class(p.epi) == EC_GLU;
    const Plan plan = plan_of(p, glu, cus);
    if (plan.kernel == K_NONE)
        return fail(MK_ERR_ARG, "gemm_i8: a launch of more than 2^32 threads");
    uint32_t o[6] = {16, glu ? 32u : 16u, 0, 0, 0, 0};
    for (const TileCost& c : kTiles)
        if (c.kernel == plan.kernel) {
            o[0] = c.bm;
            o[1] = c.bn;
            o[2] = c.stages;
        }
    if (plan.kernel == K_MIXED) {
        o[0] = o[1] = plan.whole ? 256 : 128;
        o[2] = plan.whole ? 2 : 4;
        o[3] = plan.chain ? plan.chains : 0;
        o[4] = plan.whole && plan.grid > plan.chains ? plan.side : 0;
        o[5] = plan.grid;
    } else {
        o[5] = cdiv(p.M, o[0]) * cdiv(p.N, o[1]) * p.batch;
    }
    std::copy(o, o + 6, out);
    return MK_OK;
}

} // extern "C"
