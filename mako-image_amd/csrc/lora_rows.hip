// mk_lora_rows: low-rank adapters of many requests beside a shared projection.
//
// Two launches: t = x A^T (the rows' own adapters) into the workspace, then c = base + scale t B^T. Bound by memory: x, base
// and c once each, with 2 rank flops a value. t is a few values a row, so it goes through memory in fp32, as the
// partial sums of the workgroups that share a row's K (no atomics: the second launch adds them in their order). Very few rows
// take both products in one launch, and many rows in no order are first put in the order of their adapters by one more.
// On the device: 4352 x 4096 to 12288 by rank 32 in 3 parts 75 us (x, base and c at 3.3 TB/s; 84 through single calls), 16401 x 12288 to
// 4096 by rank 64, fp32 rows, 250 to 277 us (3.4 to 3.7 TB/s), 1 row of 4096 to 4096 5.1 us.
#include "common.hpp"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace mk {

namespace {

struct LoraP {
    const uint16_t *x, *a, *b;
    const float* scale;
    const int32_t* ids;
    const void* base;
    void* c;
    float* t;       // workspace: [splits][rows][parts rank], a row's at its own number
    u32x2* perm;    // workspace: [rows], the row at each place of the tiles and its adapter, or NULL: places are rows
    int64_t ldx, ldbase, ldc;
    uint32_t rows, K, N, rank, parts, adapters;
    uint32_t splits, split_k; // workgroups that share a row's K, and the k of each
    uint32_t blocks;          // of 128 columns that a wave of the second product goes through
};

template <bool F16> __device__ inline float widen(uint16_t h) { return F16 ? h2f_bits(h) : bf2f_bits(h); }
template <bool F16> __device__ inline void widen8(const u32x4& v, float (&f)[8])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = widen<F16>(uint16_t(v[j]));
        f[2 * j + 1] = widen<F16>(uint16_t(v[j] >> 16));
    }
}
template <uint32_t CT> __device__ inline float load_c(const void* c, int64_t at)
{
    return CT == MK_F32 ? static_cast<const float*>(c)[at] : widen<CT == MK_F16>(static_cast<const uint16_t*>(c)[at]);
}
// the adapter of a row, or -1
__device__ inline int adapter_of(const LoraP& p, uint32_t row)
{
    const int id = p.ids ? p.ids[row] : 0;
    return id >= 0 && uint32_t(id) < p.adapters ? id : -1;
}
// s_waitcnt immediate: vmcnt vm, lgkmcnt 0 (vmcnt's bits 3:0 and 15:14, expcnt not waited for)
constexpr int wait_vm(int vm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4); }

constexpr uint32_t kOut = 0x80000000u; // a byte offset past every buffer resource here
constexpr int kRows = 64;              // rows of a workgroup of the second product
// the row at a place of the tiles from first on, counted from there or, in order, from row 0 (row_base), and its adapter (-1: none)
__device__ inline uint32_t row_base(const LoraP& p, uint32_t first) { return p.perm ? 0 : first; }
__device__ inline int row_at(const LoraP& p, uint32_t first, uint32_t i, uint32_t& row)
{
    if (p.perm) {
        const u32x2 v = p.perm[first + i];
        row = v[0];
        return int(v[1]);
    }
    row = i;
    return adapter_of(p, first + i);
}
// the smallest adapter above `last` among a wave's rows (a lane's row each), or INT_MAX
__device__ inline int next_adapter(int id, int last)
{
    int v = id > last ? id : 0x7fffffff;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1)
        v = min(v, __shfl_xor(v, m));
    return __builtin_amdgcn_readfirstlane(v);
}

// ------------------------------------------------------------------------------------------------------------
// rows in the order of their adapters
// ------------------------------------------------------------------------------------------------------------

// A tile goes through its steps for every adapter among its rows, so rows in no order cost as many times as there are adapters
// (4352 rows of 4096 to 12288 by rank 32, 8 adapters: 232 us like that, 106 after the sort, 78 where they are in runs already). One workgroup sorts the rows' numbers by
// counting, where more than every second tile would have a change of adapter; rows in runs keep their places. Which
// place a row gets among its adapter's depends on the order of atomics, its values do not: they are sums over k and rank alone.
constexpr uint32_t kMaxOrdered = 1024; // adapters
__global__ __launch_bounds__(1024) void order_kernel(LoraP p)
{
    __shared__ uint32_t count[kMaxOrdered + 1], sums[2][1024], changes;
    const uint32_t tid = threadIdx.x, lane = tid & 63, bins = p.adapters + 1; // the last one: rows without an adapter
    if (tid == 0)
        changes = 0;
    __syncthreads();
    // (8 loads of a thread at a time: one after the other, 16401 rows took 9 us)
    uint32_t mine = 0;
    for (uint32_t i0 = tid; i0 < p.rows; i0 += 8 * 1024) {
        int id[8], before[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t i = min(i0 + j * 1024, p.rows - 1);
            id[j] = p.ids[i];
            before[j] = p.ids[i ? i - 1 : 0];
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            mine += i0 + j * 1024 < p.rows && id[j] != before[j];
    }
    if (mine)
        atomicAdd(&changes, mine);
    __syncthreads();
    if (changes <= p.rows / (2 * kRows)) {
        for (uint32_t i = tid; i < p.rows; i += 1024)
            p.perm[i] = u32x2{i, uint32_t(adapter_of(p, i))};
        return;
    }
    for (uint32_t i = tid; i < bins; i += 1024)
        count[i] = 0;
    __syncthreads();
    // the bins' counters up by a wave's rows, one atomic a bin; a row's place among them
    auto place = [&](uint32_t i, int id) {
        const bool on = i < p.rows;
        const uint32_t bin = id >= 0 && uint32_t(id) < p.adapters ? uint32_t(id) : p.adapters;
        uint32_t at = 0;
        for (uint64_t todo = __ballot(on); todo;) {
            const int first = __builtin_ctzll(todo);
            const uint32_t b = __shfl(bin, first);
            const uint64_t same = __ballot(on && bin == b);
            uint32_t from = 0;
            if (int(lane) == first)
                from = atomicAdd(&count[b], uint32_t(__popcll(same)));
            from = __shfl(from, first);
            if (on && bin == b)
                at = from + uint32_t(__popcll(same & ((1ull << lane) - 1)));
            todo &= ~same;
        }
        return at;
    };
    auto each = [&](auto f) {
        for (uint32_t i0 = tid - lane; i0 < p.rows; i0 += 8 * 1024) {
            int id[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                id[j] = p.ids[min(i0 + j * 1024 + lane, p.rows - 1)];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (i0 + j * 1024 < p.rows)
                    f(i0 + j * 1024 + lane, id[j]);
        }
    };
    each([&](uint32_t i, int id) { place(i, id); });
    __syncthreads();
    // where each bin starts: an inclusive sum over 1024 of them, less the bin itself (the last bin of 1025 needs no more than that)
    const uint32_t own = tid < bins ? count[tid] : 0;
    sums[0][tid] = own;
    int cur = 0;
    for (uint32_t d = 1; d < 1024; d *= 2, cur ^= 1) {
        __syncthreads();
        sums[cur ^ 1][tid] = sums[cur][tid] + (tid >= d ? sums[cur][tid - d] : 0);
    }
    __syncthreads();
    if (tid < bins)
        count[tid] = sums[cur][tid] - own;
    if (tid == 0 && bins > 1024)
        count[1024] = sums[cur][1023];
    __syncthreads();
    each([&](uint32_t i, int id) {
        const uint32_t at = place(i, id);
        if (i < p.rows)
            p.perm[at] = u32x2{i, id >= 0 && uint32_t(id) < p.adapters ? uint32_t(id) : ~0u};
    });
}

// ------------------------------------------------------------------------------------------------------------
// t = x A^T
// ------------------------------------------------------------------------------------------------------------

// Few rows: a workgroup for a row and 4 of its adapter's rows, its four waves a quarter of K each.
constexpr uint32_t kVecI = 4;
template <bool F16> __global__ __launch_bounds__(256) void shrink_vec(LoraP p)
{
    const uint32_t width = p.parts * p.rank, row = blockIdx.y, i0 = blockIdx.x * kVecI, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int a = adapter_of(p, row);
    if (a < 0)
        return;
    const uint16_t* x = p.x + int64_t(row) * p.ldx;
    const uint16_t* w = p.a + (int64_t(a) * width + i0) * p.K;
    float s[kVecI] = {};
#pragma unroll 2
    for (uint32_t k = threadIdx.x * 8; k < p.K; k += 2048) {
        float xf[8];
        widen8<F16>(*reinterpret_cast<const u32x4*>(x + k), xf);
#pragma unroll
        for (uint32_t i = 0; i < kVecI; ++i) {
            float wf[8];
            widen8<F16>(*reinterpret_cast<const u32x4*>(w + int64_t(i) * p.K + k), wf);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                s[i] = fmaf(xf[j], wf[j], s[i]);
        }
    }
    __shared__ float red[4][kVecI];
#pragma unroll
    for (uint32_t i = 0; i < kVecI; ++i) {
        const float v = wave_sum(s[i]);
        if (lane == 0)
            red[wave][i] = v;
    }
    __syncthreads();
    if (threadIdx.x < kVecI)
        p.t[int64_t(row) * width + i0 + threadIdx.x] =
            (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// Very few rows: both products in one launch. A workgroup for a row, a part and 1024 of its columns makes the part's t by itself, 8
// values at a time over all of K, and goes on with its columns: A is read again for every 1024 columns, but a launch (2 to 3 us on
// the host and the device each) is saved.
constexpr uint32_t kOneThreads = 512, kOneCols = 2 * kOneThreads;
template <bool F16, uint32_t CT> __global__ __launch_bounds__(kOneThreads) void one_kernel(LoraP p)
{
    const uint32_t row = blockIdx.y, per = p.N / p.parts, chunks = (per + kOneCols - 1) / kOneCols;
    const uint32_t part = blockIdx.x / chunks, col = blockIdx.x % chunks * kOneCols + threadIdx.x * 2, n = part * per + col;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int a = adapter_of(p, row);
    __shared__ float red[kOneThreads / 64][8];
    __shared__ float st[256];
    if (a >= 0) {
        const uint16_t* x = p.x + int64_t(row) * p.ldx;
        const uint16_t* w = p.a + (int64_t(a) * p.parts + part) * p.rank * p.K;
        for (uint32_t i = 0; i < p.rank; i += 8, w += 8 * int64_t(p.K)) {
            float s[8] = {};
            for (uint32_t k = threadIdx.x * 8; k < p.K; k += kOneThreads * 8) {
                u32x4 wv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    wv[e] = *reinterpret_cast<const u32x4*>(w + int64_t(e) * p.K + k);
                float xf[8];
                widen8<F16>(*reinterpret_cast<const u32x4*>(x + k), xf);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float wf[8];
                    widen8<F16>(wv[e], wf);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        s[e] = fmaf(xf[j], wf[j], s[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                s[e] = wave_sum(s[e]);
            if (lane == 0)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    red[wave][e] = s[e];
            __syncthreads();
            if (threadIdx.x < 8) {
                float v = 0.0f;
#pragma unroll
                for (uint32_t q = 0; q < kOneThreads / 64; ++q)
                    v += red[q][threadIdx.x];
                st[i + threadIdx.x] = v;
            }
            __syncthreads();
        }
    }
    if (col >= per) // (per is a multiple of 8)
        return;
    float v[2] = {};
    if (a >= 0) {
        const uint16_t* w = p.b + (int64_t(a) * p.N + n) * p.rank;
        const float scale = p.scale ? p.scale[a] : 1.0f;
#pragma unroll 2
        for (uint32_t j = 0; j < p.rank; j += 8)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float wf[8];
                widen8<F16>(*reinterpret_cast<const u32x4*>(w + c * p.rank + j), wf);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[c] = fmaf(st[j + e], wf[e], v[c]);
            }
        v[0] *= scale;
        v[1] *= scale;
    }
    if (p.base) {
        v[0] += load_c<CT>(p.base, int64_t(row) * p.ldbase + n);
        v[1] += load_c<CT>(p.base, int64_t(row) * p.ldbase + n + 1);
    }
    const int64_t at = int64_t(row) * p.ldc + n;
    if constexpr (CT == MK_F32) {
        static_cast<float*>(p.c)[at] = v[0];
        static_cast<float*>(p.c)[at + 1] = v[1];
    } else {
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.c) + at) = pack_x2(v[0], v[1], CT == MK_F16);
    }
}

// Many rows: a tile of 64 rows by 32 NB of A's rows and one split of K. Each of the four waves takes every fourth 32 k for the
// whole tile, through three stages of LDS of its own (direct loads, two steps ahead, no barriers in the loop; nothing is read
// from LDS twice), and the waves' sums are added at the end. A tile with rows of several adapters goes through K for each.
// 16401 rows of 12288, rank 64: 117 to 134 us, 3.0 to 3.4 TB/s of x, of 3.6 to 4.0 TB/s that a reduction's reads reach. No faster: two or four
// stages, 128 rows a tile (160 us), a line of 128 bytes a row and wave, K begun elsewhere in every tile, and all tiles' steps
// shared evenly by as many workgroups as the chip holds (139 us, and more partial results to add).
constexpr int kStepK = 128;
template <bool F16, int NB> __global__ __launch_bounds__(256) void shrink_tile(LoraP p)
{
    constexpr int XB = kRows * 64, AB = NB * 2048, WB = XB + AB;   // bytes of a wave's stage
    constexpr int NX = XB / 1024, ND = WB / 1024;                 // direct loads of x, of both
    __shared__ __attribute__((aligned(16))) uint8_t s0[4 * WB], s1[4 * WB], s2[4 * WB];
    const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, hk = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t width = p.parts * p.rank, row0 = blockIdx.x * kRows, rows = min(p.rows - row0, uint32_t(kRows));
    const uint32_t split = blockIdx.y % p.splits, i0 = blockIdx.y / p.splits * (32 * NB);
    const uint32_t kb = split * p.split_k, ke = min(p.K, kb + p.split_k);
    const int steps = int((ke - kb + kStepK - 1) / kStepK);
    // lane's row of the tile, from the first row of the resource on, and its adapter
    uint32_t src;
    int mine = row_at(p, row0, min(uint32_t(lane), rows - 1), src);
    mine = uint32_t(lane) < rows ? mine : -1;

    const BufRes rx = buf_res(p.perm ? p.x : p.x + int64_t(row0) * p.ldx, uint32_t(((p.perm ? p.rows - 1 : rows - 1) * p.ldx + p.K) * 2));
    // byte offset of a lane's 16 bytes of each load, and their k: LDS rows of 64 bytes whose chunk c holds k chunk
    // c ^ ((row >> 2) & 3), so the 16-byte fragment reads of 8 rows fall on all banks
    uint32_t off[ND];
    const uint32_t kof = uint32_t(wave * 32 + ((lane & 3) ^ ((lane >> 4) & 3)) * 8); // ((row >> 2) & 3 of row 16 j + lane / 4)
#pragma unroll
    for (int j = 0; j < ND; ++j) {
        const uint32_t r = uint32_t((j < NX ? j : j - NX) * 16 + lane / 4);
        off[j] = j < NX ? uint32_t(__shfl(src, int(r))) * uint32_t(p.ldx) * 2 : min(r, width - i0 - 1) * p.K * 2;
    }
    for (int a = next_adapter(mine, -1); a != 0x7fffffff; a = next_adapter(mine, a)) {
        const BufRes ra = buf_res(p.a + (int64_t(a) * width + i0) * p.K, uint32_t(min(uint32_t(32 * NB), width - i0) * p.K * 2));
        auto issue = [&](int s, uint8_t* buf) {
            // behind the split's end: past the resource, so zeros come
            const uint32_t k = kb + uint32_t(s) * kStepK + kof;
#pragma unroll
            for (int j = 0; j < ND; ++j)
                buf_load_lds16(j < NX ? rx : ra, (lds_void*)(buf + wave * WB + j * 1024), k < ke ? off[j] + k * 2 : kOut, 0);
        };
        f32x16 acc[2][NB];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[i][j] = f32x16{};
        auto step = [&](int s, uint8_t* cur, uint8_t* into) {
            if (s >= steps)
                return;
            issue(s + 2, into);
            __builtin_amdgcn_s_waitcnt(wait_vm(2 * ND)); // step s landed, the next two may be in flight
            const uint8_t* b = cur + wave * WB;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const int at = (((ks * 2 + hk) ^ ((r32 >> 2) & 3)) << 4) + r32 * 64;
                u32x4 xf[2], af[NB];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    xf[i] = *reinterpret_cast<const u32x4*>(b + at + i * 2048);
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    af[j] = *reinterpret_cast<const u32x4*>(b + XB + at + j * 2048);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        acc[i][j] = mfma_32x32x16<F16>(af[j], xf[i], acc[i][j]);
            }
        };
        issue(0, s0);
        issue(1, s1);
        for (int s = 0; s < steps; s += 3) {
            step(s, s0, s2);
            step(s + 1, s1, s0);
            step(s + 2, s2, s1);
        }
        __builtin_amdgcn_s_waitcnt(0); // the last (unused) loads land before the LDS is reused
        // the waves' sums: a lane's values 4 g .. 4 g + 3 are A rows 8 g + 4 hk .. + 3 of x row r32
        float* red = reinterpret_cast<float*>(s0);
        constexpr int JB = 4 * WB / 16384 < NB ? 4 * WB / 16384 : NB; // 32 x 32 sums of the four waves that a stage holds
#pragma unroll
        for (int ij = 0; ij < 2 * NB; ij += JB) {
            __syncthreads();
#pragma unroll
            for (int q = ij; q < ij + JB && q < 2 * NB; ++q) {
                const f32x16& v = acc[q / NB][q % NB];
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4*>(red + ((((q - ij) * 4 + wave) * 4 + g) * 64 + lane) * 4) =
                        f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            }
            __syncthreads();
#pragma unroll
            for (int q = ij; q < ij + JB && q < 2 * NB; ++q) {
                f32x4 v = *reinterpret_cast<const f32x4*>(red + (((q - ij) * 16 + wave) * 64 + lane) * 4);
#pragma unroll
                for (int w = 1; w < 4; ++w)
                    v += *reinterpret_cast<const f32x4*>(red + ((((q - ij) * 4 + w) * 4 + wave) * 64 + lane) * 4);
                const uint32_t r = q / NB * 32 + r32, n = i0 + q % NB * 32 + wave * 8 + hk * 4;
                const uint32_t row = row_base(p, row0) + uint32_t(__shfl(int(src), int(r)));
                if (__shfl(mine, int(r)) == a && n < width)
                    *reinterpret_cast<f32x4*>(p.t + (int64_t(split) * p.rows + row) * width + n) = v;
            }
        }
        __syncthreads(); // before the next adapter's loads
    }
}

// ------------------------------------------------------------------------------------------------------------
// c = base + scale t B^T
// ------------------------------------------------------------------------------------------------------------

// the sum of the splits' partial t, 4 of a row, in their order; 8 loads at a time (one after the other, 16 splits took 8 us)
__device__ inline f32x4 load_t(const LoraP& p, uint32_t row, uint32_t i)
{
    const int64_t width = int64_t(p.parts) * p.rank, step = p.rows * width;
    const float* t = p.t + row * width + i;
    f32x4 v = *reinterpret_cast<const f32x4*>(t);
    for (uint32_t s = 1; s < p.splits; s += 8) {
        f32x4 w[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            w[j] = *reinterpret_cast<const f32x4*>(t + min(s + j, p.splits - 1) * step);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (s + j < p.splits)
                v += w[j];
    }
    return v;
}
// 4 values through a buffer resource; past it zeros come, and nothing is stored
template <class V> __device__ inline V load_v(BufRes r, uint32_t voff, uint32_t soff)
{
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (sizeof(V) == 16)
        return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, int(voff), int(soff), 0));
    else
        return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, int(voff), int(soff), 0));
#else
    return V{};
#endif
}
// (A 16-byte store's offset is in one register, with no scalar beside it: its data must not be overwritten by the very next
// instruction, and the compiler keeps them apart only in that form. With a scalar offset, the first values of the last
// store of a tile came out as what the next instruction wrote, in some lanes and now and then.) Non-temporal: c is many times a cache,
// and leaves base and x room in it (us with / without: 16384 x 4096 to 4096 by rank 16 95 / 107, 16401 x 12288 to 4096 in fp32 252 /
// 263, 4352 x 4096 to 12288 76 / 78; with the projection before and the rotary positions behind it the same). Base loaded so
// is faster where it comes from memory (241) and slower where the projection has just stored it; x loaded so is slower.
template <class V> __device__ inline void store_v(V v, BufRes r, uint32_t voff)
{
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (sizeof(V) == 16)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, int(voff), 0, 2);
    else
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), r, int(voff), 0, 2);
#endif
}

// Few rows: a thread a value.
template <bool F16, uint32_t CT> __global__ __launch_bounds__(256) void expand_vec(LoraP p)
{
    const uint32_t row = blockIdx.y, per = p.N / p.parts, groups = (per + 255) / 256;
    const uint32_t part = blockIdx.x / groups, col = blockIdx.x % groups * 256 + threadIdx.x, n = part * per + col;
    const int a = adapter_of(p, row);
    __shared__ __attribute__((aligned(16))) float st[256];
    if (a >= 0 && threadIdx.x * 4 < p.rank)
        *reinterpret_cast<f32x4*>(st + threadIdx.x * 4) = load_t(p, row, part * p.rank + threadIdx.x * 4);
    __syncthreads();
    if (col >= per)
        return;
    float v = 0.0f;
    if (a >= 0) {
        const uint16_t* w = p.b + (int64_t(a) * p.N + n) * p.rank;
#pragma unroll 2
        for (uint32_t j = 0; j < p.rank; j += 8) {
            float wf[8];
            widen8<F16>(*reinterpret_cast<const u32x4*>(w + j), wf);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v = fmaf(st[j + e], wf[e], v);
        }
        if (p.scale)
            v *= p.scale[a];
    }
    if (p.base)
        v += load_c<CT>(p.base, int64_t(row) * p.ldbase + n);
    const int64_t at = int64_t(row) * p.ldc + n;
    if constexpr (CT == MK_F32)
        static_cast<float*>(p.c)[at] = v;
    else
        static_cast<uint16_t*>(p.c)[at] = CT == MK_F16 ? f2h_bits(v) : f2bf_bits(v);
}

// Many rows: a workgroup has 64 rows of one part; its waves go through blocks of 128 columns. t is in LDS as 2 or 3 values
// of the inputs' type (v = v0 + v1 (+ v2), each the rounding of what is left: 2^-16 of t, or 2^-24 with three, for fp32
// outputs; half t after a power of two that puts the row's largest near 2^14, so that none is lost below the half range). In the product C = T B^T a wave's
// four column tiles take columns 4 j + tile: a lane then has 4 columns next to each other of each of its rows, and base and c
// go by 8 or 16 bytes a lane, 256 or 512 next to each other.
// FUSE: both 32-row halves of the tile at once, so that B is read once.
template <bool F16, uint32_t CT, bool FUSE> __global__ __launch_bounds__(256, 2) void expand_tile(LoraP p)
{
    constexpr int NV = CT == MK_F32 && !F16 ? 3 : 2;
    constexpr uint32_t SZ = CT == MK_F32 ? 4 : 2;
    typedef std::conditional_t<CT == MK_F32, u32x4, u32x2> V; // 4 values of c
    extern __shared__ __attribute__((aligned(16))) uint16_t st[]; // [NV][64][pad], then a factor a row
    __shared__ __attribute__((aligned(16))) uint32_t row_b[kRows], row_c[kRows]; // the rows' byte offsets in base and c
    const uint32_t tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, hk = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t row0 = blockIdx.x * kRows, rows = min(p.rows - row0, uint32_t(kRows));
    const uint32_t per = p.N / p.parts, span = 512 * p.blocks, groups = (per + span - 1) / span;
    const uint32_t part = blockIdx.y / groups, first = blockIdx.y % groups * span;
    const uint32_t depth = (p.rank + 15) / 16 * 16, pad = depth + 8; // (rows 16 bytes off each other's banks)
    float* factor = reinterpret_cast<float*>(st + NV * kRows * pad);
    uint32_t src;
    int mine = row_at(p, row0, min(lane, rows - 1), src);
    mine = lane < rows ? mine : -2;
    row_b[lane] = src * uint32_t(p.ldbase) * SZ; // (every wave writes the same)
    row_c[lane] = src * uint32_t(p.ldc) * SZ;
    {
        // 4 threads a row, t's values 4 (q + 4 i) .. + 3 of it in each
        const uint32_t r = tid / 4, q = tid % 4, row = row_base(p, row0) + uint32_t(__shfl(int(src), int(r)));
        const bool on = __shfl(mine, int(r)) >= 0;
        float top = 0.0f;
        if constexpr (F16) {
            if (on)
                for (uint32_t i = q * 4; i < p.rank; i += 16) {
                    const f32x4 v = load_t(p, row, part * p.rank + i);
                    top = fmaxf(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), top);
                }
            top = fmaxf(top, __shfl_xor(top, 1));
            top = fmaxf(top, __shfl_xor(top, 2));
        }
        float up = 1.0f, down = 1.0f;
        if (F16 && top > 0.0f && top < __builtin_inff()) {
            const int e = min(14 - ilogbf(top), 100);
            up = ldexpf(1.0f, e);
            down = ldexpf(1.0f, -e);
        }
        if (q == 0)
            factor[r] = down;
        for (uint32_t i = q * 4; i < depth; i += 16) {
            const f32x4 v = on && i < p.rank ? load_t(p, row, part * p.rank + i) : f32x4{};
            float rest[4] = {v[0] * up, v[1] * up, v[2] * up, v[3] * up};
#pragma unroll
            for (int s = 0; s < NV; ++s) {
                const u32x2 h{pack_x2(rest[0], rest[1], F16), pack_x2(rest[2], rest[3], F16)};
                *reinterpret_cast<u32x2*>(st + (s * kRows + r) * pad + i) = h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (an infinity's or a NaN's rest is nothing)
                    const float d = rest[e] - widen<F16>(uint16_t(h[e / 2] >> (16 * (e % 2))));
                    rest[e] = fabsf(d) < __builtin_inff() ? d : 0.0f;
                }
            }
        }
    }
    __syncthreads();
    for (int a = next_adapter(mine, -2); a != 0x7fffffff; a = next_adapter(mine, a)) {
        if (a < 0 && p.base == p.c)
            continue; // rows without an adapter, in place
        const float scale = a >= 0 && p.scale ? p.scale[a] : 1.0f;
        const uint64_t on = __ballot(mine == a); // the adapter's rows of the tile
        for (uint32_t blk = 0; blk < p.blocks; ++blk) {
            const uint32_t c0 = first + (blk * 4 + wave) * 128; // column of the part
            if (c0 >= per)
                break;
            const uint32_t col = c0 + r32 * 4;
            const bool in = col < per; // (per is a multiple of 8: all 4 of a lane's columns, or none)
            // A lane's rows of a 32-row half are 8 (i / 4) + 4 hk + i % 4. Their base and c by buffer loads and stores at the rows'
            // byte offsets; what is not the adapter's goes past the resource.
            auto row_of = [](int i) { return uint32_t(8 * (i / 4) + i % 4); };
            auto has_of = [&](uint32_t rt) { return in ? uint32_t(on >> (32 * rt)) >> (4 * hk) : 0u; };
            auto res_of = [&](const void* x, int64_t ld) {
                return buf_res(static_cast<const char*>(x) + ((p.perm ? 0 : int64_t(row0)) * ld + part * per) * SZ,
                               x ? uint32_t(((p.perm ? p.rows : rows) - 1) * ld + per) * SZ : 0u);
            };
            auto load_base = [&](uint32_t rt, V (&basev)[16]) {
                const BufRes rb = res_of(p.base, p.ldbase);
                const uint32_t has = has_of(rt);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    basev[i] = load_v<V>(rb, has >> row_of(i) & 1 ? row_b[rt * 32 + 4 * hk + row_of(i)] + col * SZ : kOut, 0);
            };
            // RT halves from half rt on at a time: what B costs is shared by them
            auto multiply = [&](uint32_t rt, auto& acc) {
                constexpr int RT = sizeof(acc) / sizeof(acc[0]);
#pragma unroll
                for (int h = 0; h < RT; ++h)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[h][t] = f32x16{};
                if (a < 0)
                    return;
                // k steps in groups of 4, 2 or 1: half wave hk takes 8 G ranks next to each other of the group's 16 G (of B and of
                // t alike), so a row of B is read by whole lines
                const uint16_t* w = p.b + (int64_t(a) * p.N + part * per + col) * p.rank;
                const uint16_t* tv = st + (rt * 32 + r32) * pad;
                auto group = [&](uint32_t k, auto g_c) {
                    constexpr int G = decltype(g_c)::value;
                    const uint32_t at = k + hk * (8 * G);
                    u32x4 bf[4][G];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int q = 0; q < G; ++q) {
                            bf[t][q] = u32x4{};
                            if (in && at + q * 8 < p.rank)
                                bf[t][q] = *reinterpret_cast<const u32x4*>(w + t * p.rank + at + q * 8);
                        }
#pragma unroll
                    for (int q = 0; q < G; ++q)
#pragma unroll
                        for (int s = NV - 1; s >= 0; --s)
#pragma unroll
                            for (int h = 0; h < RT; ++h) {
                                const u32x4 tf = *reinterpret_cast<const u32x4*>(tv + (s * kRows + h * 32) * pad + at + q * 8);
#pragma unroll
                                for (int t = 0; t < 4; ++t)
                                    acc[h][t] = mfma_32x32x16<F16>(tf, bf[t][q], acc[h][t]);
                            }
                };
                uint32_t k = 0;
                if constexpr (RT == 1)
#pragma unroll 1
                    for (; k + 64 <= depth; k += 64)
                        group(k, std::integral_constant<int, 4>{});
#pragma unroll 1
                for (; k + 32 <= depth; k += 32)
                    group(k, std::integral_constant<int, 2>{});
                if (k < depth)
                    group(k, std::integral_constant<int, 1>{});
            };
            auto finish = [&](uint32_t rt, const f32x16 (&acc)[4], const V (&basev)[16]) {
                const BufRes rc = res_of(p.c, p.ldc);
                const uint32_t has = has_of(rt);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float f = scale * factor[rt * 32 + 4 * hk + row_of(i)];
                    float v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        float o;
                        if constexpr (CT == MK_F32)
                            o = __builtin_bit_cast(float, uint32_t(basev[i][t]));
                        else
                            o = widen<CT == MK_F16>(uint16_t(basev[i][t / 2] >> (16 * (t % 2))));
                        v[t] = a >= 0 ? fmaf(acc[t][i], f, o) : o;
                    }
                    V out;
                    if constexpr (CT == MK_F32)
                        out = __builtin_bit_cast(V, f32x4{v[0], v[1], v[2], v[3]});
                    else
                        out = V{pack_x2(v[0], v[1], CT == MK_F16), pack_x2(v[2], v[3], CT == MK_F16)};
                    store_v(out, rc, has >> row_of(i) & 1 ? row_c[rt * 32 + 4 * hk + row_of(i)] + col * SZ : kOut);
                }
            };
            if constexpr (FUSE) {
                f32x16 acc[2][4];
                multiply(0, acc);
#pragma unroll
                for (uint32_t rt = 0; rt < 2; ++rt) {
                    V basev[16];
                    load_base(rt, basev);
                    finish(rt, acc[rt], basev);
                }
            } else {
#pragma unroll 1
                for (uint32_t rt = 0; rt < 2; ++rt) {
                    if (!uint32_t(on >> (32 * rt)))
                        continue;
                    V basev[16];
                    f32x16 acc[1][4];
                    load_base(rt, basev);
                    multiply(rt, acc);
                    finish(rt, acc[0], basev);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------------------

// sizes and types, for the call and for its workspace's size
mk_status check_sizes(const mk_lora_rows_args* a)
{
    if (a->dtype != MK_BF16 && a->dtype != MK_F16)
        return fail(MK_ERR_ARG, "lora_rows: x, a and b must be bf16 or f16");
    if (a->c_dtype != MK_F32 && a->c_dtype != MK_BF16 && a->c_dtype != MK_F16)
        return fail(MK_ERR_ARG, "lora_rows: base and c must be f32, bf16 or f16");
    if (!a->parts || a->parts > 4 || !a->rank || a->rank % 8 || a->rank > 256 || !a->adapters || a->adapters > 0x7fffffffu)
        return fail(MK_ERR_ARG, "lora_rows: 1 to 4 parts of rank a multiple of 8 up to 256, 1 adapter or more");
    if (!a->K || a->K % 8 || a->K > (1u << 22) || !a->N || a->N % (8 * a->parts) || a->N > (1u << 22))
        return fail(MK_ERR_ARG, "lora_rows: K must be a multiple of 8, N of 8 parts, up to 2^22");
    if (a->rows > (1u << 28)) // (64 rows a workgroup of 256: 2^30 threads)
        return fail(MK_ERR_ARG, "lora_rows: more than 2^28 rows");
    return MK_OK;
}

// How the two products run, by the sizes alone (on `cus` compute units; `room` bytes of workspace bound the splits of K).
struct Plan {
    bool one;           // both products in one launch (very few rows)
    bool order;         // rows are taken in the order of their adapters
    bool vec1, vec2;    // else a workgroup a row (few rows) or tiles of 64 rows, each
    uint32_t nb;        // the first product's tiles: 32 nb of A's rows
    uint32_t splits, split_k;
    uint32_t blocks;
    bool fuse;          // both halves of a tile share what they read of B
};
// t, and the rows' order
uint64_t bytes_of_t(const mk_lora_rows_args* a, uint32_t splits)
{
    return round_up(uint64_t(splits) * a->rows * a->parts * a->rank * 4, 16);
}
uint64_t workspace_of(const mk_lora_rows_args* a, uint32_t splits) { return bytes_of_t(a, splits) + round_up(uint64_t(a->rows) * 8, 16); }
Plan plan_of(const mk_lora_rows_args* a, uint32_t cus, uint64_t room)
{
    Plan p{};
    const uint32_t width = a->parts * a->rank, chunks = cdiv(width, 128), tiles = cdiv(a->rows, kRows);
    const uint64_t macs = uint64_t(a->rows) * width * a->K, macs2 = uint64_t(a->rows) * a->N * a->rank;
    const uint32_t per = a->N / a->parts;
    // (its 8 values of t at a time take 1.3 us for every 4096 k: us in two launches / in one, on the device alone, of 1 row of 4096 to 4096
    // by rank 16 5.7 / 5.2, of 32 by rank 32 6.9 / 9.1, of 64 by rank 16 5.9 / 5.1 in runs and 6.5 / 5.6 in no order, of 256 x 1280 to 5120 6.8 /
    // 4.7 and 9.1 / 11.6. 24 rows of 16 adapters to 3 x 4096 by rank 16 6.5 / 8.0, but 9.4 / 8.9 a call through the Python binding, whose
    // time is the host's: one launch, and a captured graph of that call is the slower for it.)
    const uint64_t again = uint64_t(a->rows) * a->parts * cdiv(per, kOneCols) * a->rank * a->K;
    p.one = a->rows <= 1024 && a->rank / 8 * cdiv(a->K, 8 * kOneThreads) <= 2 && again <= (1u << 25);
    // us by rows / by tiles in runs that are said to be grouped, and in no order (8 adapters, sorted for the tiles): 512 x 4096 to 4096 by
    // rank 16 (2^25 products each) 9.6 / 14.2, 14 / 29; 1024 (2^26) 24 / 14, 27 / 28; 512 x 1280 to 3840 by rank 32 in 3 parts (2^25.9)
    // 10 / 17, 22 / 37; 1024 (2^26.9) 17 / 17, 42 / 34; 256 x 4096 to 12288 by rank 32 in 3 parts (2^26.6) 20 / 20, 31 / 40; 2048 x 12288
    // to 4096 by rank 64 228 / 30, 261 / 59.
    p.vec1 = a->rows <= 4096 && macs < (1u << 26);
    p.vec2 = a->rows <= 4096 && macs2 < (1u << 26);
    // Where a product goes by tiles, the other one by rows or not (us in no order without / with, and in runs, where finding that out
    // is all it does: 2000 x 1280 to 5120 by rank 16 58 / 35 and 24 / 27, 2000 x 256 to 12288 99 / 46 and 35 / 38, 600 x 12288 to 640 32 / 22 and
    // 14 / 19; byte offsets from the first row on are below 2^31).
    const int64_t far = std::max(p.vec1 ? 0 : a->ldx * 2, p.vec2 ? 0 : std::max(a->base ? a->ldbase : 0, a->ldc) * (a->c_dtype == MK_F32 ? 4 : 2)) * a->rows;
    p.order = !p.one && !(p.vec1 && p.vec2) && a->ids && !a->grouped && a->adapters > 1 && a->adapters <= kMaxOrdered && a->rows <= (1u << 18) && far < (1ll << 31);
    p.nb = cdiv(cdiv(width, chunks), 32);
    p.splits = 1;
    p.split_k = uint32_t(round_up(a->K, kStepK));
    if (!p.vec1) {
        // a workgroup a compute unit at a time: the fewest rounds of the shortest splits; a split's start and end, and its
        // partial t, cost about 4 steps (us of both products with splits / without: 2048 x 12288 to 4096 by rank 64 28 / 69, 4352 x 4096
        // to 12288 by rank 32 83 / 101, 16384 x 4096 to 4096 by rank 16 109 / 110)
        const uint32_t steps = cdiv(a->K, kStepK);
        const uint64_t groups = uint64_t(tiles) * chunks;
        double best = 1e30;
        for (uint32_t s = 1; s <= 16 && s <= steps; ++s) {
            const uint32_t each = cdiv(steps, s), used = cdiv(steps, each);
            if (used > 1 && workspace_of(a, used) > room)
                break;
            const double cost = double((groups * used + cus - 1) / cus) * (each + 4.0);
            if (cost < best * 0.97) {
                best = cost;
                p.splits = used;
                p.split_k = each * kStepK;
            }
        }
    }
    // More blocks a workgroup while the chip keeps at least four workgroups a compute unit: t is split up once for all of them (us
    // with up to 4 / with 1: 16384 x 4096 to 4096 by rank 16 109 / 116, to 12288 by rank 32 in no order 320 / 333, to 12288 by rank
    // 128 402 / 391; 4352 rows have one at any rate: two there took 58 us for 54, four 77).
    p.blocks = 1;
    while (p.blocks < 4 && p.blocks * 512 < per && uint64_t(tiles) * a->parts * cdiv(per, 1024 * p.blocks) >= 4ull * cus)
        p.blocks *= 2;
    // from rank 64 on B is the most of what a tile reads (us apart / shared by its two halves: 16384 x 12288 by rank 128 430 / 383
    // with the first product, 4352 x 4096 by 64 49.3 / 47.6)
    p.fuse = a->rank >= 64;
    return p;
}

template <bool F16, uint32_t CT> void launch_one(const LoraP& p, hipStream_t s)
{
    one_kernel<F16, CT><<<dim3(p.parts * cdiv(p.N / p.parts, kOneCols), p.rows), kOneThreads, 0, s>>>(p);
}
template <bool F16> void launch_shrink(const LoraP& p, const Plan& plan, hipStream_t s)
{
    const uint32_t width = p.parts * p.rank;
    if (plan.vec1) {
        shrink_vec<F16><<<dim3(width / kVecI, p.rows), 256, 0, s>>>(p);
        return;
    }
    const dim3 grid(cdiv(p.rows, kRows), cdiv(width, 32 * plan.nb) * p.splits);
    switch (plan.nb) {
    case 1: shrink_tile<F16, 1><<<grid, 256, 0, s>>>(p); break;
    case 2: shrink_tile<F16, 2><<<grid, 256, 0, s>>>(p); break;
    case 3: shrink_tile<F16, 3><<<grid, 256, 0, s>>>(p); break;
    default: shrink_tile<F16, 4><<<grid, 256, 0, s>>>(p); break;
    }
}
template <bool F16, uint32_t CT> void launch_expand(const LoraP& p, const Plan& plan, hipStream_t s)
{
    const uint32_t per = p.N / p.parts;
    if (plan.vec2) {
        expand_vec<F16, CT><<<dim3(p.parts * cdiv(per, 256), p.rows), 256, 0, s>>>(p);
        return;
    }
    const uint32_t pad = (p.rank + 15) / 16 * 16 + 8, values = CT == MK_F32 && !F16 ? 3 : 2;
    const dim3 grid(cdiv(p.rows, kRows), p.parts * cdiv(per, 512 * p.blocks));
    const uint32_t lds = (values * pad * 2 + 4) * kRows;
    if (plan.fuse)
        expand_tile<F16, CT, true><<<grid, 256, lds, s>>>(p);
    else
        expand_tile<F16, CT, false><<<grid, 256, lds, s>>>(p);
}

} // namespace

} // namespace mk

using namespace mk;

extern "C" {

mk_status mk_lora_rows_workspace(const mk_lora_rows_args* a, uint64_t* bytes)
{
    if (!a || !bytes)
        return fail(MK_ERR_ARG, "lora_rows_workspace: null argument");
    MK_TRY(check_sizes(a));
    *bytes = 0;
    if (!a->rows)
        return MK_OK;
    uint32_t cus = 1;
    MK_TRY(compute_units(cus));
    *bytes = workspace_of(a, plan_of(a, cus, UINT64_MAX).splits);
    return MK_OK;
}

mk_status mk_lora_rows_plan(const mk_lora_rows_args* a, uint32_t cus, uint32_t* out)
{
    if (!a || !out || !cus)
        return fail(MK_ERR_ARG, "lora_rows_plan: null argument or no compute units");
    MK_TRY(check_sizes(a));
    if (!a->rows)
        return fail(MK_ERR_ARG, "lora_rows_plan: no rows");
    const Plan p = plan_of(a, cus, a->workspace ? a->workspace_bytes : UINT64_MAX);
    const uint32_t o[6] = {p.one, p.one || p.vec1 ? 0 : 32 * p.nb, p.one || p.vec2 ? 0 : 512 * p.blocks, p.one || p.vec1 ? 1 : p.splits, p.order,
                           !p.one && !p.vec2 && p.fuse};
    std::copy(o, o + 6, out);
    return MK_OK;
}

mk_status mk_lora_rows(const mk_lora_rows_args* a, void* stream)
{
    if (!a)
        return fail(MK_ERR_ARG, "lora_rows: null argument");
    MK_TRY(check_sizes(a));
    // (a tile's 64 rows of x, or 32 of c, are addressed by 31 bits)
    auto bad = [](int64_t ld, uint32_t n) { return ld < int64_t(n) || ld % 8 || ld >= (1 << 23); };
    if (bad(a->ldx, a->K) || bad(a->ldc, a->N) || (a->base && bad(a->ldbase, a->N)))
        return fail(MK_ERR_ARG, "lora_rows: ldx, ldbase and ldc must be multiples of 8 below 2^23, at least the row");
    if (a->base && a->base == a->c && a->ldbase != a->ldc)
        return fail(MK_ERR_ARG, "lora_rows: in place needs ldbase == ldc");
    if (!aligned(a->x, 16) || !aligned(a->a, 16) || !aligned(a->b, 16) || !aligned(a->base, 16) || !aligned(a->c, 16) ||
        !aligned(a->workspace, 16) || !aligned(a->scale, 4) || !aligned(a->ids, 4))
        return fail(MK_ERR_ARG, "lora_rows: operands and workspace must be 16-byte aligned (scale and ids 4)");
    if (a->grouped > 1)
        return fail(MK_ERR_ARG, "lora_rows: grouped is 0 or 1");
    if (!a->rows)
        return MK_OK;
    if (!a->x || !a->a || !a->b || !a->c)
        return fail(MK_ERR_ARG, "lora_rows: null argument (x, a, b and c are required)");
    if (!a->workspace || a->workspace_bytes < workspace_of(a, 1))
        return fail(MK_ERR_ARG, "lora_rows: the workspace holds less than (4 parts rank + 8) rows bytes");
    uint32_t cus = 1;
    MK_TRY(compute_units(cus));
    const Plan plan = plan_of(a, cus, a->workspace_bytes);
    LoraP p{static_cast<const uint16_t*>(a->x), static_cast<const uint16_t*>(a->a), static_cast<const uint16_t*>(a->b), a->scale,
            a->ids, a->base, a->c, static_cast<float*>(a->workspace),
            plan.order ? reinterpret_cast<u32x2*>(static_cast<char*>(a->workspace) + bytes_of_t(a, plan.splits)) : nullptr,
            a->ldx, a->ldbase, a->ldc, a->rows, a->K, a->N, a->rank,
            a->parts, a->adapters, plan.splits, plan.split_k, plan.blocks};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto f16_c, auto ct_c) {
        constexpr bool H = decltype(f16_c)::value;
        constexpr uint32_t CT = decltype(ct_c)::value;
        if (plan.one) {
            launch_one<H, CT>(p, s);
            return;
        }
        if (plan.order)
            order_kernel<<<1, 1024, 0, s>>>(p);
        launch_shrink<H>(p, plan, s);
        launch_expand<H, CT>(p, plan, s);
    };
    auto with_c = [&](auto f16_c) {
        if (a->c_dtype == MK_F32)
            run(f16_c, std::integral_constant<uint32_t, MK_F32>{});
        else if (a->c_dtype == MK_BF16)
            run(f16_c, std::integral_constant<uint32_t, MK_BF16>{});
        else
            run(f16_c, std::integral_constant<uint32_t, MK_F16>{});
    };
    if (a->dtype == MK_F16)
        with_c(std::true_type{});
    else
        with_c(std::false_type{});
    MK_LAUNCH_CHECK("lora_rows");
    return MK_OK;
}

} // extern "C"
