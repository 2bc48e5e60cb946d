// mk_attention_packed: softmax attention of packed documents, with causal and prefix masks, a tanh cap and a distance bias.
//
// One pass over the keys with a running reference and sum of the softmax. A wave has 32 rows (of all heads that share a key head) and makes
// S^T = K Q^T, so that a lane holds one row's scores, which are the second product's operand as they are. Tiles of 64 keys come by direct
// loads into two LDS buffers; few rows over many keys are split over workgroups and joined by a second launch. Long documents are bound
// by the issue that matrix instructions and the exponentials share (2 x 4352 rows of 32 heads of 128 555 to 570 us, 1.1 PFLOP/s), one row
// over a cache by its reads (16411 keys of 8 heads of 128 17 us, 3.9 TB/s, and 5 to join), few keys by a workgroup's start and end.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <utility>
#include <vector>

namespace mk {

namespace {

constexpr uint32_t kMaxDocs = 64; // documents a launch: they go by kernel argument, in less than 4 KB
constexpr int kKT = 64;           // keys a tile
// The exponentials' reference m moves only when a weight against it passes 2^8, in half 2^15 (below). For half weights it lies 7 under
// the largest score, whose own weight is then 2^7, unrounded: a weight loses 2^-25 below half's normal range, so 2^-32 of the largest (with
// m the largest score itself, 2^17 keys of 2^-25.5 each, 0.3% of their row, came out as nothing). bf16 has fp32's range.
constexpr float kUp = 7.0f;
template <bool F16> constexpr float kLazyP = F16 ? 32768.0f : 256.0f;
constexpr float kLeast = -3.402823466e38f; // m of rows without a score above -inf
// |m| from which on scores are rounded before m is taken off them. Below it one fma does both, exact against any m (without a bias or
// a cap: with them s - m or cap - m is rounded first, by up to half a step of m, as a score in fp32 of m's size is); from 2^31 on half
// a step of m itself, which the largest weight would be off by, no longer fits a weight's exponent (a half's from 2^26).
constexpr float kLargeM = 16777216.0f;

struct Doc {
    uint32_t q_row, q_rows, k_row, k_rows;
    int32_t q_pos;
    uint32_t block, prefix;
    uint32_t blocks; // of 32 NW rows a key head
    uint32_t splits; // workgroups that share a block's keys
    uint32_t slot;   // its first partial result in the workspace, when splits > 1
};
struct PackedP {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    int64_t ldq, ldk, ldv, ldo;
    const float* slopes;
    float* part;    // workspace: [slot][NW][32 D] sums (part_at), then [slot][NW][32][2] m and l
    float* part_ml;
    float c;        // scale log2(e); with a cap: 2 scale log2(e) / cap
    float cap;      // cap log2(e)
    uint32_t kv_heads, group, n_docs, out_f16;
    uint32_t first[kMaxDocs]; // a document's first workgroup, a multiple of 8
    uint32_t join[kMaxDocs];  // and that of the second launch
    Doc docs[kMaxDocs];
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 4 x 16 values of 16 bits from LDS, transposed: 16 lanes read 4 rows of 16 next to each other, 4 a lane, and each gets a column
__device__ inline u32x2 read_tr(const uint16_t* p)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
#else
    return u32x2{};
#endif
}

// How many of a document's keys a row at position pos sees: they are the first ones under every mask.
__device__ inline int seen_keys(const Doc& d, int64_t pos)
{
    if (d.block == 0 || pos >= int64_t(d.block))
        return int(d.k_rows);
    int64_t n = pos + 1 > int64_t(d.prefix) ? pos + 1 : int64_t(d.prefix);
    n = n < int64_t(d.k_rows) ? n : int64_t(d.k_rows);
    return int(n > 0 ? n : 0);
}
// The document of a workgroup, by its place among their first ones (`table`: at most 64, ascending, the first 0), and that first
// one. Arguments come from host memory, 2 us and more a round trip, so a lane reads each place and document in one go: a
// search by halves took several, the place and then the document two (6453 rows over three documents 21.9 us, 21.1 so).
__device__ inline Doc find_doc(const PackedP& p, const uint32_t (&table)[kMaxDocs], uint32_t item, uint32_t& first)
{
    static_assert(kMaxDocs <= 64, "one a lane");
    if (p.n_docs == 1) {
        first = 0;
        return p.docs[0];
    }
    const uint32_t lane = threadIdx.x & 63, i = min(lane, p.n_docs - 1), at = table[i];
    const Doc d = p.docs[i];
    const int of = int(__popcll(__ballot(lane < p.n_docs && at <= item))) - 1;
    auto get = [&](uint32_t v) { return uint32_t(__builtin_amdgcn_readlane(int(v), of)); };
    first = get(at);
    return Doc{get(d.q_row), get(d.q_rows), get(d.k_row), get(d.k_rows), int32_t(get(uint32_t(d.q_pos))), get(d.block), get(d.prefix),
               get(d.blocks), get(d.splits), get(d.slot)};
}

// Where 4 dims (chunk) of one of a wave's 32 rows are in its partial results: with many rows the rows of a chunk next to each
// other, as a wave holds them (1 KB a store: by rows, 16 bytes a lane 512 apart, was half as fast), with few by rows.
template <int D, int NW> __device__ inline uint32_t part_at(uint32_t chunk, uint32_t r)
{
    return NW == 1 ? r * D + chunk * 4 : (chunk * 32 + r) * 4;
}

enum { kPlain = 0, kBias = 1, kCap = 2 /* a bit each */ };

// Waves a SIMD that the registers have to leave room for. (Heads of 64 fit three, us of 20 heads, two documents of 4096, with
// three / with two: with a bias 221 / 243, capped 304 / 329, neither the same. Heads of 128 would spill.)
constexpr int waves_of(int d, int nw) { return nw == 1 ? 1 : d == 64 ? 3 : 2; }

template <int D, bool F16, int MODE, int NW>
__global__ __launch_bounds__(64 * NW, waves_of(D, NW)) __attribute__((amdgpu_waves_per_eu(waves_of(D, NW), waves_of(D, NW)))) void packed_kernel(PackedP p)
{
    constexpr int DS = D / 16, DT = D / 32, KC = D / 8; // k steps of S, 32-dim blocks of O, 16-byte chunks of a row
    constexpr int RL = kKT * KC / (64 * NW);            // direct loads a wave and operand
    constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
    // the two buffers are separate objects, so that the compiler can tell a load into one from the reads of the other
    __shared__ __attribute__((aligned(16))) uint16_t sK0[kKT * D], sK1[kKT * D], sV0[kKT * D], sV1[kKT * D];
    __shared__ int odd_tile; // 1 + the last tile in which find_odd found any
    // there: which of a lane's weights of a half are not zero, those of pair j in bits j and 16 + j (not in registers, which are full)
    __shared__ uint32_t weighty[2][64 * NW];
    auto sK = [&](int b) { return b ? sK1 : sK0; };
    auto sV = [&](int b) { return b ? sV1 : sV0; };

    const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, hk = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t doc_first;
    const Doc doc = find_doc(p, p.first, blockIdx.x, doc_first);
    // Workgroup i runs on XCD i % 8: each XCD takes a run of a document's (key head, block, split), whose blocks share keys in
    // its L2; later blocks, which see more under a causal mask, come first.
    const uint32_t each = doc.blocks * doc.splits, real = each * p.kv_heads, run = (real + 7) / 8;
    const uint32_t local = blockIdx.x - doc_first, item = local % 8 * run + local / 8;
    if (local / 8 >= run || item >= real)
        return;
    const uint32_t kvh = item / each, block = doc.blocks - 1 - item % each / doc.splits, split = item % doc.splits;

    // rows of a block: (query row, head of the group) pairs, so that all heads of a key head share its tiles
    const uint32_t rows = doc.q_rows * p.group, wg0 = block * (32 * NW), w0 = wg0 + wave * 32;
    const uint32_t wg_last = min(wg0 + 32 * NW, rows) - 1, row = min(w0 + r32, rows - 1);
    const uint32_t qi = row / p.group, head = kvh * p.group + row % p.group;
    const int64_t pos = int64_t(doc.q_pos) + qi;
    const int lim = seen_keys(doc, pos);
    const int64_t wg_pos = int64_t(doc.q_pos) + wg0 / p.group;
    const int wg_lim = seen_keys(doc, wg_pos); // of the workgroup's first row: the least
    const int wave_most = seen_keys(doc, int64_t(doc.q_pos) + min(w0 + 31, rows - 1) / p.group);
    const int all_tiles = (uint32_t(seen_keys(doc, int64_t(doc.q_pos) + wg_last / p.group)) + kKT - 1) / kKT;
    const int t_begin = int(uint64_t(all_tiles) * split / doc.splits), t_end = int(uint64_t(all_tiles) * (split + 1) / doc.splits);

    u32x4 qf[DS];
    {
        const uint16_t* Q = p.q + (int64_t(doc.q_row) + qi) * p.ldq + int64_t(head) * D;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
            qf[ds] = *reinterpret_cast<const u32x4*>(Q + ds * 16 + hk * 8);
    }
    // LDS chunks: K's so that 16 keys' fragment reads fall on all banks, V's so that the 64 bytes of 4 keys that a transposing
    // read takes do
    auto kswz = [](int key, int c) { return KC == 16 ? c ^ (key & 15) : c ^ ((key >> 1) & 7); };
    auto vswz = [](int key, int c) { return KC == 16 ? c ^ ((key & 3) << 2) : c ^ ((key & 2) << 1); };
    // A lane's byte offset of each direct load. Loads VO apart have the same swizzle, so they differ by whole rows: a scalar.
    constexpr int VO = NW == 4 ? 1 : D / 32, VK = VO * 64 * NW / KC; // VK: rows between them
    static_assert(VK % 16 == 0 && RL % VO == 0, "");
    uint32_t ok[VO], ov[VO];
#pragma unroll
    for (int i = 0; i < VO; ++i) {
        const int P = (i * NW + wave) * 64 + lane, key = P / KC, c = P % KC;
        ok[i] = (uint32_t(key) * uint32_t(p.ldk) + kswz(key, c) * 8) * 2;
        ov[i] = (uint32_t(key) * uint32_t(p.ldv) + vswz(key, c) * 8) * 2;
    }
    const uint32_t sk = VK * uint32_t(p.ldk) * 2, sv = VK * uint32_t(p.ldv) * 2;
    const uint16_t* K = p.k + int64_t(doc.k_row) * p.ldk + int64_t(kvh) * D;
    const uint16_t* V = p.v + int64_t(doc.k_row) * p.ldv + int64_t(kvh) * D;
    // a tile's resources end with the document's last key: what lies behind it comes as zeros (no tile, -1: nothing)
    auto tile_keys = [&](int t) { return t >= 0 ? min(int(doc.k_rows) - t * kKT, kKT) : 0; };
    auto res_of = [&](const uint16_t* base, int64_t ld, int t) {
        const int n = tile_keys(t);
        return buf_res(n ? base + int64_t(t) * kKT * ld : base, n ? uint32_t((n - 1) * int(ld) + D) * 2 : 0u);
    };
    // load i of tile t's 2 RL into buffer buf
    auto dma = [&](const BufRes& rk, const BufRes& rv, int buf, int i) {
        if (i < RL)
            buf_load_lds16(rk, (lds_void*)&sK(buf)[(i * NW + wave) * 512], ok[i % VO], i / VO * sk);
        else if (i < 2 * RL)
            buf_load_lds16(rv, (lds_void*)&sV(buf)[((i - RL) * NW + wave) * 512], ov[(i - RL) % VO], (i - RL) / VO * sv);
    };

    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        oacc[dt] = f32x16{};
    float m = kLeast, l = 0.0f;
    float ref = kLeast; // what the weights are first made against: m, or, where m is large, so little that they are made again
    const float slope = MODE & kBias ? p.slopes[head] * 1.4426950408889634f : 0.0f;

    // What a lane knows of a half of a tile: its row's position less the lane's first key (values r are 8 (r / 4) + r % 4 keys
    // further), and how many keys the row sees from that one on.
    struct Half {
        float rel;
        int more;
    };
    auto half_of = [&](int k0) {
        return Half{MODE & kBias ? float(pos - k0 - 4 * hk) : 0.0f, lim - k0 - 4 * hk};
    };
    // score r of a half in log2 units, less `from`
    auto score = [&](float s, const Half& h, int r, float from) {
        float x;
        if constexpr (MODE & kCap) // cap tanh(y) = cap - 2 cap / (1 + e^2y)
            x = fmaf(-2.0f * p.cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * p.c)), p.cap - from);
        else
            x = fmaf(s, p.c, -from);
        if constexpr (MODE & kBias)
            x = fmaf(-slope, fabsf(h.rel - float(8 * (r / 4) + r % 4)), x);
        return x;
    };
    auto masked = [](float x, const Half& h, int r) { return 8 * (r / 4) + r % 4 < h.more ? x : -__builtin_inff(); };
    // The weights of pair j of a half against `from` (and then `less`), packed, and their sum. The second product takes them rounded to the
    // inputs' type, the matrix instruction's: of the output's error against 64 bits of 0.0023 (16411 keys, bf16; its own rounding alone
    // 0.0016) that is 0.0016. A sum of the rounded weights changes nothing (0.0023). A second product of what the rounding left takes the
    // error away and costs half as many matrix instructions more: even one row's wave, which waits for memory, took 24.4 us for
    // 21.3 (16411 keys), 8.6 for 7.3 (77).
    auto pair = [&](const f32x16& sc, const Half& h, int j, uint32_t (&pw)[8], float& ls, float from, auto less, auto edge_c) {
        float x0 = score(sc[2 * j], h, 2 * j, from), x1 = score(sc[2 * j + 1], h, 2 * j + 1, from);
        if constexpr (std::is_same_v<decltype(less), float>) {
            x0 -= less;
            x1 -= less;
        }
        if constexpr (decltype(edge_c)::value) {
            x0 = masked(x0, h, 2 * j);
            x1 = masked(x1, h, 2 * j + 1);
        }
        const float e0 = __builtin_amdgcn_exp2f(x0), e1 = __builtin_amdgcn_exp2f(x1);
        pw[j] = pack_x2(e0, e1, F16);
        ls += e0 + e1;
    };
    // moves m up to a half's largest score (less kUp), rescales what was summed against the old one, and makes the half's weights again
    auto redo = [&](const f32x16& sc, const Half& h, uint32_t (&pw)[8], float& ls, auto edge_c) __attribute__((always_inline)) {
        f32x16 x;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = score(sc[r], h, r, 0.0f);
            if constexpr (decltype(edge_c)::value)
                x[r] = masked(x[r], h, r);
        }
        const float top = max_xor32(max16(x)), mn = fmaxf(m, F16 ? top - kUp : top), alpha = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        const bool large = fabsf(m) >= kLargeM;
        ref = large ? kLeast : m;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                oacc[dt][r] *= alpha;
        ls = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            pair(sc, h, j, pw, ls, large ? 0.0f : m, large ? m : 0.0f, edge_c);
    };
    auto read_k = [&](int buf, int kt, int ds) {
        const int key = kt * 32 + r32;
        return *reinterpret_cast<const u32x4*>(&sK(buf)[key * D + kswz(key, ds * 2 + hk) * 8]);
    };
    // V^T fragment of 16 keys (step s2 of the tile's 4) and 32 dims: slots 4 i + j of a lane are keys 16 s2 + 8 i + 4 hk + j,
    // those of its weights
    auto read_v = [&](int buf, int s2, int dt) {
        u32x4 f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int key = 16 * s2 + 8 * i + 4 * hk + ((lane & 15) >> 2), d = dt * 32 + (lane & 16) + (lane & 3) * 4;
            const u32x2 h = read_tr(&sV(buf)[key * D + vswz(key, d / 8) * 8 + d % 8]);
            f[2 * i] = h[0];
            f[2 * i + 1] = h[1];
        }
        return f;
    };

    // Infinities and NaNs of V at keys that only some of a tile's rows see must not meet the others' zero weights. Where a mask
    // cuts a tile for some row of the workgroup, V is looked through (a quarter a wave); if there are any, they are replaced by
    // zeros in LDS, and after the products each row adds those that it sees, or a NaN where its weight is zero (0 x inf), as the
    // product itself makes it in a tile that no mask cuts.
    auto find_odd = [&](int t, auto buf_c) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value, N = kKT * KC / (64 * NW);
        constexpr uint32_t ODD = F16 ? 0x04000400u : 0x00800080u; // added to an exponent of all ones: a carry into bit 15
        uint32_t any = 0;
#pragma unroll 4
        for (int i = 0; i < N; ++i) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(&sV(buf)[(i * 64 * NW + tid) * 8]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                any |= (v[e] & (EXP * 0x10001u)) + ODD;
        }
        if (any & 0x80008000u)
            odd_tile = t + 1;
        __syncthreads();
        if (odd_tile != t + 1)
            return false;
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
            u32x4* at = reinterpret_cast<u32x4*>(&sV(buf)[(i * 64 * NW + tid) * 8]);
            u32x4 v = *at;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t c = ((v[e] & (EXP * 0x10001u)) + ODD) & 0x80008000u;
                v[e] &= ~((c >> 15) * 0xffffu);
            }
            *at = v;
        }
        __syncthreads();
        return true;
    };
    auto add_odd = [&](int t) __attribute__((always_inline)) {
#pragma unroll 1
        for (int i = 0, n = tile_keys(t); i < n; ++i) {
            const int key = t * kKT + i;
            const uint16_t* v = V + int64_t(key) * p.ldv + 4 * hk;
            if (key >= lim)
                continue;
            // (key 8 (r / 4) + 4 hk + r % 4 of a half is lane half hk's value r, of its pair r / 2)
            const bool zero = !(weighty[i / 32][wave * 64 + (i & 4) * 8 + r32] >> (i % 2 * 16 + i % 32 / 8 * 2 + i % 4 / 2) & 1);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x2 h = *reinterpret_cast<const u32x2*>(v + dt * 32 + 8 * j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t x = uint16_t(h[e / 2] >> (16 * (e % 2)));
                        if ((x & EXP) == EXP)
                            oacc[dt][4 * j + e] += zero ? __builtin_nanf("") : F16 ? h2f_bits(x) : bf2f_bits(x);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };

    // One tile from buffer `buf`. Its fragment reads stream LA ahead of the products that use them, in a fixed order (fenced), and
    // the next tile's loads go out between the first products. The weights are made against the m that is there, before
    // the tile's largest score is known: those of half a between the products S^T of half b, those of half b between the
    // products P V of half a. A lane's part of their sum decides afterwards whether a half is made again against a new m:
    // a score more than 8 (in log2 units) above m puts that sum above kLazyP.
    constexpr int LA = 3, CH = 8 / DS; // fragments ahead; pairs of weights behind a product
    auto tile = [&](int t, int next, auto buf_c, auto edge_c, bool odd) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value;
        constexpr bool EDGE = decltype(edge_c)::value;
        const int k0 = t * kKT;
        const BufRes rk = res_of(K, p.ldk, next), rv = res_of(V, p.ldv, next);
        if (EDGE && k0 >= wave_most) { // no row of the wave sees the tile
#pragma unroll
            for (int i = 0; i < 2 * RL; ++i)
                dma(rk, rv, buf ^ 1, i);
            return;
        }
        u32x4 fk[2 * DS], fv[4 * DT];
        auto rd = [&](int g) {
            if (g < 2 * DS)
                fk[g] = read_k(buf, g / DS, g % DS);
            else if (g < 2 * DS + 4 * DT)
                fv[g - 2 * DS] = read_v(buf, (g - 2 * DS) / DT, (g - 2 * DS) % DT);
        };
        f32x16 s_a = f32x16{}, s_b = f32x16{};
        uint32_t pa[8], pb[8];
        float la = 0.0f, lb = 0.0f;
#pragma unroll
        for (int g = 0; g < LA; ++g)
            rd(g);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int ND = 2 * RL, PER = (ND + DS - 1) / DS;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            s_a = mfma_32x32x16<F16>(fk[ds], qf[ds], s_a);
            __builtin_amdgcn_sched_barrier(0);
            rd(ds + LA);
#pragma unroll
            for (int i = ds * PER; i < (ds + 1) * PER && i < ND; ++i)
                dma(rk, rv, buf ^ 1, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        const Half ha = half_of(k0), hb = half_of(k0 + 32);
        auto not_zero = [&](const uint32_t (&pw)[8], int half) {
            if constexpr (EDGE) {
                if (!odd)
                    return;
                uint32_t some = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    some |= __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, pw[j]), u16x2{1, 1})) << j;
                weighty[half][tid] = some;
            }
        };
        auto chunk = [&](const f32x16& sc, const Half& h, uint32_t (&pw)[8], float& ls, int c) {
#pragma unroll
            for (int j = c * CH; j < (c + 1) * CH; ++j) {
                pair(sc, h, j, pw, ls, ref, 0, edge_c);
                // (pinned here: the compiler would sink the work into the path that keeps it)
                asm volatile("" : "+v"(pw[j]), "+v"(ls));
            }
        };
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            s_b = mfma_32x32x16<F16>(fk[DS + ds], qf[ds], s_b);
            __builtin_amdgcn_sched_barrier(0);
            rd(DS + ds + LA);
            __builtin_amdgcn_sched_barrier(0);
            chunk(s_a, ha, pa, la, ds);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__any(la > kLazyP<F16>))
            redo(s_a, ha, pa, la, edge_c);
        l += la;
        not_zero(pa, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
            const int st = j / DT;
            oacc[j % DT] = mfma_32x32x16<F16>(fv[j], u32x4{pa[4 * st], pa[4 * st + 1], pa[4 * st + 2], pa[4 * st + 3]}, oacc[j % DT]);
            __builtin_amdgcn_sched_barrier(0);
            rd(2 * DS + j + LA);
            __builtin_amdgcn_sched_barrier(0);
            chunk(s_b, hb, pb, lb, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__any(lb > kLazyP<F16>))
            redo(s_b, hb, pb, lb, edge_c);
        l += lb;
        not_zero(pb, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
            const int st = j / DT;
            oacc[j % DT] = mfma_32x32x16<F16>(fv[2 * DT + j], u32x4{pb[4 * st], pb[4 * st + 1], pb[4 * st + 2], pb[4 * st + 3]}, oacc[j % DT]);
            __builtin_amdgcn_sched_barrier(0);
            rd(2 * DS + 2 * DT + j + LA);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Masks only cut the last keys off. The tiles that they cut for some row of the workgroup come first, the last one before the
    // others, then those that all rows see, in a loop of its own (one loop with a branch in it spilled registers): with a
    // bias from the tile of the first row's own position downwards and then upwards from there, so that scores fall away
    // from the start and m seldom moves (4096 rows of 20 heads of 64 upwards throughout: 348 us).
    const int edges = t_end - max(min(wg_lim / kKT, t_end), t_begin), fulls = t_end - t_begin - edges;
    const int own = !(MODE & kBias) ? fulls - 1 : max(min(int(wg_pos / kKT) - t_begin, fulls - 1), 0);
    auto tile_at = [&](int i) {
        const int j = i - edges;
        return i >= edges + fulls ? -1 : j < 0 ? t_end - 1 - i : t_begin + (j <= own ? own - j : j);
    };
    auto step = [&](int i, auto buf_c, auto edge_c) __attribute__((always_inline)) {
        const int t = tile_at(i);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        bool odd = false;
        if constexpr (decltype(edge_c)::value)
            odd = wg_lim < t * kKT + tile_keys(t) && find_odd(t, buf_c);
        tile(t, tile_at(i + 1), buf_c, edge_c, odd);
        if (decltype(edge_c)::value && odd)
            add_odd(t);
    };
    if (tid == 0)
        odd_tile = 0; // (the first step's barrier is behind it)
    if (t_begin < t_end) {
        const int t = tile_at(0);
        const BufRes rk = res_of(K, p.ldk, t), rv = res_of(V, p.ldv, t);
#pragma unroll
        for (int i = 0; i < 2 * RL; ++i)
            dma(rk, rv, 0, i);
    }
    constexpr std::integral_constant<int, 0> b0{};
    constexpr std::integral_constant<int, 1> b1{};
    int i = 0;
    for (; i + 1 < edges; i += 2) {
        step(i, b0, std::true_type{});
        step(i + 1, b1, std::true_type{});
    }
    if (i < edges) {
        step(i++, b0, std::true_type{});
        if (i < edges + fulls)
            step(i++, b1, std::false_type{});
    }
    for (; i < edges + fulls; i += 2) {
        step(i, b0, std::false_type{});
        if (i + 1 < edges + fulls)
            step(i + 1, b1, std::false_type{});
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads(); // the tiles' LDS is free

    const float lt = add_xor32(l);
    if (doc.splits > 1) {
        if (w0 + r32 >= rows)
            return; // (rows that are not there write nothing)
        const uint64_t at = (uint64_t(doc.slot) + item) * NW + wave;
        float* o = p.part + at * (32 * D);
#pragma unroll
        for (int i = 0; i < 4 * DT; ++i)
            *reinterpret_cast<f32x4*>(o + part_at<D, NW>(2 * i + hk, r32)) =
                f32x4{oacc[i / 4][4 * (i % 4)], oacc[i / 4][4 * (i % 4) + 1], oacc[i / 4][4 * (i % 4) + 2], oacc[i / 4][4 * (i % 4) + 3]};
        if (hk == 0) {
            p.part_ml[2 * (at * 32 + r32)] = m;
            p.part_ml[2 * (at * 32 + r32) + 1] = lt;
        }
        return;
    }
    // The output through LDS (32 rows a wave, 16-byte chunks XOR-ed with the row), so that whole rows of a head leave 16 bytes a
    // lane (8-byte pieces of 32 rows at a time: 4.4 us more of the 24 that 6453 x 20 heads of 64 over 77 to 231 keys took).
    // Non-temporal: nothing here reads it again, keys and queries do (6453 rows 21.6 -> 20.4 us, 4352 + 1101 + 2377 + 1801 459 -> 451).
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
    uint16_t* so = (wave & 2 ? sV0 : sK0) + (wave & 1) * (32 * D);
    auto stage = [&](auto h_c) {
        constexpr bool H = decltype(h_c)::value;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x16& a = oacc[dt];
                *reinterpret_cast<u32x2*>(so + r32 * D + ((dt * 4 + i) ^ (r32 % KC)) * 8 + 4 * hk) = u32x2{
                    pack_x2(a[4 * i] * inv, a[4 * i + 1] * inv, H), pack_x2(a[4 * i + 2] * inv, a[4 * i + 3] * inv, H)};
            }
    };
    if (p.out_f16)
        stage(std::true_type{});
    else
        stage(std::false_type{});
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0): this wave's LDS writes done
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < KC / 2; ++j) {
        const int r = j * (64 / KC) + lane / KC, c = lane % KC;
        if (w0 + r >= rows)
            continue;
        const u32x4 v = *reinterpret_cast<const u32x4*>(so + r * D + (c ^ (r % KC)) * 8);
        const uint32_t rr = w0 + r, qr = p.group == 1 ? rr : rr / p.group, hh = p.group == 1 ? kvh : kvh * p.group + rr % p.group;
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p.out + (int64_t(doc.q_row) + qr) * p.ldo + int64_t(hh) * D + c * 8));
    }
}

// The splits joined: 4 dims of a row a thread, RW rows of a wave's 32 a workgroup, its G groups every G-th split each. Many rows: as
// many as make 256 threads, in 1 group for up to 8 splits, in 4 for more; few: one, in 8 groups (16) (32 rows of 52 splits 4.0 us, 8 rows
// a workgroup 7.6).
constexpr uint32_t join_rows(int d, int nw) { return nw == 1 ? 1 : 1024 / d; }
template <int D, int NW, uint32_t G> __global__ __launch_bounds__(D / 4 * join_rows(D, NW) * G) void join_kernel(PackedP p)
{
    constexpr uint32_t RW = join_rows(D, NW), PER = NW * 32 / RW, T = D / 4 * RW; // T: threads a group
    uint32_t doc_first;
    const Doc doc = find_doc(p, p.join, blockIdx.x, doc_first);
    const uint32_t rows = doc.q_rows * p.group, at = blockIdx.x - doc_first;
    const uint32_t kvh = at / (doc.blocks * PER), bi = at / PER % doc.blocks, sub = at % PER; // (blocks as above, from the last one)
    const uint32_t g = threadIdx.x / T, q = threadIdx.x % T, chunk = q / RW;
    const uint32_t in_block = sub * RW + q % RW, row = (doc.blocks - 1 - bi) * (32 * NW) + in_block;
    if ((doc.blocks - 1 - bi) * (32 * NW) + sub * RW >= rows)
        return; // (the whole workgroup)
    const uint64_t slot = uint64_t(doc.slot) + (uint64_t(kvh) * doc.blocks + bi) * doc.splits;
    const uint32_t wave = in_block / 32, r32 = in_block % 32;
    float m = kLeast, l = 0.0f;
    f32x4 o = f32x4{};
    if (row < rows) {
        // (4 splits' loads at a time)
        constexpr uint32_t U = 4;
        for (uint32_t s0 = g; s0 < doc.splits; s0 += U * G) {
            float ms[U], ls[U];
            f32x4 os[U];
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint64_t i = (slot + min(s0 + j * G, doc.splits - 1)) * NW + wave;
                ms[j] = p.part_ml[2 * (i * 32 + r32)];
                ls[j] = p.part_ml[2 * (i * 32 + r32) + 1];
                os[j] = *reinterpret_cast<const f32x4*>(p.part + i * (32 * D) + part_at<D, NW>(chunk, r32));
            }
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                if (s0 + j * G >= doc.splits)
                    break;
                const float mn = fmaxf(m, ms[j]), a = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(ms[j] - mn);
                m = mn;
                l = l * a + w * ls[j];
                o = o * a + w * os[j];
            }
        }
    }
    if constexpr (G > 1) {
        __shared__ __attribute__((aligned(16))) f32x4 so[G - 1][T];
        __shared__ float sm[G - 1][T], sl[G - 1][T];
        if (g) {
            so[g - 1][q] = o;
            sm[g - 1][q] = m;
            sl[g - 1][q] = l;
        }
        __syncthreads();
        if (g)
            return;
#pragma unroll
        for (uint32_t i = 0; i < G - 1; ++i) {
            const float mn = fmaxf(m, sm[i][q]), a = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(sm[i][q] - mn);
            m = mn;
            l = l * a + w * sl[i][q];
            o = o * a + w * so[i][q];
        }
    }
    if (row >= rows)
        return;
    o *= l == 0.0f ? 0.0f : 1.0f / l;
    const bool h = p.out_f16;
    *reinterpret_cast<u32x2*>(p.out + (int64_t(doc.q_row) + row / p.group) * p.ldo + int64_t(kvh * p.group + row % p.group) * D + chunk * 4) =
        u32x2{pack_x2(o[0], o[1], h), pack_x2(o[2], o[3], h)};
}

// everything but the operands' addresses, for the call and for its workspace's size
mk_status check_shape(const mk_attn_packed_args* a)
{
    if (a->dtype != MK_BF16 && a->dtype != MK_F16)
        return fail(MK_ERR_ARG, "attention_packed: q, k and v must be bf16 or f16");
    if (a->out_dtype != MK_BF16 && a->out_dtype != MK_F16)
        return fail(MK_ERR_ARG, "attention_packed: output bf16 or f16");
    if (!a->heads || a->heads > 65535 || !a->kv_heads || a->heads % a->kv_heads)
        return fail(MK_ERR_ARG, "attention_packed: kv_heads must divide heads, 1 to 65535");
    if (a->d != 64 && a->d != 128)
        return fail(MK_ERR_ARG, "attention_packed: head dim must be 64 or 128");
    if (!(a->scale >= 0.0f) || std::isinf(a->scale) || !(a->cap >= 0.0f) || std::isinf(a->cap))
        return fail(MK_ERR_ARG, "attention_packed: scale and cap must be finite and not negative");
    // (the kernels' factors; and cap tanh(s / cap) is made as cap - 2 cap / (1 + e^(2 s / cap)), 16 u cap off: 2^-8 at 2^12)
    constexpr float kLog2e = 1.4426950408889634f;
    if (a->cap > 4096.0f || std::isinf(kLog2e * a->scale) || (a->cap > 0.0f && std::isinf(2.0f * kLog2e * a->scale / a->cap)))
        return fail(MK_ERR_ARG, "attention_packed: cap up to 4096, scale and scale / cap below 2^126");
    const int64_t nq = int64_t(a->heads) * a->d, nk = int64_t(a->kv_heads) * a->d;
    constexpr int64_t most = 1 << 24;
    auto bad = [](int64_t ld, int64_t n) { return ld < n || ld % 8 || ld >= most; };
    if (bad(a->ldq, nq) || bad(a->ldo, nq) || bad(a->ldk, nk) || bad(a->ldv, nk))
        return fail(MK_ERR_ARG, "attention_packed: rows must hold their heads, in multiples of 8 elements below 2^24");
    if (a->n_docs && !a->docs)
        return fail(MK_ERR_ARG, "attention_packed: null documents");
    bool sorted = true;
    uint64_t end = 0;
    for (uint32_t i = 0; i < a->n_docs; ++i) {
        const mk_attn_doc& d = a->docs[i];
        if (uint64_t(d.q_row) + d.q_rows > 0x7fffffffu || uint64_t(d.k_row) + d.k_rows > 0x7fffffffu)
            return fail(MK_ERR_ARG, "attention_packed: a document's rows end past 2^31 - 1");
        if (uint64_t(d.q_rows) * a->heads > (1u << 29)) // (128 of them a workgroup of 256: 2^30 threads)
            return fail(MK_ERR_ARG, "attention_packed: a document's q_rows times heads pass 2^29");
        if (int64_t(d.q_pos) + d.q_rows > 0x7fffffff)
            return fail(MK_ERR_ARG, "attention_packed: a document's positions end past 2^31 - 1");
        if (d.q_rows) {
            sorted = sorted && d.q_row >= end;
            end = uint64_t(d.q_row) + d.q_rows;
        }
    }
    if (!sorted) try {
        std::vector<std::pair<uint32_t, uint32_t>> spans;
        for (uint32_t i = 0; i < a->n_docs; ++i)
            if (a->docs[i].q_rows)
                spans.emplace_back(a->docs[i].q_row, a->docs[i].q_row + a->docs[i].q_rows);
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i].first < spans[i - 1].second)
                return fail(MK_ERR_ARG, "attention_packed: two documents share query rows");
    } catch (const std::bad_alloc&) {
        return fail(MK_ERR_NOMEM, "attention_packed: no memory to compare the documents");
    }
    return MK_OK;
}

// One launch: up to kMaxDocs documents from docs[next] on, the longest first, and how their keys are split.
struct Launch {
    uint32_t nw;          // waves a workgroup (32 rows each)
    uint32_t groups;      // workgroups
    uint32_t joins;       // workgroups of the second launch, 0: none
    uint32_t most_splits;
    uint64_t slots;       // partial results
};

constexpr uint64_t kMostGroups = 1u << 23; // of 256 threads: fewer than 2^32 in all

uint64_t bytes_of(const mk_attn_packed_args* a, uint64_t slots, uint32_t nw) { return slots * (32 * nw) * (a->d + 2) * 4; }

// Takes documents into p, their keys split as far as `room` bytes of workspace hold the partial results; returns how many of docs
// were looked at. With all the room that the best split needs it is the same split as with any more.
uint32_t plan_launch(const mk_attn_packed_args* a, uint32_t next, uint32_t cus, uint64_t room, PackedP& p, Launch& out)
{
    const uint32_t group = a->heads / a->kv_heads;
    uint32_t at = next, n = 0;
    uint64_t most_rows = 0, sum = 0;
    for (; at < a->n_docs && n < kMaxDocs; ++at) {
        const mk_attn_doc& d = a->docs[at];
        if (!d.q_rows)
            continue;
        sum += uint64_t(cdiv(uint64_t(d.q_rows) * group, 128)) * a->kv_heads;
        if (n && sum > kMostGroups)
            break;
        p.docs[n++] = Doc{d.q_row, d.q_rows, d.k_row, d.k_rows, d.q_pos, d.block, d.prefix, 0, 1, 0};
        most_rows = std::max(most_rows, uint64_t(d.q_rows) * group);
    }
    // longest first (at most kMaxDocs: an insertion sort)
    for (uint32_t i = 1; i < n; ++i)
        for (uint32_t j = i; j && p.docs[j].k_rows > p.docs[j - 1].k_rows; --j)
            std::swap(p.docs[j], p.docs[j - 1]);
    // One wave a workgroup where a key head has few rows in every document (us with one / with four: 1 row of 32 heads of 128 on
    // 8 over 16411 keys 22.3 / 24.4, 16 rows of 20 heads of 64 over 4096 11.8 / 13.7; 32 rows over 77 6.2 / 5.7, 32 rows of 32 heads
    // of 128 over 4096 25.1 / 22.6: four waves share a tile's loads). Single rows next to a prompt take its four waves, three of them
    // idle, in the prompt's launch (us so / in a launch of their own behind the prompt's: 31 rows over 2000 keys, 32 heads of 128 on 8, and
    // a prompt of 512 63 / 69, of 128 67 / 64, of 2048 99 / 104; 20 heads of 64, 512 86 / 106, 17 121 / 98; 7 rows over 16411 and 512 119 / 113).
    out.nw = most_rows <= 16 ? 1 : 4;
    const uint32_t resident = cus * (out.nw == 4 || a->d == 128 ? 2 : 4);
    uint64_t tiles = 0, longest = 0;
    for (uint32_t i = 0; i < n; ++i) {
        Doc& d = p.docs[i];
        d.blocks = cdiv(uint64_t(d.q_rows) * group, 32 * out.nw);
        tiles += uint64_t(d.blocks) * a->kv_heads * cdiv(d.k_rows, kKT);
        longest = std::max<uint64_t>(longest, cdiv(d.k_rows, kKT));
    }
    // How many tiles a workgroup takes at most: the part of the longest document's with the least estimated time. A tile takes about
    // 1 us (heads of 128; 0.7 of 64) where a compute unit has one workgroup; partial results cost a launch and their way to
    // memory and back, 2.5 us and 0.6 a MB. (us without splits / with 2 / with 8: 8 heads of 64 over 1024 rows 16.5 / 14.4 / 19.0, 20 of
    // 128 over 1024 21.6 / 30.2 / 43.0, over 64 of 2048 43.6 / 24.5 / 14.3.)
    auto splits_of = [](const Doc& d, uint64_t target) {
        return std::max<uint64_t>((cdiv(d.k_rows, kKT) + target - 1) / target, 1);
    };
    uint64_t target = std::max<uint64_t>(longest, 1);
    double best = 1e300;
    for (uint64_t parts = 1; room && parts <= std::max<uint64_t>(longest, 1); parts += 1 + parts / 4) {
        const uint64_t t = std::max<uint64_t>((longest + parts - 1) / parts, 1);
        double rows = 0, items = 0;
        uint64_t slots = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const Doc& d = p.docs[i];
            const uint64_t splits = splits_of(d, t), of = uint64_t(d.blocks) * a->kv_heads * splits;
            items += double(of);
            if (splits > 1) {
                rows += double(d.q_rows) * a->heads * splits;
                slots += of;
            }
        }
        if (bytes_of(a, slots, out.nw) > room)
            continue;
        // (more workgroups than the chip holds: their share, and half a workgroup for the last round's end)
        const double long_one = items <= resident ? double(t) : double(tiles) / resident + 0.5 * double(t);
        const double time = long_one * (a->d == 128 ? 1.0 : 0.7) + (rows > 0 ? 2.5 + rows * (a->d + 2) * 4 * 0.6e-6 : 0.0);
        if (time < best) {
            best = time;
            target = t;
        }
    }
    uint64_t first = 0, join = 0;
    out.slots = out.most_splits = 0;
    for (uint32_t i = 0; i < n; ++i) {
        Doc& d = p.docs[i];
        d.splits = uint32_t(splits_of(d, target));
        const uint64_t items = uint64_t(d.blocks) * a->kv_heads * d.splits;
        out.most_splits = std::max(out.most_splits, d.splits);
        p.first[i] = uint32_t(first);
        p.join[i] = uint32_t(join);
        d.slot = uint32_t(out.slots);
        first += round_up(items, 8);
        if (d.splits > 1) {
            out.slots += items;
            join += uint64_t(d.blocks) * a->kv_heads * (out.nw == 1 ? 32 : 128 * a->d / 1024);
        }
    }
    p.n_docs = n;
    out.groups = uint32_t(first);
    out.joins = uint32_t(join);
    return at - next;
}
template <int D, bool F16, int NW> void launch_mode(const PackedP& p, int mode, uint32_t groups, hipStream_t s)
{
    if (mode == kPlain)
        packed_kernel<D, F16, kPlain, NW><<<groups, 64 * NW, 0, s>>>(p);
    else if (mode == kBias)
        packed_kernel<D, F16, kBias, NW><<<groups, 64 * NW, 0, s>>>(p);
    else if (mode == kCap)
        packed_kernel<D, F16, kCap, NW><<<groups, 64 * NW, 0, s>>>(p);
    else
        packed_kernel<D, F16, kCap | kBias, NW><<<groups, 64 * NW, 0, s>>>(p);
}
template <int D> void launch_all(const PackedP& p, const Launch& l, bool f16, int mode, hipStream_t s)
{
    if (l.nw == 4)
        f16 ? launch_mode<D, true, 4>(p, mode, l.groups, s) : launch_mode<D, false, 4>(p, mode, l.groups, s);
    else
        f16 ? launch_mode<D, true, 1>(p, mode, l.groups, s) : launch_mode<D, false, 1>(p, mode, l.groups, s);
    if (!l.joins)
        return;
    if (l.nw == 1)
        join_kernel<D, 1, 1024 / D><<<l.joins, 256, 0, s>>>(p);
    else if (l.most_splits <= 8)
        join_kernel<D, 4, 1><<<l.joins, 256, 0, s>>>(p);
    else
        join_kernel<D, 4, 4><<<l.joins, 1024, 0, s>>>(p);
}
// whether a document has query rows, and (keys) one of those keys
bool any_rows(const mk_attn_packed_args* a, bool* keys = nullptr)
{
    bool any = false;
    for (uint32_t i = 0; i < a->n_docs; ++i)
        if (a->docs[i].q_rows) {
            any = true;
            if (keys && a->docs[i].k_rows)
                *keys = true;
        }
    return any;
}

} // namespace

} // namespace mk

using namespace mk;

extern "C" {

mk_status mk_attention_packed_workspace(const mk_attn_packed_args* a, uint64_t* bytes)
{
    if (!a || !bytes)
        return fail(MK_ERR_ARG, "attention_packed_workspace: null argument");
    MK_TRY(check_shape(a));
    *bytes = 0;
    if (!any_rows(a))
        return MK_OK;
    uint32_t cus = 1;
    MK_TRY(compute_units(cus));
    PackedP p;
    Launch l;
    for (uint32_t i = 0; i < a->n_docs;) {
        i += plan_launch(a, i, cus, UINT64_MAX, p, l);
        *bytes = std::max(*bytes, bytes_of(a, l.slots, l.nw)); // (launches run one after the other)
    }
    return MK_OK;
}

mk_status mk_attention_packed(const mk_attn_packed_args* a, void* stream)
{
    if (!a)
        return fail(MK_ERR_ARG, "attention_packed: null argument");
    MK_TRY(check_shape(a));
    if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) || !aligned(a->workspace, 16) ||
        !aligned(a->slopes, 4))
        return fail(MK_ERR_ARG, "attention_packed: operands and workspace must be 16-byte aligned (slopes 4)");
    bool keys = false;
    if (!any_rows(a, &keys))
        return MK_OK;
    if (!a->q || !a->out || (keys && (!a->k || !a->v)))
        return fail(MK_ERR_ARG, "attention_packed: null argument (q and out are required, k and v for documents with keys)");
    uint32_t cus = 1;
    MK_TRY(compute_units(cus));
    PackedP p;
    Launch l;
    hipStream_t s = static_cast<hipStream_t>(stream);
    constexpr float kLog2e = 1.4426950408889634f;
    const int mode = (a->cap > 0.0f ? kCap : 0) | (a->slopes ? kBias : 0);
    p.q = static_cast<const uint16_t*>(a->q);
    p.k = static_cast<const uint16_t*>(a->k);
    p.v = static_cast<const uint16_t*>(a->v);
    p.out = static_cast<uint16_t*>(a->out);
    p.ldq = a->ldq;
    p.ldk = a->ldk;
    p.ldv = a->ldv;
    p.ldo = a->ldo;
    p.slopes = a->slopes;
    p.c = mode & kCap ? 2.0f * kLog2e * a->scale / a->cap : a->scale * kLog2e;
    p.cap = a->cap * kLog2e;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.out_f16 = a->out_dtype == MK_F16;
    for (uint32_t i = 0; i < a->n_docs;) {
        i += plan_launch(a, i, cus, a->workspace ? a->workspace_bytes : 0, p, l);
        if (!l.groups)
            continue;
        p.part = static_cast<float*>(a->workspace);
        p.part_ml = p.part ? p.part + l.slots * (32 * l.nw) * a->d : nullptr;
        const bool f16 = a->dtype == MK_F16;
        a->d == 128 ? launch_all<128>(p, l, f16, mode, s) : launch_all<64>(p, l, f16, mode, s);
        MK_LAUNCH_CHECK("attention_packed");
    }
    return MK_OK;
}

} // extern "C"
