// mk_attention_packed: softmax attention of packed documents, with causal and prefix masks, a tanh cap and a distance bias.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <utility>
#include <vector>

namespace mk {

namespace {

constexpr uint32_t kMaxDocs = 96; // documents a launch: they go by kernel argument

struct Doc {
    uint32_t first; // its first item
    uint32_t q_row, q_rows, k_row, k_rows;
    int32_t q_pos;
    uint32_t block, prefix;
};
struct PackedP {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    int64_t ldq, ldk, ldv, ldo;
    const float* slopes;
    float scale, cap;
    uint32_t heads, group, n_docs, out_f16;
    Doc docs[kMaxDocs];
};

template <bool F16> __device__ inline float widen(uint16_t h) { return F16 ? h2f_bits(h) : bf2f_bits(h); }

__device__ inline bool sees(const Doc& d, int64_t pos, int64_t key)
{
    return d.block == 0 || pos >= int64_t(d.block) || key <= pos || key < int64_t(d.prefix);
}

// a wave a query row and head: a key a lane, then the head's dims a lane
template <bool F16, int D> __global__ __launch_bounds__(64) void simple_kernel(PackedP p)
{
    uint32_t di = 0;
    while (di + 1 < p.n_docs && blockIdx.x >= p.docs[di + 1].first)
        ++di;
    const Doc d = p.docs[di];
    const uint32_t i = blockIdx.x - d.first, head = blockIdx.y, lane = threadIdx.x;
    const int64_t pos = int64_t(d.q_pos) + i;
    const uint16_t* q = p.q + (int64_t(d.q_row) + i) * p.ldq + int64_t(head) * D;
    const uint16_t* k = p.k + int64_t(d.k_row) * p.ldk + int64_t(head / p.group) * D;
    const uint16_t* v = p.v + int64_t(d.k_row) * p.ldv + int64_t(head / p.group) * D;
    __shared__ float sq[D], sp[64];
    for (int e = lane; e < D; e += 64)
        sq[e] = widen<F16>(q[e]);
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f, acc[D / 64] = {};
    for (uint32_t k0 = 0; k0 < d.k_rows; k0 += 64) {
        const uint32_t key = k0 + lane;
        float s = -__builtin_inff();
        if (key < d.k_rows && sees(d, pos, key)) {
            s = 0.0f;
            for (int e = 0; e < D; ++e)
                s += sq[e] * widen<F16>(k[int64_t(key) * p.ldk + e]);
            s *= p.scale;
            if (p.cap > 0.0f)
                s = p.cap * tanhf(s / p.cap);
            if (p.slopes)
                s -= p.slopes[head] * fabsf(float(pos - int64_t(key)));
        }
        const float mn = fmaxf(m, wave_max(s)), base = mn == -__builtin_inff() ? 0.0f : mn;
        const float alpha = m == -__builtin_inff() ? 0.0f : expf(m - base), e = expf(s - base);
        l = l * alpha + wave_sum(e);
        m = mn;
        __syncthreads();
        sp[lane] = e;
        __syncthreads();
        for (int c = 0; c < D / 64; ++c) {
            acc[c] *= alpha;
            for (uint32_t j = 0; j < 64 && k0 + j < d.k_rows; ++j)
                if (sees(d, pos, k0 + j))
                    acc[c] += sp[j] * widen<F16>(v[int64_t(k0 + j) * p.ldv + c * 64 + lane]);
        }
    }
    for (int c = 0; c < D / 64; ++c) {
        const float o = l == 0.0f ? 0.0f : acc[c] / l;
        p.out[(int64_t(d.q_row) + i) * p.ldo + int64_t(head) * D + c * 64 + lane] = p.out_f16 ? f2h_bits(o) : f2bf_bits(o);
    }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

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
    return MK_OK;
}

mk_status mk_attention_packed(const mk_attn_packed_args* a, void* stream)
{
    if (!a || !a->q || !a->k || !a->v || !a->out)
        return fail(MK_ERR_ARG, "attention_packed: null argument (q, k, v and out are required)");
    MK_TRY(check_shape(a));
    if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) || !aligned(a->workspace, 16) ||
        !aligned(a->slopes, 4))
        return fail(MK_ERR_ARG, "attention_packed: operands and workspace must be 16-byte aligned (slopes 4)");
    uint64_t need = 0;
    MK_TRY(mk_attention_packed_workspace(a, &need));
    if (a->workspace && a->workspace_bytes < need)
        return fail(MK_ERR_ARG, "attention_packed: the workspace is smaller than mk_attention_packed_workspace says");
    hipStream_t s = static_cast<hipStream_t>(stream);
    PackedP p{static_cast<const uint16_t*>(a->q), static_cast<const uint16_t*>(a->k), static_cast<const uint16_t*>(a->v),
              static_cast<uint16_t*>(a->out), a->ldq, a->ldk, a->ldv, a->ldo, a->slopes, a->scale, a->cap, a->heads,
              a->heads / a->kv_heads, 0, a->out_dtype == MK_F16 ? 1u : 0u, {}};
    uint32_t items = 0;
    auto launch = [&]() {
        if (!items)
            return;
        const dim3 grid(items, p.heads);
        if (a->dtype == MK_F16)
            a->d == 128 ? simple_kernel<true, 128><<<grid, 64, 0, s>>>(p) : simple_kernel<true, 64><<<grid, 64, 0, s>>>(p);
        else
            a->d == 128 ? simple_kernel<false, 128><<<grid, 64, 0, s>>>(p) : simple_kernel<false, 64><<<grid, 64, 0, s>>>(p);
        p.n_docs = items = 0;
    };
    for (uint32_t i = 0; i < a->n_docs; ++i) {
        const mk_attn_doc& d = a->docs[i];
        if (!d.q_rows)
            continue;
        if (p.n_docs == kMaxDocs || uint64_t(items) + d.q_rows > (1u << 25))
            launch();
        p.docs[p.n_docs++] = Doc{items, d.q_row, d.q_rows, d.k_row, d.k_rows, d.q_pos, d.block, d.prefix};
        items += d.q_rows;
    }
    if (!p.n_docs)
        return MK_OK;
    launch();
    MK_LAUNCH_CHECK("attention_packed");
    return MK_OK;
}

} // extern "C"
