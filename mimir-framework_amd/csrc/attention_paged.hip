// attention_paged.hip -- attention of new tokens over a paged cache of keys and
// values (mimir_hip.h mimir_attention_paged_fwd): softmax(Q K^T * scale) V with the
// softmax fused between the products, as attention.hip, for sequences of different
// lengths whose queries share key / value heads.
#include "kvcache.hpp"

#include <math.h>

#include <algorithm>
#include <cmath>

using namespace mimir;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
    KvView c;
    KvBatch b;
    const float* q;
    float* out;
    int64_t ld_q, ld_out;
    int32_t heads, group;  // query heads, those that share a key / value head
    float qscale;          // scale * log2(e)
    int32_t causal;
};

// Element d of a cache row (index `at` among the rows of the type's buffer).
template <int DT>
__device__ __forceinline__ float element(const char* base, int64_t at, int stride, int d) {
    const int64_t i = at * stride + d;
    if constexpr (DT == MIMIR_KV_F32) return reinterpret_cast<const float*>(base)[i];
    else if constexpr (DT == MIMIR_KV_BF16)
        return __builtin_bit_cast(float, static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(base)[i]) << 16);
    else return static_cast<float>(reinterpret_cast<const int8_t*>(base)[i]);
}

constexpr int kRowChunks = kKvMaxDim / kWave;

// One query row over keys j0 .. j1 - 1 by one wave, lane l holding dimensions l + 64 c.
// Leaves the sums (without the division) and the running max (base-2 units) and sum.
template <int DT>
__device__ __forceinline__ void row_over_keys(const PagedArgs& a, int s, int kv_head, const float* q, int j0, int j1,
                                              float* acc, float* m_out, float* l_out) {
    const int lane = threadIdx.x % kWave;
    float x[kRowChunks];
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
        const int d = lane + c * kWave;
        x[c] = d < a.c.head_dim ? q[d] * a.qscale : 0.f;
        acc[c] = 0.f;
    }
    float m = -1e30f, l = 0.f;
    for (int j = j0; j < j1; ++j) {
        const auto [page, slot] = kv_slot(a.b, a.c.pages, a.c.page_div, s, j);
        if (page < 0) continue;
        const int64_t at = (static_cast<int64_t>(page) * a.c.kv_heads + kv_head) * a.c.page_size + slot;
        float part = 0.f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) {
            const int d = lane + c * kWave;
            if (d < a.c.head_dim) part += x[c] * element<DT>(a.c.k, at, a.c.stride, d);
        }
        float score = wave_sum(part);
        if constexpr (DT == MIMIR_KV_I8) score *= a.c.k_scale[at];
        const float m_new = fmaxf(m, score);
        const float alpha = __builtin_amdgcn_exp2f(m - m_new);
        const float p = __builtin_amdgcn_exp2f(score - m_new);
        m = m_new;
        l = l * alpha + p;
        const float w = DT == MIMIR_KV_I8 ? p * a.c.v_scale[at] : p;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) {
            const int d = lane + c * kWave;
            if (d < a.c.head_dim) acc[c] = acc[c] * alpha + w * element<DT>(a.c.v, at, a.c.stride, d);
        }
    }
    *m_out = m;
    *l_out = l;
}

// One wave per (token, query head).
template <int DT>
__global__ __launch_bounds__(kBlock) void paged_rows(PagedArgs a) {
    const int lane = threadIdx.x % kWave;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave;
    const int64_t t = row / a.heads;
    if (t >= a.b.tokens) return;
    const int head = static_cast<int>(row % a.heads);
    const int s = kv_sequence_of(a.b, static_cast<int>(t));
    if (s < 0) return;
    const KvSequence seq = kv_sequence(a.b, s);
    const int i = static_cast<int>(t) - seq.first;
    if (i < 0 || i >= seq.n) return;
    const int end = a.causal ? min(max(seq.len - seq.n + i + 1, 0), seq.len) : seq.len;
    float acc[kRowChunks], m, l;
    row_over_keys<DT>(a, s, head / a.group, a.q + t * a.ld_q + static_cast<int64_t>(head) * a.c.head_dim, 0, end, acc, &m, &l);
    const float inv = 1.0f / (l + 1e-9f);
    float* out = a.out + t * a.ld_out + static_cast<int64_t>(head) * a.c.head_dim;
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
        const int d = lane + c * kWave;
        if (d < a.c.head_dim) out[d] = acc[c] * inv;
    }
}

template <int DT>
int launch_rows(mimir_ctx* ctx, const PagedArgs& a) {
    const int64_t rows = static_cast<int64_t>(a.b.tokens) * a.heads, blocks = (rows + 3) / 4;
    MIMIR_REQUIRE(ctx, dispatch_fits(blocks, kBlock), "paged attention: grid of %lld workgroups exceeds the limit",
                  (long long)blocks);
    paged_rows<DT><<<static_cast<unsigned>(blocks), kBlock, 0, ctx->stream>>>(a);
    return launched(ctx, "paged_rows");
}

}  // namespace

extern "C" int mimir_attention_paged_fwd(mimir_ctx* ctx, const mimir_kv_cache* cache, const mimir_kv_batch* batch,
                                         const float* q, int64_t ld_q, float* out, int64_t ld_out, int64_t q_heads,
                                         float scale, int causal) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "paged attention";
    PagedArgs a{};
    if (int st = kv_view(ctx, what, cache, &a.c)) return st;
    if (int st = kv_batch(ctx, what, cache, batch, &a.b)) return st;
    MIMIR_REQUIRE(ctx, q_heads >= 1 && q_heads <= (1 << 20) && q_heads % cache->kv_heads == 0,
                  "%s: q_heads %lld is not a multiple of kv_heads %d", what, (long long)q_heads, cache->kv_heads);
    const int64_t width = q_heads * cache->head_dim;
    MIMIR_REQUIRE(ctx, ld_q >= width && ld_out >= width, "%s: row strides (%lld, %lld) below q_heads * head_dim = %lld", what,
                  (long long)ld_q, (long long)ld_out, (long long)width);
    MIMIR_REQUIRE(ctx, std::isfinite(scale), "%s: scale must be finite", what);
    if (batch->tokens == 0 || batch->sequences == 0 || batch->max_new == 0) return MIMIR_OK;
    MIMIR_REQUIRE(ctx, q && out, "%s: null pointer", what);
    MIMIR_ENTER(ctx);
    a.q = q;
    a.out = out;
    a.ld_q = ld_q;
    a.ld_out = ld_out;
    a.heads = static_cast<int32_t>(q_heads);
    a.group = static_cast<int32_t>(q_heads / cache->kv_heads);
    a.qscale = scale * kLog2e;
    a.causal = causal ? 1 : 0;
    if (cache->dtype == MIMIR_KV_F32) return launch_rows<MIMIR_KV_F32>(ctx, a);
    if (cache->dtype == MIMIR_KV_BF16) return launch_rows<MIMIR_KV_BF16>(ctx, a);
    return launch_rows<MIMIR_KV_I8>(ctx, a);
}
