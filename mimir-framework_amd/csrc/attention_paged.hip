// attention_paged.hip -- attention of new tokens over a paged cache of keys and
// values (mimir_hip.h mimir_attention_paged_fwd): softmax(Q K^T * scale) V with the
// softmax fused between the products, as attention.hip, for sequences of different
// lengths whose queries share key / value heads.  The two kernels are in
// attention_paged_stream.hip and attention_paged_block.hip; here are the call and the
// join of blocks whose keys several workgroups had.
#include "attention_paged.hpp"

#include <math.h>

#include <algorithm>
#include <cmath>

using namespace mimir;

namespace {

constexpr int64_t kStreamRows = 32;

// The shares of one row: brought to one max, added up and divided.  WAVES waves a
// row; the block's first run (this descriptor's) kept what it begins, the others what
// they go on with.
template <int WAVES>
__global__ __launch_bounds__(kBlock) void paged_join(PagedArgs p, PagedRuns a) {
    constexpr int kAhead = 4, kRowsOf = kBlock / kWave / WAVES;
    __shared__ float share[kBlock / kWave][kKvMaxDim + 2];
    const uint32_t groups = static_cast<uint32_t>((a.part_rows + kRowsOf - 1) / kRowsOf);
    const uint32_t first = blockIdx.x / groups;
    const PagedShared s = a.shared[first];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, d = p.c.head_dim;
    const int row = static_cast<int>(blockIdx.x % groups) * kRowsOf + wave / WAVES;
    if (s.runs <= 1) return;
    const bool mine = row < s.rows;
    float m = -1e30f, l = 0.f, acc[kRowChunks];
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) acc[c] = 0.f;
    for (int i = wave % WAVES; mine && i < s.runs; i += kAhead * WAVES) {
        float ms[kAhead], ls[kAhead], x[kAhead][kRowChunks];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = i + u * WAVES;
            ms[u] = -1e30f;
            ls[u] = 0.f;
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c) x[u][c] = 0.f;
            if (j >= s.runs) continue;
            const float* part = paged_part(a, d, first + static_cast<uint32_t>(j), j == 0, row);
            ms[u] = part[0];
            ls[u] = part[1];
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c)
                if (lane + c * kWave < d) x[u][c] = part[2 + lane + c * kWave];
        }
        float m_new = m;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) m_new = fmaxf(m_new, ms[u]);
        const float f = __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) acc[c] *= f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const float g = __builtin_amdgcn_exp2f(ms[u] - m);
            l += ls[u] * g;
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c) acc[c] += x[u][c] * g;
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) share[wave][lane + c * kWave] = acc[c];
        if (lane == 0) {
            share[wave][kKvMaxDim] = m;
            share[wave][kKvMaxDim + 1] = l;
        }
        __syncthreads();
        const int w0 = wave / WAVES * WAVES;
        if (wave != w0) return;
#pragma unroll
        for (int v = 1; v < WAVES; ++v) {
            const float mv = share[w0 + v][kKvMaxDim], m_new = fmaxf(m, mv);
            const float f = __builtin_amdgcn_exp2f(m - m_new), g = __builtin_amdgcn_exp2f(mv - m_new);
            m = m_new;
            l = l * f + share[w0 + v][kKvMaxDim + 1] * g;
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c) acc[c] = acc[c] * f + share[w0 + v][lane + c * kWave] * g;
        }
    }
    if (!mine) return;
    const float inv = 1.0f / (l + 1e-9f);
    float* out = p.out + paged_row(p, p.ld_out, s.first, s.head, s.row0 + row);
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c)
        if (lane + c * kWave < d) out[lane + c * kWave] = acc[c] * inv;
}

}  // namespace

int64_t mimir::paged_runs(mimir_ctx* ctx, const PagedArgs& p, PagedRuns* a, int64_t runs, int64_t blocks, bool split) {
    const int64_t floats = runs * 2 * a->part_rows * (p.c.head_dim + 2);
    const int64_t bytes = runs * static_cast<int64_t>(sizeof(PagedShared)) + floats * 4;
    char* work = split && bytes <= static_cast<int64_t>(kPagedWorkBytes) ? paged_work(ctx) : nullptr;
    if (!work) return blocks;
    a->shared = reinterpret_cast<PagedShared*>(work);
    a->part = reinterpret_cast<float*>(work + runs * sizeof(PagedShared));
    a->runs = static_cast<uint32_t>(runs);
    return runs;
}

int mimir::paged_join_launch(mimir_ctx* ctx, const PagedArgs& p, const PagedRuns& a) {
    if (!a.part) return MIMIR_OK;
    // Few rows: four waves each, as many runs may have shared a long sequence.
    if (a.part_rows <= 16) paged_join<4><<<a.runs * static_cast<unsigned>(a.part_rows), kBlock, 0, ctx->stream>>>(p, a);
    else paged_join<1><<<a.runs * static_cast<unsigned>((a.part_rows + 3) / 4), kBlock, 0, ctx->stream>>>(p, a);
    return launched(ctx, "paged_join");
}

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
    if (cache->pages == 0) a.b.max_len = 0;  // no keys, and no memory to point at
    MIMIR_REQUIRE(ctx, q && out, "%s: null pointer", what);
    MIMIR_ENTER(ctx);
    a.q = q;
    a.out = out;
    a.ld_q = ld_q;
    a.ld_out = ld_out;
    a.heads = static_cast<int32_t>(q_heads);
    a.group = static_cast<int32_t>(q_heads / cache->kv_heads);
    a.qscale = scale * kPagedLog2e;
    a.causal = causal ? 1 : 0;
    a.group_div = make_fastdiv(static_cast<uint32_t>(a.group));
    const int64_t rows = static_cast<int64_t>(a.b.max_new) * a.group;
    MIMIR_REQUIRE(ctx, rows <= INT32_MAX, "%s: %lld query rows of a head", what, (long long)rows);
    // Sequences with up to kStreamRows query rows of a key / value head stream their
    // keys, the others' keys go through LDS.  A batch whose sequences all have the
    // same number needs one of the two.
    const bool even = a.b.sequences * static_cast<int64_t>(a.b.max_new) == a.b.tokens;
    if (a.c.stride > kPagedBlockStride) return paged_stream_launch(ctx, a, cache->dtype, INT32_MAX);
    if (rows <= kStreamRows || !even)
        if (int st = paged_stream_launch(ctx, a, cache->dtype, kStreamRows)) return st;
    if (rows <= kStreamRows) return MIMIR_OK;
    return paged_block_launch(ctx, a, cache->dtype, kStreamRows + 1);
}
