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

// Query rows of a key / value head that the stream kernel takes, of all sequences or of
// those beside longer ones.  Where the block kernel would take as long (40 to 64 rows,
// stream / block, us): 32 sequences x 3000 keys x 4 heads of 128, bf16 90-98 / 86-88,
// 8-bit 76-82 / 92-93, fp32 162-167 / 181-185; one of 30000 x 8 heads, 64 rows, bf16
// 62 / 86, 8-bit 58 / 88, fp32 111 / 141.  Beside longer ones it has 16 rows a block, and
// so it has of fp32 heads over 128, which are the block kernel's from there on (32
// sequences x 3000 keys x 4 heads of 256, 32 rows 369 / 173, 64 720 / 234).
constexpr int64_t kStreamRows = 64, kStreamBeside = 32, kStreamWide = 16;

// The shares of a block's rows: each brought to one max, added up and divided.  LPR
// lanes hold a row, four dimensions each.  ONE: the whole workgroup takes a row at a
// time, its groups of lanes every so many of the runs (a long sequence's block may have
// hundreds); else each group a row of its own.  The block's first run, whose descriptor
// is the workgroup's, kept what it begins, the others what they go on with.  `parts`
// workgroups for each descriptor.
template <int LPR, bool ONE>
__device__ __forceinline__ void join_rows(const PagedArgs& p, const PagedRuns& a, uint32_t parts, uint32_t block,
                                          f4 (*share)[LPR], f2* stats) {
    constexpr int kAhead = 4, kGroups = kBlock / LPR, kEach = ONE ? kGroups : 1, kRowsOf = ONE ? 1 : kGroups;
    const uint32_t first = block / parts;
    const PagedShared s = a.shared[first];
    if (s.runs <= 1) return;
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, d = p.c.head_dim;
    for (int row0 = static_cast<int>(block % parts) * kRowsOf; row0 < s.rows; row0 += static_cast<int>(parts) * kRowsOf) {
        const int row = row0 + (ONE ? 0 : group);
        const bool mine = row < s.rows;
        float m = -1e30f, l = 0.f;
        f4 acc{0.f, 0.f, 0.f, 0.f};
        for (int i = ONE ? group : 0; mine && i < s.runs; i += kAhead * kEach) {
            f2 st[kAhead];
            f4 x[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int j = i + u * kEach;
                st[u] = f2{-1e30f, 0.f};
                x[u] = f4{0.f, 0.f, 0.f, 0.f};
                if (j >= s.runs) continue;
                const PagedPart part(a, d, first + static_cast<uint32_t>(j), j == 0);
                st[u] = *part.stat(row);
                if (4 * lane < d) x[u] = *reinterpret_cast<const f4*>(part.sums(row) + 4 * lane);
            }
            float m_new = m;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) m_new = fmaxf(m_new, st[u][0]);
            const float f = __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= f;
            acc *= f;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float g = __builtin_amdgcn_exp2f(st[u][0] - m);
                l += st[u][1] * g;
                acc += x[u] * g;
            }
        }
        if constexpr (ONE) {
            share[group][lane] = acc;
            if (lane == 0) stats[group] = f2{m, l};
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int v = 1; v < kGroups; ++v) {
                    const f2 st = stats[v];
                    const float m_new = fmaxf(m, st[0]);
                    const float f = __builtin_amdgcn_exp2f(m - m_new), g = __builtin_amdgcn_exp2f(st[0] - m_new);
                    m = m_new;
                    l = l * f + st[1] * g;
                    acc = acc * f + share[v][lane] * g;
                }
            }
            __syncthreads();  // the next row's shares
        }
        if (!mine || (ONE && group > 0)) continue;
        const float inv = 1.0f / (l + 1e-9f);
        float* out = p.out + paged_row(p, p.ld_out, s.first, s.head, s.row0 + row);
#pragma unroll
        for (int e = 0; e < 4; ++e)  // a row's sums may be followed by what nothing wrote
            if (4 * lane + e < d) out[4 * lane + e] = acc[e] * inv;
    }
}

// Of one launch's blocks, and of another's behind them.
template <int LPR>
__global__ __launch_bounds__(kBlock) void paged_join(PagedArgs p, PagedRuns a, uint32_t parts_a, PagedRuns b, uint32_t parts_b) {
    constexpr int kGroups = kBlock / LPR;
    __shared__ f4 share[kGroups][LPR];
    __shared__ f2 stats[kGroups];
    const uint32_t of_a = a.runs * parts_a;
    const bool first = blockIdx.x < of_a;
    const PagedRuns& r = first ? a : b;
    const uint32_t parts = first ? parts_a : parts_b, block = first ? blockIdx.x : blockIdx.x - of_a;
    if (r.many) join_rows<LPR, true>(p, r, parts, block, share, stats);
    else join_rows<LPR, false>(p, r, parts, block, share, stats);
}

template <int LPR>
void launch_join(const PagedArgs& p, const PagedRuns& a, const PagedRuns& b, hipStream_t s) {
    constexpr int kRowsOf = kBlock / LPR;
    const auto parts = [](const PagedRuns& x) {
        return static_cast<uint32_t>(x.many ? std::min(x.part_rows, 8) : (x.part_rows + kRowsOf - 1) / kRowsOf);
    };
    paged_join<LPR><<<a.runs * parts(a) + b.runs * parts(b), kBlock, 0, s>>>(p, a, parts(a), b, parts(b));
}

// Joins the blocks that several runs had keys of; a launch that cut none has no runs.
int join(mimir_ctx* ctx, const PagedArgs& p, const PagedRuns& a, const PagedRuns& b) {
    if (a.runs + b.runs == 0) return MIMIR_OK;
    if (p.c.head_dim <= 128) launch_join<32>(p, a, b, ctx->stream);
    else launch_join<64>(p, a, b, ctx->stream);
    return launched(ctx, "paged_join");
}

}  // namespace

int64_t mimir::paged_runs(mimir_ctx* ctx, const PagedArgs& p, PagedRuns* a, int64_t runs, int64_t blocks, int threads, bool split,
                          bool beside) {
    split = split || !dispatch_fits(blocks, threads);
    // No more than keep to the least length of a run (PagedWalk), by the longest costs, each block's last one shorter.
    const int64_t cost = a->extra + static_cast<int64_t>(p.b.max_len) + (p.causal ? (a->block_rows + p.group - 1) / p.group : 0);
    if (blocks < 1 << 24) runs = std::max<int64_t>(1, std::min(runs, blocks * (cost / a->least + 1)));
    a->apart = p.b.sequences <= kWave;
    a->many = a->part_rows <= 32 && runs > 4 * blocks;
    constexpr size_t kAlone = kPagedWorkBytes - kPagedBesideBytes;
    const int64_t bytes = runs * (static_cast<int64_t>(sizeof(PagedShared)) + 2 * 4 * paged_part_floats(a->part_rows, p.c.head_dim));
    if (!split || bytes > static_cast<int64_t>(beside ? kPagedBesideBytes : kAlone)) return blocks;
    char* work = paged_work(ctx);
    if (!work) return blocks;
    if (beside) work += kAlone;
    a->shared = reinterpret_cast<PagedShared*>(work);
    a->part = reinterpret_cast<float*>(work + runs * sizeof(PagedShared));
    a->runs = static_cast<uint32_t>(runs);
    return runs;
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
    MIMIR_REQUIRE(ctx, q != out, "%s: out must not be q", what);
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
    // Sequences with few query rows of a key / value head stream their keys, the others'
    // keys go through LDS, by a launch each.  A batch whose sequences all have max_new
    // tokens (or whose rows would suffice for that) has the second alone, which takes any;
    // so has one of short contexts with up to 256 (sequence, key / value head) pairs, or, of
    // fp32 heads over 64, of whose streaming workgroups a compute unit holds one, 1024.  One
    // launch / two, us, chunks of 91 tokens beside single ones, up to 100 keys before them,
    // sequences x 8 heads.  One chunk: bf16 heads of 128, 256 pairs 21 / 29, 512 27 / 36, 1024
    // 43 / 45, 1792 68 / 61; 8-bit 25 / 33, 31 / 39, 47 / 48, 76 / 62; fp32 38 / 57, 69 / 77,
    // 124 / 114, 209 / 171; fp32 heads of 64 19 / 28, 25 / 35, 38 / 43, 61 / 60, of 256 49 / 54,
    // 85 / 75, 153 / 133, 255 / 221.  A chunk to seven single tokens: bf16 28 / 36, 40 / 46,
    // 61 / 69, 100 / 105; fp32 50 / 59, 86 / 89, 150 / 160, 257 / 272, heads of 96 35 / 54,
    // 47 / 77, 73 / 130, 119 / 209.  (So the sides meet between 500 and 1800 pairs, by the
    // type and by how many chunks there are: 256 is on the low side, 1024 within it.)
    const int64_t rows = static_cast<int64_t>(a.b.max_new) * a.group;
    MIMIR_REQUIRE(ctx, rows <= INT32_MAX, "%s: %lld query rows of a head", what, (long long)rows);
    PagedRuns few{}, others{};
    const int64_t pairs = cache->dtype == MIMIR_KV_F32 && a.c.stride > 64 ? 1024 : 256;
    const int64_t streamed = cache->dtype == MIMIR_KV_F32 && a.c.stride > 128 ? kStreamWide : kStreamRows;
    if (rows <= streamed) {
        if (int st = paged_stream_launch(ctx, a, cache->dtype, INT32_MAX, false, &few)) return st;
    } else {
        const int64_t sequences = a.b.sequences;
        const bool both = sequences * a.b.max_new > a.b.tokens && (a.b.max_len > kWholeLen || sequences * a.c.kv_heads > pairs);
        if (both)
            if (int st = paged_stream_launch(ctx, a, cache->dtype, std::min(streamed, kStreamBeside), true, &few)) return st;
        if (int st = paged_block_launch(ctx, a, cache->dtype, both ? std::min(streamed, kStreamBeside) + 1 : 1, &others)) return st;
    }
    return join(ctx, a, few, others);
}
