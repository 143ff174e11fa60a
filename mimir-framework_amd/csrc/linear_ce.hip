// linear_ce.hip -- softmax cross entropy of a linear layer over a large vocabulary,
// and its gradients, without the logits in memory.
//
//   z_iv = x_i . w_v,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_i,t(i)
//   G_iv = g_i (exp(z_iv - lse_i) - [v = t(i)]),  dx = G w,  dw (+)= G^T x
//
// The reference has no loss on the device side of this path: its trainer hands
// Model::backwardPass a loss gradient (Model.cpp:7307-9153); this makes the one for
// a model's last layer.
//
// Forward: the product z = w x^T of matrix.hpp, 256 or 128 of the vocabulary by as
// many tokens a workgroup.  A lane has one token's logits in its registers, so the
// tile's maximum and sum of exp(z - maximum) cost one exchange between half waves
// and one through LDS; they go to part[tile][token] (8 bytes for 256 logits), and
// ce_finish joins them.
//
// Backward: the same product again for a piece of the vocabulary, whose epilogue
// writes G in bf16 (three planes for fp32 operands), then the two products with G.
// The logits again are a third of the backward's products: kept, they would be
// tokens x vocab values of memory from the one call to the other.  (A single call for the
// loss and its gradients could take the tokens in pieces and keep a piece's logits; with
// two, a program has the loss first and weighs it.)  G without its common
// factor (scale, and 1 / count for the mean): the factor is applied to the fp32 sums.
// Rounding G to bf16 beside bf16 operands is off by 2^-8 of a term at most, as rounding a
// layer's output gradient is, and averages out in the sums; two terms hold it to 2^-16
// (few tokens, or where the caller asks for it).
//
// Tokens without a target take no part: x's counted rows are gathered first, so the
// products run over those alone, and what stands in the others reaches nothing.
//
// Measured on MI355X, us: 2048 tokens x 4096 x 32000 bf16 forward 461 to 472; 8192 tokens
// forward and backward 7180 (products 1758, 1846, 1685, 1759); 32 tokens forward 55, the
// weights' 262 MB at 6.2 TB/s in the kernel, backward 64 for G and 76 and 73 for dx and dw;
// fp32 136, 116 and 177; 17 x 256 x 1000 fp32 10.7, two launches.
#include "matrix.hpp"

#include <algorithm>

using namespace mimir;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
// The maximum of nothing.
constexpr float kLowest = -3.40282347e38f;

// exp(z - m).  The difference first: z log2 e - m log2 e in one step is off by the rounding
// of m log2 e, so that the maximum itself would not give 1, a sum could come out below 1
// and a loss below 0, by more the larger the logits are.  (2048 tokens x 4096 x 32000 bf16
// forward 461 us, 458 in one step.)
__device__ __forceinline__ float exp_from(float z, float m) { return __builtin_amdgcn_exp2f((z - m) * kLog2e); }

// --- the counted rows --------------------------------------------------------------

struct GatherArgs {
    const void* x;
    int64_t ld_x;
    const int32_t* target;
    int64_t tokens, dim, vocab;
    uint16_t* dst;       // planes of [tokens][ld_dst]
    int64_t ld_dst, plane;
    float* raw;          // the rows as they are [tokens][dim] too (fp32), or null
    int32_t* row;        // [tokens]: the token of each gathered row
    int32_t* count;      // and a counter for ce_finish, zeroed
    const int32_t* blocks;  // how many tokens of each kGatherBlock count; null: there is one block
    float* zero_a;       // of tokens without a target: loss and lse, or null
    float* zero_b;
    void* dx;            // their gradient's rows are zeroed, or null
    int64_t ld_dx;
};

constexpr int kGatherRows = kBlock / kWave;
constexpr int64_t kGatherBlock = 8192;

__device__ __forceinline__ bool target_counts(const int32_t* target, int64_t i, int64_t vocab) {
    return static_cast<uint32_t>(target[i]) < static_cast<uint32_t>(vocab);
}

__device__ __forceinline__ int block_sum(int v, int* lds) {
#pragma unroll
    for (int s = 1; s < kWave; s *= 2) v += __shfl_xor(v, s);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) all += lds[w];
    return all;
}

// One block of tokens a workgroup.
__global__ __launch_bounds__(kBlock) void count_rows(const int32_t* target, int64_t tokens, int64_t vocab, int32_t* blocks) {
    __shared__ int lds[kBlock / kWave];
    const int64_t first = blockIdx.x * kGatherBlock;
    int mine = 0;
#pragma unroll 16
    for (int e = 0; e < kGatherBlock / kBlock; ++e) {
        const int64_t i = first + e * kBlock + threadIdx.x;
        mine += i < tokens && target_counts(target, i, vocab);
    }
    const int all = block_sum(mine, lds);
    if (threadIdx.x == 0) blocks[blockIdx.x] = all;
}

// Four tokens a workgroup, one a wave.  How many rows before its own count is found by
// reading the counts of the blocks before its own and the targets before them in it: at
// most 8 and 32 KB for 2^24 tokens, in L2.
template <bool BF16>
__global__ __launch_bounds__(kBlock) void gather_rows(GatherArgs a) {
    __shared__ int lds[kBlock / kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kGatherRows, t = t0 + wave;
    const auto counts = [&](int64_t i) { return target_counts(a.target, i, a.vocab); };
    const int64_t block = t0 / kGatherBlock;
    int mine = 0;
    for (int64_t i = threadIdx.x; i < block; i += kBlock) mine += a.blocks[i];
    for (int64_t i = block * kGatherBlock + threadIdx.x; i < t0; i += 4 * kBlock) {
        bool is[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) is[e] = i + e * kBlock < t0 && counts(i + e * kBlock);
        mine += is[0] + is[1] + is[2] + is[3];
    }
    int at = block_sum(mine, lds);
    const bool last = t0 + kGatherRows >= a.tokens;
    if (last && threadIdx.x == 0) {
        int all = at;
        for (int64_t i = t0; i < a.tokens; ++i) all += counts(i) ? 1 : 0;
        a.count[0] = all;
        a.count[1] = 0;  // ce_finish's workgroups that are done
    }
    if (t >= a.tokens) return;
    for (int64_t i = t0; i < t; ++i) at += counts(i) ? 1 : 0;
    if (counts(t)) {
        if (lane == 0) a.row[at] = static_cast<int32_t>(t);
#pragma unroll 4
        for (int64_t c = 8 * lane; c < a.ld_dst; c += 8 * kWave)
            mat_stage8<BF16>(a.x, t * a.ld_x + c, a.dim - c, a.dst + at * a.ld_dst + c, a.plane);
        if (!BF16 && a.raw)
            for (int64_t c = lane; c < a.dim; c += kWave) a.raw[at * a.dim + c] = static_cast<const float*>(a.x)[t * a.ld_x + c];
        return;
    }
    if (lane == 0 && a.zero_a) a.zero_a[t] = 0.0f, a.zero_b[t] = 0.0f;
    if (!a.dx) return;
    for (int64_t c = lane; c < a.dim; c += kWave) {
        if (BF16) static_cast<uint16_t*>(a.dx)[t * a.ld_dx + c] = 0;
        else static_cast<float*>(a.dx)[t * a.ld_dx + c] = 0.0f;
    }
}

// --- forward -----------------------------------------------------------------------

// (max, sum of exp(z - max)) of two sets; an empty one is (-infinity, 0).
__device__ __forceinline__ f2 join(f2 a, f2 b) {
    const float m = fmaxf(fmaxf(a[0], b[0]), kLowest);
    return f2{m, a[1] * exp_from(a[0], m) + b[1] * exp_from(b[0], m)};
}

struct CeStats {
    const int32_t* target;
    const int32_t* row;  // null: n itself
    f2* part;            // [tile][tokens]
    float* logit;        // [tokens]: the target's
    int64_t tokens, first;  // first: the piece's first vocabulary row
    int32_t tile0;          // and tile

    template <class S>
    __device__ __forceinline__ void run(const MatAt& at, MatAcc<S>& acc, char* lds) const {
        f2* red = reinterpret_cast<f2*>(lds);
        const bool whole = at.m0 + S::kM <= at.m;
#pragma unroll
        for (int j = 0; j < S::kBn; ++j) {
            const int32_t n = at.n0 + acc.n_of(j);
            const int64_t target = n < at.n ? target_of(n) - first - at.m0 : -1;
            // Few tiles hold any of their tokens' targets.
            if (__any(target >= 0 && target < S::kM)) {
                float hit = 0.0f;
                bool has = false;
#pragma unroll
                for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (acc.m_of(i, r) == target) hit = acc.c[i][j][r], has = true;
                if (has) logit[n] = hit;
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (at.m0 + acc.m_of(i, r) >= at.m) acc.c[i][j][r] = -__builtin_inff();
            }
            float m = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) m = fmaxf(m, acc.c[i][j][r]);
            const float top = fmaxf(m, kLowest);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += exp_from(acc.c[i][j][r], top);
            f2 v = join(f2{m, s}, f2{__shfl_xor(m, 32), __shfl_xor(s, 32)});
            if (threadIdx.x % kWave < 32) red[acc.wm * S::kN + acc.n_of(j)] = v;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < S::kN; c += S::kThreads) {
            if (at.n0 + c >= at.n) continue;
            f2 v = red[c];
#pragma unroll
            for (int w = 1; w < S::kWaveM; ++w) v = join(v, red[w * S::kN + c]);
            part[(tile0 + at.tile_m) * tokens + at.n0 + c] = v;
        }
    }
    __device__ __forceinline__ int64_t target_of(int32_t n) const { return target[row ? row[n] : n]; }
};

constexpr int kFinishTokens = 32;

struct FinishArgs {
    const f2* part;
    int64_t tokens;
    int32_t tiles;
    const float* logit;
    const int32_t* row;     // of the gathered tokens, *count of them; null: all tokens, one workgroup
    int32_t* count;         // and the counter of workgroups that are done
    const int32_t* target;  // row null
    int64_t vocab;
    float* loss;
    float* lse;
    double* sums;           // one for each workgroup
    float* mean;            // or null
};

// 32 tokens a workgroup, THREADS / 32 threads a token over the tiles.  The workgroup
// that is done last adds up all of them for the mean, in a fixed order and 64 bits.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void ce_finish(FinishArgs a) {
    constexpr int kParts = THREADS / kFinishTokens, kTogether = 4;
    __shared__ f2 red[kParts][kFinishTokens];
    __shared__ double wave_sums[THREADS / kWave];
    __shared__ bool last;
    const int t = threadIdx.x % kFinishTokens, p = threadIdx.x / kFinishTokens;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kFinishTokens + t;
    const int64_t limit = a.row ? *a.count : a.tokens;
    const bool in = n < limit && (a.row || static_cast<uint32_t>(a.target[n]) < static_cast<uint32_t>(a.vocab));
    f2 v{-__builtin_inff(), 0.0f};
    if (in)
        for (int32_t i = p; i < a.tiles; i += kTogether * kParts) {
            f2 x[kTogether];
#pragma unroll
            for (int e = 0; e < kTogether; ++e)
                x[e] = i + e * kParts < a.tiles ? a.part[(i + e * kParts) * a.tokens + n] : f2{-__builtin_inff(), 0.0f};
            v = join(v, join(join(x[0], x[1]), join(x[2], x[3])));
        }
    red[p][t] = v;
    __syncthreads();
    double sum = 0.0;
    if (p == 0 && n < limit) {
        float l = 0.0f, own = 0.0f;
        if (in) {
#pragma unroll
            for (int w = 1; w < kParts; ++w) v = join(v, red[w][t]);
            l = v[0] + logf(v[1]);
            own = l - a.logit[n];
            sum = own;
        }
        const int64_t to = a.row ? a.row[n] : n;
        a.loss[to] = own;
        a.lse[to] = l;
    }
    if (!a.mean) return;
    int32_t count = a.row ? static_cast<int32_t>(limit) : 0;
    if (threadIdx.x < kWave) {
        if (!a.row) count = __popcll(__ballot(p == 0 && in));
#pragma unroll
        for (int d = 1; d < kFinishTokens; d *= 2) sum += __shfl_xor(sum, d);
        if (threadIdx.x == 0) {
            last = !a.row;
            if (a.row) {
                __hip_atomic_store(a.sums + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last = __hip_atomic_fetch_add(a.count + 1, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int>(gridDim.x) - 1;
            }
        }
    }
    __syncthreads();
    if (!last) return;
    if (a.row) {
        sum = 0.0;
        for (uint32_t i = threadIdx.x; i < gridDim.x; i += THREADS)
            sum += __hip_atomic_load(a.sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d);
        if (threadIdx.x % kWave == 0) wave_sums[threadIdx.x / kWave] = sum;
        __syncthreads();
        for (int w = 1; w < THREADS / kWave; ++w)
            if (threadIdx.x == 0) sum += wave_sums[w];
    }
    if (threadIdx.x) return;
    a.mean[0] = static_cast<float>(sum / (count > 0 ? count : 1));
    a.mean[1] = static_cast<float>(count);
}

// --- backward ----------------------------------------------------------------------

// G of a piece of the vocabulary, PG planes of [n][ld], zeros from m on to ld.
template <int PG>
struct CeGrad {
    const int32_t* target;
    const int32_t* row;
    const float* lse;
    const float* dloss;  // null: 1
    uint16_t* g;
    int64_t ld, plane, first;
    float* raw;          // G as it is too, [n][ld_raw], zeros from m on, or null
    int64_t ld_raw;

    template <class S>
    __device__ __forceinline__ void run(const MatAt& at, MatAcc<S>& acc, char*) const {
#pragma unroll
        for (int j = 0; j < S::kBn; ++j) {
            const int32_t n = at.n0 + acc.n_of(j);
            const bool live = n < at.n;
            const int32_t t = live ? row[n] : 0;
            const int64_t hit = live ? target[t] - first - at.m0 : -1;
            const float base = live ? lse[t] : 0.0f, w = live && dloss ? dloss[t] : 1.0f;
#pragma unroll
            for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int32_t m = acc.m_of(i, 8 * h + e);
                        const float p = exp_from(acc.c[i][j][8 * h + e], base);
                        v[e] = at.m0 + m < at.m ? (p - (m == hit ? 1.0f : 0.0f)) * w : 0.0f;
                    }
                    if (PG == 3 && raw && live)
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            if (const int32_t m = at.m0 + acc.m_of(i, 8 * h + 4 * q); m < ld_raw)
                                *reinterpret_cast<f4*>(raw + n * ld_raw + m) = f4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                    const int32_t m = at.m0 + acc.m_of8(i, h);
                    uint16_t* to = g + n * ld + m;
#pragma unroll
                    for (int p = 0; p < PG; ++p) {
                        const u4 x = mat_pack8(v);
                        const u4 y = mat_exchange(x);  // every lane takes part
                        if (live && m < ld) *reinterpret_cast<u4*>(to + p * plane) = y;
                        if (p + 1 < PG)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                v[e] -= __builtin_bit_cast(float, e % 2 ? x[e / 2] & 0xffff0000u : x[e / 2] << 16);
                    }
                }
        }
    }
};

// --- the work's parts ----------------------------------------------------------------

struct Plan {
    int64_t ld, ld_g, piece;     // columns of x's and w's planes, of G's; the piece's rows of w
    int p, pg;                   // planes of x and w, of G
    bool w_direct, few;
    MatDeal deal_x, deal_w;      // dx's contraction over a piece, dw's over the tokens
    size_t x, raw_x, row, count, blocks, logit, sums, part, w, g, raw_g, partial, partial_w, total;
};

constexpr int64_t kPieceBytes = int64_t{512} << 20;
constexpr int64_t kTileM = 128;  // the smaller shape's: how many partial results a token has at most

// G of bf16 operands takes a second plane where tokens are few: up to 64 the products' time
// is the weights' bytes, and the fewer tokens a sum of dw runs over, the less its terms'
// roundings average out.  Measured, both gradients, 4096 x 32000: 33 tokens 270 us, 64 284,
// 128 322 with two planes, 129 286 with one.  With more tokens the caller chooses
// (MIMIR_NUM_TWO_TERMS): 129 tokens 290 / 386 us with one / two, 2048 1443 / 3028, 8192
// 5281 / 12372 (twice the products, in the smaller tiles).
constexpr int64_t kTwoPlaneTokens = 128;

Plan plan_of(const mimir_ctx* ctx, int type, const void* w, int64_t ld_w, int64_t tokens, int64_t dim, int64_t vocab, bool back,
             bool two_terms) {
    Plan p{};
    p.ld = mat_round(dim, 8);
    p.p = type == MIMIR_NUM_BF16 ? 1 : 3;
    p.pg = p.p == 3 ? 3 : two_terms || tokens <= kTwoPlaneTokens ? 2 : 1;
    p.w_direct = type == MIMIR_NUM_BF16 && mat_direct(w, ld_w, dim);
    // Few tokens in fp32: w's planes would be five times its bytes on the way.
    p.few = back && p.p == 3 && tokens <= kFewN && vocab <= (1 << 18) && few_direct(true, w, ld_w, dim);
    const int64_t of_row = (back ? tokens * p.pg * 2 : 0) + (p.w_direct ? 0 : p.ld * p.p * 2);
    if (ctx->tune.mat_piece > 0) p.piece = mat_round(ctx->tune.mat_piece, 8);
    else p.piece = of_row ? std::max<int64_t>(256, kPieceBytes / of_row / 256 * 256) : vocab;
    p.piece = std::min({p.few ? vocab + 8 : p.piece, mat_round(vocab, 8), int64_t{1} << 19});  // G's rows are within the operands' strides
    p.ld_g = mat_round(p.piece, 8);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t was = at;
        at += (bytes + 255) / 256 * 256;
        return was;
    };
    p.x = take(static_cast<size_t>(p.p * tokens * p.ld * 2));
    p.row = take(static_cast<size_t>(tokens * 4));
    p.count = take(8);
    p.blocks = take(static_cast<size_t>((tokens + kGatherBlock - 1) / kGatherBlock * 4));
    p.w = take(p.w_direct || p.few ? 0 : static_cast<size_t>(p.p * p.piece * p.ld * 2));
    if (back) {
        p.g = take(static_cast<size_t>(p.pg * tokens * p.ld_g * 2));
        const int64_t piece = std::min(p.piece, vocab);
        if (p.p == 3) {
            p.deal_x = mat_deal<3, 3, kCols, kRows>(ctx, dim, tokens, piece, 1, p.piece < vocab);
            p.deal_w = mat_deal<3, 3, kCols, kCols>(ctx, dim, piece, tokens, 1, false);
        } else if (p.pg == 2) {
            p.deal_x = mat_deal<1, 2, kCols, kRows>(ctx, dim, tokens, piece, 1, p.piece < vocab);
            p.deal_w = mat_deal<1, 2, kCols, kCols>(ctx, dim, piece, tokens, 1, false);
        } else {
            p.deal_x = mat_deal<1, 1, kCols, kRows>(ctx, dim, tokens, piece, 1, p.piece < vocab);
            p.deal_w = mat_deal<1, 1, kCols, kCols>(ctx, dim, piece, tokens, 1, false);
        }
        if (p.few) {
            p.raw_x = take(static_cast<size_t>(tokens * dim * 4));
            p.raw_g = take(static_cast<size_t>(tokens * mat_round(vocab, 4) * 4));
            p.deal_x.splits = few_splits(dim, vocab, 1);
            p.deal_x.partial = static_cast<size_t>(p.deal_x.splits * tokens * mat_round(dim, 4) * 4);
        }
        p.partial = take(p.deal_x.partial);
        p.partial_w = take(p.deal_w.partial);
    } else {
        p.logit = take(static_cast<size_t>(tokens * 4));
        p.sums = take(static_cast<size_t>((tokens + kFinishTokens - 1) / kFinishTokens * 8));
        const int64_t pieces = (vocab + p.piece - 1) / p.piece, tiles = (std::min(p.piece, vocab) + kTileM - 1) / kTileM;
        p.part = take(static_cast<size_t>(pieces * tiles * tokens * 8));
    }
    p.total = at;
    return p;
}

struct Call {
    int type;
    const void* x;
    int64_t ld_x;
    const void* w;
    int64_t ld_w;
    const int32_t* target;
    int64_t tokens, dim, vocab;
};

int check(mimir_ctx* ctx, const char* what, const Call& c) {
    MIMIR_REQUIRE(ctx, c.type == MIMIR_NUM_F32 || c.type == MIMIR_NUM_BF16, "%s: type %d", what, c.type);
    constexpr int64_t kMost = int64_t{1} << 24;
    MIMIR_REQUIRE(ctx, c.tokens >= 0 && c.tokens <= kMost && c.dim >= 1 && c.dim <= (1 << 18) && c.vocab >= 1 && c.vocab <= kMost,
                  "%s: tokens=%lld (0 to 2^24) dim=%lld (1 to 2^18) vocab=%lld (1 to 2^24)", what, (long long)c.tokens,
                  (long long)c.dim, (long long)c.vocab);
    MIMIR_REQUIRE(ctx, c.ld_x >= c.dim && c.ld_w >= c.dim, "%s: row strides (%lld, %lld) below dim", what, (long long)c.ld_x,
                  (long long)c.ld_w);
    return MIMIR_OK;
}

const char* rows_at(const Call& c, int64_t first) {
    return static_cast<const char*>(c.w) + first * c.ld_w * (c.type == MIMIR_NUM_BF16 ? 2 : 4);
}

// `blocks`: room for the blocks' counts, which a launch of its own makes where there is
// more than one.  Measured with / without, us, rows of 4096 bf16: 8200 tokens 32 / 26, 16384
// 51 / 47, 32768 109 / 161, 65536 196 / 391, 262144 764 / 2732.
int gather(mimir_ctx* ctx, const Call& c, GatherArgs a, int32_t* blocks) {
    if (c.tokens > kGatherBlock) {
        count_rows<<<static_cast<unsigned>((c.tokens + kGatherBlock - 1) / kGatherBlock), kBlock, 0, ctx->stream>>>(c.target, c.tokens,
                                                                                                                   c.vocab, blocks);
        if (int st = launched(ctx, "count_rows")) return st;
        a.blocks = blocks;
    }
    const auto grid = static_cast<unsigned>((c.tokens + kGatherRows - 1) / kGatherRows);
    if (c.type == MIMIR_NUM_BF16) gather_rows<true><<<grid, kBlock, 0, ctx->stream>>>(a);
    else gather_rows<false><<<grid, kBlock, 0, ctx->stream>>>(a);
    return launched(ctx, "gather_rows");
}

// The piece's rows of w as an operand, from `first` on.
int weights(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, int64_t first, int64_t rows, MatOperand* out) {
    if (p.w_direct) {
        *out = MatOperand{reinterpret_cast<const uint16_t*>(rows_at(c, first)), c.ld_w, 0};
        return MIMIR_OK;
    }
    auto* dst = reinterpret_cast<uint16_t*>(work + p.w);
    *out = MatOperand{dst, p.ld, p.piece * p.ld};
    return mat_stage(ctx, c.type, rows_at(c, first), rows, c.dim, c.ld_w, dst, p.ld, p.piece * p.ld);
}

MatArgs args_of(const MatOperand& a, const MatOperand& b, int64_t m, int64_t n, int64_t k) {
    MatArgs g{};
    g.a[0] = a;
    g.b[0] = b;
    g.m = static_cast<int32_t>(m);
    g.n = static_cast<int32_t>(n);
    g.k = static_cast<int32_t>(k);
    g.segments = g.batches = g.splits = 1;
    return g;
}

template <int P>
int forward(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, float* loss, float* lse, float* mean) {
    const MatOperand x{reinterpret_cast<const uint16_t*>(work + p.x), p.ld, c.tokens * p.ld};
    auto* row = reinterpret_cast<int32_t*>(work + p.row);
    auto* count = reinterpret_cast<int32_t*>(work + p.count);
    CeStats e{c.target, row, reinterpret_cast<f2*>(work + p.part), reinterpret_cast<float*>(work + p.logit), c.tokens, 0, 0};
    for (int64_t first = 0; first < c.vocab; first += p.piece) {
        const int64_t rows = std::min(p.piece, c.vocab - first);
        MatOperand w;
        if (int st = weights(ctx, c, p, work, first, rows, &w)) return st;
        MatArgs g = args_of(w, x, rows, c.tokens, c.dim);
        g.n_dev = count;
        e.first = first;
        using B = MatBig<P, P, kRows, kRows>;
        using S = MatSmall<P, P, kRows, kRows>;
        const bool big = mat_fills<B>(ctx, g);
        const int st = big ? mat_launch<B>(ctx, "cross entropy statistics", g, e) : mat_launch<S>(ctx, "cross entropy statistics", g, e);
        if (st) return st;
        e.tile0 += static_cast<int32_t>((rows + (big ? B::kM : S::kM) - 1) / (big ? B::kM : S::kM));
    }
    const FinishArgs f{e.part, c.tokens, e.tile0, e.logit, row, count, nullptr, 0, loss, lse, reinterpret_cast<double*>(work + p.sums), mean};
    ce_finish<kBlock><<<static_cast<unsigned>((c.tokens + kFinishTokens - 1) / kFinishTokens), kBlock, 0, ctx->stream>>>(f);
    return launched(ctx, "ce_finish");
}

// Few tokens, operands that can be read as they are: no token is gathered and no operand
// staged.
bool few_applies(const Call& c) {
    const bool fp32 = c.type == MIMIR_NUM_F32;
    return c.tokens <= kFewN && few_direct(fp32, c.x, c.ld_x, c.dim) && few_direct(fp32, c.w, c.ld_w, c.dim);
}

template <bool FP32>
int forward_few(mimir_ctx* ctx, const Call& c, float* loss, float* lse, float* mean) {
    constexpr int64_t kRowsOf = 32 * kFewBlocks;
    const int64_t tiles = (c.vocab + kRowsOf - 1) / kRowsOf;
    char* work;
    if (int st = mat_scratch(ctx, 256 + static_cast<size_t>(tiles * c.tokens * 8), &work)) return st;
    const auto operand = [](const void* p, int64_t ld) { return MatOperand{static_cast<const uint16_t*>(p), ld, 0}; };
    const MatArgs g = args_of(operand(c.w, c.ld_w), operand(c.x, c.ld_x), c.vocab, c.tokens, c.dim);
    const CeStats e{c.target, nullptr, reinterpret_cast<f2*>(work + 256), reinterpret_cast<float*>(work), c.tokens, 0, 0};
    if (int st = few_launch<FP32, kRows, false>(ctx, "cross entropy statistics", g, e)) return st;
    const FinishArgs f{e.part, c.tokens, static_cast<int32_t>(tiles), e.logit, nullptr, nullptr, c.target, c.vocab, loss, lse, nullptr, mean};
    ce_finish<1024><<<1, 1024, 0, ctx->stream>>>(f);
    return launched(ctx, "ce_finish");
}

struct Gradients {
    const float* lse;
    const float* dloss;
    const float* mean;
    float scale;
    void* dx;
    int64_t ld_dx;
    void* dw;
    int64_t ld_dw;
    int accumulate_x, accumulate_w;
};

// P planes of x and w, PG of G.
template <int P, int PG>
int backward(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, const Gradients& d) {
    const MatOperand x{reinterpret_cast<const uint16_t*>(work + p.x), p.ld, c.tokens * p.ld};
    const MatOperand gr{reinterpret_cast<const uint16_t*>(work + p.g), p.ld_g, c.tokens * p.ld_g};
    auto* row = reinterpret_cast<int32_t*>(work + p.row);
    auto* count = reinterpret_cast<int32_t*>(work + p.count);
    const int bf16 = c.type == MIMIR_NUM_BF16;
    const int64_t size = bf16 ? 2 : 4;
    MatOut ox{};
    ox.out[0] = d.dx;
    ox.ld = d.ld_dx;
    ox.row = row;
    ox.partial = reinterpret_cast<float*>(work + p.partial);
    ox.count = d.mean ? d.mean + 1 : nullptr;
    ox.alpha = d.scale;
    ox.bf16 = bf16;
    ox.accumulate = d.accumulate_x;
    MatOut ow = ox;
    ow.row = nullptr;
    ow.partial = reinterpret_cast<float*>(work + p.partial_w);
    ow.ld = d.ld_dw;
    ow.accumulate = d.accumulate_w;
    ow.last = 1;
    CeGrad<PG> e{c.target, row, d.lse, d.dloss, reinterpret_cast<uint16_t*>(work + p.g), p.ld_g, c.tokens * p.ld_g, 0,
                 p.few ? reinterpret_cast<float*>(work + p.raw_g) : nullptr, mat_round(c.vocab, 4)};
    const bool few = P == 3 && p.few;
    const auto as_is = [](const void* q, int64_t ld) { return MatOperand{static_cast<const uint16_t*>(q), ld, 0}; };

    for (int64_t first = 0; first < c.vocab; first += p.piece) {
        const int64_t rows = std::min(p.piece, c.vocab - first);
        MatOperand w = as_is(c.w, c.ld_w);
        if (!few)
            if (int st = weights(ctx, c, p, work, first, rows, &w)) return st;
        MatArgs g = args_of(w, few ? as_is(work + p.raw_x, c.dim) : x, rows, c.tokens, c.dim);
        g.n_dev = count;
        e.first = first;
        using BG = MatBig<P, P, kRows, kRows>;
        using SG = MatSmall<P, P, kRows, kRows>;
        int st = MIMIR_OK;
        if (!few) {
            st = mat_fills<BG>(ctx, g) ? mat_launch<BG>(ctx, "cross entropy gradient", g, e)
                                       : mat_launch<SG>(ctx, "cross entropy gradient", g, e);
        } else if constexpr (P == 3) {
            st = few_launch<true, kRows, false>(ctx, "cross entropy gradient", g, e);
        }
        if (st) return st;
        if (d.dx) {
            g = args_of(w, gr, c.dim, c.tokens, rows);
            g.n_dev = count;
            ox.read_partial = first > 0;
            ox.last = first + rows >= c.vocab;
            if (!few) {
                st = mat_product<P, PG, kCols, kRows>(ctx, "cross entropy dx", g, ox, p.deal_x);
            } else if constexpr (P == 3) {
                g.b[0] = as_is(work + p.raw_g, mat_round(c.vocab, 4));
                g.splits = p.deal_x.splits;
                st = few_product<kCols>(ctx, "cross entropy dx", g, ox);
            }
            if (st) return st;
        }
        if (d.dw) {
            g = args_of(x, gr, c.dim, rows, c.tokens);
            g.k_dev = count;
            ow.out[0] = static_cast<char*>(d.dw) + first * d.ld_dw * size;
            st = mat_product<P, PG, kCols, kCols>(ctx, "cross entropy dw", g, ow, p.deal_w);
            if (st) return st;
        }
    }
    return MIMIR_OK;
}

}  // namespace

extern "C" {

int mimir_linear_cross_entropy_fwd(mimir_ctx* ctx, int type, const void* x, int64_t ld_x, const void* w, int64_t ld_w,
                                   const int32_t* targets, int64_t tokens, int64_t dim, int64_t vocab, float* loss, float* lse,
                                   float* mean) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "linear cross entropy";
    const Call c{type, x, ld_x, w, ld_w, targets, tokens, dim, vocab};
    if (int st = check(ctx, what, c)) return st;
    MIMIR_REQUIRE(ctx, tokens == 0 || (x && w && targets && loss && lse), "%s: null pointer", what);
    MIMIR_REQUIRE(ctx, mat_apart({loss, lse, mean}, {x, w, targets}), "%s: an output is an input or another output", what);
    if (tokens == 0 && !mean) return MIMIR_OK;
    MIMIR_ENTER(ctx);
    if (tokens == 0) return mimir_fill_f32(ctx, mean, 2, 0.0f);
    if (few_applies(c))
        return type == MIMIR_NUM_F32 ? forward_few<true>(ctx, c, loss, lse, mean) : forward_few<false>(ctx, c, loss, lse, mean);
    const Plan p = plan_of(ctx, type, w, ld_w, tokens, dim, vocab, false, false);
    char* work;
    if (int st = mat_scratch(ctx, p.total, &work)) return st;
    auto* count = reinterpret_cast<int32_t*>(work + p.count);
    const GatherArgs a{x, ld_x, targets, tokens, dim, vocab, reinterpret_cast<uint16_t*>(work + p.x), p.ld, tokens * p.ld,
                       nullptr, reinterpret_cast<int32_t*>(work + p.row), count, nullptr, loss, lse, nullptr, 0};
    if (int st = gather(ctx, c, a, reinterpret_cast<int32_t*>(work + p.blocks))) return st;
    return p.p == 1 ? forward<1>(ctx, c, p, work, loss, lse, mean) : forward<3>(ctx, c, p, work, loss, lse, mean);
}

int mimir_linear_cross_entropy_bwd(mimir_ctx* ctx, int type, const void* x, int64_t ld_x, const void* w, int64_t ld_w,
                                   const int32_t* targets, int64_t tokens, int64_t dim, int64_t vocab, const float* lse,
                                   const float* dloss, const float* mean, float scale, void* dx, int64_t ld_dx, int accumulate_x,
                                   void* dw, int64_t ld_dw, int accumulate_w) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "linear cross entropy gradient";
    const bool two_terms = type == (MIMIR_NUM_BF16 | MIMIR_NUM_TWO_TERMS);
    if (two_terms) type = MIMIR_NUM_BF16;
    const Call c{type, x, ld_x, w, ld_w, targets, tokens, dim, vocab};
    if (int st = check(ctx, what, c)) return st;
    MIMIR_REQUIRE(ctx, (!dx || ld_dx >= dim) && (!dw || ld_dw >= dim), "%s: gradient strides (%lld, %lld) below dim", what,
                  (long long)ld_dx, (long long)ld_dw);
    MIMIR_REQUIRE(ctx, tokens == 0 || (x && w && targets && lse), "%s: null pointer", what);
    MIMIR_REQUIRE(ctx, mat_apart({dw}, {x, w, targets, lse, dloss, mean}) && mat_apart({dx, dw}, {w, targets, lse, dloss, mean}),
                  "%s: dx may be x, and no other output an input", what);
    MIMIR_REQUIRE(ctx, !dx || dx != x || ld_dx == ld_x, "%s: dx in place needs equal strides", what);
    if (!dx && !dw) return MIMIR_OK;
    MIMIR_ENTER(ctx);
    // Without tokens no input is looked at (w may be null).
    if (tokens == 0) return dw && !accumulate_w ? mat_zero(ctx, type, dw, vocab, dim, ld_dw) : MIMIR_OK;
    Plan p = plan_of(ctx, type, w, ld_w, tokens, dim, vocab, true, two_terms);
    char* work;
    if (int st = mat_scratch(ctx, p.total, &work)) return st;
    auto* count = reinterpret_cast<int32_t*>(work + p.count);
    const Gradients d{lse, dloss, mean, scale, dx, ld_dx, dw, ld_dw, accumulate_x ? 1 : 0, accumulate_w ? 1 : 0};
    const GatherArgs a{x, ld_x, targets, tokens, dim, vocab, reinterpret_cast<uint16_t*>(work + p.x), p.ld, tokens * p.ld,
                       p.few ? reinterpret_cast<float*>(work + p.raw_x) : nullptr, reinterpret_cast<int32_t*>(work + p.row), count, nullptr, nullptr, nullptr,
                       accumulate_x ? nullptr : dx, ld_dx};
    if (int st = gather(ctx, c, a, reinterpret_cast<int32_t*>(work + p.blocks))) return st;
    if (p.p == 3) return backward<3, 3>(ctx, c, p, work, d);
    return p.pg == 2 ? backward<1, 2>(ctx, c, p, work, d) : backward<1, 1>(ctx, c, p, work, d);
}

}  // extern "C"
