// gated_linear.hip -- the gated products at the head of a feed-forward block, and
// their gradients:
//
//   gate = x Wg,  up = x Wu,  y = act(gate) * up        act: SiLU or tanh-GELU
//   du = dy * act(gate),  dg = dy * up * act'(gate)
//   dx = dg Wg^T + du Wu^T,  dWg (+)= x^T dg,  dWu (+)= x^T du
//
// The reference runs them as layers of their own, on the host: two Linear layers,
// LayerOps::silu_forward / gelu_forward (LayerOps.hpp:556-581) and multiply_forward
// (:205-230).
//
// Forward: one product of matrix.hpp whose A tile is half gate columns, half up
// columns, so a lane ends with both values of its elements and gate and up are
// written only where the backward is to read them.  Backward: dg and du come from
// gate, up and dy in one pass, in bf16 (three planes for fp32 operands, two where
// tokens are few), then dx is one product over both weights' columns and dWg, dWu are
// two batches of another.  The pass is bound by its bytes (20 or 12 a value beside
// 4 or 12 written), the products by the matrix cores.
//
// Measured on MI355X, us: 2048 tokens x 4096 x 11008 bf16 forward 335 (1.10 PFLOP/s); 8192
// tokens forward and backward 4370 (forward 1562, the pass 258 = 5.6 TB/s, dx 1249, both
// weights' 1300); 1021 x 1024 x 2752 fp32 both 258; 7 tokens fp32 forward 17.4; 8 tokens x
// 4096 x 11008 forward 40 bf16 and 111 fp32, backward 106 and 210.
#include "matrix.hpp"
#include "pointwise.hpp"

using namespace mimir;

namespace {

enum : int { kSilu = MIMIR_ACT_SILU, kGelu = MIMIR_ACT_GELU };

template <int ACT>
__device__ __forceinline__ float act1(float x) {
    return ACT == kSilu ? silu1(x) : gelu1(x);
}

// act(x) and act'(x).  With s = sigmoid(v), v = x or 2u of the tanh-GELU: act = x s,
// act' = s + x s (1 - s) v'.  From e = exp(-|v|): s and 1 - s without cancellation.  v'
// of the GELU is taken at |x| <= 100: from 14 on 1 - s or s is zero.
template <int ACT>
__device__ __forceinline__ f2 act_slope(float x) {
    const float k = 2.0f * __builtin_sqrtf(2.0f / 3.14159265359f);
    const float v = ACT == kSilu ? x : k * (x + 0.044715f * x * x * x);
    const float t = fminf(fabsf(x), 100.0f);
    const float slope = ACT == kSilu ? 1.0f : k * (1.0f + 3.0f * 0.044715f * t * t);
    const float e = expf(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
    const float s = v >= 0.0f ? r : e * r;
    return f2{act1<ACT>(x), s + (x * (e * r) * r) * slope};
}

// --- forward -----------------------------------------------------------------------

template <int ACT>
struct GatedOut {
    MatOut y;
    float* gate_up;  // [n][2 * hidden], or null
    int64_t hidden;

    template <class S>
    __device__ __forceinline__ void run(const MatAt& at, MatAcc<S>& acc, char*) const {
#pragma unroll
        for (int j = 0; j < S::kBn; ++j) {
            const int32_t n = at.n0 + acc.n_of(j);
            const bool live = n < at.n;
#pragma unroll
            for (int i = 0; i < S::kSubBlocks; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f4 g[2], u[2];
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        g[e / 4][e % 4] = acc.c[i][j][8 * h + e];
                        u[e / 4][e % 4] = acc.c[i + S::kSubBlocks][j][8 * h + e];
                        v[e] = act1<ACT>(acc.c[i][j][8 * h + e]) * acc.c[i + S::kSubBlocks][j][8 * h + e];
                    }
                    if (y.bf16) {
                        const u4 x = mat_exchange(mat_pack8(v));
                        if (live) y.put8(0, n, at.m0 + acc.m_of8(i, h), at.m, x);
                    }
                    if (!live) continue;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int32_t m = at.m0 + acc.m_of(i, 8 * h + 4 * q);
                        if (m >= at.m) continue;
                        if (!y.bf16) y.put(0, n, m, at.m, f4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]}, 1.0f);
                        if (!gate_up) continue;
                        float* to = gate_up + n * 2 * hidden + m;
                        if (m + 4 <= at.m) {
                            *reinterpret_cast<f4u*>(to) = g[q];
                            *reinterpret_cast<f4u*>(to + hidden) = u[q];
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (m + e < at.m) to[e] = g[q][e], to[hidden + e] = u[q][e];
                        }
                    }
                }
        }
    }
};

// y from gate and up, eight columns a thread.
struct ActArgs {
    const float* gate_up;  // [tokens][2 * hidden]
    int64_t tokens, hidden;
    void* y;
    int64_t ld_y;
};
template <int ACT, bool BF16>
__global__ __launch_bounds__(kBlock) void gated_act(ActArgs a) {
    const int64_t of_row = (a.hidden + 7) / 8, total = a.tokens * of_row, stride = static_cast<int64_t>(gridDim.x) * kBlock;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += stride) {
        const int64_t t = i / of_row, c = i % of_row * 8;
        const float* gp = a.gate_up + t * 2 * a.hidden + c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (c + e >= a.hidden) break;
            const float v = act1<ACT>(gp[e]) * gp[a.hidden + e];
            if (BF16) static_cast<uint16_t*>(a.y)[t * a.ld_y + c + e] = static_cast<uint16_t>(pack_bf16(v, v));
            else static_cast<float*>(a.y)[t * a.ld_y + c + e] = v;
        }
    }
}

// --- backward ----------------------------------------------------------------------

struct GradArgs {
    const float* gate_up;  // at the piece's first column
    int64_t hidden;
    const void* dy;        // likewise
    int64_t ld_dy;
    uint16_t* out;         // planes of [tokens][2 * cols_out]: dg, then du
    int64_t tokens, cols, cols_out, plane;
    float* raw;            // also as they are, dg [tokens][cols] then du, or null
};

// Eight columns a thread; columns from `cols` on are zeros.
template <int ACT, bool BF16, int PG>
__global__ __launch_bounds__(kBlock) void gated_grad(GradArgs a) {
    const int64_t of_row = a.cols_out / 8, total = a.tokens * of_row, stride = static_cast<int64_t>(gridDim.x) * kBlock;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += stride) {
        const int64_t t = i / of_row, c = i % of_row * 8, left = a.cols - c;
        const float* gp = a.gate_up + t * 2 * a.hidden + c;
        const float* up = gp + a.hidden;
        float g[8], u[8], d[8];
        if (left >= 8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f4u x = __builtin_nontemporal_load(reinterpret_cast<const f4u*>(gp + 4 * h));
                const f4u y = __builtin_nontemporal_load(reinterpret_cast<const f4u*>(up + 4 * h));
#pragma unroll
                for (int e = 0; e < 4; ++e) g[4 * h + e] = x[e], u[4 * h + e] = y[e];
            }
            if constexpr (BF16) {
                const u4e x = *reinterpret_cast<const u4e*>(static_cast<const uint16_t*>(a.dy) + t * a.ld_dy + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = __builtin_bit_cast(float, e % 2 ? x[e / 2] & 0xffff0000u : x[e / 2] << 16);
            } else {
                const float* p = static_cast<const float*>(a.dy) + t * a.ld_dy + c;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f4u x = __builtin_nontemporal_load(reinterpret_cast<const f4u*>(p + 4 * h));
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[4 * h + e] = x[e];
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = e < left;
                g[e] = in ? gp[e] : 0.0f;
                u[e] = in ? up[e] : 0.0f;
                if constexpr (BF16)
                    d[e] = in ? __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(a.dy)[t * a.ld_dy + c + e]) << 16) : 0.0f;
                else
                    d[e] = in ? static_cast<const float*>(a.dy)[t * a.ld_dy + c + e] : 0.0f;
            }
        }
        float dg[8], du[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const f2 s = act_slope<ACT>(g[e]);
            du[e] = d[e] * s[0];
            dg[e] = d[e] * u[e] * s[1];
        }
        if (PG == 3 && a.raw) {
            float* to = a.raw + t * a.cols + c;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (4 * h + 4 <= left) {
                    *reinterpret_cast<f4u*>(to + 4 * h) = f4u{dg[4 * h], dg[4 * h + 1], dg[4 * h + 2], dg[4 * h + 3]};
                    *reinterpret_cast<f4u*>(to + a.tokens * a.cols + 4 * h) = f4u{du[4 * h], du[4 * h + 1], du[4 * h + 2], du[4 * h + 3]};
                } else {
#pragma unroll
                    for (int e = 4 * h; e < 4 * h + 3; ++e)
                        if (e < left) to[e] = dg[e], to[a.tokens * a.cols + e] = du[e];
                }
        }
        uint16_t* to = a.out + t * 2 * a.cols_out + c;
        const Split8 x = split8(dg), y = split8(du);
        const u4 xs[3] = {x.h, x.m, x.l}, ys[3] = {y.h, y.m, y.l};
#pragma unroll
        for (int p = 0; p < PG; ++p) {
            *reinterpret_cast<u4*>(to + p * a.plane) = xs[p];
            *reinterpret_cast<u4*>(to + a.cols_out + p * a.plane) = ys[p];
        }
    }
}

// --- the work's parts --------------------------------------------------------------

constexpr int64_t kPieceBytes = int64_t{512} << 20;
// As linear_ce.hip's.  Measured, gradients of 4096 x 11008 bf16: 64 tokens 147 us, 128 177
// with two planes, 129 153 with one; the gradients' error is 1.4 times a single rounding's
// with one, 1.0 with two.  With more tokens (MIMIR_NUM_TWO_TERMS) one / two: 129 156 / 223, 2048
// 771 / 1817, 8192 2669 / 7624.
constexpr int64_t kTwoPlaneTokens = 128;

struct Call {
    int type, act;
    const void* x;
    int64_t ld_x;
    const void* w[2];
    int64_t ld_w, tokens, dim, hidden;
};

struct Plan {
    int p, pg;
    int64_t ld_x, piece, ld_w;  // columns of x's planes; a piece's columns of the weights, their planes' columns
    bool x_direct, w_direct, few;
    bool split;                 // forward: few tiles, so the contraction is dealt out and the activation a pass of its own
    MatDeal deal_y;
    size_t gate_up;
    MatDeal deal_x, deal_w;
    size_t x, w, g, raw, partial, partial_w, total;
};

// Few tokens, weights that can be read as they are.
bool few_weights(const Call& c) {
    const bool fp32 = c.type == MIMIR_NUM_F32;
    return c.tokens <= kFewN && c.hidden <= (1 << 18) && few_direct(fp32, c.w[0], c.ld_w, c.hidden) &&
           few_direct(fp32, c.w[1], c.ld_w, c.hidden);
}
// And their rows of x: the forward is one launch.
bool few_applies(const Call& c) { return few_weights(c) && few_direct(c.type == MIMIR_NUM_F32, c.x, c.ld_x, c.dim); }


Plan plan_of(const mimir_ctx* ctx, const Call& c, bool back, bool two_terms) {
    Plan p{};
    p.p = c.type == MIMIR_NUM_BF16 ? 1 : 3;
    p.pg = p.p == 3 ? 3 : two_terms || c.tokens <= kTwoPlaneTokens ? 2 : 1;
    p.x_direct = p.p == 1 && mat_direct(c.x, c.ld_x, c.dim);
    p.w_direct = p.p == 1 && mat_direct(c.w[0], c.ld_w, c.hidden) && mat_direct(c.w[1], c.ld_w, c.hidden);
    p.ld_x = mat_round(c.dim, 8);
    // fp32: the weights' planes would be five times their bytes on the way.
    p.few = back && p.p == 3 && few_weights(c);
    const int64_t of_column = (back ? c.tokens * p.pg * 4 : 0) + (p.w_direct ? 0 : c.dim * p.p * 4);
    if (ctx->tune.mat_piece > 0) p.piece = mat_round(ctx->tune.mat_piece, 8);
    else p.piece = of_column ? std::max<int64_t>(256, kPieceBytes / of_column / 256 * 256) : c.hidden;
    p.piece = std::min({p.few ? c.hidden + 8 : p.piece, mat_round(c.hidden, 8), int64_t{1} << 18});
    p.ld_w = p.piece;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t was = at;
        at += (bytes + 255) / 256 * 256;
        return was;
    };
    p.x = take(p.x_direct ? 0 : static_cast<size_t>(p.p * c.tokens * p.ld_x * 2));
    p.w = take(p.w_direct || p.few ? 0 : static_cast<size_t>(2 * p.p * c.dim * p.ld_w * 2));
    if (!back) {
        // A contraction long enough that dealing it to several workgroups gains more than the
        // second pass, of a launch and 16 bytes an element, takes.  The fewer the tiles, the
        // more it gains, and fp32's six products a step gain more than bf16's one.  Measured,
        // us, split / whole: fp32 dim 512, 16 to 258 tiles 36 to 56 / 32 to 49; 1024, 120 tiles
        // 47 / 59, 172 64 / 65, 258 86 / 79; 2048, 250 tiles 133 / 155; 4096, 258 tiles 261 /
        // 319, 344 709 / 708.  bf16 1024, 16 tiles 18 / 15, 125 30 / 19; 2048, 43 tiles 24 / 29,
        // 86 31 to 35 / 30 to 32; 4096, 125 tiles 51 / 58, 172 66 / 64.
        const int64_t tn = p.p == 3 ? 64 : 128, tiles = (c.hidden + 63) / 64 * ((c.tokens + tn - 1) / tn);
        const int64_t least = p.p == 3 ? 1024 : 2048, most = std::min<int64_t>(c.dim / (p.p == 3 ? 8 : 32), 256);
        p.split = p.piece >= c.hidden && tiles <= most && c.dim >= least && ctx->tune.mat_big != 1;
        if (p.split) {
            p.deal_y = p.p == 3 ? mat_deal<3, 3, kCols, kRows>(ctx, c.hidden, c.tokens, c.dim, 2, false)
                                : mat_deal<1, 1, kCols, kRows>(ctx, c.hidden, c.tokens, c.dim, 2, false);
            p.partial = take(p.deal_y.partial);
            p.gate_up = take(static_cast<size_t>(2 * c.tokens * c.hidden * 4));
        }
    }
    if (back) {
        p.g = take(static_cast<size_t>(p.pg * c.tokens * 2 * p.piece * 2));
        const int64_t piece = std::min(p.piece, c.hidden);
        if (p.p == 3) {
            p.deal_x = mat_deal<3, 3, kRows, kRows>(ctx, c.dim, c.tokens, 2 * piece, 1, p.piece < c.hidden);
            p.deal_w = mat_deal<3, 3, kCols, kCols>(ctx, piece, c.dim, c.tokens, 2, false);
        } else if (p.pg == 2) {
            p.deal_x = mat_deal<1, 2, kRows, kRows>(ctx, c.dim, c.tokens, 2 * piece, 1, p.piece < c.hidden);
            p.deal_w = mat_deal<2, 1, kCols, kCols>(ctx, piece, c.dim, c.tokens, 2, false);
        } else {
            p.deal_x = mat_deal<1, 1, kRows, kRows>(ctx, c.dim, c.tokens, 2 * piece, 1, p.piece < c.hidden);
            p.deal_w = mat_deal<1, 1, kCols, kCols>(ctx, piece, c.dim, c.tokens, 2, false);
        }
        if (p.few) {
            p.raw = take(static_cast<size_t>(2 * c.tokens * c.hidden * 4));
            p.deal_x.splits = few_splits(c.dim, c.hidden, 2);
            p.deal_x.partial = static_cast<size_t>(2 * p.deal_x.splits * c.tokens * mat_round(c.dim, 4) * 4);
        }
        p.partial = take(p.deal_x.partial);
        p.partial_w = take(p.deal_w.partial);
    }
    p.total = std::max<size_t>(at, 256);
    return p;
}

int check(mimir_ctx* ctx, const char* what, const Call& c) {
    MIMIR_REQUIRE(ctx, c.type == MIMIR_NUM_F32 || c.type == MIMIR_NUM_BF16, "%s: type %d", what, c.type);
    MIMIR_REQUIRE(ctx, c.act == kSilu || c.act == kGelu, "%s: activation %d", what, c.act);
    MIMIR_REQUIRE(ctx, c.tokens >= 0 && c.tokens <= (1 << 24) && c.dim >= 1 && c.dim <= (1 << 18) && c.hidden >= 1 &&
                           c.hidden <= (1 << 20),
                  "%s: tokens=%lld (0 to 2^24) dim=%lld (1 to 2^18) hidden=%lld (1 to 2^20)", what, (long long)c.tokens,
                  (long long)c.dim, (long long)c.hidden);
    MIMIR_REQUIRE(ctx, c.ld_x >= c.dim && c.ld_w >= c.hidden, "%s: row strides (%lld, %lld) below dim, hidden", what,
                  (long long)c.ld_x, (long long)c.ld_w);
    return MIMIR_OK;
}

int inputs(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, MatOperand* x) {
    if (p.x_direct) {
        *x = MatOperand{static_cast<const uint16_t*>(c.x), c.ld_x, 0};
        return MIMIR_OK;
    }
    auto* dst = reinterpret_cast<uint16_t*>(work + p.x);
    *x = MatOperand{dst, p.ld_x, c.tokens * p.ld_x};
    return mat_stage(ctx, c.type, c.x, c.tokens, c.dim, c.ld_x, dst, p.ld_x, c.tokens * p.ld_x);
}

// Columns first .. + cols of both weights.
int weights(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, int64_t first, int64_t cols, MatOperand* w) {
    for (int i = 0; i < 2; ++i) {
        const char* at = static_cast<const char*>(c.w[i]) + first * (p.p == 1 ? 2 : 4);
        if (p.w_direct) {
            w[i] = MatOperand{reinterpret_cast<const uint16_t*>(at), c.ld_w, 0};
            continue;
        }
        const int64_t plane = c.dim * p.ld_w;
        auto* dst = reinterpret_cast<uint16_t*>(work + p.w) + i * p.p * plane;
        w[i] = MatOperand{dst, p.ld_w, plane};
        if (int st = mat_stage(ctx, c.type, at, c.dim, cols, c.ld_w, dst, p.ld_w, plane)) return st;
    }
    return MIMIR_OK;
}

MatArgs args_of(int64_t m, int64_t n, int64_t k) {
    MatArgs g{};
    g.m = static_cast<int32_t>(m);
    g.n = static_cast<int32_t>(n);
    g.k = static_cast<int32_t>(k);
    g.segments = g.batches = g.splits = 1;
    return g;
}

template <int P, int ACT>
int forward(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, void* y, int64_t ld_y, float* gate_up) {
    MatOperand x;
    if (int st = inputs(ctx, c, p, work, &x)) return st;
    const int bf16 = P == 1;
    for (int64_t first = 0; first < c.hidden; first += p.piece) {
        const int64_t cols = std::min(p.piece, c.hidden - first);
        MatArgs g = args_of(cols, c.tokens, c.dim);
        if (int st = weights(ctx, c, p, work, first, cols, g.a)) return st;
        g.b[0] = x;
        if (p.split) {
            if (!gate_up) gate_up = reinterpret_cast<float*>(work + p.gate_up);
            MatOut o{};
            o.out[0] = gate_up;
            o.out[1] = gate_up + c.hidden;
            o.ld = 2 * c.hidden;
            o.partial = reinterpret_cast<float*>(work + p.partial);
            o.alpha = 1.0f;
            o.last = 1;
            g.batches = 2;
            if (int st = mat_product<P, P, kCols, kRows>(ctx, "gated products", g, o, p.deal_y)) return st;
            const int64_t blocks = (c.tokens * ((c.hidden + 7) / 8) + kBlock - 1) / kBlock;
            gated_act<ACT, P == 1><<<static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 16)), kBlock, 0, ctx->stream>>>(
                ActArgs{gate_up, c.tokens, c.hidden, y, ld_y});
            return launched(ctx, "gated_act");
        }
        GatedOut<ACT> e{};
        e.y.out[0] = static_cast<char*>(y) + first * (bf16 ? 2 : 4);
        e.y.ld = ld_y;
        e.y.bf16 = bf16;
        e.gate_up = gate_up ? gate_up + first : nullptr;
        e.hidden = c.hidden;
        using B = MatBig<P, P, kCols, kRows, true>;
        using S = MatSmall<P, P, kCols, kRows, true>;
        const int st = mat_fills<B>(ctx, g) ? mat_launch<B>(ctx, "gated products", g, e) : mat_launch<S>(ctx, "gated products", g, e);
        if (st) return st;
    }
    return MIMIR_OK;
}

template <bool FP32, int ACT>
int forward_few(mimir_ctx* ctx, const Call& c, void* y, int64_t ld_y, float* gate_up) {
    MatArgs g = args_of(c.hidden, c.tokens, c.dim);
    for (int i = 0; i < 2; ++i) g.a[i] = MatOperand{static_cast<const uint16_t*>(c.w[i]), c.ld_w, 0};
    g.b[0] = MatOperand{static_cast<const uint16_t*>(c.x), c.ld_x, 0};
    GatedOut<ACT> e{};
    e.y.out[0] = y;
    e.y.ld = ld_y;
    e.y.bf16 = !FP32;
    e.gate_up = gate_up;
    e.hidden = c.hidden;
    return few_launch<FP32, kCols, true>(ctx, "gated products", g, e);
}

struct Gradients {
    const float* gate_up;
    const void* dy;
    int64_t ld_dy;
    void* dx;
    int64_t ld_dx;
    void* dw[2];
    int64_t ld_dw;
    int accumulate_x, accumulate_w;
};

template <int P, int PG, int ACT>
int backward(mimir_ctx* ctx, const Call& c, const Plan& p, char* work, const Gradients& d) {
    MatOperand x{};
    if (d.dw[0])
        if (int st = inputs(ctx, c, p, work, &x)) return st;
    const int bf16 = P == 1;
    const int64_t size = bf16 ? 2 : 4;
    auto* planes = reinterpret_cast<uint16_t*>(work + p.g);
    const int64_t ld_g = 2 * p.piece, plane = c.tokens * ld_g;
    MatOut ox{};
    ox.out[0] = d.dx;
    ox.ld = d.ld_dx;
    ox.partial = reinterpret_cast<float*>(work + p.partial);
    ox.alpha = 1.0f;
    ox.bf16 = bf16;
    ox.accumulate = d.accumulate_x;
    MatOut ow = ox;
    ow.partial = reinterpret_cast<float*>(work + p.partial_w);
    ow.ld = d.ld_dw;
    ow.accumulate = d.accumulate_w;
    ow.last = 1;
    for (int64_t first = 0; first < c.hidden; first += p.piece) {
        const int64_t cols = std::min(p.piece, c.hidden - first);
        const GradArgs a{d.gate_up + first, c.hidden, static_cast<const char*>(d.dy) + first * size, d.ld_dy,
                         planes, c.tokens, cols, p.piece, plane, p.few ? reinterpret_cast<float*>(work + p.raw) : nullptr};
        const int64_t blocks = (c.tokens * (p.piece / 8) + kBlock - 1) / kBlock;
        const auto grid = static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 16));
        gated_grad<ACT, P == 1, PG><<<grid, kBlock, 0, ctx->stream>>>(a);
        if (int st = launched(ctx, "gated_grad")) return st;
        const MatOperand dg{planes, ld_g, plane}, du{planes + p.piece, ld_g, plane};
        if (d.dx) {
            MatArgs g = args_of(c.dim, c.tokens, cols);
            ox.read_partial = first > 0;
            ox.last = first + cols >= c.hidden;
            g.segments = 2;
            int st = MIMIR_OK;
            if (P == 3 && p.few) {
                for (int i = 0; i < 2; ++i) {
                    g.a[i] = MatOperand{static_cast<const uint16_t*>(c.w[i]), c.ld_w, 0};
                    g.b[i] = MatOperand{reinterpret_cast<const uint16_t*>(a.raw + i * c.tokens * c.hidden), c.hidden, 0};
                }
                g.splits = p.deal_x.splits;
                if constexpr (P == 3) st = few_product<kRows>(ctx, "gated dx", g, ox);
            } else if (st = weights(ctx, c, p, work, first, cols, g.a); st == MIMIR_OK) {
                g.b[0] = dg;
                g.b[1] = du;
                st = mat_product<P, PG, kRows, kRows>(ctx, "gated dx", g, ox, p.deal_x);
            }
            if (st) return st;
        }
        if (d.dw[0]) {
            MatArgs g = args_of(cols, c.dim, c.tokens);
            g.a[0] = dg;
            g.a[1] = du;
            g.b[0] = x;
            g.batches = 2;
            for (int i = 0; i < 2; ++i) ow.out[i] = static_cast<char*>(d.dw[i]) + first * size;
            if (int st = mat_product<PG, P, kCols, kCols>(ctx, "gated dw", g, ow, p.deal_w)) return st;
        }
    }
    return MIMIR_OK;
}

}  // namespace

extern "C" {

int mimir_gated_linear_fwd(mimir_ctx* ctx, int type, int act, const void* x, int64_t ld_x, const void* w_gate, const void* w_up,
                           int64_t ld_w, int64_t tokens, int64_t dim, int64_t hidden, void* y, int64_t ld_y, float* gate_up) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "gated products";
    const Call c{type, act, x, ld_x, {w_gate, w_up}, ld_w, tokens, dim, hidden};
    if (int st = check(ctx, what, c)) return st;
    MIMIR_REQUIRE(ctx, ld_y >= hidden, "%s: row stride %lld below hidden", what, (long long)ld_y);
    if (tokens == 0) return MIMIR_OK;
    MIMIR_REQUIRE(ctx, x && w_gate && w_up && y, "%s: null pointer", what);
    MIMIR_REQUIRE(ctx, mat_apart({y, gate_up}, {x, w_gate, w_up}), "%s: an output is an input or another output", what);
    MIMIR_ENTER(ctx);
    if (few_applies(c)) {
        if (type == MIMIR_NUM_F32) return act == kSilu ? forward_few<true, kSilu>(ctx, c, y, ld_y, gate_up) : forward_few<true, kGelu>(ctx, c, y, ld_y, gate_up);
        return act == kSilu ? forward_few<false, kSilu>(ctx, c, y, ld_y, gate_up) : forward_few<false, kGelu>(ctx, c, y, ld_y, gate_up);
    }
    const Plan p = plan_of(ctx, c, false, false);
    char* work;
    if (int st = mat_scratch(ctx, p.total, &work)) return st;
    if (p.p == 3) return act == kSilu ? forward<3, kSilu>(ctx, c, p, work, y, ld_y, gate_up) : forward<3, kGelu>(ctx, c, p, work, y, ld_y, gate_up);
    return act == kSilu ? forward<1, kSilu>(ctx, c, p, work, y, ld_y, gate_up) : forward<1, kGelu>(ctx, c, p, work, y, ld_y, gate_up);
}

int mimir_gated_linear_bwd(mimir_ctx* ctx, int type, int act, const void* x, int64_t ld_x, const void* w_gate, const void* w_up,
                           int64_t ld_w, int64_t tokens, int64_t dim, int64_t hidden, const float* gate_up, const void* dy,
                           int64_t ld_dy, void* dx, int64_t ld_dx, int accumulate_x, void* dw_gate, void* dw_up, int64_t ld_dw,
                           int accumulate_w) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "gated products' gradient";
    const bool two_terms = type == (MIMIR_NUM_BF16 | MIMIR_NUM_TWO_TERMS);
    if (two_terms) type = MIMIR_NUM_BF16;
    const Call c{type, act, x, ld_x, {w_gate, w_up}, ld_w, tokens, dim, hidden};
    if (int st = check(ctx, what, c)) return st;
    MIMIR_REQUIRE(ctx, !dw_gate == !dw_up, "%s: dw_gate and dw_up go together", what);
    MIMIR_REQUIRE(ctx, ld_dy >= hidden && (!dx || ld_dx >= dim) && (!dw_gate || ld_dw >= hidden),
                  "%s: row strides of dy, dx, dw (%lld, %lld, %lld) below hidden, dim, hidden", what, (long long)ld_dy,
                  (long long)ld_dx, (long long)ld_dw);
    if (!dx && !dw_gate) return MIMIR_OK;
    MIMIR_REQUIRE(ctx, tokens == 0 || (x && w_gate && w_up && gate_up && dy), "%s: null pointer", what);
    MIMIR_REQUIRE(ctx, mat_apart({dx, dw_gate, dw_up}, {x, w_gate, w_up, gate_up, dy}), "%s: an output is an input or another output", what);
    if (tokens == 0 && !dw_gate) return MIMIR_OK;
    MIMIR_ENTER(ctx);
    if (tokens == 0) {
        if (accumulate_w) return MIMIR_OK;
        if (int st = mat_zero(ctx, type, dw_gate, dim, hidden, ld_dw)) return st;
        return mat_zero(ctx, type, dw_up, dim, hidden, ld_dw);
    }
    const Plan p = plan_of(ctx, c, true, two_terms);
    char* work;
    if (int st = mat_scratch(ctx, p.total, &work)) return st;
    const Gradients d{gate_up, dy, ld_dy, dx, ld_dx, {dw_gate, dw_up}, ld_dw, accumulate_x ? 1 : 0, accumulate_w ? 1 : 0};
    const auto run = [&](auto a) {
        constexpr int ACT = decltype(a)::value;
        if (p.p == 3) return backward<3, 3, ACT>(ctx, c, p, work, d);
        return p.pg == 2 ? backward<1, 2, ACT>(ctx, c, p, work, d) : backward<1, 1, ACT>(ctx, c, p, work, d);
    };
    return act == kSilu ? run(std::integral_constant<int, kSilu>{}) : run(std::integral_constant<int, kGelu>{});
}

}  // extern "C"
