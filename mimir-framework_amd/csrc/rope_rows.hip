// rope_rows.hip -- rotary positions of packed tokens, each at its own position:
// pairs half a rotated part apart or side by side, part of a head or all of it,
// forward and the transposed rotation of a gradient; and the host tables of
// scaled frequencies.  (Su et al. 2021, "RoFormer"; the scalings: Chen et al. 2023,
// position interpolation, and Peng et al. 2023, "YaRN", whose ramp by turns is
// BY_PARTS.)
//
// Bound by HBM: every element is read once and written once; the positions and
// their table rows are shared by the heads of a token and stay in L2.  A "slot" is
// two vectors of one head row (kvcache.hpp unit_place): four pairs, or eight
// dimensions that are copied.  The
// products are taken in double (kvcache.hpp rotate_pair): 8 operations on pairs
// that cost 32 bytes of HBM, a tenth of the time those take.
#include "common.hpp"
#include "fastdiv.hpp"
#include "internal.hpp"
#include "kvcache.hpp"

#include <math.h>

#include <algorithm>

using namespace mimir;

namespace {

struct RowsArgs {
    const float* q;
    float* q_out;
    const float* k;
    float* k_out;
    int64_t ld_q, ld_q_out, ld_k, ld_k_out;
    const int32_t* positions;
    const float* cos_tab;
    const float* sin_tab;
    int64_t table_rows;
    uint32_t q_slots, slots;  // q's, then k's
    FastDiv unit_div, q_div, k_div;  // units of a head row, heads of a token
    int32_t head_dim, half, interleaved;
    float sign;  // of sin: -1 turns back
};

// W elements of a row (one 16-byte vector, or one float), and whether they lie in it.
template <int W>
struct Half {
    float x[W];
    __device__ __forceinline__ void load(const float* p, bool in) {
        if (!in) return;
        if constexpr (W == 4) {
            const f4 v = *reinterpret_cast<const f4*>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = v[e];
        } else {
            x[0] = *p;
        }
    }
    template <bool KEEP, bool ACC>
    __device__ __forceinline__ void store(float* p, bool in) {
        if (!in) return;
        if constexpr (W == 4) {
            f4 v{x[0], x[1], x[2], x[3]};
            if constexpr (ACC) v = *reinterpret_cast<const f4*>(p) + v;
            st_out<KEEP, ACC ? kStoreNt : kStoreThrough>(p, v);
        } else {
            float v = x[0];
            if constexpr (ACC) v = *p + v;
            if constexpr (KEEP) *p = v;
            else st_stream(p, v);
        }
    }
};

// W: elements per half of a slot, 4 where every row is whole 16-byte vectors and the
// rotated part a multiple of 8, else 1 for all of a row (8192 tokens x 40 heads of 128, of
// which 128 dimensions are rotated 48 us, 124 63; heads of 96 39 us = 6.5 TB/s, of 100 54
// = 4.9 TB/s, of 99 57 = 4.6 TB/s; the same inputs each time, in part from the caches).  A
// thread has one slot: 8192 tokens x 40 heads of 128 take 58 us = 5.8 TB/s (a copy of
// as many bytes 53), with two slots a thread 61, four 61, eight 89.  The loads leave
// their lines in the caches, where the projection before may have put them (4099
// tokens x 32 heads: 22 us, non-temporal 26; the larger case 58 and 57).
template <int W, bool KEEP, bool ACC>
__global__ __launch_bounds__(kBlock) void rope_rows(RowsArgs a) {
    const uint32_t slot = blockIdx.x * kBlock + threadIdx.x;
    if (slot >= a.slots) return;
    const bool is_q = slot < a.q_slots;
    const uint32_t local = is_q ? slot : slot - a.q_slots;
    const uint32_t row = fastdiv(local, a.unit_div);
    const int unit = static_cast<int>(local - row * a.unit_div.d);
    const FastDiv& heads = is_q ? a.q_div : a.k_div;
    const uint32_t t = fastdiv(row, heads);
    const int64_t col = static_cast<int64_t>(row - t * heads.d) * a.head_dim;
    const auto [d0, d1, pairs] = unit_place<W>(unit, a.half, a.interleaved, a.head_dim);
    const float* x = (is_q ? a.q + t * a.ld_q : a.k + t * a.ld_k) + col;
    float* y = (is_q ? a.q_out + t * a.ld_q_out : a.k_out + t * a.ld_k_out) + col;
    const bool two = d1 < a.head_dim;
    Half<W> lo, hi;
    lo.load(x + d0, true);
    hi.load(x + d1, two);
    const int64_t p = a.positions[t];
    if (p < 0 || p >= a.table_rows) {
        if constexpr (ACC) return;
#pragma unroll
        for (int e = 0; e < W; ++e) lo.x[e] = hi.x[e] = 0.f;
    } else if (pairs) {
        float c[W], s[W];
        unit_turns<W>(a.cos_tab, a.sin_tab, p * a.half, unit, a.half, a.interleaved, c, s);
#pragma unroll
        for (int e = 0; e < W; ++e) s[e] *= a.sign;
        unit_rotate<W>(lo.x, hi.x, c, s, a.interleaved);
    }
    lo.template store<KEEP, ACC>(y + d0, true);
    hi.template store<KEEP, ACC>(y + d1, two);
}

template <int W, bool ACC>
int launch(mimir_ctx* ctx, const RowsArgs& a) {
    unsigned blocks;
    if (!grid_for(a.slots, kBlock, kBlock, &blocks)) return fail(ctx, MIMIR_EINVAL, "RoPE: grid exceeds the limit");
    if (ctx->keep_outputs) rope_rows<W, true, ACC><<<blocks, kBlock, 0, ctx->stream>>>(a);
    else rope_rows<W, false, ACC><<<blocks, kBlock, 0, ctx->stream>>>(a);
    return launched(ctx, "rope_rows");
}

int rope_rows_run(mimir_ctx* ctx, const char* what, const float* q, int64_t ld_q, float* q_out, int64_t ld_q_out,
                  int64_t q_heads, const float* k, int64_t ld_k, float* k_out, int64_t ld_k_out, int64_t k_heads,
                  int64_t tokens, int64_t head_dim, const int32_t* positions, const mimir_rope* rope, bool back, bool acc) {
    if (!ctx) return MIMIR_EINVAL;
    constexpr int64_t kMost = int64_t{1} << 30;
    MIMIR_REQUIRE(ctx, tokens >= 0 && tokens < kMost && head_dim >= 1 && head_dim <= (1 << 16) && (!q || q_heads >= 0) &&
                           (!k || k_heads >= 0),
                  "%s: invalid shape (tokens=%lld q_heads=%lld k_heads=%lld head_dim=%lld)", what, (long long)tokens,
                  (long long)q_heads, (long long)k_heads, (long long)head_dim);
    if (int st = rope_check(ctx, what, rope, head_dim)) return st;
    const int64_t qh = q ? q_heads : 0, kh = k ? k_heads : 0;
    MIMIR_REQUIRE(ctx, qh <= (1 << 20) && kh <= (1 << 20), "%s: too many heads", what);
    MIMIR_REQUIRE(ctx, (!qh || (ld_q >= qh * head_dim && ld_q_out >= qh * head_dim)) &&
                           (!kh || (ld_k >= kh * head_dim && ld_k_out >= kh * head_dim)),
                  "%s: row strides (%lld, %lld, %lld, %lld) below heads * head_dim", what, (long long)ld_q, (long long)ld_q_out,
                  (long long)ld_k, (long long)ld_k_out);
    if (tokens == 0 || qh + kh == 0) return MIMIR_OK;
    MIMIR_REQUIRE(ctx, positions && (!qh || q_out) && (!kh || k_out), "%s: null pointer", what);
    MIMIR_REQUIRE(ctx, (!qh || q != q_out || ld_q == ld_q_out) && (!kh || k != k_out || ld_k == ld_k_out),
                  "%s: in place needs equal strides", what);
    MIMIR_REQUIRE(ctx, !acc || ((!qh || q != q_out) && (!kh || k != k_out)), "%s: an in-place gradient cannot accumulate", what);
    MIMIR_ENTER(ctx);
    const bool vec = head_dim % 4 == 0 && rope->rot_dim % 8 == 0 && aligned16(rope->cos_tab) && aligned16(rope->sin_tab) &&
                     (!qh || (ld_q % 4 == 0 && ld_q_out % 4 == 0 && aligned16(q) && aligned16(q_out))) &&
                     (!kh || (ld_k % 4 == 0 && ld_k_out % 4 == 0 && aligned16(k) && aligned16(k_out)));
    const int64_t w = vec ? 4 : 1, units = (head_dim + 2 * w - 1) / (2 * w);
    // A launch counts its slots in 32 bits: more tokens than that go in several.
    const int64_t most = std::max<int64_t>(1, (int64_t{1} << 31) / ((qh + kh) * units));
    MIMIR_REQUIRE(ctx, (qh + kh) * units <= (int64_t{1} << 31), "%s: row too wide", what);
    for (int64_t t = 0; t < tokens; t += most) {
        const int64_t n = std::min(most, tokens - t);
        RowsArgs a{qh ? q + t * ld_q : nullptr, qh ? q_out + t * ld_q_out : nullptr, kh ? k + t * ld_k : nullptr,
                   kh ? k_out + t * ld_k_out : nullptr, ld_q, ld_q_out, ld_k, ld_k_out, positions + t, rope->cos_tab,
                   rope->sin_tab, rope->table_rows, static_cast<uint32_t>(n * qh * units),
                   static_cast<uint32_t>(n * (qh + kh) * units), make_fastdiv(static_cast<uint32_t>(units)),
                   make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(qh, 1))),
                   make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(kh, 1))), static_cast<int32_t>(head_dim),
                   rope->rot_dim / 2, rope->interleaved ? 1 : 0, back ? -1.f : 1.f};
        const int st = vec ? (acc ? launch<4, true>(ctx, a) : launch<4, false>(ctx, a))
                           : (acc ? launch<1, true>(ctx, a) : launch<1, false>(ctx, a));
        if (st) return st;
    }
    return MIMIR_OK;
}

}  // namespace

int mimir::rope_check(mimir_ctx* ctx, const char* what, const mimir_rope* rope, int64_t head_dim) {
    MIMIR_REQUIRE(ctx, rope, "%s: null rope", what);
    MIMIR_REQUIRE(ctx, rope->rot_dim > 0 && rope->rot_dim % 2 == 0 && rope->rot_dim <= head_dim,
                  "%s: rot_dim %d is not an even number from 2 to head_dim %lld", what, rope->rot_dim, (long long)head_dim);
    MIMIR_REQUIRE(ctx, rope->table_rows >= 0 && (rope->table_rows == 0 || (rope->cos_tab && rope->sin_tab)),
                  "%s: no tables of %lld rows", what, (long long)rope->table_rows);
    return MIMIR_OK;
}

extern "C" {

int mimir_rope_table_scaled(int64_t first, int64_t rows, int64_t rot_dim, double theta,
                            const mimir_rope_scaling* scaling, float* cos_tab, float* sin_tab) {
    if (first < 0 || rows < 0 || rot_dim <= 0 || (rot_dim & 1) || !(theta > 0.0) || !std::isfinite(theta)) return MIMIR_EINVAL;
    if (rows > 0 && (!cos_tab || !sin_tab)) return MIMIR_EINVAL;
    const mimir_rope_scaling none{MIMIR_ROPE_SCALE_NONE, 1.0, 1.0, 0.0, 1.0, 1.0};
    const mimir_rope_scaling& z = scaling ? *scaling : none;
    if (z.kind < MIMIR_ROPE_SCALE_NONE || z.kind > MIMIR_ROPE_SCALE_BY_PARTS || !std::isfinite(z.magnitude)) return MIMIR_EINVAL;
    if (z.kind != MIMIR_ROPE_SCALE_NONE && !(z.factor > 0.0 && std::isfinite(z.factor))) return MIMIR_EINVAL;
    if (z.kind == MIMIR_ROPE_SCALE_BASE && rot_dim <= 2) return MIMIR_EINVAL;
    if (z.kind == MIMIR_ROPE_SCALE_BY_PARTS &&
        !(z.original_len > 0.0 && std::isfinite(z.original_len) && z.low < z.high && std::isfinite(z.low) && std::isfinite(z.high)))
        return MIMIR_EINVAL;
    const int64_t half = rot_dim / 2;
    const double d = static_cast<double>(rot_dim);
    const double base = z.kind == MIMIR_ROPE_SCALE_BASE ? theta * pow(z.factor, d / (d - 2.0)) : theta;
    const auto frequency = [&](int64_t i) {
        double f = 1.0 / pow(base, static_cast<double>(2 * i) / d);
        if (z.kind == MIMIR_ROPE_SCALE_LINEAR) f /= z.factor;
        if (z.kind == MIMIR_ROPE_SCALE_BY_PARTS) {
            const double turns = z.original_len * f / 6.283185307179586476925;
            const double g = std::min(1.0, std::max(0.0, (turns - z.low) / (z.high - z.low)));
            f = (1.0 - g) * f / z.factor + g * f;
        }
        return f;
    };
    // Nothing is written of a table that would have values which are no numbers.
    if (rows > 0) {
        if (first > INT64_MAX - rows || !std::isfinite(static_cast<float>(z.magnitude))) return MIMIR_EINVAL;
        for (int64_t i = 0; i < half; ++i)
            if (const double f = frequency(i); !std::isfinite(f) || !std::isfinite(static_cast<double>(first + rows - 1) * f))
                return MIMIR_EINVAL;
    }
    for (int64_t i = 0; i < half; ++i) {
        const double f = frequency(i);
        for (int64_t p = 0; p < rows; ++p) {
            const double a = static_cast<double>(first + p) * f;
            cos_tab[p * half + i] = static_cast<float>(cos(a) * z.magnitude);
            sin_tab[p * half + i] = static_cast<float>(sin(a) * z.magnitude);
        }
    }
    return MIMIR_OK;
}

int mimir_rope_rows_fwd(mimir_ctx* ctx, const float* q, int64_t ld_q, float* q_out, int64_t ld_q_out, int64_t q_heads,
                        const float* k, int64_t ld_k, float* k_out, int64_t ld_k_out, int64_t k_heads, int64_t tokens,
                        int64_t head_dim, const int32_t* positions, const mimir_rope* rope) {
    return rope_rows_run(ctx, "RoPE rows", q, ld_q, q_out, ld_q_out, q_heads, k, ld_k, k_out, ld_k_out, k_heads, tokens,
                         head_dim, positions, rope, false, false);
}

int mimir_rope_rows_bwd(mimir_ctx* ctx, const float* dq, int64_t ld_dq, float* dq_in, int64_t ld_dq_in, int64_t q_heads,
                        const float* dk, int64_t ld_dk, float* dk_in, int64_t ld_dk_in, int64_t k_heads, int64_t tokens,
                        int64_t head_dim, const int32_t* positions, const mimir_rope* rope, int accumulate) {
    return rope_rows_run(ctx, "RoPE rows backward", dq, ld_dq, dq_in, ld_dq_in, q_heads, dk, ld_dk, dk_in, ld_dk_in, k_heads,
                         tokens, head_dim, positions, rope, true, accumulate != 0);
}

}  // extern "C"
