// kvcache.hip -- the paged key/value cache: new tokens' keys and values written
// into their pages (keys and queries rotated on the way), and read back.
//
// Bound by HBM: q, k and v are read from it once and written once, in the cache's type.
// LPR lanes hold a head row, eight elements each (two vectors, kvcache.hpp
// unit_place), so that the largest absolute value of an 8-bit row is a few lane
// exchanges away.  Of a row with fewer elements than that (unrotated heads of 80 have 10
// units for 16 lanes) the lanes behind the last unit load and store vectors of its second
// half once more, the same values to the same places.  A workgroup takes rows of one token, whose
// sequence its waves search in token_start while the row is on its way.  Prompts of
// 9270 tokens x 32 + 2 x 8 heads of 128 into an 8-bit cache and read back (500 MB): 68
// and 17 us, 85 in turn = 5.9 TB/s; steps of 48 tokens 4 and 3, launch to launch 9.5.
//
// Numerics.  Rotation in double, rounded once (rotate_pair).  An 8-bit code is the
// exact quotient x * 127 / max rounded to nearest even: the fp32 quotient is off by
// at most 127 * 2^-23 < 2^-16, so only where it comes within 2^-12 of the border
// between two codes does it need the double one, which is exact enough to see a tie
// (both operands of the comparison are integers of 49 bits).
#include "kvcache.hpp"

#include <math.h>

#include <algorithm>

using namespace mimir;

namespace {

struct AppendArgs {
    KvView c;
    KvBatch b;
    const float* q;
    float* q_out;
    const float* k;
    const float* v;
    int64_t ld_q, ld_q_out, ld_kv;
    const float* cos_tab;
    const float* sin_tab;
    int32_t q_heads, half, interleaved;
    uint32_t parts;  // workgroups per token
};

// Largest bit pattern over aligned groups of LPR lanes; of absolute values it is the
// largest value, with infinities and NaN above all others.
template <int LPR>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    const auto step = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    v = step(v, __builtin_amdgcn_update_dpp(0, v, kDppQuadXor1, 0xF, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(0, v, kDppQuadXor2, 0xF, 0xF, false));
    v = step(v, __builtin_amdgcn_update_dpp(0, v, kDppRowHalfMirror, 0xF, 0xF, false));
    if constexpr (LPR >= 16) v = step(v, __builtin_amdgcn_update_dpp(0, v, kDppRowMirror, 0xF, 0xF, false));
    if constexpr (LPR >= 32) v = step(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
    return v;
}

// The code of x in a row whose largest absolute value is `most` (finite, above 0);
// inv = 127 / most.
__device__ __forceinline__ int code_of(float x, float most, float inv) {
    const float t = x * inv;
    float c = rintf(t);
    // The second test: a quotient that fp32 could not hold, or has lost bits of.
    if (fabsf(t - c) > 0.5f - 0x1p-12f || !(most > 0x1p-100f))
        c = static_cast<float>(rint(static_cast<double>(x) * 127.0 / static_cast<double>(most)));
    return static_cast<int>(c);
}

// Stores W elements of a cache row, `at` elements in.
template <int DT, int W>
__device__ __forceinline__ void put(char* row, int at, const float* x) {
    if constexpr (DT == MIMIR_KV_F32) {
        float* p = reinterpret_cast<float*>(row) + at;
        if constexpr (W == 4) *reinterpret_cast<f4*>(p) = f4{x[0], x[1], x[2], x[3]};
        else *p = x[0];
    } else if constexpr (DT == MIMIR_KV_BF16) {
        __bf16* p = reinterpret_cast<__bf16*>(row) + at;
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        if constexpr (W == 4)
            *reinterpret_cast<b4*>(p) = b4{static_cast<__bf16>(x[0]), static_cast<__bf16>(x[1]), static_cast<__bf16>(x[2]),
                                           static_cast<__bf16>(x[3])};
        else *p = static_cast<__bf16>(x[0]);
    }
}

// W: elements per vector, 4 where every row of q, k, v and q_out is whole 16-byte
// vectors and half the rotated part too; UN units of 2 W elements per lane.  (Of one
// element, 128 of 128 dimensions rotated and 124, prompts of 9270 tokens x 32 + 2 x 8
// heads written and read back: fp32 99 and 128 us, bf16 90 and 119, 8-bit 86 and 118.)  A workgroup has rows of one token:
// several tokens each kept fewer loads in flight (prompts of 9270 tokens x 48 heads of
// 128, 8-bit: 91 us written and read back, with two 94, four 101, eight 123).
template <int DT, int LPR, int W, bool KEEP>
__global__ __launch_bounds__(kBlock) void kv_append(AppendArgs a) {
    constexpr int UN = 4 / W;  // 8 elements a lane
    const uint32_t t = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const int d = a.c.head_dim, row = static_cast<int>(part * (blockDim.x / LPR)) + group;
    const bool is_q = row < a.q_heads, is_k = !is_q && row < a.q_heads + a.c.kv_heads;
    const bool mine = row < a.q_heads + 2 * a.c.kv_heads;
    const int head = is_q ? row : row - a.q_heads - (is_k ? 0 : a.c.kv_heads);
    const int half = is_q || is_k ? a.half : 0;  // values are not rotated
    const int64_t ld = is_q ? a.ld_q : a.ld_kv;
    const float* x = (is_q ? a.q : is_k ? a.k : a.v) + t * ld + static_cast<int64_t>(head) * d;
    float lo[UN][W], hi[UN][W];
    UnitPlace at[UN];
#pragma unroll
    for (int n = 0; n < UN; ++n) {
        at[n] = unit_place<W>(lane + n * LPR, half, a.interleaved, a.c.stride);
#pragma unroll
        for (int e = 0; e < W; ++e) lo[n][e] = hi[n][e] = 0.f;
        if (mine) {
            if constexpr (W == 4) {
                if (at[n].d0 < d) {
                    const f4 v = ld4<true>(x + at[n].d0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) lo[n][e] = v[e];
                }
                if (at[n].d1 < d) {
                    const f4 v = ld4<true>(x + at[n].d1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) hi[n][e] = v[e];
                }
            } else {
                if (at[n].d0 < d) lo[n][0] = x[at[n].d0];
                if (at[n].d1 < d) hi[n][0] = x[at[n].d1];
            }
        }
    }

    int s;
    kv_sequences_of<1>(a.b, static_cast<int>(t), &s);
    const KvToken tok = kv_token(a.b, a.c, s, static_cast<int>(t));
    if (!tok.in) return;  // the whole workgroup
#pragma unroll
    for (int n = 0; n < UN; ++n) {
        if (!at[n].turned || tok.position < 0) continue;
        float c[W], sn[W];
        unit_turns<W>(a.cos_tab, a.sin_tab, static_cast<int64_t>(tok.position) * a.half, lane + n * LPR, a.half, a.interleaved,
                      c, sn);
        unit_rotate<W>(lo[n], hi[n], c, sn, a.interleaved);
    }
    if (is_q) {
        float* y = a.q_out + t * a.ld_q_out + static_cast<int64_t>(head) * d;
#pragma unroll
        for (int n = 0; n < UN; ++n) {
            if (tok.position < 0) {
#pragma unroll
                for (int e = 0; e < W; ++e) lo[n][e] = hi[n][e] = 0.f;
            }
            // Written through (85 us for prompts of 9270 tokens, plain stores 91), or kept
            // (mimir_ctx_set_output_caching).
            if constexpr (W == 4) {
                if (at[n].d0 < d) st_out<KEEP, kStoreThrough>(y + at[n].d0, f4{lo[n][0], lo[n][1], lo[n][2], lo[n][3]});
                if (at[n].d1 < d) st_out<KEEP, kStoreThrough>(y + at[n].d1, f4{hi[n][0], hi[n][1], hi[n][2], hi[n][3]});
            } else {
                if (at[n].d0 < d) y[at[n].d0] = lo[n][0];
                if (at[n].d1 < d) y[at[n].d1] = hi[n][0];
            }
        }
        return;
    }
    const bool held = mine && tok.page >= 0;
    const int64_t slot = held ? (static_cast<int64_t>(tok.page) * a.c.kv_heads + head) * a.c.page_size + tok.slot : 0;
    if constexpr (DT == MIMIR_KV_I8) {
        uint32_t bits = 0;  // all lanes of the group come here together
#pragma unroll
        for (int n = 0; n < UN; ++n)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                bits = max(bits, __builtin_bit_cast(uint32_t, lo[n][e]) & 0x7fffffffu);
                bits = max(bits, __builtin_bit_cast(uint32_t, hi[n][e]) & 0x7fffffffu);
            }
        bits = lanes_max<LPR>(bits);
        if (!held) return;
        const bool finite = bits < 0x7f800000u;
        const float most = __builtin_bit_cast(float, bits), inv = 127.f / most;
        char* out = (is_k ? a.c.k : a.c.v) + slot * a.c.stride;
        if (lane == 0) (is_k ? a.c.k_scale : a.c.v_scale)[slot] = finite ? most / 127.f : __builtin_nanf("");
        const bool codes = finite && bits > 0;
#pragma unroll
        for (int n = 0; n < UN; ++n) {
            uint32_t l = 0, h = 0;
            if (codes) {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    l |= static_cast<uint32_t>(code_of(lo[n][e], most, inv) & 0xff) << (8 * e);
                    h |= static_cast<uint32_t>(code_of(hi[n][e], most, inv) & 0xff) << (8 * e);
                }
            }
            if constexpr (W == 4) {
                if (at[n].d0 < a.c.stride) *reinterpret_cast<uint32_t*>(out + at[n].d0) = l;
                if (at[n].d1 < a.c.stride) *reinterpret_cast<uint32_t*>(out + at[n].d1) = h;
            } else {
                if (at[n].d0 < a.c.stride) out[at[n].d0] = static_cast<char>(l);
                if (at[n].d1 < a.c.stride) out[at[n].d1] = static_cast<char>(h);
            }
        }
    } else {
        if (!held) return;
        char* out = (is_k ? a.c.k : a.c.v) + slot * a.c.stride * (DT == MIMIR_KV_F32 ? 4 : 2);
#pragma unroll
        for (int n = 0; n < UN; ++n) {
            if (at[n].d0 < a.c.stride) put<DT, W>(out, at[n].d0, lo[n]);
            if (at[n].d1 < a.c.stride) put<DT, W>(out, at[n].d1, hi[n]);
        }
    }
}

struct ReadArgs {
    KvView c;
    KvBatch b;
    float* k_out;
    float* v_out;
    int64_t ld_out;
    int32_t kinds;   // outputs: keys, values or both
    uint32_t parts;  // workgroups per token
};

// Four elements of a cache row, as the type's bits.
template <int DT>
__device__ __forceinline__ u4 get(const char* row, int at) {
    if constexpr (DT == MIMIR_KV_F32) return *reinterpret_cast<const u4*>(row + 4 * at);
    else if constexpr (DT == MIMIR_KV_BF16) {
        const uint64_t w = *reinterpret_cast<const uint64_t*>(row + 2 * at);
        return u4{static_cast<uint32_t>(w), static_cast<uint32_t>(w >> 32), 0, 0};
    } else return u4{*reinterpret_cast<const uint32_t*>(row + at), 0, 0, 0};
}

template <int DT>
__device__ __forceinline__ f4 value_of(u4 w, float scale) {
    if constexpr (DT == MIMIR_KV_F32) return __builtin_bit_cast(f4, w);
    else if constexpr (DT == MIMIR_KV_BF16)
        return __builtin_bit_cast(f4, u4{w[0] << 16, w[0] & 0xffff0000u, w[1] << 16, w[1] & 0xffff0000u});
    else {
        f4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(static_cast<int8_t>(w[0] >> (8 * e))) * scale;
        return x;
    }
}

// LPR lanes per row, two vectors of four elements each (unit_place); T tokens, the
// same row of each.  VEC: 16-byte stores.
template <int DT, int LPR, bool VEC, int T>
__global__ __launch_bounds__(kBlock) void kv_read(ReadArgs a) {
    constexpr int kGroups = kBlock / LPR;
    const uint32_t t0 = blockIdx.x / a.parts * T, part = blockIdx.x % a.parts;
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    int s[T];
    KvToken tok[T];
    kv_sequences_of<T>(a.b, static_cast<int>(t0), s);
#pragma unroll
    for (int i = 0; i < T; ++i) tok[i] = kv_token(a.b, a.c, s[i], static_cast<int>(t0) + i);
    const int row = static_cast<int>(part) * kGroups + group;
    if (row >= a.kinds * a.c.kv_heads) return;
    const bool is_k = a.k_out && row < a.c.kv_heads;
    const int head = row % a.c.kv_heads;
    const auto [d0, d1, turned] = unit_place<4>(lane, 0, false, a.c.stride);
    if (d1 >= a.c.stride) return;
    u4 lo[T], hi[T];
    float scale[T];
#pragma unroll
    for (int i = 0; i < T; ++i) {
        lo[i] = hi[i] = u4{0, 0, 0, 0};
        scale[i] = 0.f;
        if (tok[i].page < 0) continue;
        const int64_t at = (static_cast<int64_t>(tok[i].page) * a.c.kv_heads + head) * a.c.page_size + tok[i].slot;
        const char* in = (is_k ? a.c.k : a.c.v) + at * a.c.stride * (DT == MIMIR_KV_F32 ? 4 : DT == MIMIR_KV_BF16 ? 2 : 1);
        lo[i] = get<DT>(in, d0);
        hi[i] = get<DT>(in, d1);
        if constexpr (DT == MIMIR_KV_I8) scale[i] = (is_k ? a.c.k_scale : a.c.v_scale)[at];
    }
#pragma unroll
    for (int i = 0; i < T; ++i) {
        if (!tok[i].in) continue;
        float* y = (is_k ? a.k_out : a.v_out) + (t0 + i) * a.ld_out + static_cast<int64_t>(head) * a.c.head_dim;
        const f4 l = value_of<DT>(lo[i], scale[i]), h = value_of<DT>(hi[i], scale[i]);
        if constexpr (VEC) {
            if (d0 < a.c.head_dim) st_stream(y + d0, l);
            if (d1 < a.c.head_dim) st_stream(y + d1, h);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (d0 + e < a.c.head_dim) y[d0 + e] = l[e];
                if (d1 + e < a.c.head_dim) y[d1 + e] = h[e];
            }
        }
    }
}

// f(LPR) for rows of `stride` elements, eight to a lane.
template <class Fn>
int with_lanes(int stride, Fn&& f) {
    if (stride <= 64) return f(std::integral_constant<int, 8>{});
    if (stride <= 128) return f(std::integral_constant<int, 16>{});
    return f(std::integral_constant<int, 32>{});
}

// Tokens of a workgroup where there are enough for the GPU.
constexpr int kTokens = 4;
bool several_tokens(int64_t tokens, int64_t parts) { return tokens / kTokens * parts >= 2048; }

template <class Fn>
int with_type(int dtype, Fn&& f) {
    if (dtype == MIMIR_KV_F32) return f(std::integral_constant<int, MIMIR_KV_F32>{});
    if (dtype == MIMIR_KV_BF16) return f(std::integral_constant<int, MIMIR_KV_BF16>{});
    return f(std::integral_constant<int, MIMIR_KV_I8>{});
}

}  // namespace

int mimir::kv_view(mimir_ctx* ctx, const char* what, const mimir_kv_cache* c, KvView* out) {
    MIMIR_REQUIRE(ctx, c, "%s: null cache", what);
    MIMIR_REQUIRE(ctx, c->dtype >= MIMIR_KV_F32 && c->dtype <= MIMIR_KV_I8, "%s: cache type %d", what, c->dtype);
    MIMIR_REQUIRE(ctx, c->page_size >= kKvPad && c->page_size % kKvPad == 0 && c->page_size <= (1 << 20),
                  "%s: page_size %d is not a multiple of 16 up to 2^20", what, c->page_size);
    MIMIR_REQUIRE(ctx, c->kv_heads >= 1 && c->kv_heads <= (1 << 16) && c->head_dim >= 1 && c->head_dim <= kKvMaxDim,
                  "%s: kv_heads %d, head_dim %d (1 to %d)", what, c->kv_heads, c->head_dim, kKvMaxDim);
    MIMIR_REQUIRE(ctx, c->pages >= 0 && c->pages < (int64_t{1} << 31), "%s: %lld pages", what, (long long)c->pages);
    const bool scaled = c->dtype == MIMIR_KV_I8;
    MIMIR_REQUIRE(ctx, c->pages == 0 || (c->k && c->v && (!scaled || (c->k_scale && c->v_scale))), "%s: null cache buffer", what);
    MIMIR_REQUIRE(ctx, aligned16(c->k) && aligned16(c->v) && (!scaled || (aligned16(c->k_scale) && aligned16(c->v_scale))),
                  "%s: cache buffers must be 16-byte aligned", what);
    *out = KvView{static_cast<char*>(c->k), static_cast<char*>(c->v), c->k_scale, c->v_scale, c->pages, c->kv_heads, c->head_dim,
                  kv_stride(c->head_dim), c->page_size, make_fastdiv(static_cast<uint32_t>(c->page_size))};
    return MIMIR_OK;
}

int mimir::kv_batch(mimir_ctx* ctx, const char* what, const mimir_kv_cache* c, const mimir_kv_batch* b, KvBatch* out) {
    MIMIR_REQUIRE(ctx, b, "%s: null batch", what);
    constexpr int64_t kMost = int64_t{1} << 30;
    MIMIR_REQUIRE(ctx, b->sequences >= 0 && b->sequences < kMost && b->tokens >= 0 && b->tokens < kMost && b->max_new >= 0 &&
                           b->max_new < kMost && b->max_len >= 0 && b->max_len < kMost,
                  "%s: invalid batch (sequences=%lld tokens=%lld max_new=%lld max_len=%lld)", what, (long long)b->sequences,
                  (long long)b->tokens, (long long)b->max_new, (long long)b->max_len);
    MIMIR_REQUIRE(ctx, b->ld_pages >= 0 && (b->max_len + c->page_size - 1) / c->page_size <= b->ld_pages,
                  "%s: max_len %lld does not fit %lld pages of %d", what, (long long)b->max_len, (long long)b->ld_pages,
                  c->page_size);
    MIMIR_REQUIRE(ctx, b->sequences == 0 || (b->token_start && b->kv_len && (b->max_len == 0 || b->page_table)),
                  "%s: null batch array", what);
    // No sequence has more rows than there are, whatever the bound.
    *out = KvBatch{b->token_start, b->kv_len, b->page_table, b->ld_pages, static_cast<int32_t>(b->sequences),
                   static_cast<int32_t>(b->tokens), static_cast<int32_t>(std::min(b->max_new, b->tokens)),
                   static_cast<int32_t>(b->max_len)};
    return MIMIR_OK;
}

extern "C" {

int mimir_kv_cache_bytes(const mimir_kv_cache* c, size_t* kv_bytes, size_t* scale_bytes) {
    if (!c || !kv_bytes || !scale_bytes || c->dtype < MIMIR_KV_F32 || c->dtype > MIMIR_KV_I8 || c->page_size < kKvPad ||
        c->page_size % kKvPad || c->page_size > (1 << 20) || c->pages < 0 || c->pages >= (int64_t{1} << 31) || c->kv_heads < 1 ||
        c->kv_heads > (1 << 16) || c->head_dim < 1 || c->head_dim > kKvMaxDim)
        return MIMIR_EINVAL;
    // pages * heads * slots < 2^67: checked before the product.
    const double most = static_cast<double>(c->pages) * c->kv_heads * c->page_size * kv_stride(c->head_dim) * 4.0;
    if (most >= 9e18) return MIMIR_EINVAL;
    const size_t slots = static_cast<size_t>(c->pages) * static_cast<size_t>(c->kv_heads) * static_cast<size_t>(c->page_size);
    *kv_bytes = slots * static_cast<size_t>(kv_stride(c->head_dim) * kv_element_bytes(c->dtype));
    *scale_bytes = c->dtype == MIMIR_KV_I8 ? slots * sizeof(float) : 0;
    return MIMIR_OK;
}

int mimir_kv_append(mimir_ctx* ctx, const mimir_kv_cache* cache, const mimir_kv_batch* batch, const float* k,
                    const float* v, int64_t ld_kv, const mimir_rope* rope, const float* q, int64_t ld_q, float* q_out,
                    int64_t ld_q_out, int64_t q_heads) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "KV append";
    AppendArgs a{};
    if (int st = kv_view(ctx, what, cache, &a.c)) return st;
    if (int st = kv_batch(ctx, what, cache, batch, &a.b)) return st;
    const int64_t d = cache->head_dim;
    MIMIR_REQUIRE(ctx, ld_kv >= cache->kv_heads * d, "%s: row stride %lld below kv_heads * head_dim", what, (long long)ld_kv);
    MIMIR_REQUIRE(ctx, rope || !q, "%s: q without rope", what);
    if (rope) {
        if (int st = rope_check(ctx, what, rope, d)) return st;
        MIMIR_REQUIRE(ctx, batch->max_len <= rope->table_rows, "%s: max_len %lld exceeds the %lld-row table", what,
                      (long long)batch->max_len, (long long)rope->table_rows);
    }
    MIMIR_REQUIRE(ctx, !q || (q_heads >= 1 && q_heads <= (1 << 20)), "%s: q_heads %lld", what, (long long)q_heads);
    const int64_t qh = q ? q_heads : 0;
    MIMIR_REQUIRE(ctx, !q || (ld_q >= qh * d && ld_q_out >= qh * d), "%s: q strides (%lld, %lld) below q_heads * head_dim", what,
                  (long long)ld_q, (long long)ld_q_out);
    if (batch->tokens == 0 || batch->sequences == 0) return MIMIR_OK;
    MIMIR_REQUIRE(ctx, k && v && (!q || q_out), "%s: null pointer", what);
    MIMIR_REQUIRE(ctx, !q || q != q_out || ld_q == ld_q_out, "%s: in place needs equal strides", what);
    MIMIR_ENTER(ctx);
    a.q = q;
    a.q_out = q_out;
    a.k = k;
    a.v = v;
    a.ld_q = ld_q;
    a.ld_q_out = ld_q_out;
    a.ld_kv = ld_kv;
    a.cos_tab = rope ? rope->cos_tab : nullptr;
    a.sin_tab = rope ? rope->sin_tab : nullptr;
    a.q_heads = static_cast<int32_t>(qh);
    a.half = rope ? rope->rot_dim / 2 : 0;
    a.interleaved = rope && rope->interleaved ? 1 : 0;
    const bool vec = d % 4 == 0 && a.half % 4 == 0 && ld_kv % 4 == 0 && aligned16(k) && aligned16(v) &&
                     (!rope || (aligned16(rope->cos_tab) && aligned16(rope->sin_tab))) &&
                     (!q || (ld_q % 4 == 0 && ld_q_out % 4 == 0 && aligned16(q) && aligned16(q_out)));
    const int64_t rows = qh + 2 * cache->kv_heads;
    return with_type(cache->dtype, [&](auto dt) {
        return with_lanes(a.c.stride, [&](auto lpr) {
            constexpr int LPR = decltype(lpr)::value, DT = decltype(dt)::value;
            // Half the threads where they leave fewer without a row.
            constexpr int64_t kGroups = kBlock / LPR;
            const auto parts_of = [&](int64_t groups) { return (rows + groups - 1) / groups; };
            const bool small = parts_of(kGroups / 2) < 2 * parts_of(kGroups);
            a.parts = static_cast<uint32_t>(parts_of(small ? kGroups / 2 : kGroups));
            const int threads = small ? kBlock / 2 : kBlock;
            const int64_t blocks = batch->tokens * a.parts;
            MIMIR_REQUIRE(ctx, dispatch_fits(blocks, threads), "%s: grid of %lld workgroups exceeds the limit", what,
                          (long long)blocks);
            const auto grid = static_cast<unsigned>(blocks);
            if (vec && ctx->keep_outputs) kv_append<DT, LPR, 4, true><<<grid, threads, 0, ctx->stream>>>(a);
            else if (vec) kv_append<DT, LPR, 4, false><<<grid, threads, 0, ctx->stream>>>(a);
            else kv_append<DT, LPR, 1, true><<<grid, threads, 0, ctx->stream>>>(a);
            return launched(ctx, "kv_append");
        });
    });
}

int mimir_kv_read(mimir_ctx* ctx, const mimir_kv_cache* cache, const mimir_kv_batch* batch, float* k_out, float* v_out,
                  int64_t ld_out) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "KV read";
    ReadArgs a{};
    if (int st = kv_view(ctx, what, cache, &a.c)) return st;
    if (int st = kv_batch(ctx, what, cache, batch, &a.b)) return st;
    MIMIR_REQUIRE(ctx, ld_out >= static_cast<int64_t>(cache->kv_heads) * cache->head_dim,
                  "%s: row stride %lld below kv_heads * head_dim", what, (long long)ld_out);
    if (batch->tokens == 0 || batch->sequences == 0 || (!k_out && !v_out)) return MIMIR_OK;
    MIMIR_ENTER(ctx);
    a.k_out = k_out;
    a.v_out = v_out;
    a.ld_out = ld_out;
    a.kinds = (k_out ? 1 : 0) + (v_out ? 1 : 0);
    const bool vec = cache->head_dim % 4 == 0 && ld_out % 4 == 0 && aligned16(k_out) && aligned16(v_out);
    return with_type(cache->dtype, [&](auto dt) {
        return with_lanes(a.c.stride, [&](auto lpr) {
            constexpr int LPR = decltype(lpr)::value, DT = decltype(dt)::value;
            constexpr int64_t kGroups = kBlock / LPR;
            a.parts = static_cast<uint32_t>((static_cast<int64_t>(a.kinds) * cache->kv_heads + kGroups - 1) / kGroups);
            const bool many = several_tokens(batch->tokens, a.parts);
            const int64_t blocks = (many ? (batch->tokens + kTokens - 1) / kTokens : batch->tokens) * a.parts;
            MIMIR_REQUIRE(ctx, dispatch_fits(blocks, kBlock), "%s: grid of %lld workgroups exceeds the limit", what,
                          (long long)blocks);
            const auto grid = static_cast<unsigned>(blocks);
            if (vec && many) kv_read<DT, LPR, true, kTokens><<<grid, kBlock, 0, ctx->stream>>>(a);
            else if (vec) kv_read<DT, LPR, true, 1><<<grid, kBlock, 0, ctx->stream>>>(a);
            else if (many) kv_read<DT, LPR, false, kTokens><<<grid, kBlock, 0, ctx->stream>>>(a);
            else kv_read<DT, LPR, false, 1><<<grid, kBlock, 0, ctx->stream>>>(a);
            return launched(ctx, "kv_read");
        });
    });
}

}  // extern "C"
