// kvcache.hpp -- the paged key/value cache and packed batches as the kernels see
// them (mimir_hip.h mimir_kv_cache, mimir_kv_batch), and the host's checks of both.
#pragma once

#include "common.hpp"
#include "fastdiv.hpp"
#include "internal.hpp"
#include "kvindex.hpp"

namespace mimir {

// A row of the cache is padded to this many elements, so that every type's rows
// are whole 16-byte vectors.
constexpr int kKvPad = 16;
constexpr int kKvMaxDim = 256;

struct KvView {
    char* k;
    char* v;
    float* k_scale;
    float* v_scale;
    int64_t pages;
    int32_t kv_heads, head_dim, stride, page_size;
    FastDiv page_div;
};

// Which sequences have rows t .. t + T - 1, searched by a whole wave (every lane gets
// the answers): the last one that starts at or before each.  -1: none has it.
template <int T>
__device__ __forceinline__ void kv_sequences_of(const KvBatch& b, int t, int* found) {
    const int lane = threadIdx.x & (kWave - 1);
    // Starts at or before t by 64 places at a time: there are lo to hi of them.  (A token
    // each of 4096 sequences written and read back: 49 us, searched from the first on 104.)
    int lo = 0, hi = b.sequences + 1;
    while (hi - lo > kWave) {
        const int apart = (hi - lo + kWave - 1) / kWave, s = lo + min(lane, (hi - lo - 1) / apart) * apart;
        const bool in = lo + lane * apart < hi;
        const int n = __popcll(__ballot(in && b.token_start[s] <= t));
        hi = n * apart < hi - lo ? lo + n * apart : hi;
        lo = n > 0 ? lo + (n - 1) * apart + 1 : lo;
    }
#pragma unroll
    for (int i = 0; i < T; ++i) found[i] = lo;  // starts at or before t + i
    for (int s = lo + lane; __any(s <= b.sequences); s += kWave) {
        const bool in = s <= b.sequences;
        const int start = b.token_start[min(s, b.sequences)];
#pragma unroll
        for (int i = 0; i < T; ++i) found[i] += __popcll(__ballot(in && start <= t + i));
        if (!__all(in && start <= t + T - 1)) break;
    }
#pragma unroll
    for (int i = 0; i < T; ++i) found[i] = found[i] >= 1 && found[i] <= b.sequences ? found[i] - 1 : -1;
}

// Where token t of sequence s (kv_sequences_of) stands: its position (below 0 for
// tokens that the cache has no room for), page and slot.  Not `in`: no token.
struct KvToken {
    bool in;
    int32_t position, page, slot;
};

__device__ __forceinline__ KvToken kv_token(const KvBatch& b, const KvView& c, int s, int t) {
    if (s < 0) return KvToken{false, -1, -1, 0};
    const KvSequence q = kv_sequence(b, s);
    const int i = t - q.first, position = q.len - q.n + i;
    if (i < 0 || i >= q.n) return KvToken{false, -1, -1, 0};
    const KvSlot at = kv_slot(b, c.pages, c.page_div, s, position);
    return KvToken{true, position, at.page, at.slot};
}

inline int kv_element_bytes(int dtype) { return dtype == MIMIR_KV_F32 ? 4 : dtype == MIMIR_KV_BF16 ? 2 : 1; }
inline int kv_stride(int head_dim) { return (head_dim + kKvPad - 1) / kKvPad * kKvPad; }

// MIMIR_OK and the view, or the error.
int kv_view(mimir_ctx* ctx, const char* what, const mimir_kv_cache* cache, KvView* out);
int kv_batch(mimir_ctx* ctx, const char* what, const mimir_kv_cache* cache, const mimir_kv_batch* batch, KvBatch* out);

// --- rotation ----------------------------------------------------------------

// A pair turned by (c, s), each result computed in double (the products are exact
// there) and rounded once, so that what is stored in fewer bits than fp32 does not
// depend on how the compiler contracts the products.
__device__ __forceinline__ void rotate_pair(float& x0, float& x1, float c, float s) {
    const double a = x0, b = x1, cd = c, sd = s;
    x0 = static_cast<float>(a * cd - b * sd);
    x1 = static_cast<float>(b * cd + a * sd);
}

// A unit: two vectors of W elements of a head row, for one lane.  Unit u of the
// rotated part holds vectors u and u + (half of the part), which for pairs half the
// part apart are the pairs' two elements, and otherwise W / 2 pairs each (W = 1: the
// pair itself); the rest of the row is halved the same way.  So lanes side by side
// read and write one run of memory with each vector.
struct UnitPlace {
    int d0, d1;  // first elements
    bool turned;
};

template <int W>
__device__ __forceinline__ UnitPlace unit_place(int u, int half, bool interleaved, int width) {
    if (u * W < half) return W == 1 && interleaved ? UnitPlace{2 * u, 2 * u + 1, true} : UnitPlace{u * W, half + u * W, true};
    const int rest = (width - 2 * half) / W, d = 2 * half + (u - half / W) * W;
    return UnitPlace{d, d + (rest + 1) / 2 * W, false};
}

// cos and sin of a turned unit's W pairs; `row`: the position's first pair.
template <int W>
__device__ __forceinline__ void unit_turns(const float* cos_tab, const float* sin_tab, int64_t row, int u, int half,
                                           bool interleaved, float* c, float* s) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
        const int pair = W == 1 || !interleaved ? u * W + e : (e < W / 2 ? 0 : half / 2) + u * W / 2 + e % ((W + 1) / 2);
        c[e] = cos_tab[row + pair];
        s[e] = sin_tab[row + pair];
    }
}

template <int W>
__device__ __forceinline__ void unit_rotate(float* lo, float* hi, const float* c, const float* s, bool interleaved) {
    if (W > 1 && interleaved) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) {
            rotate_pair(lo[2 * e], lo[2 * e + 1], c[e], s[e]);
            rotate_pair(hi[2 * e], hi[2 * e + 1], c[W / 2 + e], s[W / 2 + e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) rotate_pair(lo[e], hi[e], c[e], s[e]);
    }
}

// MIMIR_OK, or why these tables do not fit heads of head_dim.
int rope_check(mimir_ctx* ctx, const char* what, const mimir_rope* rope, int64_t head_dim);

}  // namespace mimir
