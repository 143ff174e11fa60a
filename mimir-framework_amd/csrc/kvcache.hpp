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

// Which sequence has row t, searched by a whole wave (every lane gets the
// answer): the last one that starts at or before t.  -1: none has it.
__device__ __forceinline__ int kv_sequence_of(const KvBatch& b, int t) {
    int below = 0;  // starts at or before t
    for (int s = threadIdx.x & (kWave - 1); __any(s <= b.sequences); s += kWave) {
        const bool in = s <= b.sequences && b.token_start[min(s, b.sequences)] <= t;
        const int n = __popcll(__ballot(in));
        below += n;
        if (n < kWave) break;
    }
    return below >= 1 && below <= b.sequences ? below - 1 : -1;
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

// MIMIR_OK, or why these tables do not fit heads of head_dim.
int rope_check(mimir_ctx* ctx, const char* what, const mimir_rope* rope, int64_t head_dim);

}  // namespace mimir
