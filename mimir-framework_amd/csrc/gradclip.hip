// gradclip.hip -- the norm of many gradients and their clipping by it:
//
//   norm = sqrt(sum over all tensors of x^2),  out = x * min(1, max_norm / (norm + 1e-6))
//
// The reference has neither on the device; its optimisers work on host vectors.
//
// Both are bound by the bytes: once over the tensors for the norm, once more, with
// the writes, for the clipping.  Chunks of 8192 elements are dealt round a grid that
// the GPU holds at once; a workgroup finds its chunk's tensor in the list, which the
// kernel's arguments carry (kTensors of them a launch: no table in memory, none to
// keep).  Each leaves one sum in 64 bits -- squares of fp32's whole range, whose
// rounding no order of the tensors shows -- and every workgroup of the clipping adds
// those up itself, in the same order, instead of a launch that does (which joins them
// where they are more than one launch leaves).  The clipping
// goes through its chunks from the last to the first: what the norm's pass has left
// in the Infinity Cache is read from there.
//
// Measured on MI355X: 369 M values in 44 tensors (738 MB), norm 116 us = 6.3 TB/s, clipping
// 275 us = 5.4; 30 tensors of 3.4 M values in all 4.6 and 6.4 us.
#include "common.hpp"
#include "internal.hpp"
#include "matrix.hpp"

#include <math.h>

using namespace mimir;

namespace {

constexpr int kTensors = 96;        // of a launch: 2.7 KB of arguments
constexpr int64_t kChunk = 8192;    // elements
constexpr int kWorkgroups = 2048;   // eight a CU

struct List {
    const void* in[kTensors];
    void* out[kTensors];
    int64_t n[kTensors];
    int32_t first[kTensors + 1];  // chunk
    uint32_t bf16[kTensors / 32], vec[kTensors / 32];
    int32_t count;
};

struct Chunk {
    int tensor;
    int64_t at, n;
};

__device__ __forceinline__ Chunk chunk_of(const List& l, int32_t c) {
    int lo = 0, hi = l.count - 1;  // the last tensor whose first chunk is not after c
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (l.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    const int64_t at = static_cast<int64_t>(c - l.first[lo]) * kChunk;
    return Chunk{lo, at, min(kChunk, l.n[lo] - at)};
}

__device__ __forceinline__ float bf16_at(uint32_t pair, int high) {
    return __builtin_bit_cast(float, high ? pair & 0xffff0000u : pair << 16);
}

// f(element, vector) for the workgroup's vectors of `wide` elements of p[0, n): the N of
// a whole chunk are loaded before the first is used.
template <int N, class V, class T, class F>
__device__ __forceinline__ void with_vectors(const T* p, int wide, int64_t n, F&& f) {
    const int64_t first = wide * threadIdx.x, next = wide * kBlock;
    if (n == kChunk) {
        V v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = *reinterpret_cast<const V*>(p + first + j * next);
#pragma unroll
        for (int j = 0; j < N; ++j) f(first + j * next, v[j]);
        return;
    }
    for (int64_t i = first; i < n; i += next) f(i, *reinterpret_cast<const V*>(p + i));
}

__device__ __forceinline__ double block_sum64(double v, double* lds) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) s += lds[w];
    return s;
}

__device__ __forceinline__ double square(float x) { return static_cast<double>(x) * static_cast<double>(x); }

__global__ __launch_bounds__(kBlock) void norm_sums(List l, double* sums) {
    __shared__ double lds[kBlock / kWave];
    double s[4] = {};
    for (int32_t c = blockIdx.x; c < l.first[l.count]; c += gridDim.x) {
        const Chunk k = chunk_of(l, c);
        const bool bf16 = l.bf16[k.tensor / 32] >> (k.tensor % 32) & 1, vec = l.vec[k.tensor / 32] >> (k.tensor % 32) & 1;
        int64_t done = 0;
        if (bf16) {
            const uint16_t* p = static_cast<const uint16_t*>(l.in[k.tensor]) + k.at;
            if (vec) {
                done = k.n / 8 * 8;
                with_vectors<4, u4>(p, 8, done, [&](int64_t, u4 v) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[e % 4] += square(bf16_at(v[e / 2], e % 2));
                });
            }
            for (int64_t i = done + threadIdx.x; i < k.n; i += kBlock) s[0] += square(bf16_at(p[i], 0));
        } else {
            const float* p = static_cast<const float*>(l.in[k.tensor]) + k.at;
            if (vec) {
                done = k.n / 4 * 4;
                with_vectors<8, f4>(p, 4, done, [&](int64_t, f4 v) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] += square(v[e]);
                });
            }
            for (int64_t i = done + threadIdx.x; i < k.n; i += kBlock) s[0] += square(p[i]);
        }
    }
    const double all = block_sum64((s[0] + s[1]) + (s[2] + s[3]), lds);
    if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

__device__ __forceinline__ double total_of(const double* sums, int32_t count, double* lds) {
    double s = 0.0;
    for (int32_t i = threadIdx.x; i < count; i += kBlock) s += sums[i];
    return block_sum64(s, lds);
}

__global__ __launch_bounds__(kBlock) void sums_join(const double* sums, int32_t count, double* total) {
    __shared__ double lds[kBlock / kWave];
    const double s = total_of(sums, count, lds);
    if (threadIdx.x == 0) *total = s;
}

__global__ __launch_bounds__(kBlock) void norm_join(const double* sums, int32_t count, float* norm) {
    __shared__ double lds[kBlock / kWave];
    const double n = sqrt(total_of(sums, count, lds));
    if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

__global__ __launch_bounds__(kBlock) void clip(List l, const double* sums, int32_t count, float max_norm, float* norm) {
    __shared__ double lds[kBlock / kWave];
    const double n = sqrt(total_of(sums, count, lds));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
    // An infinite max_norm clips nothing, also where the norm is infinite.
    const double ratio = isinf(max_norm) && !isnan(n) ? 2.0 : static_cast<double>(max_norm) / (n + 1e-6);
    // A NaN stays one.  A factor that fp32 does not hold with all its bits, of elements
    // near fp32's largest, multiplies in 64 bits.
    const bool tiny = ratio < 0x1p-126;
    const float by = ratio > 1.0 ? 1.0f : static_cast<float>(ratio);
    const auto scaled = [&](float x) { return tiny ? static_cast<float>(static_cast<double>(x) * ratio) : x * by; };
    const int32_t chunks = l.first[l.count];
    for (int32_t c = chunks - 1 - static_cast<int32_t>(blockIdx.x); c >= 0; c -= gridDim.x) {
        const Chunk k = chunk_of(l, c);
        if (by == 1.0f && l.in[k.tensor] == l.out[k.tensor]) continue;
        const bool bf16 = l.bf16[k.tensor / 32] >> (k.tensor % 32) & 1, vec = l.vec[k.tensor / 32] >> (k.tensor % 32) & 1;
        int64_t done = 0;
        if (bf16) {
            const uint16_t* p = static_cast<const uint16_t*>(l.in[k.tensor]) + k.at;
            uint16_t* q = static_cast<uint16_t*>(l.out[k.tensor]) + k.at;
            if (vec) {
                done = k.n / 8 * 8;
                with_vectors<4, u4>(p, 8, done, [&](int64_t i, u4 v) {
                    u4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = pack_bf16(scaled(bf16_at(v[e], 0)), scaled(bf16_at(v[e], 1)));
                    st_stream(q + i, y);
                });
            }
            for (int64_t i = done + threadIdx.x; i < k.n; i += kBlock) {
                const float y = scaled(bf16_at(p[i], 0));
                q[i] = static_cast<uint16_t>(pack_bf16(y, y));
            }
        } else {
            const float* p = static_cast<const float*>(l.in[k.tensor]) + k.at;
            float* q = static_cast<float*>(l.out[k.tensor]) + k.at;
            if (vec) {
                done = k.n / 4 * 4;
                with_vectors<8, f4>(p, 4, done, [&](int64_t i, f4 v) { st_stream(q + i, f4{scaled(v[0]), scaled(v[1]), scaled(v[2]), scaled(v[3])}); });
            }
            for (int64_t i = done + threadIdx.x; i < k.n; i += kBlock) q[i] = scaled(p[i]);
        }
    }
}

struct Launch {
    List list;
    int grid;
};

// f(Launch, sums before it) for each launch's tensors.
template <class Fn>
int with_lists(mimir_ctx* ctx, const char* what, const mimir_tensor* t, int64_t count, int64_t launches, bool clipping, Fn&& f) {
    int64_t before = 0, i = 0;
    while (i < count) {
        Launch a{};
        int64_t chunks = 0;
        for (; i < count && a.list.count < kTensors; ++i) {
            if (t[i].n == 0) continue;
            const int k = a.list.count;
            const int64_t more = (t[i].n + kChunk - 1) / kChunk;
            if (chunks + more > INT32_MAX - kWorkgroups) {
                if (k > 0) break;
                return fail(ctx, MIMIR_EINVAL, "%s: a tensor of %lld elements", what, (long long)t[i].n);
            }
            a.list.in[k] = t[i].data;
            a.list.out[k] = clipping ? t[i].out : nullptr;
            a.list.n[k] = t[i].n;
            a.list.first[k] = static_cast<int32_t>(chunks);
            if (t[i].type == MIMIR_NUM_BF16) a.list.bf16[k / 32] |= 1u << (k % 32);
            if (aligned16(t[i].data) && (!clipping || aligned16(t[i].out))) a.list.vec[k / 32] |= 1u << (k % 32);
            chunks += more;
            a.list.first[++a.list.count] = static_cast<int32_t>(chunks);
        }
        if (a.list.count == 0) continue;
        // The sums of up to eight launches together stay as many as one's; more of them
        // take 256 workgroups each, one a CU.
        a.grid = static_cast<int>(std::min<int64_t>(chunks, std::max<int64_t>(256, kWorkgroups / launches)));
        f(a, before);
        if (int st = launched(ctx, what)) return st;
        before += a.grid;
    }
    return MIMIR_OK;
}

int check(mimir_ctx* ctx, const char* what, const mimir_tensor* t, int64_t count, bool clipping) {
    MIMIR_REQUIRE(ctx, count >= 0 && count <= (1 << 20), "%s: %lld tensors (0 to 2^20)", what, (long long)count);
    MIMIR_REQUIRE(ctx, count == 0 || t, "%s: null list", what);
    for (int64_t i = 0; i < count; ++i) {
        MIMIR_REQUIRE(ctx, t[i].type == MIMIR_NUM_F32 || t[i].type == MIMIR_NUM_BF16, "%s: tensor %lld of type %d", what, (long long)i,
                      (int)t[i].type);
        MIMIR_REQUIRE(ctx, t[i].n >= 0 && t[i].n <= (int64_t{1} << 40), "%s: tensor %lld of %lld elements", what, (long long)i,
                      (long long)t[i].n);
        MIMIR_REQUIRE(ctx, t[i].n == 0 || (t[i].data && (!clipping || t[i].out)), "%s: tensor %lld is null", what, (long long)i);
        const uintptr_t size = t[i].type == MIMIR_NUM_BF16 ? 2 : 4;
        MIMIR_REQUIRE(ctx, reinterpret_cast<uintptr_t>(t[i].data) % size == 0 && reinterpret_cast<uintptr_t>(t[i].out) % size == 0,
                      "%s: tensor %lld is not aligned to its elements", what, (long long)i);
    }
    return MIMIR_OK;
}

// The launches' sums, and how many.
int sums_of(mimir_ctx* ctx, const char* what, const mimir_tensor* t, int64_t count, int64_t* launches, double** sums, int32_t* have) {
    *launches = (count + kTensors - 1) / kTensors + 1;
    char* work;
    if (int st = mat_scratch(ctx, sizeof(double) * static_cast<size_t>(*launches * kWorkgroups), &work)) return st;
    *sums = reinterpret_cast<double*>(work);
    *have = 0;
    return with_lists(ctx, what, t, count, *launches, false, [&](const Launch& a, int64_t before) {
        norm_sums<<<static_cast<unsigned>(a.grid), kBlock, 0, ctx->stream>>>(a.list, *sums + before);
        *have = static_cast<int32_t>(before + a.grid);
    });
}

}  // namespace

extern "C" {

int mimir_grad_norm(mimir_ctx* ctx, const mimir_tensor* tensors, int64_t count, float* norm) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "gradients' norm";
    if (int st = check(ctx, what, tensors, count, false)) return st;
    MIMIR_REQUIRE(ctx, norm, "%s: null norm", what);
    MIMIR_ENTER(ctx);
    int64_t launches;
    double* sums;
    int32_t have;
    if (int st = sums_of(ctx, what, tensors, count, &launches, &sums, &have)) return st;
    norm_join<<<1, kBlock, 0, ctx->stream>>>(sums, have, norm);
    return launched(ctx, "norm_join");
}

int mimir_grad_clip(mimir_ctx* ctx, const mimir_tensor* tensors, int64_t count, float max_norm, float* norm) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "gradients' clipping";
    if (int st = check(ctx, what, tensors, count, true)) return st;
    MIMIR_REQUIRE(ctx, max_norm >= 0.0f, "%s: max_norm %g", what, (double)max_norm);
    MIMIR_ENTER(ctx);
    int64_t launches;
    double* sums;
    int32_t have;
    if (int st = sums_of(ctx, what, tensors, count, &launches, &sums, &have)) return st;
    if (have == 0) return norm ? mimir_fill_f32(ctx, norm, 1, 0.0f) : MIMIR_OK;
    // Each workgroup of each launch adds the sums up.  More of them than one launch leaves
    // are added once, in the same order, to the place behind them (sums_of counts one more
    // launch than there are).  With / without,
    // us: 3000 tensors of 64 elements 314 / 318, 20000 1859 / 3397, 100000 7737 / 49105.
    if (have > kWorkgroups) {
        sums_join<<<1, kBlock, 0, ctx->stream>>>(sums, have, sums + have);
        if (int st = launched(ctx, "sums_join")) return st;
        sums += have;
        have = 1;
    }
    return with_lists(ctx, what, tensors, count, launches, true, [&](const Launch& a, int64_t before) {
        clip<<<static_cast<unsigned>(a.grid), kBlock, 0, ctx->stream>>>(a.list, sums, have, max_norm, before ? nullptr : norm);
    });
}

}  // extern "C"
