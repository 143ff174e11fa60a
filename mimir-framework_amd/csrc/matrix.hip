// matrix.hip -- what the products of matrix.hpp need beside themselves: operands
// split or copied into planes of bf16, slices of a split contraction joined, a gradient
// of no tokens, scratch.
#include "matrix.hpp"

using namespace mimir;

namespace {

// Eight columns a thread: 32 bytes of fp32 read, 16 written to each of three planes.
template <bool BF16>
__global__ __launch_bounds__(kBlock) void stage_rows(const void* src, int64_t rows, int64_t cols, int64_t ld, uint16_t* dst,
                                                      int64_t ld_dst, int64_t plane) {
    const int64_t of_row = ld_dst / 8, total = rows * of_row, stride = static_cast<int64_t>(gridDim.x) * kBlock;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += stride) {
        const int64_t r = i / of_row, c = i % of_row * 8;
        mat_stage8<BF16>(src, r * ld + c, cols - c, dst + r * ld_dst + c, plane);
    }
}

__global__ __launch_bounds__(kBlock) void join_slices(MatOut o, MatArgs g, MatTileSize tile) {
    const int64_t n = g.n_dev ? min(g.n, *g.n_dev) : g.n, slice = n * o.ld_partial;
    const int32_t splits = g.splits_of(mat_tiles_of(tile, g.m, n, 1));
    const float by = o.factor();
    const int64_t of_row = (g.m + 3) / 4, one = n * of_row, stride = static_cast<int64_t>(gridDim.x) * kBlock;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < one * g.batches; i += stride) {
        const int64_t batch = i / one, r = i % one / of_row, c = i % one % of_row * 4;
        const float* p = o.partial + batch * slice + r * o.ld_partial + c;
        f4 v{};
        for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f4*>(p + s * g.batches * slice);
        o.put(static_cast<int>(batch), r, static_cast<int32_t>(c), g.m, v, by);
    }
}

// Eight columns a thread.
template <class T>
__global__ __launch_bounds__(kBlock) void zero_rows(T* p, int64_t rows, int64_t cols, int64_t ld) {
    typedef uint32_t V __attribute__((ext_vector_type(2 * sizeof(T)), aligned(sizeof(T))));
    const int64_t of_row = (cols + 7) / 8, total = rows * of_row, stride = static_cast<int64_t>(gridDim.x) * kBlock;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += stride) {
        const int64_t c = i % of_row * 8;
        T* q = p + i / of_row * ld + c;
        if (c + 8 <= cols) *reinterpret_cast<V*>(q) = V{};
        else
            for (int64_t e = 0; e < cols - c; ++e) q[e] = T{};
    }
}

unsigned grid_of(int64_t items) {
    const int64_t b = (items + kBlock - 1) / kBlock;
    return static_cast<unsigned>(b < 1 ? 1 : b > 65536 ? 65536 : b);
}

}  // namespace

int mimir::mat_stage(mimir_ctx* ctx, int type, const void* src, int64_t rows, int64_t cols, int64_t ld, uint16_t* dst,
                     int64_t ld_dst, int64_t plane) {
    const unsigned grid = grid_of(rows * (ld_dst / 8));
    if (type == MIMIR_NUM_BF16) stage_rows<true><<<grid, kBlock, 0, ctx->stream>>>(src, rows, cols, ld, dst, ld_dst, plane);
    else stage_rows<false><<<grid, kBlock, 0, ctx->stream>>>(src, rows, cols, ld, dst, ld_dst, plane);
    return launched(ctx, "stage_rows");
}

int mimir::mat_zero(mimir_ctx* ctx, int type, void* p, int64_t rows, int64_t cols, int64_t ld) {
    const unsigned grid = grid_of(rows * ((cols + 7) / 8));
    if (type == MIMIR_NUM_BF16) zero_rows<<<grid, kBlock, 0, ctx->stream>>>(static_cast<uint16_t*>(p), rows, cols, ld);
    else zero_rows<<<grid, kBlock, 0, ctx->stream>>>(static_cast<float*>(p), rows, cols, ld);
    return launched(ctx, "zero_rows");
}

int mimir::mat_join(mimir_ctx* ctx, const MatOut& o, const MatArgs& g, MatTileSize tile) {
    join_slices<<<grid_of(static_cast<int64_t>(g.n) * ((g.m + 3) / 4) * g.batches), kBlock, 0, ctx->stream>>>(o, g, tile);
    return launched(ctx, "join_slices");
}

int mimir::mat_scratch(mimir_ctx* ctx, size_t bytes, char** out) {
    void* p = nullptr;
    const int st = captured_scratch(ctx, bytes, &p);
    *out = static_cast<char*>(p);
    return st;
}
