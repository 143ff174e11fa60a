// attention_paged_block.hip -- attention over a paged cache for many query rows per
// key / value head (prompts, and chunks of them): tiles of 32 keys in LDS.
#include "attention_paged.hpp"

#include <math.h>

#include <algorithm>

using namespace mimir;

namespace {

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_s4;

constexpr int kTile = 32;     // keys of a tile, and query rows of a wave
constexpr int kXcds = 8;

// A tile's keys and values in LDS: planes of rows of DP bf16 (fp32: three terms of
// each).  A key row is padded so that 16 rows' 16-byte reads touch every bank once; a
// value row, read four dimensions of four keys at a time and transposed on the way
// (ds_read_b64_tr_b16), so that four rows' 32 dimensions do.
template <int DT, int DP>
struct BlockTile {
    static constexpr int kPlanes = DT == MIMIR_KV_F32 ? 3 : 1;
    static constexpr int kKeyRow = 2 * DP + 16;
    static constexpr int kValueRow = DP % 64 == 32 ? 2 * DP : 2 * DP + 64;
    static_assert(kValueRow / 4 % 32 == 16, "four rows' reads in different banks");
    static constexpr int kKeyPlane = kTile * kKeyRow, kValuePlane = kTile * kValueRow;
    static constexpr int kValuesAt = kPlanes * kKeyPlane;
    static constexpr int kScalesAt = kValuesAt + kPlanes * kValuePlane;  // 8-bit: 32 of the keys, 32 of the values
    static constexpr int kBytes = kScalesAt + (DT == MIMIR_KV_I8 ? 2 * kTile * 4 : 0);
};

// Eight elements of a row on their way from memory to LDS.
template <int DT>
struct RowItem {
    static constexpr int kVecs = DT == MIMIR_KV_F32 ? 2 : 1;
    u4 v[kVecs];
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (DT == MIMIR_KV_I8) {
            const u2 x = *reinterpret_cast<const u2*>(p);
            v[0] = u4{x[0], x[1], 0, 0};
        } else {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) v[i] = reinterpret_cast<const u4*>(p)[i];
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = u4{0, 0, 0, 0};
    }
    __device__ __forceinline__ void stash(char* lds, int plane) const {
        if constexpr (DT == MIMIR_KV_F32) {
            const f4 a = __builtin_bit_cast(f4, v[0]), b = __builtin_bit_cast(f4, v[1]);
            const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            const Split8 s = split8(x);
            *reinterpret_cast<u4*>(lds) = s.h;
            *reinterpret_cast<u4*>(lds + plane) = s.m;
            *reinterpret_cast<u4*>(lds + 2 * plane) = s.l;
        } else if constexpr (DT == MIMIR_KV_BF16) {
            *reinterpret_cast<u4*>(lds) = v[0];
        } else {
            *reinterpret_cast<u4*>(lds) = bytes_bf16(v[0][0], v[0][1]);
        }
    }
};

// c += a b, a's planes in LDS.
template <int PLANES>
__device__ __forceinline__ f16v mfma_planes(const u4* a, const Split8& b, f16v c) {
    if constexpr (PLANES == 3) return mfma_split(Split8{a[0], a[1], a[2]}, b, c);
    c = mfma_bf16(a[0], b.l, c);
    c = mfma_bf16(a[0], b.m, c);
    return mfma_bf16(a[0], b.h, c);
}

template <int DT, int DP, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void paged_block(PagedArgs p, PagedRuns a) {
    using Tile = BlockTile<DT, DP>;
    constexpr int kThreads = WAVES * kWave, kC = DP / 16, kDb = DP / 32;
    constexpr int kElement = DT == MIMIR_KV_F32 ? 4 : DT == MIMIR_KV_BF16 ? 2 : 1;
    constexpr int kItems = (kTile * (DP / 8) + kThreads - 1) / kThreads;
    __shared__ __attribute__((aligned(16))) char lds[2 * Tile::kBytes];
    __shared__ PagedChunk chunk;

    // Each XCD takes runs that follow each other, whose keys it has in its L2.
    const uint32_t at = a.runs % kXcds == 0 && gridDim.x == a.runs ? blockIdx.x % kXcds * (a.runs / kXcds) + blockIdx.x / kXcds : blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    for (PagedWalk walk(p, a, at, &chunk); walk.more();) {
    int tid = static_cast<int>(threadIdx.x);
    asm volatile("" : "+v"(tid));  // what follows from it is computed for each block, not held in registers across them
    const int lane = tid % kWave;
    const PagedPiece w = walk.next(p, a);
    const int k0 = w.k0, k1 = w.k1;
    const int li = lane % 32, hf = lane / 32;
    const int wave_rows = min(w.rows - wave * kTile, kTile);  // below 1: a wave that only moves tiles
    const bool in = li < wave_rows;
    const int my_row = w.row0 + wave * kTile + max(0, min(li, wave_rows - 1));
    const int my_end = min(row_end(p, w.seq, min(my_row, w.row0 + w.rows - 1)), k1);
    const int wave_end = wave_rows > 0 ? min(k1, row_end(p, w.seq, w.row0 + wave * kTile + wave_rows - 1)) : k0;
    const auto q_row = [&](int row) { return p.q + paged_row(p, p.ld_q, w.seq.first, w.head, row); };
    // Row of the block: its output, or where its sums are kept.
    const auto out_row = [&](int row) {
        return w.whole ? p.out + paged_row(p, p.ld_out, w.seq.first, w.head, w.row0 + row)
                       : paged_part(a, p.c.head_dim, walk.index, w.begins, row) + 2;
    };

    // This lane's query values, times scale * log2(e).
    Split8 q[kC];
    {
        const float* row = q_row(min(my_row, w.row0 + w.rows - 1));
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = 16 * c + 8 * hf + e;
                x[e] = d < p.c.head_dim ? row[d] * p.qscale : 0.f;
            }
            q[c] = split8(x);
        }
    }

    // Tiles in, one item (eight dimensions of a key) at a time.
    const int tiles = (k1 - k0 + kTile - 1) / kTile;
    const scalar_i32 table = (scalar_i32)(p.b.page_table + w.s * p.b.ld_pages);
    const int row_bytes = p.c.stride * kElement;
    struct Pages {
        int page[2], slot[2];
    };
    const auto find = [&](int t) {
        Pages g;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = k0 + t * kTile + kHalf * u, i = max(min(j, (k1 - 1) & -kHalf), 0);
            const uint32_t entry = fastdiv(static_cast<uint32_t>(i), p.c.page_div);
            const int page = j < k1 ? table[entry] : -1;
            g.page[u] = page < p.c.pages ? page : -1;
            g.slot[u] = i - static_cast<int>(entry) * p.c.page_size;
        }
        return g;
    };
    const auto cache_row = [&](const Pages& g, int u) {
        return (static_cast<int64_t>(max(g.page[u], 0)) * p.c.kv_heads + w.head) * p.c.page_size + g.slot[u];
    };
    RowItem<DT> ki[kItems], vi[kItems];
    float scale = 0.f;
    const auto load = [&](int t, const Pages& g) {
        const int64_t r0 = cache_row(g, 0), r1 = cache_row(g, 1);
#pragma unroll
        for (int n = 0; n < kItems; ++n) {
            const int id = tid + n * kThreads, row = id / (DP / 8), d = 8 * (id % (DP / 8));
            if (row >= kTile) continue;
            const int u = row / kHalf;
            const int64_t off = ((u ? r1 : r0) + row % kHalf) * row_bytes + min(d, p.c.stride - 8) * kElement;
            ki[n].load(p.c.k + off);
            vi[n].load(p.c.v + off);
            // Dimensions past the row, and values of keys that are not there.
            if (d >= p.c.stride) ki[n].clear();
            if (d >= p.c.stride || k0 + t * kTile + row >= k1 || (u ? g.page[1] : g.page[0]) < 0) vi[n].clear();
        }
        if constexpr (DT == MIMIR_KV_I8) {
            if (tid < 2 * kTile) {
                const int row = tid % kTile, u = row / kHalf;
                const int64_t at = (u ? r1 : r0) + row % kHalf;
                scale = (tid < kTile ? p.c.k_scale : p.c.v_scale)[at];
                if (k0 + t * kTile + row >= k1 || (u ? g.page[1] : g.page[0]) < 0) scale = 0.f;
            }
        }
    };
    const auto stash = [&](char* buf) {
#pragma unroll
        for (int n = 0; n < kItems; ++n) {
            const int id = tid + n * kThreads, row = id / (DP / 8), at = 16 * (id % (DP / 8));
            if (row >= kTile) continue;
            ki[n].stash(buf + row * Tile::kKeyRow + at, Tile::kKeyPlane);
            vi[n].stash(buf + Tile::kValuesAt + row * Tile::kValueRow + at, Tile::kValuePlane);
        }
        if constexpr (DT == MIMIR_KV_I8)
            if (tid < 2 * kTile) reinterpret_cast<float*>(buf + Tile::kScalesAt)[tid] = scale;
    };

    f16v o[kDb];
#pragma unroll
    for (int d = 0; d < kDb; ++d) o[d] = f16v{};
    float m_run = -1e30f, l_run = 0.f;

    Pages g0{}, g1{}, g2{};  // of the tile in LDS, the one in registers, the next
    if (tiles > 0) {
        g0 = find(0);
        load(0, g0);
        g1 = find(1);
        stash(lds);
        load(1, g1);
        g2 = find(2);
    }
    __syncthreads();
    // A lane's part of a transposed read: key 4 hf + (lane % 16) / 4, dimensions
    // 16 (lane / 16 % 2) + 4 (lane % 4) on.
    const int v_lane = (4 * hf + lane % 16 / 4) * Tile::kValueRow + (lane / 16 % 2 * 16 + 4 * (lane % 4)) * 2;
    for (int t = 0; t < tiles; ++t) {
        const char* cur = lds + (t & 1) * Tile::kBytes;
        char* const next = lds + ((t + 1) & 1) * Tile::kBytes;
        const int key = k0 + t * kTile;
        if (key < wave_end) {
            f16v s = f16v{};
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                u4 k[Tile::kPlanes];
#pragma unroll
                for (int n = 0; n < Tile::kPlanes; ++n)
                    k[n] = *reinterpret_cast<const u4*>(cur + n * Tile::kKeyPlane + li * Tile::kKeyRow + 32 * c + 16 * hf);
                s = mfma_planes<Tile::kPlanes>(k, q[c], s);
            }
            // Past the last tile the stash rewrites a buffer that is not read again.
            stash(next);
            __builtin_amdgcn_s_setprio(0);
            load(t + 2, g2);
            if constexpr (DT == MIMIR_KV_I8) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f4 x = *reinterpret_cast<const f4*>(cur + Tile::kScalesAt + (2 * r + 4 * hf) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r + e] *= x[e];
                }
            }
            if (g0.page[0] < 0 || g0.page[1] < 0 || __any(key + kTile > my_end)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = key + 8 * (r / 4) + 4 * hf + r % 4;
                    s[r] = j < my_end && g0.page[r / 8] >= 0 ? s[r] : -INFINITY;
                }
            }
            float top = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
            if (__any(top > m_run + kPagedSlack)) {
                const float m_new = fmaxf(m_run, fmaxf(top, __shfl_xor(top, 32)));
                const float f = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= f;
#pragma unroll
                for (int d = 0; d < kDb; ++d) o[d] *= f;
            }
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_amdgcn_exp2f(s[r] - m_run);
                sum += s[r];
            }
            l_run += sum;
            if constexpr (DT == MIMIR_KV_I8) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f4 x = *reinterpret_cast<const f4*>(cur + Tile::kScalesAt + (kTile + 2 * r + 4 * hf) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r + e] *= x[e];
                }
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[8 * c + e];
                const Split8 pw = split8(x);
#pragma unroll
                for (int d = 0; d < kDb; ++d) {
                    u4 v[Tile::kPlanes];
#pragma unroll
                    for (int n = 0; n < Tile::kPlanes; ++n) {
                        const char* at = cur + Tile::kValuesAt + n * Tile::kValuePlane + v_lane + 16 * c * Tile::kValueRow + 64 * d;
                        const u2 x0 = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at));
                        const u2 x1 = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + 8 * Tile::kValueRow)));
                        v[n] = u4{x0[0], x0[1], x1[0], x1[1]};
                    }
                    o[d] = mfma_planes<Tile::kPlanes>(v, pw, o[d]);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        } else {
            stash(next);
            load(t + 2, g2);
        }
        g0 = g1;
        g1 = g2;
        g2 = find(t + 3);
        __syncthreads();
    }

    // The wave's rows out: lane (li, hf) holds dimensions 32 d + 8 (r / 4) + 4 hf + r % 4.
    if (wave_rows <= 0) continue;
    const float l_tot = l_run + __shfl_xor(l_run, 32);
    const int row = my_row - w.row0, d_all = p.c.head_dim;
    float* const out = out_row(row);
    const float inv = w.whole ? 1.0f / (l_tot + 1e-9f) : 1.0f;
    const bool vec = w.whole && d_all % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.ld_out % 4 == 0;
    float check = l_tot - l_tot;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d0 = 32 * d + 8 * (r / 4) + 4 * hf;
            const f4 x{o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv};
#pragma unroll
            for (int e = 0; e < 4; ++e) check += x[e] - x[e];
            if (!in) continue;
            if (vec) {
                if (d0 < d_all) *reinterpret_cast<f4*>(out + d0) = x;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d0 + e < d_all) out[d0 + e] = x[e];
            }
        }
    if (!w.whole && in && hf == 0) {
        out[-2] = m_run;
        out[-1] = l_tot;
    }
    // Rows that came out NaN or infinite, again in fp32 (as paged_stream).
    const uint64_t ballot = __ballot(check != check && in);
    for (uint32_t bad = static_cast<uint32_t>(ballot | ballot >> 32); bad; bad &= bad - 1) {
        const int r = wave * kTile + __builtin_ctz(bad), full = w.row0 + r;
        float acc[kRowChunks], m, l;
        row_over_keys<DT>(p, w.s, w.head, q_row(full), k0, min(k1, row_end(p, w.seq, full)), acc, &m, &l);
        float* const to = out_row(r);
        const float f = w.whole ? 1.0f / (l + 1e-9f) : 1.0f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c)
            if (lane + c * kWave < d_all) to[lane + c * kWave] = acc[c] * f;
        if (!w.whole && lane == 0) {
            to[-2] = m;
            to[-1] = l;
        }
    }
    }
}

template <int DT, int DP, int WAVES>
int launch(mimir_ctx* ctx, const PagedArgs& p, PagedRuns a) {
    a.block_rows = a.part_rows = WAVES * kTile;
    const int64_t rows = static_cast<int64_t>(p.b.max_new) * p.group;
    const int64_t blocks = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads * ((rows + a.block_rows - 1) / a.block_rows);
    const int64_t runs = ctx->tune.attn_splits > 0 ? ctx->tune.attn_splits : 2048 / WAVES;
    const int64_t grid = paged_runs(ctx, p, &a, runs, blocks, true);
    MIMIR_REQUIRE(ctx, dispatch_fits(grid, WAVES * kWave), "paged attention: grid of %lld workgroups exceeds the limit",
                  (long long)grid);
    paged_block<DT, DP, WAVES><<<static_cast<unsigned>(grid), WAVES * kWave, 0, ctx->stream>>>(p, a);
    if (int st = launched(ctx, "paged_block")) return st;
    return paged_join_launch(ctx, p, a);
}

template <int DT, int DP>
int launch_waves(mimir_ctx* ctx, const PagedArgs& p, const PagedRuns& a) {
    int waves = static_cast<int64_t>(p.b.max_new) * p.group <= 4 * kTile ? 4 : 8;
    if (ctx->tune.attn_waves == 4 || ctx->tune.attn_waves == 8) waves = ctx->tune.attn_waves;
    return waves == 4 ? launch<DT, DP, 4>(ctx, p, a) : launch<DT, DP, 8>(ctx, p, a);
}

template <int DT>
int launch_dim(mimir_ctx* ctx, const PagedArgs& p, const PagedRuns& a) {
    if (p.c.stride <= 64) return launch_waves<DT, 64>(ctx, p, a);
    if (p.c.stride <= 96) return launch_waves<DT, 96>(ctx, p, a);
    return launch_waves<DT, 128>(ctx, p, a);
}

}  // namespace

int mimir::paged_block_launch(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t least_rows) {
    PagedRuns a{};
    a.extra = 4 * kTile;
    a.grain = kTile;
    a.least_rows = static_cast<int32_t>(least_rows);
    a.most_rows = INT32_MAX;
    if (dtype == MIMIR_KV_F32) return launch_dim<MIMIR_KV_F32>(ctx, p, a);
    if (dtype == MIMIR_KV_BF16) return launch_dim<MIMIR_KV_BF16>(ctx, p, a);
    return launch_dim<MIMIR_KV_I8>(ctx, p, a);
}
