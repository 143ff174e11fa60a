// attention_paged_block.hip -- attention over a paged cache for many query rows per
// key / value head (prompts, and chunks of them): tiles of 32 keys in LDS.
//
// A workgroup has 128 or 256 query rows, the tokens' heads that share a key / value
// head side by side, 32 a wave; every tile of keys and values is read from the cache
// and converted once for all of them.
// - Scores: S^T = K Q^T by v_mfma_f32_32x32x16_bf16 (split.hpp has the lanes' parts).
//   A lane's query row, 8 of 16 dimensions, is split into its three terms once and
//   stays in registers; the keys' planes come from LDS, 16 bytes a read.
// - Output: O^T = V^T P^T, the weights straight from the scores' registers.  Values
//   lie in LDS as in the cache, rows of dimensions, and are transposed as they are
//   read (ds_read_b64_tr_b16), in the order of keys that the scores come out in.
// - Tile t is computed while t + 1 goes from registers to LDS and t + 2 comes from
//   memory; one barrier a tile.
// - Heads over 128: a row's queries and sums would not fit one wave's registers, so two
//   waves (fp32: four) share 32 rows, a half (a quarter) of the dimensions each.  Their
//   scores meet in LDS, in one order for all, and each wave does the row's softmax.
//   Keys and values have one buffer each: a tile's values come in beside its scores'
//   products, the next one's keys after them; two barriers a tile.
// - Causal: a wave passes over tiles behind its last row's keys.  Rows' ends inside a
//   tile, and pages that are none, are looked at only where there are any.
//
// 512 tokens of one sequence over 8812 keys, 32 heads on 8 of 128, bf16, 201 to 212 us =
// 340 to 357 TFLOP/s of fp32 work, 1020 to 1070 of bf16 MFMAs, which are busy 46% of
// the cycles at 2.1 GHz beside 5.4 VALU operations each; a library product of 8192 x
// 8192 bf16 runs at 1390.  Prompts (4 of up to 2048, 16 heads): fp32 240 to 253 us, bf16
// 156, 8-bit 163; heads of 64 135, 101, 113.
// What the other half of the cycles goes to has not been taken apart.  In the built code
// each load of a tile stands in a loop over lanes (a descriptor's length, at most the keys
// of a half, is a vector value to the compiler), which cuts the tile's instructions into
// pieces that are not scheduled together; 167 to 212 scalar values are kept in vector
// registers' lanes, and 1 to 11 vector registers of the instances of 128 and 256
// dimensions (fp32: 96 and 128) in memory.
// Measured on the way: a lane's query row in loads of 4 bytes instead of 16 cost 12 us
// a block, page numbers looked at for each tile instead of once a block 6 us of 219,
// and waves that all multiply the values in the tile they were scored in 7% of the
// whole.  Two accumulators in turns for the scores: no change.  Heads of 256, 4 prompts of
// 1440 tokens, 8 heads, by streamed blocks of 16 (fp32) or 32 rows and by these: fp32 1243
// and 321 us, bf16 392 and 172, 8-bit 343 and 196; 512 tokens over 4512 keys, 16 heads on
// 4, fp32 995 and 280, bf16 235 and 131, 8-bit 159 and 149.
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
    static constexpr int kScalesAt = kPlanes * kKeyPlane;  // 8-bit: 32 of the keys, 32 of the values, beside the keys
    static constexpr int kKeyBytes = kScalesAt + (DT == MIMIR_KV_I8 ? 2 * kTile * 4 : 0);
    static constexpr int kValueBytes = kPlanes * kValuePlane;
};

// Eight elements of a row on their way from memory to LDS.
template <int DT>
struct RowItem {
    static constexpr int kVecs = DT == MIMIR_KV_F32 ? 2 : 1;
    u4 v[kVecs];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rows, uint32_t off) {
        if constexpr (DT == MIMIR_KV_I8) {
            const u2 x = __builtin_amdgcn_raw_buffer_load_b64(rows, off, 0, 0);
            v[0] = u4{x[0], x[1], 0, 0};
        } else {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(rows, off + 16 * i, 0, 0);
        }
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

// Value buffers of a workgroup, and workgroups of a CU: one of eight waves, or two of
// four where the tiles leave room.  (160 KiB of LDS; fp32 heads of 128: 113 KiB.)
template <int DT, int DP, int WAVES>
struct BlockShape {
    using Tile = BlockTile<DT, DP>;
    // Waves that share 32 rows, a part of the dimensions each: where a row's queries and
    // sums would not fit one's registers.
    static constexpr int kShare = DP == 256 ? (DT == MIMIR_KV_F32 ? 4 : 2) : 1;
    static constexpr int kDims = DP / kShare, kRows = WAVES / kShare * kTile;
    static constexpr int kValueBufs = WAVES == 8 ? 3 : 2;
    static constexpr int kParts = WAVES * kWave * 16 * 4;  // scores of the dimensions of each wave
    static constexpr int kBytes = kShare == 1 ? 2 * Tile::kKeyBytes + kValueBufs * Tile::kValueBytes
                                              : Tile::kKeyBytes + Tile::kValueBytes + kParts;
    static constexpr int kResident = WAVES == 8 || kBytes + sizeof(PagedChunk) > 80 * 1024 ? 1 : 2;
};

template <int DT, int DP, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, (WAVES / 4 * BlockShape<DT, DP, WAVES>::kResident)) void paged_block(PagedArgs p,
                                                                                                              PagedRuns a) {
    using Tile = BlockTile<DT, DP>;
    using Shape = BlockShape<DT, DP, WAVES>;
    constexpr int kThreads = WAVES * kWave, kC = Shape::kDims / 16, kDb = Shape::kDims / 32;
    constexpr bool kShared = Shape::kShare > 1;
    constexpr int kElement = DT == MIMIR_KV_F32 ? 4 : DT == MIMIR_KV_BF16 ? 2 : 1;
    // Eight waves: the second four, which share the SIMDs with the first, multiply a
    // tile's values one tile later, so that one's softmax runs beside the other's products;
    // the values stay that much longer.
    constexpr bool kStagger = WAVES == 8 && !kShared;
    __shared__ __attribute__((aligned(16))) char lds[Shape::kBytes];
    char* const values = lds + (kShared ? 1 : 2) * Tile::kKeyBytes;
    __shared__ PagedChunk chunk;
    __shared__ uint32_t bad[WAVES];  // shared: the rows that came out NaN or infinite of each wave

    // Each XCD takes runs that follow each other, whose keys it has in its L2.
    const bool dealt = a.runs % kXcds == 0 && gridDim.x == a.runs;
    const uint32_t at = dealt ? blockIdx.x % kXcds * (a.runs / kXcds) + blockIdx.x / kXcds : blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int group = wave / Shape::kShare, d_wave = wave % Shape::kShare * Shape::kDims;  // its rows, its dimensions
    for (PagedWalk walk(p, a, at, &chunk); walk.more();) {
        int tid = static_cast<int>(threadIdx.x);
        asm volatile("" : "+v"(tid));  // what follows from it is computed for each block, not held in registers across them
        const int lane = tid % kWave;
        const PagedPiece w = walk.next(p, a);
        if (w.rows <= 0) return;
        const int k0 = w.k0, k1 = w.k1;
        const int li = lane % 32, hf = lane / 32;
        const int wave_rows = min(w.rows - group * kTile, kTile);  // below 1: a wave that only moves tiles
        const bool in = li < wave_rows;
        const int my_row = w.row0 + group * kTile + max(0, min(li, wave_rows - 1));
        const int my_end = min(row_end(p, w.seq, min(my_row, w.row0 + w.rows - 1)), k1);
        const int first_end = uniform(my_end);  // the wave's first row's, none sees fewer
        const int wave_end = wave_rows > 0 ? min(k1, row_end(p, w.seq, w.row0 + group * kTile + wave_rows - 1)) : k0;
        const auto q_row = [&](int row) { return p.q + paged_row(p, p.ld_q, w.seq.first, w.head, row); };
        const PagedPart part(a, p.c.head_dim, walk.index, w.begins);
        // Row of the block: its output, or where its sums are kept.
        const auto out_row = [&](int row) {
            return w.whole ? p.out + paged_row(p, p.ld_out, w.seq.first, w.head, w.row0 + row)
                           : part.sums(row);
        };

        // Tiles in, one item (eight dimensions of a key) at a time.
        const int tiles = (k1 - k0 + kTile - 1) / kTile;
        const scalar_i32 table = (scalar_i32)(p.b.page_table + w.s * p.b.ld_pages);
        const int row_bytes = p.c.stride * kElement;
        const auto pages = static_cast<uint32_t>(p.c.pages);
        const auto there = [&](int j) {  // the half of a tile from key j on
            const auto i = static_cast<uint32_t>(max(min(j, (k1 - 1) & -kHalf), 0));
            return static_cast<uint32_t>(table[fastdiv(i, p.c.page_div)]) < pages;
        };
        // Whether a page of these keys is none.
        bool holes = false;
        if (tiles > 0) {
            const int32_t* entries = p.b.page_table + w.s * p.b.ld_pages;
            const auto last = static_cast<int>(fastdiv(static_cast<uint32_t>(k1 - 1), p.c.page_div));
            for (int e = static_cast<int>(fastdiv(static_cast<uint32_t>(k0), p.c.page_div)) + lane; e <= last; e += kWave)
                holes = holes || static_cast<uint32_t>(entries[e]) >= pages;
            holes = __any(holes);
        }
        // A thread's items: eight dimensions of a row.  An item's rows are, for a wave, of
        // one half of the tile; what lies past a row's dimensions or the half's keys reads
        // as zeros.
        constexpr int kLanes = DP == 64 ? 8 : DP == 256 ? 32 : 16;
        constexpr int kItems = (kTile * kLanes + kThreads - 1) / kThreads;
        static_assert(kWave / kLanes <= kHalf && kHalf % (kWave / kLanes) == 0, "a wave's rows in one half");
        static_assert(kItems == 1 || (kItems == 2 && kThreads == kHalf * kLanes), "an item a half");
        constexpr int kMovers = kItems == 2 ? WAVES : kHalf * kLanes / kWave;  // waves that share a half
        const int d_mine = 8 * (tid % kLanes);
        const auto row_of = [&](int n) { return (tid + n * kThreads) / kLanes; };
        const auto half_of = [&](int n) { return kItems == 2 ? n : wave / kMovers; };
        const auto mine = static_cast<uint32_t>(row_of(0) % kHalf * row_bytes + d_mine * kElement);
        const uint32_t off = d_mine < p.c.stride ? mine : kOutside;
        const int64_t head_rows = static_cast<int64_t>(w.head) * p.c.page_size;
        const int64_t page_rows = static_cast<int64_t>(p.c.kv_heads) * p.c.page_size;
        const bool mover = kItems == 2 || half_of(0) < 2;
        // Where an item's half stands, and how many of its keys are there.
        struct Halves {
            int page[kItems], slot[kItems], keys[kItems];
        };
        const auto find = [&](int t) {
            Halves g;
#pragma unroll
            for (int n = 0; n < kItems; ++n) {
                const int j = k0 + t * kTile + kHalf * half_of(n), i = max(min(j, (k1 - 1) & -kHalf), 0);
                const uint32_t entry = fastdiv(static_cast<uint32_t>(i), p.c.page_div);
                g.page[n] = table[entry];
                g.slot[n] = i - static_cast<int>(entry) * p.c.page_size;
                g.keys[n] = max(min(k1 - j, kHalf), 0);
            }
            return g;
        };
        RowItem<DT> ki[kItems], vi[kItems];
        float scale[kItems];
        const int scales = wave % kMovers;  // 8-bit: 0, the keys' scales are this wave's to move, 1, the values'
        const auto load = [&](const Halves& g, bool keys_too, bool values_too) {
            if (!mover) return;
#pragma unroll
            for (int n = 0; n < kItems; ++n) {
                const bool has = static_cast<uint32_t>(g.page[n]) < pages;
                const int64_t row = (has ? g.page[n] : 0) * page_rows + head_rows + g.slot[n];
                const int keys = has ? g.keys[n] : 0;
                const int64_t at = row * row_bytes;
                if (keys_too) ki[n].load(__builtin_amdgcn_make_buffer_rsrc(p.c.k + at, 0, keys * row_bytes, kBufferWord3), off);
                if (values_too) vi[n].load(__builtin_amdgcn_make_buffer_rsrc(p.c.v + at, 0, keys * row_bytes, kBufferWord3), off);
                if constexpr (DT == MIMIR_KV_I8)
                    if (scales < 2 && (scales ? values_too : keys_too))
                        scale[n] = buffer_f1(buffer_of((scales ? p.c.v_scale : p.c.k_scale) + row, 4 * keys),
                                             static_cast<uint32_t>(4 * (lane % kHalf)));
            }
        };
        // Both kinds' scales stand beside the keys.
        const auto stash = [&](char* key_buf, char* value_buf, bool keys_too, bool values_too) {
            if (!mover) return;
#pragma unroll
            for (int n = 0; n < kItems; ++n) {
                if (d_mine < DP) {
                    if (keys_too) ki[n].stash(key_buf + row_of(n) * Tile::kKeyRow + 2 * d_mine, Tile::kKeyPlane);
                    if (values_too) vi[n].stash(value_buf + row_of(n) * Tile::kValueRow + 2 * d_mine, Tile::kValuePlane);
                }
                if constexpr (DT == MIMIR_KV_I8)
                    if (scales < 2 && (scales ? values_too : keys_too) && lane < kHalf)
                        reinterpret_cast<float*>(key_buf + Tile::kScalesAt)[scales * kTile + half_of(n) * kHalf + lane] = scale[n];
            }
        };

        Halves to{};  // of the tile after the one in registers, which is after the one in LDS
        if (tiles > 0) {
            load(find(0), true, true);
            to = find(1);
        }
        // This lane's query values, times scale * log2(e).
        Split8 q[kC];
        {
            const float* row = q_row(min(my_row, w.row0 + w.rows - 1)) + d_wave + 8 * hf;
            const int left = p.c.head_dim - d_wave - 8 * hf;  // of the row from there on
            if (p.c.head_dim % 4 == 0) {
                f4u x[kC][2];
#pragma unroll
                for (int c = 0; c < kC; ++c)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        x[c][i] = 16 * c + 4 * i < left ? reinterpret_cast<const f4u*>(row + 16 * c)[i] : f4u{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const f4u a = x[c][0] * p.qscale, b = x[c][1] * p.qscale;
                    const float y[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
                    q[c] = split8(y);
                }
            } else {
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = 16 * c + e < left ? row[16 * c + e] * p.qscale : 0.f;
                    q[c] = split8(x);
                }
            }
        }

        f16v o[kDb];
#pragma unroll
        for (int d = 0; d < kDb; ++d) o[d] = f16v{};
        float m_run = -1e30f, l_run = 0.f;

        Halves later{};  // shared: the values follow a tile behind the keys
        if (tiles > 0) {
            stash(lds, values, true, !kShared);
            load(to, true, !kShared);
            later = to;
            to = find(2);
        }
        __syncthreads();
        // A lane's part of a transposed read: key 4 hf + (lane % 16) / 4, dimensions
        // 16 (lane / 16 % 2) + 4 (lane % 4) on.
        const int v_lane = (4 * hf + lane % 16 / 4) * Tile::kValueRow + (d_wave + lane / 16 % 2 * 16 + 4 * (lane % 4)) * 2;
        f16v s;  // scores of a tile, then its weights
        // o += V^T P^T over a tile's keys.  Values are read one operand ahead of their
        // products, and the second half's weights are split beside the first half's.
        const auto weigh = [&](const char* buf) {
            const auto read = [&](int i, u4* v) {
                const char* const at = buf + v_lane + 16 * (i / kDb) * Tile::kValueRow + 64 * (i % kDb);
#pragma unroll
                for (int n = 0; n < Tile::kPlanes; ++n) {
                    const u2 x0 = __builtin_bit_cast(
                        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + n * Tile::kValuePlane)));
                    const u2 x1 = __builtin_bit_cast(
                        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + n * Tile::kValuePlane + 8 * Tile::kValueRow)));
                    v[n] = u4{x0[0], x0[1], x1[0], x1[1]};
                }
            };
            const auto split = [&](int c) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[8 * c + e];
                return split8(x);
            };
            __builtin_amdgcn_s_setprio(1);
            u4 v[2][Tile::kPlanes];
            read(0, v[0]);
            Split8 pw = split(0), pn;
#pragma unroll
            for (int i = 0; i < 2 * kDb; ++i) {
                if (i + 1 < 2 * kDb) read(i + 1, v[(i + 1) % 2]);
                if (i == 0) pn = split(1);
                if (i == kDb) pw = pn;
                o[i % kDb] = mfma_planes<Tile::kPlanes>(v[i % 2], pw, o[i % kDb]);
            }
            if constexpr (Tile::kPlanes == 1) {
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 44, 0);
#pragma unroll
                for (int i = 0; i < 2 * kDb; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
                    for (int n = 0; n < 3; ++n) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        if (i < kDb) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                    }
                }
            }
            __builtin_amdgcn_s_setprio(0);
        };
        // S^T = K Q^T over the wave's dimensions, 8-bit: times the keys' scales.
        const auto scores = [&](const char* cur) {
            const auto read = [&](int c, u4* k) {
#pragma unroll
                for (int n = 0; n < Tile::kPlanes; ++n)
                    k[n] = *reinterpret_cast<const u4*>(cur + n * Tile::kKeyPlane + li * Tile::kKeyRow + 2 * d_wave + 32 * c +
                                                        16 * hf);
            };
            s = f16v{};
            __builtin_amdgcn_s_setprio(1);
            u4 k[2][Tile::kPlanes];
            read(0, k[0]);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                if (c + 1 < kC) read(c + 1, k[(c + 1) % 2]);
                s = mfma_planes<Tile::kPlanes>(k[c % 2], q[c], s);
            }
            if constexpr (Tile::kPlanes == 1) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        };
        const auto scaled = [&](const char* of) {  // the keys' or the values' scales
            if constexpr (DT == MIMIR_KV_I8) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f4 x = *reinterpret_cast<const f4*>(of + (2 * r + 4 * hf) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r + e] *= x[e];
                }
            }
        };
        // Scores of the tile from `key` on to weights.
        const auto soften = [&](int key, const char* cur) {
            if (holes || key + kTile > first_end) {
                const bool first = !holes || there(key), second = !holes || there(key + kHalf);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = key + 8 * (r / 4) + 4 * hf + r % 4;
                    s[r] = j < my_end && (r < 8 ? first : second) ? s[r] : -INFINITY;
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
            scaled(cur + Tile::kScalesAt + kTile * 4);
        };
        if constexpr (kShared) {
            // One buffer each: a tile's values come in beside its scores' products, the next
            // tile's keys when all waves have those.
            f4* const parts = reinterpret_cast<f4*>(values + Tile::kValueBytes);  // [wave][four scores][lane]
            for (int t = 0; t < tiles; ++t) {
                const int key = k0 + t * kTile;
                const bool active = key < wave_end;
                stash(lds, values, false, true);
                load(later, false, true);
                if (active) {
                    scores(lds);
                    scaled(lds + Tile::kScalesAt);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        parts[(4 * wave + r) * kWave + lane] = f4{s[4 * r], s[4 * r + 1], s[4 * r + 2], s[4 * r + 3]};
                }
                __syncthreads();
                stash(lds, values, true, false);
                load(to, true, false);
                if (active) {
                    s = f16v{};
#pragma unroll
                    for (int g = 0; g < Shape::kShare; ++g)  // in one order for all
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const f4 x = parts[(4 * (group * Shape::kShare + g) + r) * kWave + lane];
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[4 * r + e] += x[e];
                        }
                    soften(key, lds);
                    weigh(values);
                }
                later = to;
                to = find(t + 3);
                __syncthreads();
            }
        } else {
            const bool late = kStagger && wave >= WAVES / 2;
            char *v_old = values, *v_cur = values, *v_next = values + Tile::kValueBytes;
            for (int t = 0; t < tiles + (kStagger ? 1 : 0); ++t) {
                const char* cur = lds + (t & 1) * Tile::kKeyBytes;
                char* const next = lds + ((t + 1) & 1) * Tile::kKeyBytes;
                const int key = k0 + t * kTile;
                if (kStagger && late && t > 0 && key - kTile < wave_end) weigh(v_old);
                const bool active = key < wave_end;
                if (active) scores(cur);
                if (t < tiles) {  // past the last tile the stash rewrites buffers that are not read again
                    stash(next, v_next, true, true);
                    load(to, true, true);
                }
                if (active) {
                    scaled(cur + Tile::kScalesAt);
                    soften(key, cur);
                    if (!late) weigh(v_cur);
                }
                // Not in the late waves' turn: it is a block's first where there are no keys, whose
                // sequence may have no page table.
                if (t < tiles) to = find(t + 3);
                char* const v_free = kStagger ? v_old : v_cur;
                v_old = v_cur;
                v_cur = v_next;
                v_next = kStagger && t == 0 ? values + 2 * Tile::kValueBytes : v_free;
                __syncthreads();
            }
        }

        // The wave's rows out: lane (li, hf) holds dimensions 32 d + 8 (r / 4) + 4 hf + r % 4 of its own.
        if (!kShared && wave_rows <= 0) continue;
        const float l_tot = l_run + __shfl_xor(l_run, 32);
        const int row = my_row - w.row0, d_all = p.c.head_dim;
        float* const out = out_row(row);
        const float inv = w.whole ? 1.0f / (l_tot + 1e-9f) : 1.0f;
        const bool vec = d_all % 4 == 0 && (!w.whole || ((reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.ld_out % 4 == 0));
        float check = l_tot - l_tot;
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d0 = d_wave + 32 * d + 8 * (r / 4) + 4 * hf;
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
        if (!w.whole && in && hf == 0 && d_wave == 0) *part.stat(row) = f2{m_run, l_tot};
        // Rows that came out NaN or infinite, again in fp32 (as paged_stream).
        const uint64_t ballot = __ballot(check != check && in);
        auto again = static_cast<uint32_t>(ballot | ballot >> 32);
        if constexpr (kShared) {  // by the first of the waves, when all have written theirs
            if (lane == 0) bad[wave] = again;
            __syncthreads();
            if (d_wave > 0) continue;
#pragma unroll
            for (int g = 1; g < Shape::kShare; ++g) again |= uniform(bad[wave + g]);
        }
        for (; again; again &= again - 1) {
            const int r = group * kTile + __builtin_ctz(again), full = w.row0 + r;
            float acc[kRowChunks], m, l;
            row_over_keys<DT>(p, w.s, w.head, q_row(full), k0, min(k1, row_end(p, w.seq, full)), acc, &m, &l);
            float* const to = out_row(r);
            const float f = w.whole ? 1.0f / (l + 1e-9f) : 1.0f;
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c)
                if (lane + c * kWave < d_all) to[lane + c * kWave] = acc[c] * f;
            if (!w.whole && lane == 0) *part.stat(r) = f2{m, l};
        }
    }
}

template <int DT, int DP, int WAVES>
int launch(mimir_ctx* ctx, const PagedArgs& p, PagedRuns a, PagedRuns* left) {
    a.block_rows = a.part_rows = BlockShape<DT, DP, WAVES>::kRows;
    const int64_t rows = static_cast<int64_t>(p.b.max_new) * p.group;
    a.row_blocks = static_cast<int32_t>((rows + a.block_rows - 1) / a.block_rows);
    const int64_t blocks = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads * a.row_blocks;
    const int64_t runs = ctx->tune.paged_runs > 0 ? ctx->tune.paged_runs : 256 * BlockShape<DT, DP, WAVES>::kResident;
    const int64_t grid = paged_runs(ctx, p, &a, runs, blocks, WAVES * kWave, p.b.max_len > kWholeLen, false);
    MIMIR_REQUIRE(ctx, dispatch_fits(grid, WAVES * kWave), "paged attention: grid of %lld workgroups exceeds the limit",
                  (long long)grid);
    paged_block<DT, DP, WAVES><<<static_cast<unsigned>(grid), WAVES * kWave, 0, ctx->stream>>>(p, a);
    *left = a;
    return launched(ctx, "paged_block");
}

template <int DT, int DP>
int launch_waves(mimir_ctx* ctx, const PagedArgs& p, const PagedRuns& a, PagedRuns* left) {
    // Four for few rows and for short contexts; where a compute unit holds but one of four,
    // only if those are one round (fp32 heads of 128, four / eight: one prompt of 250 tokens
    // 38 / 44 us, 30 of up to 100 58 / 44).
    const int64_t rows = static_cast<int64_t>(p.b.max_new) * p.group;
    const int64_t blocks = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads * ((rows + 4 * kTile - 1) / (4 * kTile));
    int waves = rows <= 4 * kTile || (p.b.max_len <= kWholeLen && (BlockShape<DT, DP, 4>::kResident == 2 || blocks <= 256)) ? 4 : 8;
    if (ctx->tune.attn_waves == 4 || ctx->tune.attn_waves == 8) waves = ctx->tune.attn_waves;
    return waves == 4 ? launch<DT, DP, 4>(ctx, p, a, left) : launch<DT, DP, 8>(ctx, p, a, left);
}

template <int DT>
int launch_dim(mimir_ctx* ctx, const PagedArgs& p, const PagedRuns& a, PagedRuns* left) {
    if (p.c.stride <= 64) return launch_waves<DT, 64>(ctx, p, a, left);
    if (p.c.stride <= 96) return launch_waves<DT, 96>(ctx, p, a, left);
    if (p.c.stride <= 128) return launch_waves<DT, 128>(ctx, p, a, left);
    return launch<DT, 256, 8>(ctx, p, a, left);
}

}  // namespace

int mimir::paged_block_launch(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t least_rows, PagedRuns* left) {
    PagedRuns a{};
    a.extra = 4 * kTile;
    a.least = 5 * kTile;
    a.slack = 8 * kTile;
    a.grain = kTile;
    a.least_rows = static_cast<int32_t>(least_rows);
    a.most_rows = INT32_MAX;
    if (dtype == MIMIR_KV_F32) return launch_dim<MIMIR_KV_F32>(ctx, p, a, left);
    if (dtype == MIMIR_KV_BF16) return launch_dim<MIMIR_KV_BF16>(ctx, p, a, left);
    return launch_dim<MIMIR_KV_I8>(ctx, p, a, left);
}
