// attention_paged.hip -- attention of new tokens over a paged cache of keys and
// values (mimir_hip.h mimir_attention_paged_fwd): softmax(Q K^T * scale) V with the
// softmax fused between the products, as attention.hip, for sequences of different
// lengths whose queries share key / value heads.
#include "kvcache.hpp"
#include "split.hpp"

#include <math.h>

#include <algorithm>
#include <cmath>

using namespace mimir;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
    KvView c;
    KvBatch b;
    const float* q;
    float* out;
    int64_t ld_q, ld_out;
    int32_t heads, group;  // query heads, those that share a key / value head
    float qscale;          // scale * log2(e)
    int32_t causal;
};

// Element d of a cache row (index `at` among the rows of the type's buffer).
template <int DT>
__device__ __forceinline__ float element(const char* base, int64_t at, int stride, int d) {
    const int64_t i = at * stride + d;
    if constexpr (DT == MIMIR_KV_F32) return reinterpret_cast<const float*>(base)[i];
    else if constexpr (DT == MIMIR_KV_BF16)
        return __builtin_bit_cast(float, static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(base)[i]) << 16);
    else return static_cast<float>(reinterpret_cast<const int8_t*>(base)[i]);
}

constexpr int kRowChunks = kKvMaxDim / kWave;

// One query row over keys j0 .. j1 - 1 by one wave, lane l holding dimensions l + 64 c.
// Leaves the sums (without the division) and the running max (base-2 units) and sum.
template <int DT>
__device__ __forceinline__ void row_over_keys(const PagedArgs& a, int s, int kv_head, const float* q, int j0, int j1,
                                              float* acc, float* m_out, float* l_out) {
    const int lane = threadIdx.x % kWave;
    float x[kRowChunks];
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
        const int d = lane + c * kWave;
        x[c] = d < a.c.head_dim ? q[d] * a.qscale : 0.f;
        acc[c] = 0.f;
    }
    float m = -1e30f, l = 0.f;
    for (int j = j0; j < j1; ++j) {
        const auto [page, slot] = kv_slot(a.b, a.c.pages, a.c.page_div, s, j);
        if (page < 0) continue;
        const int64_t at = (static_cast<int64_t>(page) * a.c.kv_heads + kv_head) * a.c.page_size + slot;
        float part = 0.f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) {
            const int d = lane + c * kWave;
            if (d < a.c.head_dim) part += x[c] * element<DT>(a.c.k, at, a.c.stride, d);
        }
        float score = wave_sum(part);
        if constexpr (DT == MIMIR_KV_I8) score *= a.c.k_scale[at];
        const float m_new = fmaxf(m, score);
        const float alpha = __builtin_amdgcn_exp2f(m - m_new);
        const float p = __builtin_amdgcn_exp2f(score - m_new);
        m = m_new;
        l = l * alpha + p;
        const float w = DT == MIMIR_KV_I8 ? p * a.c.v_scale[at] : p;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) {
            const int d = lane + c * kWave;
            if (d < a.c.head_dim) acc[c] = acc[c] * alpha + w * element<DT>(a.c.v, at, a.c.stride, d);
        }
    }
    *m_out = m;
    *l_out = l;
}

// ---------------------------------------------------------------------------
// Few query rows per key / value head: keys and values straight to registers
// ---------------------------------------------------------------------------

typedef float f4r __attribute__((ext_vector_type(4)));

// Memory that a kernel only reads, at addresses that a wave shares.
typedef const __attribute__((address_space(4))) int32_t* scalar_i32;

constexpr int kRows = 16;     // query rows of a tile: (token, head of the group) pairs
constexpr int kHalf = 16;     // keys that stand in one page
constexpr int kNt = 2;        // a buffer load's non-temporal bit
constexpr int kStreamWaves = 4;
constexpr float kMaxSlack = 8.0f;  // as attention.hip: the running max may lag by this many base-2 units

__device__ __forceinline__ f4r mfma16(u4 a, u4 b, f4r c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// c += a b, b a split (split.hpp), a exact in bf16 or a split itself: the small terms first.
__device__ __forceinline__ f4r mfma16_split(u4 a, const Split8& b, f4r c) {
    c = mfma16(a, b.l, c);
    c = mfma16(a, b.m, c);
    return mfma16(a, b.h, c);
}
__device__ __forceinline__ f4r mfma16_split(const Split8& a, const Split8& b, f4r c) {
    c = mfma16(a.l, b.h, c);
    c = mfma16(a.h, b.l, c);
    c = mfma16(a.m, b.m, c);
    c = mfma16(a.m, b.h, c);
    c = mfma16(a.h, b.m, c);
    return mfma16(a.h, b.h, c);
}

// The two's complement bytes of a dword as floats, and pairs of small whole numbers
// (exact in bf16, so their floats' upper halves) packed.
__device__ __forceinline__ float byte_float(uint32_t w, int i) {
    return static_cast<float>(static_cast<int32_t>(w << (24 - 8 * i)) >> 24);
}
__device__ __forceinline__ uint32_t pack_high(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ u4 bytes_bf16(uint32_t lo, uint32_t hi) {
    u4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        r[i] = pack_high(byte_float(lo, 2 * i), byte_float(lo, 2 * i + 1));
        r[2 + i] = pack_high(byte_float(hi, 2 * i), byte_float(hi, 2 * i + 1));
    }
    return r;
}

// How a type's K rows feed the scores.  A lane (key li, slot group hg) takes 16-byte
// vectors, the four groups of a key side by side; step c is a product over 32
// dimensions, of which slot e of group hg is dim(c, hg, e).
template <int DT, int DP>
struct Kind;

template <int DP>
struct Kind<MIMIR_KV_F32, DP> {
    static constexpr int kHalves = 2;  // of a step
    static constexpr int kBytes = 4, kVecs = DP / 16;  // K vectors of a lane per half
    typedef Split8 Operand;
    static __device__ __forceinline__ int first(int v, int hg) { return 16 * v + 4 * hg; }
    static __device__ __forceinline__ int dim(int c, int hg, int e) { return 32 * c + 16 * (e / 4) + 4 * hg + e % 4; }
    static __device__ __forceinline__ Operand operand(const u4* raw, int c) {
        const f4 a = __builtin_bit_cast(f4, raw[2 * c]), b = __builtin_bit_cast(f4, raw[2 * c + 1]);
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return split8(x);
    }
};
template <int DP>
struct Kind<MIMIR_KV_BF16, DP> {
    static constexpr int kHalves = 2;  // of a step
    static constexpr int kBytes = 2, kVecs = DP / 32;
    typedef u4 Operand;
    static __device__ __forceinline__ int first(int v, int hg) { return 32 * v + 8 * hg; }
    static __device__ __forceinline__ int dim(int c, int hg, int e) { return 32 * c + 8 * hg + e; }
    static __device__ __forceinline__ Operand operand(const u4* raw, int c) { return raw[c]; }
};
template <int DP>
struct Kind<MIMIR_KV_I8, DP> {
    static constexpr int kHalves = 2;  // of a step
    static constexpr int kBytes = 1, kVecs = DP / 64;
    typedef u4 Operand;
    static __device__ __forceinline__ int first(int v, int hg) { return 64 * v + 16 * hg; }
    static __device__ __forceinline__ int dim(int c, int hg, int e) { return 64 * (c / 2) + 16 * hg + 8 * (c % 2) + e; }
    static __device__ __forceinline__ Operand operand(const u4* raw, int c) {
        return bytes_bf16(raw[c / 2][2 * (c % 2)], raw[c / 2][2 * (c % 2) + 1]);
    }
};

// A lane's share of the values of 32 keys: ND dimensions (its li-th run of them) of
// the keys 4 hg + {0..3} of both halves, raw; and the operand of output tile t, whose
// row li is dimension li * ND + t.
template <int DT, int ND>
struct Values {
    static constexpr int kBytes = DT == MIMIR_KV_F32 ? 4 : DT == MIMIR_KV_BF16 ? 2 : 1;
    static constexpr int kWords = ND * kBytes / 4;
    uint32_t w[8][kWords];
    __device__ __forceinline__ void load(int key, __amdgpu_buffer_rsrc_t rows, uint32_t off, uint32_t row) {
        if constexpr (kWords % 4 == 0) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const u4 x = __builtin_amdgcn_raw_buffer_load_b128(rows, off + 16 * i, row, kNt);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[key][4 * i + e] = x[e];
            }
        } else if constexpr (kWords == 2) {
            const u2 x = __builtin_amdgcn_raw_buffer_load_b64(rows, off, row, kNt);
            w[key][0] = x[0];
            w[key][1] = x[1];
        } else {
            static_assert(kWords == 1, "one word, two or whole vectors");
            w[key][0] = __builtin_amdgcn_raw_buffer_load_b32(rows, off, row, kNt);
        }
    }
    __device__ __forceinline__ void clear(int key) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[key][i] = 0;
    }
    __device__ __forceinline__ auto operand(int t) const {
        if constexpr (DT == MIMIR_KV_F32) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_bit_cast(float, w[e][t]);
            return split8(x);
        } else {
            u4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == MIMIR_KV_BF16)
                    r[i] = __builtin_amdgcn_perm(w[2 * i + 1][t / 2], w[2 * i][t / 2], t % 2 ? 0x07060302u : 0x05040100u);
                else
                    r[i] = pack_high(byte_float(w[2 * i][t / 4], t % 4), byte_float(w[2 * i + 1][t / 4], t % 4));
            }
            return r;
        }
    }
};

// Waves of a SIMD.
constexpr int stream_waves(int dtype, int dp) {
    return dp == 256 ? 1 : dtype == MIMIR_KV_F32 ? (dp == 128 ? 1 : 2) : dp == 128 ? 2 : 4;
}

struct StreamArgs {
    PagedArgs p;
    // Blocks that several workgroups have keys of: which (first workgroup, number of
    // them; by sequence, head and rows), and their sums, [workgroup][2][row][max, sum,
    // head_dim sums].  Null: blocks are not divided.
    int2* shared;
    float* part;
    uint32_t grain;     // keys that are not divided among workgroups
    uint32_t extra;     // what a block costs besides its keys, in grains
    uint32_t groups;    // workgroups
    int32_t row_blocks; // of the sequence with the most rows
    int32_t rows;       // rows of a block that are kept in `part`
    int32_t most_rows;  // sequences with more query rows than this are another kernel's
};

// The work: a block is 16 query rows of one key / value head of a sequence against
// its keys, and costs its keys' grains and `extra`; all blocks' costs in order
// (sequence, head, rows) are dealt to the workgroups in equal runs, so that sequences
// of any lengths fill the GPU evenly.  A run may begin and end inside a block.  Every
// wave works out its run from the sequences' lengths, 64 of them at a time.
struct StreamChunk {
    int base;         // its first sequence
    uint32_t before;  // costs of those ahead
    KvSequence seq;   // the lane's sequence: its part of the batch, a block's cost, its
    uint32_t cost, blocks, sum;  // blocks, the costs up to it
};

__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// Cost of a block of a sequence, and its blocks (0: another kernel's, or none).
__device__ __forceinline__ uint32_t stream_cost(const StreamArgs& a, const KvSequence& q, uint32_t* blocks) {
    const int64_t rows = static_cast<int64_t>(q.n) * a.p.group;
    *blocks = rows > 0 && rows <= a.most_rows
                  ? static_cast<uint32_t>((rows + kRows - 1) / kRows) * static_cast<uint32_t>(a.p.c.kv_heads)
                  : 0;
    return a.extra + max(1u, (static_cast<uint32_t>(q.len) + a.grain - 1) / a.grain);
}

__device__ __forceinline__ StreamChunk stream_chunk(const StreamArgs& a, int base, uint32_t before) {
    const int lane = static_cast<int>(threadIdx.x % kWave);
    StreamChunk c{base, before, KvSequence{0, 0, 0}, 0, 0, 0};
    if (base + lane < a.p.b.sequences) {
        c.seq = kv_sequence(a.p.b, base + lane);
        c.cost = stream_cost(a, c.seq, &c.blocks);
    }
    c.sum = c.cost * c.blocks;
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) {
        const uint32_t y = static_cast<uint32_t>(__shfl_up(static_cast<int>(c.sum), x));
        if (lane >= x) c.sum += y;
    }
    return c;
}

struct StreamBlock {
    int s, head, row0, rows;  // sequence, key / value head, first row and rows of the block
    int end;                  // keys that some row of it sees
    uint32_t index;           // of its sequence's blocks
    uint32_t first, cost;     // its run of all costs
    KvSequence seq;
};

__device__ __forceinline__ void stream_rows(const StreamArgs& a, uint32_t blocks, StreamBlock* w) {
    const uint32_t row_blocks = max(1u, blocks / static_cast<uint32_t>(a.p.c.kv_heads));
    w->head = static_cast<int>(w->index / row_blocks);
    w->row0 = static_cast<int>(w->index % row_blocks) * kRows;
    w->rows = w->index < blocks ? min(w->seq.n * a.p.group - w->row0, kRows) : 0;
    const int last = (w->row0 + max(w->rows, 1) - 1) / a.p.group;
    w->end = a.p.causal ? min(max(w->seq.len - w->seq.n + last + 1, 0), w->seq.len) : w->seq.len;
}

// The block that x (below the total) falls in; `c` moves on to its chunk.
__device__ __forceinline__ StreamBlock stream_locate(const StreamArgs& a, uint32_t x, StreamChunk* c) {
    for (;;) {
        const uint32_t to = c->before + lane_of(c->sum, kWave - 1);
        if (x < to || c->base + kWave >= a.p.b.sequences) break;
        *c = stream_chunk(a, c->base + kWave, to);
    }
    const uint64_t above = __ballot(c->before + c->sum > x);
    const int lane = above ? __builtin_ctzll(above) : kWave - 1;
    StreamBlock w;
    w.s = c->base + lane;
    w.seq = KvSequence{static_cast<int>(lane_of(c->seq.first, lane)), static_cast<int>(lane_of(c->seq.n, lane)),
                       static_cast<int>(lane_of(c->seq.len, lane))};
    w.cost = lane_of(c->cost, lane);
    const uint32_t blocks = lane_of(c->blocks, lane);
    const uint32_t start = c->before + lane_of(c->sum, lane) - w.cost * blocks;
    w.index = (x - start) / w.cost;
    w.first = start + w.index * w.cost;
    stream_rows(a, blocks, &w);
    return w;
}

// Keys that row `row` (of all its sequence's) sees.
__device__ __forceinline__ int row_end(const PagedArgs& a, const KvSequence& q, int row) {
    return a.causal ? min(max(q.len - q.n + row / a.group + 1, 0), q.len) : q.len;
}

// Where a workgroup keeps the sums of a block that it shares with others: the block
// that its run begins in (0) or the one that it ends in (1).
__device__ __forceinline__ float* stream_part(const StreamArgs& a, uint32_t group, bool ends, int row) {
    return a.part + ((static_cast<int64_t>(group) * 2 + (ends ? 1 : 0)) * a.rows + row) * (a.p.c.head_dim + 2);
}

template <int DT, int DP>
__global__ __launch_bounds__(kStreamWaves * kWave, stream_waves(DT, DP)) void paged_stream(StreamArgs a) {
    using K = Kind<DT, DP>;
    constexpr int ND = DP / 16, kSteps = DP / 32, H = K::kHalves;
    typedef float Share[kRows][DP + 2];
    __shared__ __attribute__((aligned(16))) char lds[sizeof(Share) * kStreamWaves];
    Share* const share = reinterpret_cast<Share*>(lds);  // after the keys
    u4* const q_lds = reinterpret_cast<u4*>(lds);        // [step][term][lane], during them
    static_assert(kSteps * 3 * kWave * sizeof(u4) <= sizeof lds, "the queries fit");
    __shared__ uint32_t bad;
    const PagedArgs& p = a.p;
    StreamChunk chunk = stream_chunk(a, 0, 0);
    uint32_t total = lane_of(chunk.sum, kWave - 1);
    for (int base = kWave; base < p.b.sequences; base += kWave)
        total += lane_of(stream_chunk(a, base, 0).sum, kWave - 1);
    const uint32_t run = (total + a.groups - 1) / a.groups;
    const auto end = static_cast<uint32_t>(min(static_cast<uint64_t>(total), (static_cast<uint64_t>(blockIdx.x) + 1) * run));
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    for (uint64_t from = static_cast<uint64_t>(blockIdx.x) * run; from < end;) {
    int tid = static_cast<int>(threadIdx.x);
    asm volatile("" : "+v"(tid));  // what follows from it is computed for each block, not held in registers across them
    const int lane = tid % kWave, li = lane % 16, hg = lane / 16;
    const StreamBlock w = stream_locate(a, static_cast<uint32_t>(from), &chunk);
    const uint32_t x0 = static_cast<uint32_t>(from) - w.first, x1 = min(w.cost, end - w.first);
    from = w.first + x1;
    const bool whole = x0 == 0 && x1 == w.cost;  // no other workgroup has keys of the block
    const auto keys_to = [&](uint32_t x) {
        return static_cast<int>(min(static_cast<uint64_t>(x > a.extra ? x - a.extra : 0) * a.grain, static_cast<uint64_t>(w.end)));
    };
    const int k0 = keys_to(x0), k1 = keys_to(x1);
    if (a.part && x0 == 0 && tid == 0)
        a.shared[static_cast<int64_t>(w.s) * a.row_blocks * p.c.kv_heads + w.index] =
            int2{static_cast<int>(blockIdx.x), static_cast<int>((w.first + w.cost - 1) / run - blockIdx.x) + 1};
    const int my_row = w.row0 + min(li, w.rows - 1);
    const int my_end = min(row_end(p, w.seq, my_row), k1);
    const auto q_row = [&](int row) {
        return p.q + (w.seq.first + row / p.group) * p.ld_q + static_cast<int64_t>(w.head * p.group + row % p.group) * p.c.head_dim;
    };
    // The queries' loads go out ahead of the first keys', their terms follow those.
    constexpr int kOwn = (kSteps + kStreamWaves - 1) / kStreamWaves;
    float qx[kOwn][8];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const float* row = q_row(my_row);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = K::dim(wave + i * kStreamWaves, hg, e);
            qx[i][e] = d < p.c.head_dim ? row[d] : 0.f;
        }
    }

    // Where the halves of a step stand; one without a page (or past the keys) takes
    // the first page's address, and its keys count as unseen.
    struct Step {
        int page[H], slot[H];
        __device__ __forceinline__ bool has(int u, const KvView& c) const { return page[u] >= 0 && page[u] < c.pages; }
        // Row of the cache.
        __device__ __forceinline__ int64_t at(int u, const KvView& c, int head) const {
            return (static_cast<int64_t>(has(u, c) ? page[u] : 0) * c.kv_heads + head) * c.page_size + slot[u];
        }
    };
    // The table through scalar loads: a vector load's wait would be one for the keys
    // and values in flight before it too.
    const scalar_i32 table = (scalar_i32)(p.b.page_table + w.s * p.b.ld_pages);
    const auto find = [&](int key) {
        Step st;
#pragma unroll
        for (int u = 0; u < H; ++u) {
            const int j = key + kHalf * u;
            const int i = min(j, (k1 - 1) & -kHalf);
            const uint32_t entry = fastdiv(static_cast<uint32_t>(i), p.c.page_div);
            st.page[u] = j < k1 ? table[entry] : -1;
            st.slot[u] = i - static_cast<int>(entry) * p.c.page_size;
        }
        return st;
    };
    const int row_bytes = p.c.stride * K::kBytes;
    const auto half_rows = [&](const char* base, int64_t at) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base) + at * row_bytes, 0, kHalf * row_bytes, kBufferWord3);
    };
    uint32_t k_off[K::kVecs];
#pragma unroll
    for (int v = 0; v < K::kVecs; ++v)
        k_off[v] = static_cast<uint32_t>((li * p.c.stride + min(K::first(v, hg), p.c.stride - 16 / K::kBytes)) * K::kBytes);
    const uint32_t v_off = static_cast<uint32_t>((4 * hg * p.c.stride + min(li * ND, p.c.stride - ND)) * K::kBytes);

    u4 kr[H][K::kVecs];
    Values<DT, ND> vr[H / 2];
    f4 ks[H], vs[H];
    const auto load_k = [&](const Step& st) {
#pragma unroll
        for (int u = 0; u < H; ++u) {
            const int64_t at = st.at(u, p.c, w.head);
            const __amdgpu_buffer_rsrc_t rows = half_rows(p.c.k, at);
#pragma unroll
            for (int v = 0; v < K::kVecs; ++v) kr[u][v] = __builtin_amdgcn_raw_buffer_load_b128(rows, k_off[v], 0, kNt);
            if constexpr (DT == MIMIR_KV_I8) ks[u] = *reinterpret_cast<const f4*>(p.c.k_scale + at + 4 * hg);
        }
    };
    const auto load_v = [&](const Step& st) {
#pragma unroll
        for (int u = 0; u < H; ++u) {
            const int64_t at = st.at(u, p.c, w.head);
            const __amdgpu_buffer_rsrc_t rows = half_rows(p.c.v, at);
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[u / 2].load(4 * (u % 2) + e, rows, v_off, e * row_bytes);
            if constexpr (DT == MIMIR_KV_I8) vs[u] = *reinterpret_cast<const f4*>(p.c.v_scale + at + 4 * hg);
        }
    };

    f4r o[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t) o[t] = f4r{0.f, 0.f, 0.f, 0.f};
    float m_run = -1e30f, l_run = 0.f;  // the max is the row's, the sum this lane's share

    constexpr int kKeys = kHalf * H, kStep = kKeys * kStreamWaves;
    int key = k0 + wave * kKeys;
    Step st{}, nx{}, after{};  // this step's, and the next two's, found a step ahead of their loads
    if (key < k1) {
        st = find(key);
        load_k(st);
        load_v(st);
        nx = find(key + kStep);
    }
    __syncthreads();  // the last block's sums and flags are read
    if (tid == 0) bad = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int c = wave + i * kStreamWaves;
        if (c >= kSteps) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) qx[i][e] *= p.qscale;
        const Split8 x = split8(qx[i]);
        q_lds[(3 * c) * kWave + lane] = x.h;
        q_lds[(3 * c + 1) * kWave + lane] = x.m;
        q_lds[(3 * c + 2) * kWave + lane] = x.l;
    }
    __syncthreads();
    // One step.  more: the next one's loads are issued in between, K's once the scores
    // have read this one's, V's at the end; compiled apart from the last step, so that
    // the waits for loads in flight count them.
    const auto step = [&](auto more) {
        int at = lane;
        asm volatile("" : "+v"(at));  // read here in each step, not held in registers across them
        const u4* const mine = q_lds + at;
        f4r s[H];
#pragma unroll
        for (int u = 0; u < H; ++u) s[u] = f4r{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            const Split8 q{mine[(3 * c) * kWave], mine[(3 * c + 1) * kWave], mine[(3 * c + 2) * kWave]};
#pragma unroll
            for (int u = 0; u < H; ++u) s[u] = mfma16_split(K::operand(kr[u], c), q, s[u]);
            if constexpr (DT == MIMIR_KV_F32) __builtin_amdgcn_sched_barrier(0);  // few terms at a time
        }
        if constexpr (DT == MIMIR_KV_I8) {
#pragma unroll
            for (int u = 0; u < H; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[u][r] *= ks[u][r];
        }
        if constexpr (decltype(more)::value) {
            load_k(nx);
            after = find(key + 2 * kStep);  // here, where no LDS read waits for it
        }

        float x[4 * H];
#pragma unroll
        for (int e = 0; e < 4 * H; ++e) x[e] = s[e / 4][e % 4];
        // Rows whose keys end inside the step, and halves that are not there: the
        // weights are 0 and, where no row of the tile sees a key, so are its values
        // (what is stored there may be anything).
        bool edge = __any(key + kKeys > my_end);
#pragma unroll
        for (int u = 0; u < H; ++u) edge = edge || !st.has(u, p.c);
        if (edge) {
#pragma unroll
            for (int e = 0; e < 4 * H; ++e) {
                const int u = e / 4, j = key + kHalf * u + 4 * hg + e % 4;
                x[e] = st.has(u, p.c) && j < my_end ? x[e] : -INFINITY;
                if (!st.has(u, p.c) || j >= k1) {
                    vr[u / 2].clear(e % 8);
                    if constexpr (DT == MIMIR_KV_I8) vs[u][e % 4] = 0.f;
                }
            }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 4 * H; ++e) top = fmaxf(top, x[e]);
        if (__any(top > m_run + kMaxSlack)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float m_new = fmaxf(m_run, top);
            const float f = __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= f;
#pragma unroll
            for (int t = 0; t < ND; ++t) o[t] *= f;
        }
#pragma unroll
        for (int e = 0; e < 4 * H; ++e) {
            x[e] = __builtin_amdgcn_exp2f(x[e] - m_run);
            l_run += x[e];
            if constexpr (DT == MIMIR_KV_I8) x[e] *= vs[e / 4][e % 4];
        }
#pragma unroll
        for (int h = 0; h < H / 2; ++h) {
            const Split8 pw = split8(x + 8 * h);
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                o[t] = mfma16_split(vr[h].operand(t), pw, o[t]);
                if constexpr (DT == MIMIR_KV_F32)
                    if (t % 2 == 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (decltype(more)::value) load_v(nx);
    };
    for (; key + kStep < k1; key += kStep) {
        step(std::true_type{});
        st = nx;
        nx = after;
    }
    if (key < k1) step(std::false_type{});

    // The waves' shares of the rows.  Lane (li, hg) holds dimensions (4 hg + r) ND + t.
    __syncthreads();
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < ND; ++t) share[wave][li][(4 * hg + r) * ND + t] = o[t][r];
    if (hg == 0) {
        share[wave][li][DP] = m_run;
        share[wave][li][DP + 1] = l_run;
    }
    __syncthreads();
    const auto out_row = [&](int row) {  // row of the block
        const int r = w.row0 + row;
        return p.out + (w.seq.first + r / p.group) * p.ld_out + static_cast<int64_t>(w.head * p.group + r % p.group) * p.c.head_dim;
    };
    const auto part_row = [&](int row) { return stream_part(a, blockIdx.x, x0 == 0, row); };
    for (int x = tid; x < w.rows * p.c.head_dim; x += kStreamWaves * kWave) {
        const int row = x / p.c.head_dim, d = x % p.c.head_dim;
        float m = share[0][row][DP];
#pragma unroll
        for (int v = 1; v < kStreamWaves; ++v) m = fmaxf(m, share[v][row][DP]);
        float l = 0.f, sum = 0.f;
#pragma unroll
        for (int v = 0; v < kStreamWaves; ++v) {
            const float f = __builtin_amdgcn_exp2f(share[v][row][DP] - m);
            l += share[v][row][DP + 1] * f;
            sum += share[v][row][d] * f;
        }
        if (!(fabsf(sum) < INFINITY) || !(l < INFINITY)) atomicOr(&bad, 1u << row);
        if (whole) {
            out_row(row)[d] = sum * (1.0f / (l + 1e-9f));
        } else {
            float* part = part_row(row);
            part[2 + d] = sum;
            if (d == 0) {
                part[0] = m;
                part[1] = l;
            }
        }
    }
    __syncthreads();
    // Rows that came out NaN or infinite, again in fp32: an operand had no bf16 split
    // (split.hpp), or a value that the row does not see is not finite.
    if (bad == 0) continue;
    for (int row = wave; row < w.rows; row += kStreamWaves) {
        if (!(bad >> row & 1)) continue;
        float acc[kRowChunks], m, l;
        row_over_keys<DT>(p, w.s, w.head, q_row(w.row0 + row), k0, min(k1, row_end(p, w.seq, w.row0 + row)), acc, &m, &l);
        const float inv = whole ? 1.0f / (l + 1e-9f) : 1.0f;
        float* out = whole ? out_row(row) : part_row(row) + 2;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) {
            const int d = lane + c * kWave;
            if (d < p.c.head_dim) out[d] = acc[c] * inv;
        }
        if (!whole && lane == 0) {
            out[-2] = m;
            out[-1] = l;
        }
    }
    }
}

// The shares of one row of a block that several workgroups had keys of: brought to
// one max, added up by four waves and divided.
__global__ __launch_bounds__(kBlock) void paged_join(StreamArgs a) {
    constexpr int kWaves = kBlock / kWave, kAhead = 4;
    __shared__ float share[kWaves][kKvMaxDim + 2];
    const int row = static_cast<int>(blockIdx.x % static_cast<uint32_t>(a.rows));
    const uint32_t rest = blockIdx.x / static_cast<uint32_t>(a.rows);
    const uint32_t most = static_cast<uint32_t>(a.row_blocks) * static_cast<uint32_t>(a.p.c.kv_heads);
    const int2 run = a.shared[rest];  // means nothing where the sequence has no such block
    StreamBlock w;
    w.s = static_cast<int>(rest / most);
    w.index = rest % most;
    w.seq = kv_sequence(a.p.b, w.s);
    uint32_t blocks;
    stream_cost(a, w.seq, &blocks);
    stream_rows(a, blocks, &w);
    if (row >= w.rows || run.y <= 1) return;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, d = a.p.c.head_dim;
    float m = -1e30f, l = 0.f, acc[kRowChunks];
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) acc[c] = 0.f;
    for (int i = wave; i < run.y; i += kAhead * kWaves) {
        float ms[kAhead], ls[kAhead], x[kAhead][kRowChunks];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = i + u * kWaves;
            ms[u] = -1e30f;
            ls[u] = 0.f;
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c) x[u][c] = 0.f;
            if (j >= run.y) continue;
            // The first workgroup's run ends in the block, the others' begin.
            const float* part = stream_part(a, static_cast<uint32_t>(run.x + j), j == 0, row);
            ms[u] = part[0];
            ls[u] = part[1];
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c)
                if (lane + c * kWave < d) x[u][c] = part[2 + lane + c * kWave];
        }
        float m_new = m;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) m_new = fmaxf(m_new, ms[u]);
        const float f = __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) acc[c] *= f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const float g = __builtin_amdgcn_exp2f(ms[u] - m);
            l += ls[u] * g;
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c) acc[c] += x[u][c] * g;
        }
    }
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) share[wave][lane + c * kWave] = acc[c];
    if (lane == 0) {
        share[wave][kKvMaxDim] = m;
        share[wave][kKvMaxDim + 1] = l;
    }
    __syncthreads();
    const int x = static_cast<int>(threadIdx.x);
    if (x >= d) return;
    float top = share[0][kKvMaxDim];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = fmaxf(top, share[v][kKvMaxDim]);
    float sum = 0.f, all = 0.f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
        const float f = __builtin_amdgcn_exp2f(share[v][kKvMaxDim] - top);
        sum += share[v][x] * f;
        all += share[v][kKvMaxDim + 1] * f;
    }
    const int r = w.row0 + row;
    a.p.out[(w.seq.first + r / a.p.group) * a.p.ld_out + static_cast<int64_t>(w.head * a.p.group + r % a.p.group) * d + x] =
        sum * (1.0f / (all + 1e-9f));
}
static_assert(kKvMaxDim <= kBlock, "a thread per dimension");

template <int DT>
void launch_stream_dim(const StreamArgs& a, unsigned grid, hipStream_t s) {
    constexpr int kThreads = kStreamWaves * kWave;
    if (a.p.c.stride <= 64) paged_stream<DT, 64><<<grid, kThreads, 0, s>>>(a);
    else if (a.p.c.stride <= 128) paged_stream<DT, 128><<<grid, kThreads, 0, s>>>(a);
    else paged_stream<DT, 256><<<grid, kThreads, 0, s>>>(a);
}

// What a block costs a workgroup besides its keys (its queries, the first keys' way
// in, the sums' way out), in steps of 128 keys.
constexpr int64_t kStreamExtra = 2;

// Workgroups that the GPU holds at once.
int64_t stream_resident(int dtype, int stride) {
    // Two a compute unit where registers allow them: measured (256 / 512 / 1024 workgroups, us), 64 sequences x
    // 4096 keys x 8 heads x 128: 8-bit 112 / 99 / 105, bf16 168 / 162 / 170; heads of 64: 8-bit 76 / 60 / 60, bf16
    // 88 / 87 / 92, fp32 183 / 168 / 174; heads of 256, one a unit: bf16 120 / 131 / 145.
    return 256 * std::min(2, stream_waves(dtype, stride <= 64 ? 64 : stride <= 128 ? 128 : 256));
}

int launch_stream(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t most_rows) {
    StreamArgs a{};
    a.p = p;
    a.most_rows = static_cast<int32_t>(most_rows);
    const int64_t rows = std::min(static_cast<int64_t>(p.b.max_new) * p.group, most_rows);
    a.row_blocks = static_cast<int32_t>((rows + kRows - 1) / kRows);
    a.rows = static_cast<int32_t>(std::min<int64_t>(rows, kRows));
    const int64_t blocks = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads * a.row_blocks;
    a.groups = static_cast<uint32_t>(ctx->tune.decode_splits > 0 ? ctx->tune.decode_splits : stream_resident(dtype, p.c.stride));
    // A grain is a step of the four waves, or as many as keep the sum of all in 31 bits.
    const int64_t len = std::max<int64_t>(p.b.max_len, 1);
    int64_t grain = 2 * kHalf * kStreamWaves;
    const auto grains = [&] { return (len + grain - 1) / grain; };
    // Blocks of up to two steps are not worth a join.
    const int64_t words = 2 * blocks + static_cast<int64_t>(a.groups) * 2 * a.rows * (p.c.head_dim + 2);
    float* work = grains() > 2 && words * 4 <= static_cast<int64_t>(kFixedWorkBytes) ? fixed_work(ctx) : nullptr;
    int64_t grid = blocks;
    if (work) {
        a.extra = kStreamExtra;
        while ((grains() + kStreamExtra) * blocks >= (int64_t{1} << 31) && grains() > 1) grain *= 2;
        a.shared = reinterpret_cast<int2*>(work);
        a.part = work + 2 * blocks;
        grid = std::min<int64_t>(a.groups, blocks * (grains() + kStreamExtra));
    } else {  // a workgroup per block
        grain *= grains();
        a.groups = static_cast<uint32_t>(std::min<int64_t>(blocks, INT32_MAX));
    }
    a.grain = static_cast<uint32_t>(grain);
    MIMIR_REQUIRE(ctx, dispatch_fits(grid, kStreamWaves * kWave) && dispatch_fits(blocks * a.rows, kBlock),
                  "paged attention: grid of %lld workgroups exceeds the limit", (long long)blocks);
    if (dtype == MIMIR_KV_F32) launch_stream_dim<MIMIR_KV_F32>(a, static_cast<unsigned>(grid), ctx->stream);
    else if (dtype == MIMIR_KV_BF16) launch_stream_dim<MIMIR_KV_BF16>(a, static_cast<unsigned>(grid), ctx->stream);
    else launch_stream_dim<MIMIR_KV_I8>(a, static_cast<unsigned>(grid), ctx->stream);
    if (int st = launched(ctx, "paged_stream")) return st;
    if (!a.part) return MIMIR_OK;
    paged_join<<<static_cast<unsigned>(blocks * a.rows), kBlock, 0, ctx->stream>>>(a);
    return launched(ctx, "paged_join");
}

// ---------------------------------------------------------------------------
// Many query rows per key / value head: tiles of 32 keys in LDS
// ---------------------------------------------------------------------------

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_s4;

constexpr int kTile = 32;     // keys of a tile, and query rows of a wave
constexpr int kXcds = 8;

struct BlockArgs {
    PagedArgs p;
    float* part;         // [split][block][row][head_dim sums, max, sum], null: one split
    uint32_t pairs;      // sequences x key / value heads
    int32_t row_blocks;  // row blocks of the sequence with the most rows
    int32_t splits, span;  // splits of a block's keys, keys of each (a multiple of kTile)
    int32_t least_rows;  // sequences with fewer query rows than this are another kernel's
};

struct BlockWork {
    int s, head, row0, rows;  // sequence, key / value head, first row, rows from it on
    int end;                  // keys that some row of the block sees
    KvSequence seq;
};

__device__ __forceinline__ BlockWork block_work(const BlockArgs& a, uint32_t pair, int rb, int block_rows) {
    BlockWork w;
    w.s = static_cast<int>(pair / static_cast<uint32_t>(a.p.c.kv_heads));
    w.head = static_cast<int>(pair % static_cast<uint32_t>(a.p.c.kv_heads));
    w.seq = kv_sequence(a.p.b, w.s);
    const int64_t all = static_cast<int64_t>(w.seq.n) * a.p.group;
    w.row0 = rb * block_rows;
    w.rows = all >= a.least_rows ? static_cast<int>(min(all - w.row0, static_cast<int64_t>(block_rows))) : 0;
    w.end = row_end(a.p, w.seq, w.row0 + max(w.rows, 1) - 1);
    return w;
}

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
__global__ __launch_bounds__(WAVES * kWave, 2) void paged_block(BlockArgs a) {
    using Tile = BlockTile<DT, DP>;
    constexpr int kThreads = WAVES * kWave, kRowsOf = WAVES * kTile, kC = DP / 16, kDb = DP / 32;
    constexpr int kElement = DT == MIMIR_KV_F32 ? 4 : DT == MIMIR_KV_BF16 ? 2 : 1;
    constexpr int kItems = (kTile * (DP / 8) + kThreads - 1) / kThreads;
    __shared__ __attribute__((aligned(16))) char lds[2 * Tile::kBytes];
    const PagedArgs& p = a.p;

    // Where a (sequence, head) count divides by the XCDs, each owns an eighth of them,
    // whose keys stay in its L2; the longest blocks come first.
    uint32_t pair, idx = blockIdx.x, owned = a.pairs;
    if (a.pairs % kXcds == 0) {
        owned = a.pairs / kXcds;
        idx = blockIdx.x / kXcds;
    }
    pair = idx % owned + (a.pairs % kXcds == 0 ? blockIdx.x % kXcds * owned : 0);
    const int split = static_cast<int>(idx / owned % static_cast<uint32_t>(a.splits));
    const int rb = a.row_blocks - 1 - static_cast<int>(idx / owned / static_cast<uint32_t>(a.splits));
    const BlockWork w = block_work(a, pair, rb, kRowsOf);
    const int k0 = split * a.span, k1 = min(w.end, k0 + a.span);
    if (w.rows <= 0 || (split > 0 && k0 >= w.end)) return;
    const bool whole = w.end <= a.span;

    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave), lane = threadIdx.x % kWave;
    const int li = lane % 32, hf = lane / 32;
    const int wave_rows = min(w.rows - wave * kTile, kTile);  // below 1: a wave that only moves tiles
    const bool in = li < wave_rows;
    const int my_row = w.row0 + wave * kTile + max(0, min(li, wave_rows - 1));
    const int my_end = min(row_end(p, w.seq, min(my_row, w.row0 + w.rows - 1)), k1);
    const int wave_end = wave_rows > 0 ? min(k1, row_end(p, w.seq, w.row0 + wave * kTile + wave_rows - 1)) : k0;
    const auto q_row = [&](int row) {
        return p.q + (w.seq.first + row / p.group) * p.ld_q + static_cast<int64_t>(w.head * p.group + row % p.group) * p.c.head_dim;
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
            const int id = static_cast<int>(threadIdx.x) + n * kThreads, row = id / (DP / 8), d = 8 * (id % (DP / 8));
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
            if (threadIdx.x < 2 * kTile) {
                const int row = threadIdx.x % kTile, u = row / kHalf;
                const int64_t at = (u ? r1 : r0) + row % kHalf;
                scale = (threadIdx.x < kTile ? p.c.k_scale : p.c.v_scale)[at];
                if (k0 + t * kTile + row >= k1 || (u ? g.page[1] : g.page[0]) < 0) scale = 0.f;
            }
        }
    };
    const auto stash = [&](char* buf) {
#pragma unroll
        for (int n = 0; n < kItems; ++n) {
            const int id = static_cast<int>(threadIdx.x) + n * kThreads, row = id / (DP / 8), at = 16 * (id % (DP / 8));
            if (row >= kTile) continue;
            ki[n].stash(buf + row * Tile::kKeyRow + at, Tile::kKeyPlane);
            vi[n].stash(buf + Tile::kValuesAt + row * Tile::kValueRow + at, Tile::kValuePlane);
        }
        if constexpr (DT == MIMIR_KV_I8)
            if (threadIdx.x < 2 * kTile) reinterpret_cast<float*>(buf + Tile::kScalesAt)[threadIdx.x] = scale;
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
            if (__any(top > m_run + kMaxSlack)) {
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
    if (wave_rows <= 0) return;
    const float l_tot = l_run + __shfl_xor(l_run, 32);
    const int row = my_row - w.row0;
    const int d_all = p.c.head_dim;
    float* const out = whole ? p.out + (w.seq.first + my_row / p.group) * p.ld_out + static_cast<int64_t>(w.head * p.group + my_row % p.group) * d_all
                             : a.part + ((static_cast<int64_t>(split) * a.pairs * a.row_blocks + static_cast<int64_t>(pair) * a.row_blocks + rb) * kRowsOf + row) * (d_all + 2);
    const float inv = whole ? 1.0f / (l_tot + 1e-9f) : 1.0f;
    const bool vec = whole ? d_all % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.ld_out % 4 == 0 : false;
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
    if (!whole && in && hf == 0) {
        out[d_all] = m_run;
        out[d_all + 1] = l_tot;
    }
    // Rows that came out NaN or infinite, again in fp32 (as paged_stream).
    const uint64_t ballot = __ballot(check != check && in);
    for (uint32_t bad = static_cast<uint32_t>(ballot | ballot >> 32); bad; bad &= bad - 1) {
        const int r = wave * kTile + __builtin_ctz(bad), full = w.row0 + r;
        float acc[kRowChunks], m, l;
        row_over_keys<DT>(p, w.s, w.head, q_row(full), k0, min(k1, row_end(p, w.seq, full)), acc, &m, &l);
        float* const to = whole ? p.out + (w.seq.first + full / p.group) * p.ld_out + static_cast<int64_t>(w.head * p.group + full % p.group) * d_all
                                : a.part + ((static_cast<int64_t>(split) * a.pairs * a.row_blocks + static_cast<int64_t>(pair) * a.row_blocks + rb) * kRowsOf + r) * (d_all + 2);
        const float f = whole ? 1.0f / (l + 1e-9f) : 1.0f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c)
            if (lane + c * kWave < d_all) to[lane + c * kWave] = acc[c] * f;
        if (!whole && lane == 0) {
            to[d_all] = m;
            to[d_all + 1] = l;
        }
    }
}

// The splits of one row, a wave per row.
__global__ __launch_bounds__(kBlock) void paged_block_join(BlockArgs a, int block_rows) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave;
    const int64_t all = static_cast<int64_t>(a.pairs) * a.row_blocks * block_rows;
    if (at >= all) return;
    const int row = static_cast<int>(at % block_rows), rb = static_cast<int>(at / block_rows % a.row_blocks);
    const BlockWork w = block_work(a, static_cast<uint32_t>(at / block_rows / a.row_blocks), rb, block_rows);
    if (row >= w.rows || w.end <= a.span) return;
    const int d = a.p.c.head_dim, n = (w.end + a.span - 1) / a.span, lane = threadIdx.x % kWave;
    const float* part = a.part + at * (d + 2);
    const int64_t step = all * (d + 2);
    float m = -1e30f, l = 0.f, acc[kRowChunks];
    for (int s = 0; s < n; ++s) m = fmaxf(m, part[s * step + d]);
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) acc[c] = 0.f;
    for (int s = 0; s < n; ++s) {
        const float f = __builtin_amdgcn_exp2f(part[s * step + d] - m);
        l += part[s * step + d + 1] * f;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c)
            if (lane + c * kWave < d) acc[c] += part[s * step + lane + c * kWave] * f;
    }
    const float inv = 1.0f / (l + 1e-9f);
    const int r = w.row0 + row;
    float* out = a.p.out + (w.seq.first + r / a.p.group) * a.p.ld_out + static_cast<int64_t>(w.head * a.p.group + r % a.p.group) * d;
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c)
        if (lane + c * kWave < d) out[lane + c * kWave] = acc[c] * inv;
}

template <int DT, int DP, int WAVES>
int launch_block_waves(mimir_ctx* ctx, BlockArgs a) {
    constexpr int kRowsOf = WAVES * kTile;
    const int64_t rows = static_cast<int64_t>(a.p.b.max_new) * a.p.group;
    a.row_blocks = static_cast<int32_t>((rows + kRowsOf - 1) / kRowsOf);
    const int64_t blocks = static_cast<int64_t>(a.pairs) * a.row_blocks, d = a.p.c.head_dim;
    const int64_t tiles = std::max<int64_t>(1, (a.p.b.max_len + kTile - 1) / kTile);
    // Keys are split until the workgroups fill the GPU, in parts of 256 and more.
    constexpr int64_t kTarget = 2048 / WAVES;
    int64_t splits = std::min(kTarget / std::max<int64_t>(blocks, 1), tiles / 8);
    if (ctx->tune.attn_splits > 0) splits = ctx->tune.attn_splits;
    splits = std::min(splits, static_cast<int64_t>(kFixedWorkBytes / 4) / (blocks * kRowsOf * (d + 2)));
    a.part = splits > 1 ? fixed_work(ctx) : nullptr;
    if (!a.part) splits = 1;
    a.span = static_cast<int32_t>((tiles + splits - 1) / splits * kTile);
    a.splits = static_cast<int32_t>((tiles * kTile + a.span - 1) / a.span);
    MIMIR_REQUIRE(ctx, dispatch_fits(blocks * a.splits, WAVES * kWave) && dispatch_fits((blocks * kRowsOf + 3) / 4, kBlock),
                  "paged attention: grid of %lld workgroups exceeds the limit", (long long)(blocks * a.splits));
    paged_block<DT, DP, WAVES><<<static_cast<unsigned>(blocks * a.splits), WAVES * kWave, 0, ctx->stream>>>(a);
    if (int st = launched(ctx, "paged_block")) return st;
    if (a.splits == 1) return MIMIR_OK;
    paged_block_join<<<static_cast<unsigned>((blocks * kRowsOf + 3) / 4), kBlock, 0, ctx->stream>>>(a, kRowsOf);
    return launched(ctx, "paged_block_join");
}

template <int DT, int DP>
int launch_block_dim(mimir_ctx* ctx, const BlockArgs& a) {
    const int64_t rows = static_cast<int64_t>(a.p.b.max_new) * a.p.group;
    const int64_t blocks8 = static_cast<int64_t>(a.pairs) * ((rows + 8 * kTile - 1) / (8 * kTile));
    int waves = blocks8 < 512 ? 4 : 8;
    if (ctx->tune.attn_waves == 4 || ctx->tune.attn_waves == 8) waves = ctx->tune.attn_waves;
    return waves == 4 ? launch_block_waves<DT, DP, 4>(ctx, a) : launch_block_waves<DT, DP, 8>(ctx, a);
}

template <int DT>
int launch_block_type(mimir_ctx* ctx, const BlockArgs& a) {
    if (a.p.c.stride <= 64) return launch_block_dim<DT, 64>(ctx, a);
    if (a.p.c.stride <= 96) return launch_block_dim<DT, 96>(ctx, a);
    return launch_block_dim<DT, 128>(ctx, a);
}

constexpr int64_t kStreamRows = 32;

// The widest heads (padded) of the block kernel: its queries' terms are registers.
constexpr int kBlockStride = 128;

int launch_block(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t least_rows) {
    BlockArgs a{};
    a.p = p;
    const int64_t pairs = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads;
    MIMIR_REQUIRE(ctx, pairs < (int64_t{1} << 31), "paged attention: too many heads");
    a.pairs = static_cast<uint32_t>(pairs);
    a.least_rows = static_cast<int32_t>(least_rows);
    if (dtype == MIMIR_KV_F32) return launch_block_type<MIMIR_KV_F32>(ctx, a);
    if (dtype == MIMIR_KV_BF16) return launch_block_type<MIMIR_KV_BF16>(ctx, a);
    return launch_block_type<MIMIR_KV_I8>(ctx, a);
}

}  // namespace

extern "C" int mimir_attention_paged_fwd(mimir_ctx* ctx, const mimir_kv_cache* cache, const mimir_kv_batch* batch,
                                         const float* q, int64_t ld_q, float* out, int64_t ld_out, int64_t q_heads,
                                         float scale, int causal) {
    if (!ctx) return MIMIR_EINVAL;
    const char* what = "paged attention";
    PagedArgs a{};
    if (int st = kv_view(ctx, what, cache, &a.c)) return st;
    if (int st = kv_batch(ctx, what, cache, batch, &a.b)) return st;
    MIMIR_REQUIRE(ctx, q_heads >= 1 && q_heads <= (1 << 20) && q_heads % cache->kv_heads == 0,
                  "%s: q_heads %lld is not a multiple of kv_heads %d", what, (long long)q_heads, cache->kv_heads);
    const int64_t width = q_heads * cache->head_dim;
    MIMIR_REQUIRE(ctx, ld_q >= width && ld_out >= width, "%s: row strides (%lld, %lld) below q_heads * head_dim = %lld", what,
                  (long long)ld_q, (long long)ld_out, (long long)width);
    MIMIR_REQUIRE(ctx, std::isfinite(scale), "%s: scale must be finite", what);
    if (batch->tokens == 0 || batch->sequences == 0 || batch->max_new == 0) return MIMIR_OK;
    if (cache->pages == 0) a.b.max_len = 0;  // no keys, and no memory to point at
    MIMIR_REQUIRE(ctx, q && out, "%s: null pointer", what);
    MIMIR_ENTER(ctx);
    a.q = q;
    a.out = out;
    a.ld_q = ld_q;
    a.ld_out = ld_out;
    a.heads = static_cast<int32_t>(q_heads);
    a.group = static_cast<int32_t>(q_heads / cache->kv_heads);
    a.qscale = scale * kLog2e;
    a.causal = causal ? 1 : 0;
    const int64_t rows = static_cast<int64_t>(a.b.max_new) * a.group;
    MIMIR_REQUIRE(ctx, rows <= INT32_MAX, "%s: %lld query rows of a head", what, (long long)rows);
    // Sequences with up to kStreamRows query rows of a key / value head stream their
    // keys, the others' keys go through LDS.  A batch whose sequences all have the
    // same number needs one of the two.
    const bool even = a.b.sequences * static_cast<int64_t>(a.b.max_new) == a.b.tokens;
    if (a.c.stride > kBlockStride) return launch_stream(ctx, a, cache->dtype, INT32_MAX);
    if (rows <= kStreamRows || !even)
        if (int st = launch_stream(ctx, a, cache->dtype, kStreamRows)) return st;
    if (rows <= kStreamRows) return MIMIR_OK;
    return launch_block(ctx, a, cache->dtype, kStreamRows + 1);
}
