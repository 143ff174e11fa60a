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
constexpr int kKeys = 32;     // keys of a step: two halves of 16, each inside one page
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
    static constexpr int kBytes = 2, kVecs = DP / 32;
    typedef u4 Operand;
    static __device__ __forceinline__ int first(int v, int hg) { return 32 * v + 8 * hg; }
    static __device__ __forceinline__ int dim(int c, int hg, int e) { return 32 * c + 8 * hg + e; }
    static __device__ __forceinline__ Operand operand(const u4* raw, int c) { return raw[c]; }
};
template <int DP>
struct Kind<MIMIR_KV_I8, DP> {
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
    __device__ __forceinline__ void load(int key, const char* p) {
        if constexpr (kWords % 4 == 0) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const u4 x = reinterpret_cast<const u4*>(p)[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[key][4 * i + e] = x[e];
            }
        } else if constexpr (kWords == 2) {
            const u2 x = *reinterpret_cast<const u2*>(p);
            w[key][0] = x[0];
            w[key][1] = x[1];
        } else {
            static_assert(kWords == 1, "one word, two or whole vectors");
            w[key][0] = *reinterpret_cast<const uint32_t*>(p);
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

struct StreamArgs {
    PagedArgs p;
    float* part;       // [block][split][row][max, sum, head_dim sums], null: one split
    uint32_t blocks;   // sequences x key / value heads x row blocks
    int32_t row_blocks;
    int32_t rows;      // rows of a block that are kept in `part`
    int32_t splits, span;  // splits of a sequence's keys, keys of each (a multiple of 128)
    int32_t most_rows; // sequences with more query rows than this are another kernel's
};

// What a workgroup of the stream kernel (and its part of the join) has to do.
struct StreamWork {
    int s, head, row0, rows;  // sequence, key / value head, first row and rows of the block
    int end;                  // keys that some row of it sees
    KvSequence seq;
};

__device__ __forceinline__ StreamWork stream_work(const StreamArgs& a, uint32_t block) {
    StreamWork w;
    const uint32_t rb = block % static_cast<uint32_t>(a.row_blocks), sh = block / static_cast<uint32_t>(a.row_blocks);
    w.s = static_cast<int>(sh / static_cast<uint32_t>(a.p.c.kv_heads));
    w.head = static_cast<int>(sh % static_cast<uint32_t>(a.p.c.kv_heads));
    w.seq = kv_sequence(a.p.b, w.s);
    const int64_t all = static_cast<int64_t>(w.seq.n) * a.p.group;
    w.row0 = static_cast<int>(rb) * kRows;
    w.rows = all > a.most_rows ? 0 : static_cast<int>(min(all - w.row0, static_cast<int64_t>(kRows)));
    const int last = (w.row0 + max(w.rows, 1) - 1) / a.p.group;
    w.end = a.p.causal ? min(max(w.seq.len - w.seq.n + last + 1, 0), w.seq.len) : w.seq.len;
    return w;
}

// Keys that row `row` (of all its sequence's) sees.
__device__ __forceinline__ int row_end(const PagedArgs& a, const KvSequence& q, int row) {
    return a.causal ? min(max(q.len - q.n + row / a.group + 1, 0), q.len) : q.len;
}

template <int DT, int DP>
__global__ __launch_bounds__(kStreamWaves * kWave, DP == 256 ? 1 : DT == MIMIR_KV_F32 ? (DP == 128 ? 2 : 3) : DP == 128 ? 3 : 4) void paged_stream(StreamArgs a) {
    using K = Kind<DT, DP>;
    constexpr int ND = DP / 16, kSteps = DP / 32;
    typedef float Share[kRows][DP + 2];
    __shared__ __attribute__((aligned(16))) char lds[sizeof(Share) * kStreamWaves];
    Share* const share = reinterpret_cast<Share*>(lds);  // after the keys
    u4* const q_lds = reinterpret_cast<u4*>(lds);        // [step][term][lane], during them
    static_assert(kSteps * 3 * kWave * sizeof(u4) <= sizeof lds, "the queries fit");
    __shared__ uint32_t bad;
    const PagedArgs& p = a.p;
    // The XCDs take workgroups in turn: blocks first, so that each gets whole splits'
    // worth of them, the splits that every sequence has ahead of those few have.
    const uint32_t split = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
    const StreamWork w = stream_work(a, block);
    const int k0 = static_cast<int>(split) * a.span, k1 = min(w.end, k0 + a.span);
    if (w.rows <= 0 || (split > 0 && k0 >= w.end)) return;
    const bool whole = a.part == nullptr || w.end <= a.span;  // no other split has keys

    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave), lane = threadIdx.x % kWave;
    const int li = lane % 16, hg = lane / 16;
    if (threadIdx.x == 0) bad = 0;
    const int my_row = w.row0 + min(li, w.rows - 1);
    const int my_end = min(row_end(p, w.seq, my_row), k1);
    const auto q_row = [&](int row) {
        return p.q + (w.seq.first + row / p.group) * p.ld_q + static_cast<int64_t>(w.head * p.group + row % p.group) * p.c.head_dim;
    };

    const auto query = [&](const float* row, int c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = K::dim(c, hg, e);
            x[e] = d < p.c.head_dim ? row[d] * p.qscale : 0.f;
        }
        return split8(x);
    };
    for (int c = wave; c < kSteps; c += kStreamWaves) {
        const Split8 x = query(q_row(my_row), c);
        q_lds[(3 * c) * kWave + lane] = x.h;
        q_lds[(3 * c + 1) * kWave + lane] = x.m;
        q_lds[(3 * c + 2) * kWave + lane] = x.l;
    }
    __syncthreads();

    // Where the two halves of a step stand; a half without a page (or past the
    // keys) takes the first page's address, and its keys count as unseen.
    struct Step {
        int64_t at[2];  // rows of the cache
        bool has[2];
    };
    // The table through scalar loads: a vector load's wait would be one for the keys
    // and values in flight before it too.
    const scalar_i32 table = (scalar_i32)(p.b.page_table + w.s * p.b.ld_pages);
    const auto find = [&](int key) {
        Step st;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = key + 16 * u;
            const int i = min(j, (k1 - 1) & -16);
            const uint32_t entry = fastdiv(static_cast<uint32_t>(i), p.c.page_div);
            const int page = table[entry];
            st.has[u] = j < k1 && page >= 0 && page < p.c.pages;
            st.at[u] = (static_cast<int64_t>(st.has[u] ? page : 0) * p.c.kv_heads + w.head) * p.c.page_size + i -
                       static_cast<int>(entry) * p.c.page_size;
        }
        return st;
    };
    const int64_t row_bytes = static_cast<int64_t>(p.c.stride) * K::kBytes;
    uint32_t k_off[K::kVecs], v_off;
#pragma unroll
    for (int v = 0; v < K::kVecs; ++v)
        k_off[v] = static_cast<uint32_t>((li * p.c.stride + min(K::first(v, hg), p.c.stride - 16 / K::kBytes)) * K::kBytes);
    v_off = static_cast<uint32_t>((4 * hg * p.c.stride + min(li * ND, p.c.stride - ND)) * K::kBytes);

    u4 kr[2][K::kVecs];
    Values<DT, ND> vr;
    f4 ks[2], vs[2];
    const auto load_k = [&](const Step& st) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* base = p.c.k + st.at[u] * row_bytes;
#pragma unroll
            for (int v = 0; v < K::kVecs; ++v) kr[u][v] = *reinterpret_cast<const u4*>(base + k_off[v]);
            if constexpr (DT == MIMIR_KV_I8) ks[u] = *reinterpret_cast<const f4*>(p.c.k_scale + st.at[u] + 4 * hg);
        }
    };
    const auto load_v = [&](const Step& st) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* base = p.c.v + st.at[u] * row_bytes;
#pragma unroll
            for (int e = 0; e < 4; ++e) vr.load(4 * u + e, base + v_off + e * row_bytes);
            if constexpr (DT == MIMIR_KV_I8) vs[u] = *reinterpret_cast<const f4*>(p.c.v_scale + st.at[u] + 4 * hg);
        }
    };

    f4r o[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t) o[t] = f4r{0.f, 0.f, 0.f, 0.f};
    float m_run = -1e30f, l_run = 0.f;  // the max is the row's, the sum this lane's share

    constexpr int kStep = kKeys * kStreamWaves;
    int key = k0 + wave * kKeys;
    Step st{}, nx{};  // this step's, and the next one's, found a step ahead of its loads
    if (key < k1) {
        st = find(key);
        load_k(st);
        load_v(st);
        nx = find(key + kStep);
    }
    // One step.  more: the next one's loads are issued in between, K's once the scores
    // have read this one's, V's at the end; compiled apart from the last step, so that
    // the waits for loads in flight count them.
    const auto step = [&](auto more) {
        int at = lane;
        asm volatile("" : "+v"(at));  // read here in each step, not held in registers across them
        const u4* const mine = q_lds + at;
        f4r s[2] = {f4r{0.f, 0.f, 0.f, 0.f}, f4r{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            const Split8 q{mine[(3 * c) * kWave], mine[(3 * c + 1) * kWave], mine[(3 * c + 2) * kWave]};
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] = mfma16_split(K::operand(kr[u], c), q, s[u]);
        }
        f4 scale[2];
        if constexpr (DT == MIMIR_KV_I8) {
            scale[0] = ks[0];
            scale[1] = ks[1];
        }
        if constexpr (decltype(more)::value) load_k(nx);

        float x[8];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * u + r] = DT == MIMIR_KV_I8 ? s[u][r] * scale[u][r] : s[u][r];
        // Rows whose keys end inside the step, and halves that are not there: the
        // weights are 0 and, where no row of the tile sees a key, so are its values
        // (what is stored there may be anything).
        const bool edge = !st.has[0] || !st.has[1] || __any(key + kKeys > my_end);
        if (edge) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = key + 16 * u + 4 * hg + r;
                    x[4 * u + r] = st.has[u] && j < my_end ? x[4 * u + r] : -INFINITY;
                    if (!st.has[u] || j >= k1) {
                        vr.clear(4 * u + r);
                        if constexpr (DT == MIMIR_KV_I8) vs[u][r] = 0.f;
                    }
                }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
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
        for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_amdgcn_exp2f(x[e] - m_run);
            l_run += x[e];
            if constexpr (DT == MIMIR_KV_I8) x[e] *= vs[e / 4][e % 4];
        }
        const Split8 pw = split8(x);
#pragma unroll
        for (int t = 0; t < ND; ++t) o[t] = mfma16_split(vr.operand(t), pw, o[t]);
        if constexpr (decltype(more)::value) load_v(nx);
    };
    for (; key + kStep < k1; key += kStep) {
        const Step after = find(key + 2 * kStep);
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
    const auto part_row = [&](int row) {
        return a.part + ((static_cast<int64_t>(block) * a.splits + split) * a.rows + row) * (p.c.head_dim + 2);
    };
    for (int x = threadIdx.x; x < w.rows * p.c.head_dim; x += kStreamWaves * kWave) {
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
    if (bad == 0) return;
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

// The splits of one row: brought to one max, added up by four waves and divided.
__global__ __launch_bounds__(kBlock) void paged_join(StreamArgs a) {
    __shared__ float share[kBlock / kWave][kKvMaxDim];
    const auto block = blockIdx.x / static_cast<uint32_t>(a.rows);
    const int row = static_cast<int>(blockIdx.x % static_cast<uint32_t>(a.rows));
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const StreamWork w = stream_work(a, block);
    if (row >= w.rows || w.end <= a.span) return;
    const int d = a.p.c.head_dim, n = (w.end + a.span - 1) / a.span;
    const float* part = a.part + (static_cast<int64_t>(block) * a.splits * a.rows + row) * (d + 2);
    const int64_t step = static_cast<int64_t>(a.rows) * (d + 2);
    float m = -1e30f, l = 0.f, acc[kRowChunks];
    for (int s = lane; s < n; s += kWave) m = fmaxf(m, part[s * step]);
    m = wave_max(m);
    for (int s = lane; s < n; s += kWave) l += part[s * step + 1] * __builtin_amdgcn_exp2f(part[s * step] - m);
    l = wave_sum(l);
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) acc[c] = 0.f;
#pragma unroll 4
    for (int s = wave; s < n; s += kBlock / kWave) {
        const float f = __builtin_amdgcn_exp2f(part[s * step] - m);
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c)
            if (lane + c * kWave < d) acc[c] += part[s * step + 2 + lane + c * kWave] * f;
    }
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) share[wave][lane + c * kWave] = acc[c];
    __syncthreads();
    const int x = static_cast<int>(threadIdx.x);
    if (x >= d) return;
    const int r = w.row0 + row;
    a.p.out[(w.seq.first + r / a.p.group) * a.p.ld_out + static_cast<int64_t>(w.head * a.p.group + r % a.p.group) * d + x] =
        ((share[0][x] + share[1][x]) + (share[2][x] + share[3][x])) * (1.0f / (l + 1e-9f));
}
static_assert(kKvMaxDim <= kBlock && kBlock / kWave == 4, "a thread per dimension, four waves");

template <int DT>
void launch_stream_dim(const StreamArgs& a, unsigned grid, hipStream_t s) {
    constexpr int kThreads = kStreamWaves * kWave;
    if (a.p.c.stride <= 64) paged_stream<DT, 64><<<grid, kThreads, 0, s>>>(a);
    else if (a.p.c.stride <= 128) paged_stream<DT, 128><<<grid, kThreads, 0, s>>>(a);
    else paged_stream<DT, 256><<<grid, kThreads, 0, s>>>(a);
}

int launch_stream(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t most_rows) {
    StreamArgs a{};
    a.p = p;
    a.most_rows = static_cast<int32_t>(most_rows);
    const int64_t rows = std::min(static_cast<int64_t>(p.b.max_new) * p.group, most_rows);
    a.row_blocks = static_cast<int32_t>((rows + kRows - 1) / kRows);
    a.rows = static_cast<int32_t>(std::min<int64_t>(rows, kRows));
    const int64_t blocks = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads * a.row_blocks;
    constexpr int64_t kGrain = kKeys * kStreamWaves, kTarget = 2048;
    const int64_t grains = std::max<int64_t>(1, (p.b.max_len + kGrain - 1) / kGrain);
    int64_t splits = std::min(grains, std::max<int64_t>(1, kTarget / blocks));
    if (ctx->tune.decode_splits > 0) splits = std::min<int64_t>(grains, ctx->tune.decode_splits);
    const int64_t floats = blocks * a.rows * (p.c.head_dim + 2);
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, kFixedWorkBytes / 4 / floats));
    a.part = splits > 1 ? fixed_work(ctx) : nullptr;
    if (!a.part) splits = 1;
    a.span = static_cast<int32_t>((grains + splits - 1) / splits * kGrain);
    a.splits = static_cast<int32_t>((grains * kGrain + a.span - 1) / a.span);
    if (a.splits == 1) a.part = nullptr;
    MIMIR_REQUIRE(ctx, dispatch_fits(blocks * a.splits, kStreamWaves * kWave) && dispatch_fits(blocks * a.rows, kBlock),
                  "paged attention: grid of %lld workgroups exceeds the limit", (long long)(blocks * a.splits));
    a.blocks = static_cast<uint32_t>(blocks);
    const auto grid = static_cast<unsigned>(blocks * a.splits);
    if (dtype == MIMIR_KV_F32) launch_stream_dim<MIMIR_KV_F32>(a, grid, ctx->stream);
    else if (dtype == MIMIR_KV_BF16) launch_stream_dim<MIMIR_KV_BF16>(a, grid, ctx->stream);
    else launch_stream_dim<MIMIR_KV_I8>(a, grid, ctx->stream);
    if (int st = launched(ctx, "paged_stream")) return st;
    if (!a.part) return MIMIR_OK;
    paged_join<<<static_cast<unsigned>(blocks * a.rows), kBlock, 0, ctx->stream>>>(a);
    return launched(ctx, "paged_join");
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
    return launch_stream(ctx, a, cache->dtype, std::min<int64_t>(static_cast<int64_t>(a.b.max_new) * a.group, INT32_MAX));
}
