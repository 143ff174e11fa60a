// attention_paged_stream.hip -- attention over a paged cache for few query rows per
// key / value head (single tokens, a few of them, and the heads that share keys):
// keys and values straight to registers.
//
// A wave takes 32 keys at a time, its workgroup's four waves side by side (a step of
// 128), against 16 query rows, or twice 16 that share the keys' way in.
// - Scores: S^T = K Q^T by v_mfma_f32_16x16x32_bf16, keys as rows.  Lane (li, hg)
//   supplies key li's slots and query li's, 8 of 32 dimensions each; which dimensions
//   a slot stands for is free as long as both sides agree, so a lane loads 16 bytes
//   of a key at a time whatever the type (Kind).  It receives the scores of row li
//   and the keys 4 hg + {0..3} of both halves: its softmax is its own, the max alone
//   is shared with the other three lanes of the row, and only when it has grown by
//   more than kPagedSlack.
// - Output: O^T = V^T P^T over the 32 keys in that order, so the weights feed it as
//   they are; a lane loads the same keys' values, ND dimensions each (Values).
// - Entries of bf16 and 8 bits are exact in one bf16 term, fp32 ones take three, as
//   the queries and weights do: 3 or 6 MFMAs for a product of fp32 precision.  The
//   8-bit scales multiply scores and weights instead of elements.
// - The queries' terms are in LDS (registers they would not fit beside two steps of
//   keys); the four waves' sums are brought to one max there at the end.  No instance
//   keeps vector registers in memory: a form that did (fp32 heads of 256, 100 bytes a
//   lane) gave wrong scores, of which the cause was not found.
//
// Loads: buffer loads without a bounds check in the code (the descriptor of a half of
// 16 keys ends with its keys, what lies behind reads as zero), non-temporal: nothing
// is read twice.  The next step's keys are asked for when the scores have read this
// one's, its values at the end; page numbers two steps ahead through scalar loads.
//
// Bound by memory: 64 sequences x 4096 keys x 8 heads of 128, bf16, 162 us = 6.6 TB/s
// (a copy: 6.4); 8-bit 5.4 TB/s, 64 bytes a lane and step in flight being half as
// many (64 keys a step: no change; fewer instructions: within 10% without any
// arithmetic); fp32, 2048 keys, 5.7 TB/s.  One sequence of 131002 keys 92 us =
// 5.8 TB/s, of them 7 us the join.  Short ones by latency: 101 keys 7 us, a step
// about 1.1 us, the lengths, pages, keys and sums one after the other.
#include "attention_paged.hpp"

#include <math.h>

#include <algorithm>

using namespace mimir;

namespace {

typedef float f4r __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;     // query rows of a tile: (token, head of the group) pairs
constexpr int kNt = 2;        // a buffer load's non-temporal bit
constexpr int kStreamWaves = 4;

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
constexpr int stream_waves(int dtype, int dp, int tiles) {
    return dp == 256 ? 1 : dtype == MIMIR_KV_F32 ? (dp == 128 ? 1 : 2) : dp == 128 || tiles == 2 ? 2 : 4;
}

// TILES: of 16 rows, that share the keys' and values' way in.
template <int DT, int DP, int TILES>
__global__ __launch_bounds__(kStreamWaves * kWave, stream_waves(DT, DP, TILES)) void paged_stream(PagedArgs p, PagedRuns a) {
    using K = Kind<DT, DP>;
    constexpr int ND = DP / 16, kSteps = DP / 32, H = K::kHalves, R = TILES;
    typedef float Share[kRows * R][DP + 2];
    __shared__ __attribute__((aligned(16))) char lds[sizeof(Share) * kStreamWaves];
    Share* const share = reinterpret_cast<Share*>(lds);  // after the keys
    u4* const q_lds = reinterpret_cast<u4*>(lds);        // [tile][step][term][lane], during them
    static_assert(R * kSteps * 3 * kWave * sizeof(u4) <= sizeof lds, "the queries fit");
    __shared__ uint32_t bad;
    __shared__ PagedChunk chunk;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    for (PagedWalk walk(p, a, blockIdx.x, &chunk); walk.more();) {
        int tid = static_cast<int>(threadIdx.x);
        asm volatile("" : "+v"(tid));  // what follows from it is computed for each block, not held in registers across them
        const int lane = tid % kWave, li = lane % 16, hg = lane / 16;
        const PagedPiece w = walk.next(p, a);
        if (w.rows <= 0) return;
        const int k0 = w.k0, k1 = w.k1;
        int my_row[R], my_end[R];
#pragma unroll
        for (int n = 0; n < R; ++n) {
            my_row[n] = w.row0 + min(kRows * n + li, w.rows - 1);
            my_end[n] = min(row_end(p, w.seq, my_row[n]), k1);
        }
        const auto q_row = [&](int row) { return p.q + paged_row(p, p.ld_q, w.seq.first, w.head, row); };
        // The queries' loads go out ahead of the first keys', their terms follow those.
        constexpr int kOwn = (kSteps + kStreamWaves - 1) / kStreamWaves;
        float qx[R][kOwn][8];
#pragma unroll
        for (int n = 0; n < R; ++n) {
            const float* row = q_row(my_row[n]);
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (p.c.head_dim % 4 == 0) {
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const int d = K::dim(wave + i * kStreamWaves, hg, e);
                        const f4u x = d < p.c.head_dim ? *reinterpret_cast<const f4u*>(row + d) : f4u{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int u = 0; u < 4; ++u) qx[n][i][e + u] = x[u];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = K::dim(wave + i * kStreamWaves, hg, e);
                        qx[n][i][e] = d < p.c.head_dim ? row[d] : 0.f;
                    }
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
        // A half's rows; `keys` of them are there, the others read as zeros.
        const auto half_rows = [&](char* base, int64_t at, int keys) {
            return __builtin_amdgcn_make_buffer_rsrc(base + at * row_bytes, 0, keys * row_bytes, kBufferWord3);
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
                const __amdgpu_buffer_rsrc_t rows = half_rows(p.c.k, at, kHalf);
#pragma unroll
                for (int v = 0; v < K::kVecs; ++v) kr[u][v] = __builtin_amdgcn_raw_buffer_load_b128(rows, k_off[v], 0, kNt);
                if constexpr (DT == MIMIR_KV_I8) ks[u] = *reinterpret_cast<const f4*>(p.c.k_scale + at + 4 * hg);
            }
        };
        const auto load_v = [&](const Step& st, int key_of) {
#pragma unroll
            for (int u = 0; u < H; ++u) {
                const int64_t at = st.at(u, p.c, w.head);
                const int keys = st.has(u, p.c) ? min(k1 - (key_of + kHalf * u), kHalf) : 0;
                const __amdgpu_buffer_rsrc_t rows = half_rows(p.c.v, at, keys);
#pragma unroll
                for (int e = 0; e < 4; ++e) vr[u / 2].load(4 * (u % 2) + e, rows, v_off, e * row_bytes);
                if constexpr (DT == MIMIR_KV_I8)
                    vs[u] = buffer_f4(buffer_of(p.c.v_scale + at, 4 * keys), static_cast<uint32_t>(16 * hg));
            }
        };

        f4r o[R][ND];
        float m_run[R], l_run[R];  // the max is the row's, the sum this lane's share
#pragma unroll
        for (int n = 0; n < R; ++n) {
            m_run[n] = -1e30f;
            l_run[n] = 0.f;
#pragma unroll
            for (int t = 0; t < ND; ++t) o[n][t] = f4r{0.f, 0.f, 0.f, 0.f};
        }

        constexpr int kKeys = kHalf * H, kStep = kKeys * kStreamWaves;
        int key = k0 + wave * kKeys;
        Step st{}, nx{}, after{};  // this step's, and the next two's, found a step ahead of their loads
        if (key < k1) {
            st = find(key);
            load_k(st);
            load_v(st, key);
            nx = find(key + kStep);
        }
        __syncthreads();  // the last block's sums and flags are read
        if (tid == 0) bad = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int c = wave + i * kStreamWaves;
            if (c >= kSteps) break;
#pragma unroll
            for (int n = 0; n < R; ++n) {
#pragma unroll
                for (int e = 0; e < 8; ++e) qx[n][i][e] *= p.qscale;
                const Split8 x = split8(qx[n][i]);
                u4* const to = q_lds + 3 * (n * kSteps + c) * kWave + lane;
                to[0] = x.h;
                to[kWave] = x.m;
                to[2 * kWave] = x.l;
            }
        }
        __syncthreads();
        // One step.  more: the next one's loads are issued in between, K's once the scores
        // have read this one's, V's at the end; compiled apart from the last step, so that
        // the waits for loads in flight count them.
        const auto step = [&](auto more) {
            int at = lane;
            asm volatile("" : "+v"(at));  // read here in each step, not held in registers across them
            const u4* const mine = q_lds + at;
            f4r s[R][H];
#pragma unroll
            for (int n = 0; n < R; ++n)
#pragma unroll
                for (int u = 0; u < H; ++u) s[n][u] = f4r{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                typename K::Operand k[H];
#pragma unroll
                for (int u = 0; u < H; ++u) k[u] = K::operand(kr[u], c);
#pragma unroll
                for (int n = 0; n < R; ++n) {
                    const u4* const x = mine + 3 * (n * kSteps + c) * kWave;
                    const Split8 q{x[0], x[kWave], x[2 * kWave]};
#pragma unroll
                    for (int u = 0; u < H; ++u) s[n][u] = mfma16_split(k[u], q, s[n][u]);
                }
                if constexpr (DT == MIMIR_KV_F32) __builtin_amdgcn_sched_barrier(0);  // few terms at a time
            }
            if constexpr (DT == MIMIR_KV_I8) {
#pragma unroll
                for (int n = 0; n < R; ++n)
#pragma unroll
                    for (int u = 0; u < H; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[n][u][r] *= ks[u][r];
            }
            if constexpr (decltype(more)::value) {
                load_k(nx);
                after = find(key + 2 * kStep);  // here, where no LDS read waits for it
            }

            bool holes = false;
#pragma unroll
            for (int u = 0; u < H; ++u) holes = holes || !st.has(u, p.c);
            Split8 pw[R][H / 2];
#pragma unroll
            for (int n = 0; n < R; ++n) {
                float x[4 * H];
#pragma unroll
                for (int e = 0; e < 4 * H; ++e) x[e] = s[n][e / 4][e % 4];
                // Rows whose keys end inside the step, and halves that are not there: the
                // weights are 0 (and values of keys that no row sees were read as zeros).
                if (holes || __any(key + kKeys > my_end[n])) {
#pragma unroll
                    for (int e = 0; e < 4 * H; ++e) {
                        const int u = e / 4, j = key + kHalf * u + 4 * hg + e % 4;
                        x[e] = st.has(u, p.c) && j < my_end[n] ? x[e] : -INFINITY;
                    }
                }
                float top = x[0];
#pragma unroll
                for (int e = 1; e < 4 * H; ++e) top = fmaxf(top, x[e]);
                if (__any(top > m_run[n] + kPagedSlack)) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float m_new = fmaxf(m_run[n], top);
                    const float f = __builtin_amdgcn_exp2f(m_run[n] - m_new);
                    m_run[n] = m_new;
                    l_run[n] *= f;
#pragma unroll
                    for (int t = 0; t < ND; ++t) o[n][t] *= f;
                }
#pragma unroll
                for (int e = 0; e < 4 * H; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(x[e] - m_run[n]);
                    l_run[n] += x[e];
                    if constexpr (DT == MIMIR_KV_I8) x[e] *= vs[e / 4][e % 4];
                }
#pragma unroll
                for (int h = 0; h < H / 2; ++h) pw[n][h] = split8(x + 8 * h);
            }
#pragma unroll
            for (int h = 0; h < H / 2; ++h)
#pragma unroll
                for (int t = 0; t < ND; ++t) {
                    const auto v = vr[h].operand(t);
#pragma unroll
                    for (int n = 0; n < R; ++n) o[n][t] = mfma16_split(v, pw[n][h], o[n][t]);
                    if constexpr (DT == MIMIR_KV_F32)
                        if (t % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                }
            if constexpr (decltype(more)::value) load_v(nx, key + kStep);
        };
        for (; key + kStep < k1; key += kStep) {
            step(std::true_type{});
            st = nx;
            nx = after;
        }
        if (key < k1) step(std::false_type{});

        // The waves' shares of the rows.  Lane (li, hg) holds dimensions (4 hg + r) ND + t.
        __syncthreads();
#pragma unroll
        for (int n = 0; n < R; ++n) {
            l_run[n] += __shfl_xor(l_run[n], 16);
            l_run[n] += __shfl_xor(l_run[n], 32);
            float* const to = share[wave][kRows * n + li];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < ND; ++t) to[(4 * hg + r) * ND + t] = o[n][t][r];
            if (hg == 0) {
                to[DP] = m_run[n];
                to[DP + 1] = l_run[n];
            }
        }
        __syncthreads();
        const auto out_row = [&](int row) { return p.out + paged_row(p, p.ld_out, w.seq.first, w.head, w.row0 + row); };
        const PagedPart part(a, p.c.head_dim, walk.index, w.begins);
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
            if (w.whole) {
                out_row(row)[d] = sum * (1.0f / (l + 1e-9f));
            } else {
                part.sums(row)[d] = sum;
                if (d == 0) *part.stat(row) = f2{m, l};
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
            const float inv = w.whole ? 1.0f / (l + 1e-9f) : 1.0f;
            float* out = w.whole ? out_row(row) : part.sums(row);
#pragma unroll
            for (int c = 0; c < kRowChunks; ++c) {
                const int d = lane + c * kWave;
                if (d < p.c.head_dim) out[d] = acc[c] * inv;
            }
            if (!w.whole && lane == 0) *part.stat(row) = f2{m, l};
        }
    }
}

template <int DT, int TILES>
void launch_dim(const PagedArgs& p, const PagedRuns& a, unsigned grid, hipStream_t s) {
    constexpr int kThreads = kStreamWaves * kWave;
    if (p.c.stride <= 64) paged_stream<DT, 64, TILES><<<grid, kThreads, 0, s>>>(p, a);
    else if (p.c.stride <= 128) paged_stream<DT, 128, TILES><<<grid, kThreads, 0, s>>>(p, a);
    else if constexpr (!(DT == MIMIR_KV_F32 && TILES == 2)) paged_stream<DT, 256, TILES><<<grid, kThreads, 0, s>>>(p, a);
}
template <int DT>
void launch_tiles(const PagedArgs& p, const PagedRuns& a, int tiles, unsigned grid, hipStream_t s) {
    if (tiles == 1) launch_dim<DT, 1>(p, a, grid, s);
    else launch_dim<DT, 2>(p, a, grid, s);
}

// Workgroups that the GPU holds at once.
int64_t stream_resident(int dtype, int stride, int tiles) {
    // Two a compute unit where registers allow them: measured (256 / 512 / 1024 workgroups, us), 64 sequences x
    // 4096 keys x 8 heads x 128: 8-bit 112 / 99 / 105, bf16 168 / 162 / 170; heads of 64: 8-bit 76 / 60 / 60, bf16
    // 88 / 87 / 92, fp32 183 / 168 / 174; heads of 256, one a unit: bf16 120 / 131 / 145.
    return 256 * std::min(2, stream_waves(dtype, stride <= 64 ? 64 : stride <= 128 ? 128 : 256, tiles));
}

}  // namespace

int mimir::paged_stream_launch(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t most_rows, bool beside, PagedRuns* left) {
    constexpr uint32_t kStep = 2 * kHalf * kStreamWaves;
    const int64_t rows = std::min(static_cast<int64_t>(p.b.max_new) * p.group, most_rows);
    // A sequence's second tile shares the first one's keys, unless other sequences have more rows
    // than this kernel takes: then single tokens are what most have.  (Wide fp32 heads,
    // of which two tiles are more than the registers hold, come with one at most.)
    const int tiles = rows > kRows && !beside ? 2 : 1;
    MIMIR_REQUIRE(ctx, tiles == 1 || dtype != MIMIR_KV_F32 || p.c.stride <= 128, "paged attention: %lld rows of a wide head",
                  (long long)rows);
    PagedRuns a{};
    // The queries, the first keys' way in, the sums' way out take as long whatever a key's bytes.  Two / three / four
    // steps, 64 ragged sequences of up to 8191 keys, us: 8-bit heads of 128 115 / 109 / 109, of 64 75 / 67 / 64, bf16
    // of 128, up to 4096, 96 / 97 / 99, fp32 209 / 214 / 217.
    const int64_t key_bytes = 2 * static_cast<int64_t>(p.c.stride) * kv_element_bytes(dtype);
    a.extra = (key_bytes >= 512 ? 2 : key_bytes >= 256 ? 3 : 4) * kStep;
    a.least = 3 * kStep;
    a.slack = 2 * kStep;
    a.grain = kStep;
    a.block_rows = kRows * tiles;
    a.least_rows = 1;
    a.most_rows = static_cast<int32_t>(most_rows);
    a.part_rows = static_cast<int32_t>(std::min<int64_t>(rows, a.block_rows));
    a.row_blocks = static_cast<int32_t>((rows + a.block_rows - 1) / a.block_rows);
    const int64_t blocks = static_cast<int64_t>(p.b.sequences) * p.c.kv_heads * a.row_blocks;
    const int64_t runs = ctx->tune.paged_runs > 0 ? ctx->tune.paged_runs : stream_resident(dtype, p.c.stride, tiles);
    // Short blocks are not worth a join, by the bytes of one where they do not fill the GPU.  Whole / cut, us, two
    // sequences x 8 heads: bf16 heads of 128, 500 keys 10 / 14, 1000 18 / 16; fp32 500 23 / 21, 1000 41 / 28; fp32
    // heads of 256 500 57 / 42; 32 sequences, fp32 heads of 128 and 256, 500 keys 30 / 34, 70 / 74.
    const bool small = p.b.max_len * key_bytes <= 448 * 1024 || 2 * blocks >= runs;
    const bool whole = small && p.b.max_len <= static_cast<int64_t>(8 * kStep);
    const int64_t grid = paged_runs(ctx, p, &a, runs, blocks, kStreamWaves * kWave, !whole, beside);
    MIMIR_REQUIRE(ctx, dispatch_fits(grid, kStreamWaves * kWave), "paged attention: grid of %lld workgroups exceeds the limit",
                  (long long)grid);
    if (dtype == MIMIR_KV_F32) launch_tiles<MIMIR_KV_F32>(p, a, tiles, static_cast<unsigned>(grid), ctx->stream);
    else if (dtype == MIMIR_KV_BF16) launch_tiles<MIMIR_KV_BF16>(p, a, tiles, static_cast<unsigned>(grid), ctx->stream);
    else launch_tiles<MIMIR_KV_I8>(p, a, tiles, static_cast<unsigned>(grid), ctx->stream);
    *left = a;
    return launched(ctx, "paged_stream");
}
