// matrix.hpp -- the wide products of a training step (a linear layer's cross
// entropy, linear_ce.hip, and the gated products of a feed-forward block,
// gated_linear.hip) on the bf16 matrix cores, with what follows a product done
// on its registers (an Epi).
//
//   C[n][m] = sum_k A(m, k) B(n, k)
//
// A and B are planes of bf16 in memory: one for bf16 values, three for fp32
// (split.hpp: x = h + m + l, six products), two for a value held closer than
// bf16 beside a bf16 operand.  An operand is kRows (element (r, k) at r * ld + k)
// or kCols (at k * ld + r): a matrix has one layout for every product it is in,
// and no transposed copy is made.
//
// A workgroup computes BM x BN of C, WGM x WGN waves of 32 x 32 blocks.  A step
// takes BK of the contraction: its tiles go from memory to one of two LDS
// buffers by buffer loads that write LDS, while the products of the step before
// run from the other; one barrier a step.  Those loads put the 16 bytes of lane l
// at 16 l of a wave's kilobyte, so the order that keeps reads off each other's
// banks is made by what each lane asks for: 16-byte chunk c of row r stands at
// chunk c ^ swizzle(r).  kRows operands are read in ds_read_b128, kCols ones four
// values of four k at a time by ds_read_b64_tr_b16, which transposes them.  Both
// give lane l row l % 32 and k = 8 (l / 32) .. + 7 of a 32 x 16 operand.
//
// A lane of the product holds one n (l % 32) and, in its 16 registers, m =
// 8 (r / 4) + 4 (l / 32) + r % 4: reductions over m stay in registers, and four
// values of one row of C[n][m] are stored at a time.
//
// Every load's row and k are compared with the operand's own (kOutside, which
// reads zeros), so operands may end anywhere; a chunk of 8 lies within a row, ld
// is a multiple of 8 and the operand 16-byte aligned.
//
// Bound by the power of the matrix cores.  Measured on MI355X (bf16, 8192 tokens, 4096 x
// 32000): with the cross entropy's statistics 1758 us = 1.22 PFLOP/s, with its gradient 1846,
// the gradient's products 1685 (A across the contraction) and 1759 us (both); the library's
// product of this shape 1492 us.  2048 tokens 440 to 475 us = 1.13 to 1.22, the library 445.
// The matrix cores are busy 55 to 60% of the
// cycles at 1.9 GHz; without its global loads the kernel takes 0.83, without its LDS reads
// 0.90 of the time, at lower clocks the fuller they are.  fp32, 614 x 1024 x 32000: 225 to
// 260 us = 155 to 179 TFLOP/s, where fp32 matrix instructions peak at 157; with the cross
// entropy's gradient, stored in three planes, 294.
#pragma once

#include "internal.hpp"
#include "matdeal.hpp"
#include "split.hpp"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace mimir {

enum : int { kRows = 0, kCols = 1 };

struct MatOperand {
    const uint16_t* p;
    int64_t ld;     // elements between rows in memory
    int64_t plane;  // elements between planes
};

struct MatArgs {
    // With two segments the contraction runs over (a[0], b[0]), then (a[1], b[1]);
    // with two batches, or a dual A, a[1] is the second's and b[1] is not read.
    MatOperand a[2], b[2];
    int32_t m, n, k;        // k of one segment
    const int32_t* n_dev;   // not null: n is at most this
    const int32_t* k_dev;   // not null: k is at most this
    int32_t segments, batches;
    int32_t fill, splits;   // how the contraction is split (mat_splits; n may be known on the device alone)

    __device__ __forceinline__ int32_t splits_of(int64_t tiles) const { return mat_splits(fill, splits, tiles * batches); }
};

struct MatAt {
    int32_t m0, n0, m, n;  // the tile's first, and the limits
    int32_t batch, split, splits, tile_m;
    int32_t slice;  // split * batches + batch
};

// Every workgroup runs it once; a workgroup of 64 * WGM * WGN threads.
template <int BM, int BN, int WGM, int WGN, int BK, int PA, int PB, int KA, int KB, bool DUAL = false>
struct MatShape {
    static constexpr int kM = BM, kN = BN, kWaveM = WGM, kWaveN = WGN, kK = BK, kPa = PA, kPb = PB, kKindA = KA, kKindB = KB;
    static constexpr bool kDual = DUAL;
    static constexpr int kWaves = WGM * WGN, kThreads = kWave * kWaves;
    static constexpr int kBm = BM / WGM / 32, kBn = BN / WGN / 32;  // 32 x 32 blocks of a wave
    static constexpr int kSubs = DUAL ? 2 : 1, kSubRows = BM / kSubs, kSubBlocks = kBm / kSubs;
    static constexpr int kPlaneA = BM * BK * 2, kPlaneB = BN * BK * 2;  // bytes
    static constexpr int kStage = PA * kPlaneA + PB * kPlaneB;
    static constexpr int kLds = 2 * kStage;
    static_assert(kLds <= 160 * 1024 && kBm % kSubs == 0 && BK % 16 == 0);
};

// --- one operand's tile: R rows by BK --------------------------------------------

template <int R, int BK, int KIND>
__device__ __forceinline__ constexpr int mat_swizzle(int i) {
    // kRows, of row i: 16 rows' same chunk in the 16 places of the 64 banks.  kCols, of k
    // i: four k's 64 bytes (32 values) in different banks.
    if (KIND == kRows) return BK == 64 ? (i >> 1) & 7 : (i >> 2) & 3;
    return R == 64 ? 4 * ((i >> 1) & 1) : 4 * (i & 3);
}

// LDS writes of 16 bytes a lane, behind each other from `lds` (uniform) on.  In asm:
// the compiler would wait for a builtin's load before any later LDS read, since it
// does not tell the two buffers apart.  The kernel waits itself (mat_landed); nothing
// else in it uses m0, which no clobber list can name.  The s_nop: one wait state from m0
// to the load, and five from a lane read that the compiler may have made for an operand
// just before, which it does not keep apart from assembly.
__device__ __forceinline__ void load_to_lds(uint32_t lds, uint32_t voff, __amdgpu_buffer_rsrc_t rs, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rs), "s"(soff)
                 : "memory");
}
// All but the last N of the wave's loads are there.
template <int N>
__device__ __forceinline__ void mat_landed() {
    static_assert(N < 64);
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

template <int R, int BK, int P, int KIND, int WAVES>
struct MatTile {
    static constexpr int kBytes = R * BK * 2;
    static constexpr int kLoads = kBytes / 1024 / WAVES;  // of a wave, a plane
    static_assert(kLoads >= 1 && kBytes % (1024 * WAVES) == 0);
    static constexpr int kLanes = KIND == kRows ? BK / 8 : R / 8;  // 16-byte chunks of a row of the tile
    static constexpr int kRowsOf = kWave / kLanes;                // rows of the tile in a wave's kilobyte
    // kRows: every load has other rows, each at its own limit, and the same k.  kCols:
    // every load has other k's and the same rows.
    uint32_t off[KIND == kRows ? kLoads : 1];
    int32_t k_mine;

    __device__ __forceinline__ void init(int64_t ld, int32_t rows) {
        const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
        const int r = lane / kLanes, slot = lane % kLanes;
        if constexpr (KIND == kRows) {
            // Loads are WAVES * kRowsOf rows apart, a multiple of the swizzle's 16.
            const int chunk = slot ^ mat_swizzle<R, BK, KIND>(wave * kRowsOf + r);
            k_mine = 8 * chunk;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int row = (j * WAVES + wave) * kRowsOf + r;
                off[j] = row < rows ? static_cast<uint32_t>(row * ld * 2 + 16 * chunk) : kOutside;
            }
        } else {
            k_mine = wave * kRowsOf + r;  // load j: + j * WAVES * kRowsOf, a multiple of the swizzle's four
            const int chunk = slot ^ mat_swizzle<R, BK, KIND>(k_mine);
            off[0] = 8 * chunk < rows ? static_cast<uint32_t>(k_mine * ld * 2 + 16 * chunk) : kOutside;
        }
    }
    static_assert(KIND == kRows || (WAVES * kRowsOf) % 4 == 0 || kLoads == 1);
    static_assert(KIND == kCols || (WAVES * kRowsOf) % 16 == 0);

    // A step from `at` (bytes; the tile's first row, the step's first k) on, `left` of its
    // k inside the contraction, for wave `wave` (uniform).
    __device__ __forceinline__ void load(uint32_t lds, uint64_t at, int64_t plane, uint32_t next, int32_t left, uint32_t wave) const {
        constexpr int kNext = WAVES * kRowsOf;  // kCols: k's from one load to the next, `next` bytes
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                reinterpret_cast<void*>(at + p * plane), 0, 0x7fffffff, kBufferWord3);
            const uint32_t to = lds + p * kBytes + wave * 1024;
            if (left >= BK) {
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    load_to_lds(to + j * WAVES * 1024, off[KIND == kRows ? j : 0], rs, KIND == kRows ? 0 : j * next);
            } else {
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    load_to_lds(to + j * WAVES * 1024,
                                k_mine + (KIND == kRows ? 0 : j * kNext) < left ? off[KIND == kRows ? j : 0] : kOutside, rs,
                                KIND == kRows ? 0 : j * next);
            }
        }
    }
    // Bytes from one load of a step to the next (kCols).
    static __device__ __forceinline__ uint32_t next_of(int64_t ld) { return static_cast<uint32_t>(WAVES * kRowsOf * ld * 2); }
};

// Where the next step of an operand is, in registers: a step's loads are issued without
// a look at the kernel's arguments, whose latency the matrix cores would wait out.
struct MatStream {
    uint64_t at;
    int64_t step, plane;  // bytes
};

template <int KIND, int BK>
__device__ __forceinline__ MatStream mat_stream(const MatOperand& o, int32_t row0, int32_t k0) {
    const int64_t first = KIND == kRows ? row0 * o.ld + k0 : k0 * o.ld + row0;
    return MatStream{reinterpret_cast<uint64_t>(o.p) + 2 * first, KIND == kRows ? 2 * BK : 2 * BK * o.ld, 2 * o.plane};
}

typedef int16_t s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_tr;

// A lane's part of a 32 x 16 operand in a tile.
template <int R, int BK, int KIND>
struct MatRead {
    static constexpr int kBytes = R * BK * 2;

    // Rows row0 .. + 31 (a multiple of 32), k 16 c .. + 15.
    static __device__ __forceinline__ u4 get(const char* tile, int row0, int c, int p) {
        const int lane = threadIdx.x % kWave, li = lane % 32, hf = lane / 32;
        const char* base = tile + p * kBytes;
        if constexpr (KIND == kRows) {
            const int chunk = (2 * c + hf) ^ mat_swizzle<R, BK, KIND>(li);
            return *reinterpret_cast<const u4*>(base + (row0 + li) * (BK * 2) + 16 * chunk);
        } else {
            const int q = lane % 16 / 4;                                   // k % 4
            const int k = 16 * c + 8 * hf + q;
            const int chunk = (row0 / 8 + 2 * (lane / 16 % 2) + lane % 4 / 2);
            const char* a = base + k * (2 * R) + 16 * (chunk ^ mat_swizzle<R, BK, KIND>(k)) + 8 * (lane % 2);
            const char* b = base + (k + 4) * (2 * R) + 16 * (chunk ^ mat_swizzle<R, BK, KIND>(k + 4)) + 8 * (lane % 2);
            const u2 x = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr)a));
            const u2 y = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr)b));
            return u4{x[0], x[1], y[0], y[1]};
        }
    }
};

// --- the product ------------------------------------------------------------------

constexpr int kMatXcds = 8;
constexpr int kMatGroup = 4;  // n tiles that neighbours in the order share

// Workgroup -> tile.  Workgroups go to the XCDs round-robin; each XCD takes a
// contiguous run of the tiles that there are (n may be known on the device alone),
// four n tiles beside each other for each m, so that the 32 tiles in flight on an
// XCD read 8 tiles of A and 4 of B.
template <class S>
__device__ __forceinline__ bool mat_tile_of(const MatArgs& g, MatAt* at) {
    at->m = g.m;
    at->n = g.n_dev ? __builtin_amdgcn_readfirstlane(min(g.n, *g.n_dev)) : g.n;
    const uint32_t tiles_m = (g.m + S::kM / S::kSubs - 1) / (S::kM / S::kSubs), tiles_n = (at->n + S::kN - 1) / S::kN;
    const uint32_t one = tiles_m * tiles_n;
    at->splits = g.splits_of(one);
    const uint32_t total = one * g.batches * at->splits;
    const uint32_t per = (total + kMatXcds - 1) / kMatXcds;
    const uint32_t i = (blockIdx.x % kMatXcds) * per + blockIdx.x / kMatXcds;
    if (blockIdx.x / kMatXcds >= per || i >= total) return false;
    const uint32_t r = i % one, z = i / one;
    at->batch = z % g.batches;
    at->split = z / g.batches;
    at->slice = z;
    const uint32_t group = r / (kMatGroup * tiles_m), first = group * kMatGroup, wide = min(tiles_n - first, uint32_t{kMatGroup});
    const uint32_t in = r - group * kMatGroup * tiles_m;
    at->tile_m = in / wide;
    at->m0 = at->tile_m * (S::kM / S::kSubs);
    at->n0 = (first + in % wide) * S::kN;
    return true;
}

// A wave's blocks of C, and which they are.
template <class S>
struct MatAcc {
    f16v c[S::kBm][S::kBn];
    int wm, wn;  // the wave
    // First row (m, within the tile or, dual, within its half) of block i, first column (n) of block j.
    __device__ __forceinline__ int row(int i) const {
        return wm * (S::kSubRows / S::kWaveM) + 32 * (i % S::kSubBlocks);
    }
    __device__ __forceinline__ int col(int j) const { return wn * (S::kN / S::kWaveN) + 32 * j; }
    // m of register r of block i, within the tile.
    __device__ __forceinline__ int m_of(int i, int r) const {
        return row(i) + 8 * (r / 4) + 4 * (threadIdx.x % kWave / 32) + r % 4;
    }
    // First m of the eight that a lane has of registers 8 h .. + 7 after mat_exchange.
    __device__ __forceinline__ int m_of8(int i, int h) const {
        return row(i) + 16 * h + 8 * (threadIdx.x % kWave / 32);
    }
    __device__ __forceinline__ int n_of(int j) const { return col(j) + threadIdx.x % 32; }
};

// Every wave's LDS reads before it are done and every wave's landed loads can be read
// after it; loads still out stay out (__syncthreads would wait for them).
__device__ __forceinline__ void mat_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

// Eight registers of a block as bf16, in their order.
__device__ __forceinline__ u4 mat_pack8(const float* v) {
    return u4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
}
// mat_pack8's values, four of them m 4 hf .. and four 8 + 4 hf .. of a row, as eight
// consecutive ones: the half waves trade (hf: lane / 32).
__device__ __forceinline__ u4 mat_exchange(u4 x) {
    const auto a = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
    return u4{a[0], b[0], a[1], b[1]};
}

// Reads spread between the products of the chunk before.
template <class S>
__device__ __forceinline__ void mat_interleave() {
    constexpr int kPairs = S::kPa == 3 ? 6 : S::kPa + S::kPb - 1;
    constexpr int kReads = S::kPa * S::kBm * (S::kKindA == kCols ? 2 : 1) + S::kPb * S::kBn * (S::kKindB == kCols ? 2 : 1);
    constexpr int kMfma = kPairs * S::kBm * S::kBn;
    constexpr int kEach = (kReads + kMfma - 1) / kMfma;
#pragma unroll
    for (int i = 0; i < kMfma; ++i) {
        if (i * kEach < kReads) __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
}

template <class S, class Epi>
__global__ __launch_bounds__(S::kThreads, S::kThreads == 512 ? 2 : 1) void mat_kernel(MatArgs g, Epi epi) {
    __shared__ __attribute__((aligned(1024))) char lds[S::kLds];
    MatAt at;
    if (!mat_tile_of<S>(g, &at)) return;
    const int32_t k = g.k_dev ? __builtin_amdgcn_readfirstlane(min(g.k, *g.k_dev)) : g.k;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    MatAcc<S> acc;
    acc.wm = wave / S::kWaveN;
    acc.wn = wave % S::kWaveN;

    using TileA = MatTile<S::kSubRows, S::kK, S::kPa, S::kKindA, S::kWaves>;
    using TileB = MatTile<S::kN, S::kK, S::kPb, S::kKindB, S::kWaves>;
    TileA ta;
    TileB tb;
    ta.init(g.a[0].ld, g.m - at.m0);
    tb.init(g.b[0].ld, at.n - at.n0);
    // Steps of this workgroup: the split's share of all segments' steps.
    const int32_t of_one = (k + S::kK - 1) / S::kK, all = of_one * g.segments;
    const int32_t begin = static_cast<int32_t>(static_cast<int64_t>(all) * at.split / at.splits);
    const int32_t end = static_cast<int32_t>(static_cast<int64_t>(all) * (at.split + 1) / at.splits);
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    const uint32_t next_a = __builtin_amdgcn_readfirstlane(TileA::next_of(g.a[0].ld));
    const uint32_t next_b = __builtin_amdgcn_readfirstlane(TileB::next_of(g.b[0].ld));
    MatStream sa[S::kSubs], sb;
    int32_t fetched = begin, left = 0, until = 0;  // the next step to load; its k's left; the segment's end
    const auto seek = [&]() {
        const int seg = g.segments > 1 && fetched >= of_one;
        const int32_t k0 = (fetched - seg * of_one) * S::kK;
        until = (seg + 1) * of_one;
        left = k - k0;
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s)
            sa[s] = mat_stream<S::kKindA, S::kK>(g.a[S::kDual ? s : g.segments > 1 ? seg : at.batch], at.m0, k0);
        sb = mat_stream<S::kKindB, S::kK>(g.b[seg], at.n0, k0);
    };
    const auto load = [&](int buf) {
        const uint32_t to = base + buf * S::kStage;
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s) {
            ta.load(to + s * S::kPa * TileA::kBytes, sa[s].at, sa[s].plane, next_a, left, wave);
            sa[s].at += sa[s].step;
        }
        tb.load(to + S::kPa * S::kPlaneA, sb.at, sb.plane, next_b, left, wave);
        sb.at += sb.step;
        left -= S::kK;
        if (++fetched == until && fetched < end) seek();
    };

#pragma unroll
    for (int i = 0; i < S::kBm; ++i)
#pragma unroll
        for (int j = 0; j < S::kBn; ++j) acc.c[i][j] = f16v{};
    // Three planes: the five small products of a split have sums of their own, 2^-8 the
    // size, so that the sum proper rounds once for 16 of the contraction and not six
    // times (errors against float64 of sums of 1024: 1.2e-6 -> 0.5e-6).
    constexpr bool kTwoSums = S::kPa == 3;
    f16v low[kTwoSums ? S::kBm : 1][kTwoSums ? S::kBn : 1];
    if constexpr (kTwoSums) {
#pragma unroll
        for (int i = 0; i < S::kBm; ++i)
#pragma unroll
            for (int j = 0; j < S::kBn; ++j) low[i][j] = f16v{};
    }
    // Operands of 16 of the contraction, read one ahead of their products.
    u4 a[2][S::kBm][S::kPa], b[2][S::kBn][S::kPb];
    const auto read = [&](int buf, int c, int to) {
        const char* la = lds + buf * S::kStage;
        const char* lb = la + S::kPa * S::kPlaneA;
#pragma unroll
        for (int p = 0; p < S::kPb; ++p)
#pragma unroll
            for (int j = 0; j < S::kBn; ++j) b[to][j][p] = MatRead<S::kN, S::kK, S::kKindB>::get(lb, acc.col(j), c, p);
#pragma unroll
        for (int p = 0; p < S::kPa; ++p)
#pragma unroll
            for (int i = 0; i < S::kBm; ++i)
                a[to][i][p] = MatRead<S::kSubRows, S::kK, S::kKindA>::get(la + (i / S::kSubBlocks) * S::kPa * TileA::kBytes,
                                                                          acc.row(i), c, p);
    };
    // The small products first (mfma_split's order where both have three planes).
    const auto multiply = [&](int at) {
        constexpr int kLast = (S::kPa > S::kPb ? S::kPa : S::kPb) - 1;
#pragma unroll
        for (int sum = kLast; sum >= 0; --sum)
#pragma unroll
            for (int pa = S::kPa - 1; pa >= 0; --pa) {
                const int pb = sum - pa;
                if (pb < 0 || pb >= S::kPb) continue;
#pragma unroll
                for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                    for (int j = 0; j < S::kBn; ++j) {
                        f16v& to = kTwoSums && sum > 0 ? low[kTwoSums ? i : 0][kTwoSums ? j : 0] : acc.c[i][j];
                        to = mfma_bf16(a[at][i][pa], b[at][j][pb], to);
                    }
            }
    };
    constexpr int kChunks = S::kK / 16;
    static_assert(kChunks % 2 == 0);
    // Loads are a step ahead of the products.
    if (begin < end) {
        seek();
        load(0);
        mat_landed<0>();
        mat_barrier();
        read(0, 0, 0);
    }
    int buf = 0;
    for (int32_t step = begin; step < end; ++step) {
        // The buffer is the step before's, which every wave has read (the last barrier).
        if (fetched < end) load(buf ^ 1);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            if (c + 1 < kChunks) {
                read(buf, c + 1, (c + 1) & 1);
            } else if (step + 1 < end) {
                mat_landed<0>();
                mat_barrier();
                read(buf ^ 1, 0, 0);
            }
            multiply(c & 1);
            mat_interleave<S>();
        }
        buf ^= 1;
    }
    if constexpr (kTwoSums) {
#pragma unroll
        for (int i = 0; i < S::kBm; ++i)
#pragma unroll
            for (int j = 0; j < S::kBn; ++j) acc.c[i][j] += low[i][j];
    }
    __syncthreads();  // the epilogue may use the LDS
    epi.template run<S>(at, acc, lds);
}

template <class S>
int64_t mat_tiles(const MatArgs& g) {
    const int64_t tm = S::kM / S::kSubs;
    return (g.m + tm - 1) / tm * ((g.n + S::kN - 1) / S::kN) * g.batches;
}

// The two shapes of a product with PA and PB planes: a CU's workgroup of eight waves
// where such tiles fill most of the GPU, else four waves, two or more to a CU.
template <int PA, int PB, int KA, int KB, bool DUAL = false>
using MatBig = std::conditional_t<PA == 3, MatShape<256, 128, 4, 2, 32, 3, 3, KA, KB, DUAL>,
                                  MatShape<256, 256, 2, 4, 64, PA, PB, KA, KB, DUAL>>;
template <int PA, int PB, int KA, int KB, bool DUAL = false>
using MatSmall = std::conditional_t<PA == 3, MatShape<128, 64, 2, 2, 32, 3, 3, KA, KB, DUAL>,
                                    MatShape<128, 128, 2, 2, 64, PA, PB, KA, KB, DUAL>>;
// A contraction of a few steps is over before a workgroup's stores are: smaller
// stages, so that more workgroups share a CU.
// Measured, both gradients, us, these / the others: cross entropy bf16 4096 x 32000, 9
// tokens' dw alone 75 / 154, 65 tokens 290 / 362, 128 322 / 383, 256 342 / 340, 400 452 / 435,
// 512 499 / 465; gated 4096 x 11008, 65 tokens 152 / 207, 256 183 / 203, 512 266 / 268, 700
// 345 / 333.  Three planes gain nothing by it (134 us against the larger tiles' 121 for 2 x
// 4096 x 11008).
template <int PA, int PB, int KA, int KB>
using MatThin = MatShape<128, 128, 2, 2, 32, PA, PB, KA, KB>;
constexpr int64_t kMatThinK = 256;
// More than 128 larger tiles are one round of the GPU's CUs where four times as many
// smaller ones are two rounds of two to a CU; up to 128 they are one round of both.
// Measured, a cross entropy's forward, us, larger / smaller tiles: bf16 512 x 4096 x 16384,
// 128 larger tiles, 98 / 82, x 17000, 134 of them, 97 / 125; 64 x 4096 x 32000, 125, 104 / 81;
// 1024 x 1024 x 8192, 128, 41 / 33, x 8500, 136, 42 / 46; fp32 512 x 2048 x 8192, 128, 163 /
// 141, x 8500, 136, 165 / 204; 256 x 512 x 16384, 128, 63 / 56, x 17000, 134, 65 / 74.
constexpr int64_t kMatBigTiles = 129;
template <class S>
bool mat_fills(const mimir_ctx* ctx, const MatArgs& g) {
    return ctx->tune.mat_big >= 0 ? ctx->tune.mat_big == 1 : mat_tiles<S>(g) >= kMatBigTiles;
}

// The byte offsets within a tile fit 31 bits.
inline bool mat_ld_fits(int64_t ld) { return ld < (int64_t{1} << 20); }

template <class S, class Epi>
int mat_launch(mimir_ctx* ctx, const char* what, const MatArgs& g, const Epi& epi) {
    // Fewer n than there may be have fewer tiles and more splits: `fill` workgroups at most.
    const int64_t grid = mat_round(std::max<int64_t>(mat_tiles<S>(g), g.fill), kMatXcds);
    MIMIR_REQUIRE(ctx, dispatch_fits(grid, S::kThreads), "%s: grid of %lld workgroups exceeds the limit", what, (long long)grid);
    mat_kernel<S, Epi><<<static_cast<unsigned>(grid), S::kThreads, 0, ctx->stream>>>(g, epi);
    return launched(ctx, what);
}

// Vectors at an address that is a multiple of their elements' size: gfx950 loads and
// stores them as it does aligned ones.
typedef uint32_t u4e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2e __attribute__((ext_vector_type(2), aligned(2)));

// --- products of few tokens ---------------------------------------------------------
//
// Up to 32 n: the time is A's bytes (the weights').  A workgroup has a tile of C, or
// one of the slices of its contraction (MatOut's): of each segment, `splits`.  Each wave of a workgroup has its
// own share of the contraction and its own ring of LDS stages, filled as mat_kernel's
// are, so nothing waits for another wave before the end, where the waves' sums meet in
// LDS.  FP32: both operands are fp32 in memory and are split as they are read from LDS
// (their planes would be five times the bytes on the way).  Of each wave's three stages
// two are on their way: 4 waves of 2 x 8 KB of A a CU are 17 MB in flight on the GPU.
// Measured: 32 x 4096 x 32000 bf16 42 us in the kernel, 6.2 TB/s (75 behind a step whose
// gradients, as large, are on their way to memory); 17 x 4096 x 32000 fp32 128 us, 4.1 TB/s;
// kCols operands, whose tiles are 64 or 128 bytes of each row, 8 x 4096 x 11008, both
// weights: bf16 40 us = 4.5 TB/s, fp32 111 = 3.2.

constexpr int kFewN = 32;

// 32 rows of a raw fp32 operand, BK = 32: kRows 128 bytes a row, kCols 128 bytes a k.
// Rows begin at any float.  Where a row ends inside a 16-byte chunk, the chunk's last
// floats of the row were loaded, so that nothing behind it is read: they stand at the
// chunk's end.  kRows, TAIL: `left` k's of the tile are inside.  kCols: the lane's column stands `shift` floats further (few_shift).
template <int KIND, bool TAIL>
__device__ __forceinline__ Split8 few_read32(const char* tile, int c, int left, int shift) {
    const int lane = threadIdx.x % kWave, li = lane % 32, hf = lane / 32;
    float x[8];
    if constexpr (KIND == kRows) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 16 * c + 8 * hf + 4 * h;
            f4 v = *reinterpret_cast<const f4*>(tile + li * 128 + 16 * (k / 4 ^ mat_swizzle<32, 64, kRows>(li)));
            if (TAIL && left % 4 && k < left && k + 4 > left) {
                const int by = 4 - left % 4;
                v = f4{by == 1 ? v[1] : by == 2 ? v[2] : v[3], by == 1 ? v[2] : by == 2 ? v[3] : 0.0f, by == 1 ? v[3] : 0.0f, 0.0f};
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * h + e] = v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const float*>(tile + (16 * c + 8 * hf + e) * 128 + 4 * (li + shift));
    }
    return split8(x);
}
// Of the lane's column, `rows` columns left of the matrix: those in its last, cut chunk.
__device__ __forceinline__ int few_shift(int32_t rows) {
    const int li = threadIdx.x % 32;
    return rows < 32 && rows % 4 && li < rows && li >= rows - rows % 4 ? 4 - rows % 4 : 0;
}
// Bytes that a load of the chunk from `at` on goes back where only `left` are left.
__device__ __forceinline__ uint32_t few_back(int32_t at, int32_t left) {
    return left - at < 4 ? 4 * (4 - (left - at)) : 0;
}

// The same of bf16, BK = 64: kCols 64 bytes a k.
template <int KIND>
__device__ __forceinline__ u4 few_read16(const char* tile, int c) {
    if constexpr (KIND == kRows) {
        return MatRead<32, 64, kRows>::get(tile, 0, c, 0);
    } else {
        const int lane = threadIdx.x % kWave;
        const char* a = tile + (16 * c + 8 * (lane / 32) + lane % 16 / 4) * 64 + 32 * (lane / 16 % 2) + 8 * (lane % 4);
        const u2 x = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr)a));
        const u2 y = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr)(a + 4 * 64)));
        return u4{x[0], x[1], y[0], y[1]};
    }
}

// WAVES waves, BLOCKS blocks of 32 rows of A (DUAL: half of them of a[0], half of a[1]).
template <int WAVES, int BLOCKS, int STAGES, bool FP32, int KA, bool DUAL>
struct FewShape {
    static constexpr int kM = 32 * BLOCKS, kN = kFewN, kWaveN = 1, kThreads = kWave * WAVES, kKindA = KA;
    static constexpr bool kDual = DUAL;
    static constexpr int kSubs = DUAL ? 2 : 1, kSubRows = kM / kSubs, kSubBlocks = 1;
    // The epilogue: a block (DUAL: one of each) a wave.
    static constexpr int kBm = kSubs, kBn = 1, kWaveM = BLOCKS / kSubs;
    static constexpr int kK = FP32 ? 32 : 64;
    static constexpr int kTile = 4096;  // bytes of 32 rows of kK
    static constexpr int kStage = (BLOCKS + 1) * kTile, kRing = STAGES * kStage, kLds = WAVES * kRing;
    static_assert(kLds <= 160 * 1024 && kWaveM <= WAVES && WAVES * BLOCKS * 4096 <= kLds);
};

template <int WAVES, int BLOCKS, int STAGES, bool FP32, int KA, bool DUAL, class Epi>
__global__ __launch_bounds__(kWave* WAVES, 1) void few_kernel(MatArgs g, Epi epi) {
    using S = FewShape<WAVES, BLOCKS, STAGES, FP32, KA, DUAL>;
    constexpr int kSize = FP32 ? 4 : 2, kChunk = 16 / kSize;  // bytes of an element, elements of 16 bytes
    // Offsets count from here before their row's step, so that those that go back stay positive.
    constexpr int kBefore = FP32 ? 16 : 0;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLds];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    MatAt at{};
    const uint32_t tiles = (g.m + S::kM / S::kSubs - 1) / (S::kM / S::kSubs);
    at.m = g.m;
    at.n = g.n_dev ? __builtin_amdgcn_readfirstlane(min(g.n, *g.n_dev)) : g.n;
    // Neighbouring tiles on one XCD, as mat_tile_of deals them: kCols tiles are 128 bytes
    // of each row, and their neighbours read the next.
    const uint32_t total = gridDim.x, per = (total + kMatXcds - 1) / kMatXcds, full = total - (per - 1) * kMatXcds;
    const uint32_t xcd = blockIdx.x % kMatXcds;  // the first `full` of them have `per` workgroups, the others one less
    const uint32_t id = xcd * per - (xcd > full ? xcd - full : 0) + blockIdx.x / kMatXcds;
    at.tile_m = id % tiles;
    at.slice = id / tiles;  // of the contraction: split of segment
    const int seg = DUAL ? 0 : at.slice % g.segments;
    at.m0 = at.tile_m * (S::kM / S::kSubs);

    // Rows of 128 bytes: eight lanes a row.  kCols bf16: 64 bytes of 32 values a k, four lanes.
    constexpr bool kWide = KA == kRows || FP32;
    constexpr int kLanesA = kWide ? 8 : 4, kRowsOfA = kWave / kLanesA, kLoads = S::kTile / 1024;
    const int ra = lane / kLanesA, slot_a = lane % kLanesA, rb = lane / 8, slot_b = lane % 8;
    int shift[BLOCKS];  // kCols fp32: of the lane's column in each block
    uint32_t off_a[BLOCKS][KA == kRows ? kLoads : 1], off_b[kLoads];
    int32_t k_a[KA == kRows ? kLoads : 1], k_b[kLoads];
    const int64_t lda = g.a[0].ld * kSize, ldb = g.b[0].ld * kSize;  // bytes
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int row = j * 8 + rb, chunk = slot_b ^ mat_swizzle<32, 64, kRows>(row);
        k_b[j] = kChunk * chunk;
        off_b[j] = row < at.n ? static_cast<uint32_t>(row * ldb + 16 * chunk + kBefore) : kOutside;
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const int32_t rows = g.m - at.m0 - 32 * (DUAL ? b % (BLOCKS / 2) : b);  // of this block on
        shift[b] = FP32 && KA == kCols ? few_shift(rows) : 0;
        if constexpr (KA == kRows) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int row = j * 8 + ra, chunk = slot_a ^ mat_swizzle<32, 64, kRows>(row);
                k_a[j] = kChunk * chunk;
                off_a[b][j] = row < rows ? static_cast<uint32_t>(row * lda + 16 * chunk + kBefore) : kOutside;
            }
        } else {
            k_a[0] = ra;
            off_a[b][0] = kChunk * slot_a < rows ? static_cast<uint32_t>(ra * lda + 16 * slot_a + kBefore) : kOutside;
            if constexpr (FP32)
                if (kChunk * slot_a < rows) off_a[b][0] -= few_back(kChunk * slot_a, rows);
        }
    }

    // The wave's share of its segment's steps, `splits` workgroups to a tile.
    const int32_t all = (g.k + S::kK - 1) / S::kK, parts = WAVES * g.splits, part_of = at.slice / g.segments * WAVES + wave;
    const int32_t begin = static_cast<int32_t>(static_cast<int64_t>(all) * part_of / parts);
    const int32_t end = static_cast<int32_t>(static_cast<int64_t>(all) * (part_of + 1) / parts);
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds)) + wave * S::kRing;
    uint64_t pa[BLOCKS], pb = reinterpret_cast<uint64_t>(g.b[seg].p) + int64_t{begin} * 128;
    const int64_t step_a = KA == kRows ? 128 : S::kK * lda;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const MatOperand& o = g.a[DUAL ? b / (BLOCKS / 2) : seg];
        const int64_t row = at.m0 + 32 * (DUAL ? b % (BLOCKS / 2) : b);
        pa[b] = reinterpret_cast<uint64_t>(o.p) + (KA == kRows ? row * lda : row * kSize) + begin * step_a;
    }
    int32_t fetched = begin;
    const auto load = [&](int stage) {
        const int32_t left = g.k - fetched * S::kK;
        const uint32_t to = base + stage * S::kStage;
        const auto rsrc = [](uint64_t p) {
            return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(p - kBefore), 0, 0x7fffffff, kBufferWord3);
        };
        // A chunk's offset in the last step, which its row may end in.
        const auto tail = [&](uint32_t off, int32_t k) { return k < left && off != kOutside ? off - (FP32 ? few_back(k, left) : 0) : kOutside; };
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const auto rs = rsrc(pa[b]);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                if constexpr (KA == kRows)
                    load_to_lds(to + b * S::kTile + j * 1024, left >= S::kK ? off_a[b][j] : tail(off_a[b][j], k_a[j]), rs, 0);
                else
                    load_to_lds(to + b * S::kTile + j * 1024, k_a[0] + j * kRowsOfA < left ? off_a[b][0] : kOutside, rs,
                                __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(j * kRowsOfA * lda)));
            }
            pa[b] += step_a;
        }
        const auto rs = rsrc(pb);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            load_to_lds(to + BLOCKS * S::kTile + j * 1024, left >= S::kK ? off_b[j] : tail(off_b[j], k_b[j]), rs, 0);
        pb += 128;
        ++fetched;
    };

    f16v acc[BLOCKS], low[FP32 ? BLOCKS : 1];  // low: as mat_kernel's
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) acc[b] = f16v{};
    if constexpr (FP32) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) low[b] = f16v{};
    }
    constexpr int kLater = (STAGES - 2) * (BLOCKS + 1) * kLoads;
    for (int i = 0; i < STAGES - 1 && fetched < end; ++i) load(i);
    int buf = 0;
    for (int32_t step = begin; step < end; ++step) {
        if (step + STAGES - 1 <= end) mat_landed<kLater>();
        else mat_landed<0>();
        const char* tile = lds + wave * S::kRing + buf * S::kStage;
        const char* tb = tile + BLOCKS * S::kTile;
        const int32_t inside = g.k - step * S::kK;
        const auto multiply = [&](auto tail) {
            constexpr bool kTail = decltype(tail)::value;
#pragma unroll
            for (int c = 0; c < S::kK / 16; ++c) {
                if constexpr (FP32) {
                    const Split8 x = few_read32<kRows, kTail>(tb, c, inside, 0);
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b) {
                        const Split8 y = few_read32<KA, kTail>(tile + b * S::kTile, c, inside, KA == kCols ? shift[b] : 0);
                        low[b] = mfma_bf16(y.l, x.h, low[b]);
                        low[b] = mfma_bf16(y.h, x.l, low[b]);
                        low[b] = mfma_bf16(y.m, x.m, low[b]);
                        low[b] = mfma_bf16(y.m, x.h, low[b]);
                        low[b] = mfma_bf16(y.h, x.m, low[b]);
                        acc[b] = mfma_bf16(y.h, x.h, acc[b]);
                    }
                } else {
                    const u4 x = MatRead<32, 64, kRows>::get(tb, 0, c, 0);
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b) acc[b] = mfma_bf16(few_read16<KA>(tile + b * S::kTile, c), x, acc[b]);
                }
            }
        };
        if (FP32 && inside < S::kK) multiply(std::true_type{});
        else multiply(std::false_type{});
        // The stage that was read is the next to be filled: its reads are in registers.
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        if (fetched < end) load(buf ? buf - 1 : STAGES - 1);
        buf = buf + 1 < STAGES ? buf + 1 : 0;
    }
    if constexpr (FP32) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) acc[b] += low[b];
    }
    __syncthreads();
    float* part = reinterpret_cast<float*>(lds);  // [wave][block][register][lane]
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) part[((wave * BLOCKS + b) * 16 + r) * kWave + lane] = acc[b][r];
    __syncthreads();
    MatAcc<S> sum;
    sum.wm = wave;
    sum.wn = 0;
    if (wave < S::kWaveM) {
#pragma unroll
        for (int i = 0; i < S::kBm; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v += part[((w * BLOCKS + i * S::kWaveM + wave) * 16 + r) * kWave + lane];
                sum.c[i][0][r] = v;
            }
    } else {
        at.n = 0;  // no part of the result
#pragma unroll
        for (int i = 0; i < S::kBm; ++i) sum.c[i][0] = f16v{};
    }
    __syncthreads();  // the epilogue may use the LDS
    epi.template run<S>(at, sum, lds);
}


// Operands that few_kernel takes as they are: fp32 rows of at least a chunk, bf16 ones in
// whole, aligned chunks.
inline bool few_direct(bool fp32, const void* p, int64_t ld, int64_t cols) {
    if (fp32) return cols >= 4 && mat_ld_fits(ld);
    return aligned16(p) && ld % 8 == 0 && cols % 8 == 0 && mat_ld_fits(ld);
}

// Four waves have a CU's LDS to themselves.  Two workgroups of two waves sharing it are
// slower, also where tiles number a little more than the CUs (32 x 4096 x 32000 bf16, 500
// tiles: 68 us against 55).
constexpr int kFewBlocks = 2;
template <bool FP32, int KA, bool DUAL, class Epi>
int few_launch(mimir_ctx* ctx, const char* what, const MatArgs& g, const Epi& epi) {
    constexpr int64_t kRowsOf = 32 * kFewBlocks / (DUAL ? 2 : 1);
    const int64_t grid = (g.m + kRowsOf - 1) / kRowsOf * g.segments * g.splits;
    MIMIR_REQUIRE(ctx, dispatch_fits(grid, 4 * kWave), "%s: grid of %lld workgroups exceeds the limit", what, (long long)grid);
    few_kernel<4, kFewBlocks, 3, FP32, KA, DUAL, Epi><<<static_cast<unsigned>(grid), 4 * kWave, 0, ctx->stream>>>(g, epi);
    return launched(ctx, what);
}

// --- C as a result -----------------------------------------------------------------

// out[row(n)][m] (+)= alpha * sum, sum over the pieces and splits of the contraction
// that fp32 slices hold (`partial`, one for each split and batch, row n at n * ld_partial).
// A lane has four m's of a row: one 16-byte (fp32) or 8-byte (bf16) store.
struct MatOut {
    void* out[2];             // of each batch
    int64_t ld;
    const int32_t* row;       // not null: the row of n
    float* partial;           // [splits][batches][n][ld_partial], not null if read or written
    int64_t ld_partial;       // mat_slice_ld(m): mat_product and few_product set it
    const float* count;       // not null: alpha is divided by max(count, 1)
    float alpha;
    int32_t bf16, accumulate;
    int32_t read_partial;     // pieces before this one have left their sums
    int32_t last;             // this piece's sums go to out, not to partial

    __device__ __forceinline__ float factor() const { return count ? alpha / fmaxf(*count, 1.0f) : alpha; }
    __device__ __forceinline__ void put(int batch, int64_t n, int32_t m, int32_t limit, f4 v, float by) const {
        const int64_t r = row ? row[n] : n;
        if (bf16) {
            uint16_t* p = static_cast<uint16_t*>(out[batch]) + r * ld + m;
            f4 old{};
            if (m + 4 <= limit) {
                if (accumulate) {
                    const u2e t = *reinterpret_cast<const u2e*>(p);
                    old = f4{__builtin_bit_cast(float, t[0] << 16), __builtin_bit_cast(float, t[0] & 0xffff0000u),
                             __builtin_bit_cast(float, t[1] << 16), __builtin_bit_cast(float, t[1] & 0xffff0000u)};
                }
                v = v * by + old;
                *reinterpret_cast<u2e*>(p) = u2e{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
                return;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e < limit) {
                    const float x = v[e] * by + (accumulate ? __builtin_bit_cast(float, static_cast<uint32_t>(p[e]) << 16) : 0.0f);
                    p[e] = static_cast<uint16_t>(pack_bf16(x, x));
                }
            return;
        }
        float* p = static_cast<float*>(out[batch]) + r * ld + m;
        if (m + 4 <= limit) {
            f4u* q = reinterpret_cast<f4u*>(p);
            *q = accumulate ? v * by + *q : v * by;
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m + e < limit) p[e] = accumulate ? v[e] * by + p[e] : v[e] * by;
    }

    // Eight consecutive bf16 of a row, nothing to add.
    __device__ __forceinline__ void put8(int batch, int64_t n, int32_t m, int32_t limit, u4 v) const {
        uint16_t* p = static_cast<uint16_t*>(out[batch]) + (row ? row[n] : n) * ld + m;
        if (m + 8 <= limit) {
            *reinterpret_cast<u4e*>(p) = v;
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (m + e < limit) p[e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e % 2)));
    }

    template <class S>
    __device__ __forceinline__ void run(const MatAt& at, MatAcc<S>& acc, char*) const {
        const float by = factor();
        const int64_t slice = at.n * ld_partial;
        const bool plain = bf16 && last && !read_partial && !accumulate;
#pragma unroll
        for (int j = 0; j < S::kBn; ++j) {
            const int32_t n = at.n0 + acc.n_of(j);
            const bool live = n < at.n;
            if (plain) {
#pragma unroll
                for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = acc.c[i][j][8 * h + e] * by;
                        const u4 x = mat_exchange(mat_pack8(v));
                        if (live) put8(at.batch, n, at.m0 + acc.m_of8(i, h), at.m, x);
                    }
                continue;
            }
            if (!live) continue;
#pragma unroll
            for (int i = 0; i < S::kBm; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int32_t m = at.m0 + acc.m_of(i, 4 * q);
                    if (m >= at.m) continue;
                    f4 v{acc.c[i][j][4 * q], acc.c[i][j][4 * q + 1], acc.c[i][j][4 * q + 2], acc.c[i][j][4 * q + 3]};
                    // ld_partial is a multiple of four: a whole vector, past m too.
                    f4* p = reinterpret_cast<f4*>(partial + at.slice * slice + n * ld_partial + m);
                    if (read_partial) v += *p;
                    if (last) put(at.batch, n, m, at.m, v, by);
                    else *p = v;
                }
        }
    }
};

// --- operands from a caller's matrices (matrix.hip) --------------------------------

// Whether bf16 rows can be an operand as they are.
inline bool mat_direct(const void* p, int64_t ld, int64_t cols) {
    return aligned16(p) && ld % 8 == 0 && cols % 8 == 0 && mat_ld_fits(ld);
}

// Eight values from element `at` of src on, `left` of them in the row, to dst, `plane`
// elements to the next plane.
template <bool BF16>
__device__ __forceinline__ void mat_stage8(const void* src, int64_t at, int64_t left, uint16_t* dst, int64_t plane) {
    if constexpr (BF16) {
        const uint16_t* p = static_cast<const uint16_t*>(src) + at;
        u4 v{};
        if (left >= 8) {
            v = *reinterpret_cast<const u4e*>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) v[e / 2] |= static_cast<uint32_t>(p[e]) << (16 * (e % 2));
        }
        *reinterpret_cast<u4*>(dst) = v;
    } else {
        const float* p = static_cast<const float*>(src) + at;
        float x[8];
        if (left >= 8) {
            const f4u a = *reinterpret_cast<const f4u*>(p), b = *reinterpret_cast<const f4u*>(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = e < left ? p[e] : 0.0f;
        }
        const Split8 s = split8(x);
        *reinterpret_cast<u4*>(dst) = s.h;
        *reinterpret_cast<u4*>(dst + plane) = s.m;
        *reinterpret_cast<u4*>(dst + 2 * plane) = s.l;
    }
}

// dst [planes][.][ld_dst]: `rows` rows of `cols`, split into planes (fp32: three,
// bf16: one), zeros up to ld_dst (a multiple of 8, at least cols).  plane: elements
// between planes.
int mat_stage(mimir_ctx* ctx, int type, const void* src, int64_t rows, int64_t cols, int64_t ld, uint16_t* dst, int64_t ld_dst,
              int64_t plane);
// A matrix of zeros.
int mat_zero(mimir_ctx* ctx, int type, void* p, int64_t rows, int64_t cols, int64_t ld);
// mat_deal_of for the shapes of these planes and layouts.
template <class BIG, class SMALL, bool HAS_BIG, bool HAS_THIN>
MatDeal mat_deal(const mimir_ctx* ctx, int64_t m, int64_t n, int64_t k, int64_t batches, bool more) {
    return mat_deal_of({{BIG::kM, BIG::kN}, {SMALL::kM, SMALL::kN}, HAS_BIG, HAS_THIN, kMatBigTiles, kMatThinK, ctx->tune.mat_big}, m, n, k,
                       batches, more);
}
template <int PA, int PB, int KA, int KB>
MatDeal mat_deal(const mimir_ctx* ctx, int64_t m, int64_t n, int64_t k, int64_t batches, bool more) {
    using S = MatSmall<PA, PB, KA, KB>;
    if constexpr (PA == PB) return mat_deal<MatBig<PA, PB, KA, KB>, S, true, PA != 3>(ctx, m, n, k, batches, more);
    else return mat_deal<S, S, false, true>(ctx, m, n, k, batches, more);
}

// The sum of the splits' slices into out (MatOut's fields say how) for a product of g in
// tiles of `tile`.
int mat_join(mimir_ctx* ctx, const MatOut& o, const MatArgs& g, MatTileSize tile);

// An fp32 product of few n into MatOut through slices: workgroups for about two for each
// CU, each wave with at least four steps of 32.
inline int few_splits(int64_t m, int64_t k, int segments) {
    const int64_t tiles = (m + 63) / 64 * segments, steps = (k + 31) / 32;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(tiles, 1), steps / 16, 64})));
}
template <int KA>
int few_product(mimir_ctx* ctx, const char* what, MatArgs g, MatOut o) {
    const int32_t last = o.last, splits = g.splits, segments = g.segments;
    o.ld_partial = mat_slice_ld(g.m);
    o.last = last && splits * segments == 1;
    if (int st = few_launch<true, KA, false>(ctx, what, g, o)) return st;
    if (!last || o.last) return MIMIR_OK;
    o.last = 1;
    g.splits = splits * segments;  // mat_join's: as many slices, whatever the tiles
    g.segments = 1;
    g.fill = INT32_MAX;
    return mat_join(ctx, o, g, MatTileSize{1 << 24, 1 << 24});
}

// C as a result.  o.last: these are the contraction's last pieces.
template <int PA, int PB, int KA, int KB>
int mat_product(mimir_ctx* ctx, const char* what, MatArgs g, MatOut o, const MatDeal& d) {
    g.splits = d.splits;
    g.fill = d.fill;
    o.ld_partial = mat_slice_ld(g.m);
    const int32_t last = o.last;
    if (d.splits > 1) o.last = 0;
    int st = MIMIR_OK;
    using S = MatSmall<PA, PB, KA, KB>;
    MatTileSize tile{S::kM, S::kN};
    if constexpr (PA == PB) {
        using B = MatBig<PA, PB, KA, KB>;
        if (d.big) tile = MatTileSize{B::kM, B::kN};
    }
    MIMIR_REQUIRE(ctx, (o.last && !o.read_partial) || mat_slice_bytes(d, tile, g.m, g.n, g.batches) <= d.partial,
                  "%s: %d x %d in %zu bytes of slices", what, g.m, g.n, d.partial);
    if constexpr (PA == PB)
        if (d.big) st = mat_launch<MatBig<PA, PB, KA, KB>>(ctx, what, g, o);
    if constexpr (PA != 3)
        if (d.thin) st = mat_launch<MatThin<PA, PB, KA, KB>>(ctx, what, g, o);
    if (!d.thin && !d.big) st = mat_launch<S>(ctx, what, g, o);
    if (st || d.splits == 1 || !last) return st;
    o.last = 1;
    return mat_join(ctx, o, g, tile);
}

// Whether no output is one of the inputs or another output.
inline bool mat_apart(std::initializer_list<const void*> outputs, std::initializer_list<const void*> inputs) {
    for (auto o = outputs.begin(); o != outputs.end(); ++o) {
        if (!*o) continue;
        if (std::find(inputs.begin(), inputs.end(), *o) != inputs.end() || std::find(o + 1, outputs.end(), *o) != outputs.end()) return false;
    }
    return true;
}

// The context's scratch of at least `bytes`, also while its stream is being captured
// (captured_scratch).
int mat_scratch(mimir_ctx* ctx, size_t bytes, char** out);

}  // namespace mimir
