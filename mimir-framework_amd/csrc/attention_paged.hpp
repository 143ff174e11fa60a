// attention_paged.hpp -- what the kernels of attention over a paged cache share:
// their arguments, how the work is dealt to workgroups, the conversion of cache
// entries, and one query row in plain fp32.
#pragma once

#include "kvcache.hpp"
#include "split.hpp"

namespace mimir {

constexpr float kPagedLog2e = 1.4426950408889634f;
// As attention.hip: the running max may lag by this many base-2 units.
constexpr float kPagedSlack = 8.0f;
constexpr int kHalf = 16;  // keys in a row that surely stand in one page

struct PagedArgs {
    KvView c;
    KvBatch b;
    const float* q;
    float* out;
    int64_t ld_q, ld_out;
    int32_t heads, group;  // query heads, those that share a key / value head
    FastDiv group_div;
    float qscale;          // scale * log2(e)
    int32_t causal;
};

// Memory that a kernel only reads, at addresses that a wave shares: scalar loads.
typedef const __attribute__((address_space(4))) int32_t* scalar_i32;

// --- the work --------------------------------------------------------------------
// A block is `block_rows` query rows ((token, head of the group) pairs) of one key /
// value head of a sequence, against the keys that its last row sees.  It costs those
// keys and `extra`.  All blocks' costs, in order of sequence, head and rows, are dealt
// to the workgroups in equal runs, so that sequences of any lengths fill the GPU
// evenly; a run may begin and end inside a block, whose parts paged_join adds up.
// Every wave works out its run from the sequences' lengths, 64 of them at a time.
// Sequences of 1 to 8191 keys, 64 of them x 8 heads, 8-bit: 109 us, with as many parts
// a sequence for all 210.  One sequence of 3000 keys: 20 us, with runs that end where
// blocks do 16; chunks of 217 tokens of 3 sequences over 2700 to 3200 keys 94 and 92.

// A block that a run begins and others go on with.
struct PagedShared {
    int32_t runs;                      // how many have keys of it; 0: none but this one
    int32_t first, row0, rows, head;   // its sequence's first token, its rows, its key / value head
    int32_t pad[3];
};

struct PagedRuns {
    // Blocks that several runs have keys of, by the run that begins them, and their
    // sums (PagedPart).  Null: a run is one whole block.
    PagedShared* shared;
    float* part;
    uint32_t runs;
    uint32_t extra;      // what a block costs besides its keys, in keys
    uint32_t least;      // length of a run at least
    uint32_t slack;      // how much longer a run may be for all to be of one block
    uint32_t grain;      // blocks are cut at multiples of this many keys, a power of two
    int32_t block_rows;
    int32_t part_rows;   // rows of a block that `part` has room for
    int32_t least_rows, most_rows;  // of a sequence's; those with fewer or more are another kernel's
    int32_t many;        // a block may have many runs (paged_join)
    int32_t apart;       // no run need have parts of two blocks (PagedWalk)
    int32_t row_blocks;  // of a sequence with as many rows as the host allows
};

__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    return static_cast<uint64_t>(lane_of(static_cast<uint32_t>(v >> 32), lane)) << 32 | lane_of(static_cast<uint32_t>(v), lane);
}

// Costs of a sequence's row blocks, the same for each of its heads: row block i costs
// base + slope (i + 1), since a causal block's keys end `slope` later than the one
// before it (at the sequence's end at the latest; the last one's cost is too high by
// what it lacks).
struct PagedCost {
    uint32_t base, slope, blocks;
    __device__ __forceinline__ uint64_t ahead(uint32_t i) const {
        return static_cast<uint64_t>(i) * base + static_cast<uint64_t>(slope) * i * (i + 1) / 2;
    }
};

__device__ __forceinline__ PagedCost paged_cost(const PagedArgs& p, const PagedRuns& a, const KvSequence& q) {
    const int64_t rows = static_cast<int64_t>(q.n) * p.group;
    PagedCost c{1, 0, 0};  // base of a sequence without blocks
    if (rows > 0 && rows >= a.least_rows && rows <= a.most_rows)
        c.blocks = static_cast<uint32_t>((rows + a.block_rows - 1) / a.block_rows);
    c.base = a.extra + static_cast<uint32_t>(p.causal ? max(q.len - q.n, 0) : q.len);
    c.slope = p.causal ? static_cast<uint32_t>((a.block_rows + p.group - 1) / p.group) : 0;
    return c;
}

// 64 sequences in LDS, one a lane.
struct PagedChunk {
    uint64_t sum[kWave];  // costs up to the sequence, of this chunk's
    KvSequence seq[kWave];
    PagedCost cost[kWave];
};

// The lanes' sums up to each.
__device__ __forceinline__ uint64_t lanes_up_to(uint64_t sum) {
    const int lane = static_cast<int>(threadIdx.x % kWave);
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) {
        const auto y = static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(sum), x));
        if (lane >= x) sum += y;
    }
    return sum;
}

// The costs of the sequences from `base` on up to the lane's; wave 0 writes them down.
// The lane's own is left in `cost`.
__device__ __forceinline__ uint64_t paged_chunk(const PagedArgs& p, const PagedRuns& a, int base, PagedChunk* chunk,
                                                PagedCost* cost) {
    const int lane = static_cast<int>(threadIdx.x % kWave);
    KvSequence seq{0, 0, 0};
    *cost = PagedCost{1, 0, 0};
    if (base + lane < p.b.sequences) {
        seq = kv_sequence(p.b, base + lane);
        *cost = paged_cost(p, a, seq);
    }
    const uint64_t sum = lanes_up_to(cost->ahead(cost->blocks) * static_cast<uint32_t>(p.c.kv_heads));
    if (threadIdx.x < kWave) {
        chunk->sum[lane] = sum;
        chunk->seq[lane] = seq;
        chunk->cost[lane] = *cost;
    }
    return sum;
}

// Keys that row `row` (of all its sequence's) sees.
__device__ __forceinline__ int row_end(const PagedArgs& p, const KvSequence& q, int row) {
    if (!p.causal) return q.len;
    return min(max(q.len - q.n + static_cast<int>(fastdiv(static_cast<uint32_t>(row), p.group_div)) + 1, 0), q.len);
}

// A run's part of a block.
struct PagedPiece {
    int s, head, row0, rows;  // sequence, key / value head, first row and rows of the block
    KvSequence seq;
    int k0, k1;               // keys
    bool whole, begins;       // all of the block's keys; the first of them
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}

__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 | uniform(static_cast<uint32_t>(x));
}

// x / y without the long way of a 64-bit division: its rounding is put right by the
// remainder (a quotient of up to 53 bits is off by 1 at most).
__device__ __forceinline__ uint64_t quotient(uint64_t x, uint64_t y) {
    auto q = static_cast<uint64_t>(static_cast<double>(x) / static_cast<double>(y));
    if (q * y > x) --q;
    else if (x - q * y >= y) ++q;
    return q;
}

// The pieces of one run, in order.  All waves of the workgroup walk together.
struct PagedWalk {
    PagedChunk* chunk;
    int base;                  // of the chunk: its first sequence, the costs ahead of it
    uint64_t before;
    uint64_t from, end, run;   // what is left of the run, the length of all runs
    uint32_t index;

    __device__ __forceinline__ PagedWalk(const PagedArgs& p, const PagedRuns& a, uint32_t index_, PagedChunk* chunk_)
        : chunk(chunk_), base(0), before(0), index(index_) {
        if (!a.part) {  // one block, found without the lengths of the others
            from = 0;
            end = run = 1;
            return;
        }
        PagedCost cost;
        const int lane = static_cast<int>(threadIdx.x % kWave), each = (p.b.sequences + kWave - 1) / kWave;
        uint64_t mine = 0, sum;  // costs of a lane's sequences, up to them
        if (each <= 1) {
            sum = paged_chunk(p, a, 0, chunk, &cost);
        } else {
#pragma unroll 4
            for (int i = 0; i < each; ++i) {
                const int s = lane * each + i;
                if (s >= p.b.sequences) break;
                const PagedCost one = paged_cost(p, a, kv_sequence(p.b, s));
                mine += one.ahead(one.blocks) * static_cast<uint32_t>(p.c.kv_heads);
            }
            sum = lanes_up_to(mine);
        }
        uint64_t total = lane_of(sum, kWave - 1);
        run = uniform(max(quotient(total + a.runs - 1, a.runs), static_cast<uint64_t>(a.least)));
        if (a.apart) total = set_apart(p, a, total, cost);
        from = uniform(min(total, run * index));
        end = uniform(min(total, from + run));
        // A run of nothing begins no block; the others say so as they end.
        if (from >= end && threadIdx.x == 0) a.shared[index].runs = 0;
        if (each > 1 && from < end) {  // the chunk from the sequences of the lane on that the run begins in
            const int at = __builtin_ctzll(__ballot(sum > from));
            base = uniform(at * each);
            before = uniform(lane_of(sum, at) - lane_of(mine, at));
            paged_chunk(p, a, base, chunk, &cost);
        }
        __syncthreads();
    }
    // With fewer blocks than half the runs, a block's cost may be rounded up to whole
    // runs: a second part costs its run a way in and out.  With these runs if there are
    // enough, or somewhat longer ones (by `slack`, or half).  The total.
    __device__ __forceinline__ uint64_t set_apart(const PagedArgs& p, const PagedRuns& a, uint64_t total, PagedCost cost) {
        const int lane = static_cast<int>(threadIdx.x % kWave);
        const uint64_t each = cost.base + static_cast<uint64_t>(cost.slope) * cost.blocks;  // the sequence's last block's
        const uint64_t count = static_cast<uint64_t>(cost.blocks) * static_cast<uint32_t>(p.c.kv_heads);
        const uint64_t all = lane_of(lanes_up_to(count), kWave - 1);
        if (2 * all > a.runs || all == 0) return total;
        uint64_t whole = quotient(each + run - 1, run);
        if (lane_of(lanes_up_to(whole * count), kWave - 1) > a.runs) {
            const uint64_t most = lane_of(lanes_up_to(each * count), kWave - 1), left = a.runs - all;
            const uint64_t longer = uniform(quotient(most + left - 1, left));
            if (longer > run + min(static_cast<uint64_t>(a.slack), run / 2)) return total;
            run = max(run, longer);
            whole = quotient(each + run - 1, run);
        }
        cost.slope = 0;
        cost.base = static_cast<uint32_t>(whole * run);
        const uint64_t sum = lanes_up_to(whole * run * count);
        if (threadIdx.x < kWave) {
            chunk->sum[lane] = sum;
            chunk->cost[lane] = cost;
        }
        return lane_of(sum, kWave - 1);
    }
    __device__ __forceinline__ bool more() const { return from < end; }

    // A piece without rows has nothing to do.
    __device__ __forceinline__ PagedPiece next(const PagedArgs& p, const PagedRuns& a) {
        if (!a.part) {
            from = end;
            PagedPiece w;
            const uint32_t pair = index / static_cast<uint32_t>(a.row_blocks), heads = static_cast<uint32_t>(p.c.kv_heads);
            w.s = static_cast<int>(pair / heads);
            w.head = static_cast<int>(pair % heads);
            w.seq = kv_sequence(p.b, w.s);
            w.row0 = static_cast<int>(index % static_cast<uint32_t>(a.row_blocks)) * a.block_rows;
            const int64_t all = static_cast<int64_t>(w.seq.n) * p.group;
            const bool ours = all >= a.least_rows && all <= a.most_rows;
            w.rows = ours ? static_cast<int>(min(all - w.row0, static_cast<int64_t>(a.block_rows))) : 0;
            w.k0 = 0;
            w.k1 = w.rows > 0 ? row_end(p, w.seq, w.row0 + w.rows - 1) : 0;
            w.whole = w.begins = true;
            return w;
        }
        const int mine = static_cast<int>(threadIdx.x % kWave);
        uint64_t sum;
        for (;;) {
            sum = chunk->sum[mine];
            const uint64_t to = before + lane_of(sum, kWave - 1);
            if (from < to || base + kWave >= p.b.sequences) break;
            __syncthreads();  // all waves have read it
            base += kWave;
            before = uniform(to);
            PagedCost cost;
            paged_chunk(p, a, base, chunk, &cost);
            __syncthreads();
        }
        const uint64_t above = __ballot(before + sum > from);
        const int lane = above ? __builtin_ctzll(above) : 0;
        PagedPiece w;
        w.s = base + lane;
        w.seq = KvSequence{uniform(chunk->seq[lane].first), uniform(chunk->seq[lane].n), uniform(chunk->seq[lane].len)};
        const PagedCost cost{uniform(chunk->cost[lane].base), uniform(chunk->cost[lane].slope), uniform(chunk->cost[lane].blocks)};
        const uint64_t head_cost = cost.ahead(cost.blocks);
        uint64_t first = before + lane_of(sum, lane) - head_cost * static_cast<uint32_t>(p.c.kv_heads);
        w.head = uniform(static_cast<int>(quotient(from - first, head_cost)));
        first += head_cost * static_cast<uint32_t>(w.head);
        uint32_t lo = 0, hi = cost.blocks;  // row block lo begins at or before `from`, hi after it
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (first + cost.ahead(mid) <= from) lo = mid;
            else hi = mid;
        }
        lo = uniform(lo);
        first = uniform(first + cost.ahead(lo));
        w.row0 = static_cast<int>(lo) * a.block_rows;
        w.rows = min(w.seq.n * p.group - w.row0, a.block_rows);
        const int keys = row_end(p, w.seq, w.row0 + w.rows - 1);
        const uint64_t all = static_cast<uint64_t>(cost.base) + static_cast<uint64_t>(cost.slope) * (lo + 1);
        const uint64_t x0 = from - first, x1 = min(all, end - first);
        // The same for the run that ends here and the one that begins, and never less for more.
        const auto cut = [&](uint64_t x) {
            const auto at = static_cast<uint32_t>(keys * (static_cast<double>(x) / static_cast<double>(all)));
            return x >= all ? keys : min(keys, static_cast<int>((at + a.grain / 2) & -a.grain));
        };
        w.k0 = uniform(cut(x0));
        w.k1 = uniform(cut(x1));
        w.begins = x0 == 0;
        w.whole = w.begins && x1 == all;
        if (threadIdx.x == 0 && w.begins && !w.whole)
            a.shared[index] = PagedShared{static_cast<int32_t>(quotient(first + all - 1, run) - index) + 1, w.seq.first, w.row0,
                                          w.rows, w.head, {}};
        from = uniform(first + x1);
        // None that a later run goes on with.
        if (threadIdx.x == 0 && from >= end && (w.whole || !w.begins)) a.shared[index].runs = 0;
        return w;
    }
};

// Where a run keeps the sums of a block that it shares with others, the one that it
// begins or goes on with: a max and a sum per row, then rows of head_dim sums from
// 16-byte boundaries on.
__host__ __device__ inline int64_t paged_part_stats(int part_rows) {
    return (2 * static_cast<int64_t>(part_rows) + 3) & ~int64_t{3};
}
__host__ __device__ inline int64_t paged_part_stride(int head_dim) { return (head_dim + 3) & ~3; }
__host__ __device__ inline int64_t paged_part_floats(int part_rows, int head_dim) {
    return paged_part_stats(part_rows) + part_rows * paged_part_stride(head_dim);
}
struct PagedPart {
    float* at;
    int32_t rows;
    int64_t stride;
    __device__ __forceinline__ PagedPart(const PagedRuns& a, int head_dim, uint32_t run, bool begins)
        : at(a.part + (static_cast<int64_t>(run) * 2 + (begins ? 1 : 0)) * paged_part_floats(a.part_rows, head_dim)),
          rows(a.part_rows), stride(paged_part_stride(head_dim)) {}
    __device__ __forceinline__ f2* stat(int row) const { return reinterpret_cast<f2*>(at) + row; }
    __device__ __forceinline__ float* sums(int row) const { return at + paged_part_stats(rows) + row * stride; }
};

// Row `row` of a sequence's (token, head) rows in q and out.
__device__ __forceinline__ int64_t paged_row(const PagedArgs& p, int64_t ld, int first, int head, int row) {
    const auto t = static_cast<int>(fastdiv(static_cast<uint32_t>(row), p.group_div));
    return (first + static_cast<int64_t>(t)) * ld + static_cast<int64_t>(head * p.group + row - t * p.group) * p.c.head_dim;
}

// --- entries ---------------------------------------------------------------------

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

// Elements d .. d + 3 (d a multiple of 4) of a cache row (index `at` among the rows of
// the type's buffer), and element d alone.
template <int DT>
__device__ __forceinline__ f4 elements(const char* base, int64_t at, int stride, int d) {
    const int64_t i = at * stride + d;
    if constexpr (DT == MIMIR_KV_F32) return *reinterpret_cast<const f4*>(base + 4 * i);
    if constexpr (DT == MIMIR_KV_BF16) {
        const u2 x = *reinterpret_cast<const u2*>(base + 2 * i);
        const u4 w{x[0] << 16, x[0] & 0xffff0000u, x[1] << 16, x[1] & 0xffff0000u};
        return __builtin_bit_cast(f4, w);
    }
    const uint32_t x = *reinterpret_cast<const uint32_t*>(base + i);
    return f4{byte_float(x, 0), byte_float(x, 1), byte_float(x, 2), byte_float(x, 3)};
}
template <int DT>
__device__ __forceinline__ float element(const char* base, int64_t at, int stride, int d) {
    const int64_t i = at * stride + d;
    if constexpr (DT == MIMIR_KV_F32) return reinterpret_cast<const float*>(base)[i];
    else if constexpr (DT == MIMIR_KV_BF16)
        return __builtin_bit_cast(float, static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(base)[i]) << 16);
    else return static_cast<float>(reinterpret_cast<const int8_t*>(base)[i]);
}

constexpr int kRowChunks = kKvMaxDim / kWave;

// One query row over keys j0 .. j1 - 1 by one wave: 64 keys at a time, a lane each for
// the scores; then lane l has dimensions l + 64 c of the sums.  Leaves those (without
// the division) and the running max (base-2 units) and sum.
template <int DT>
__device__ __forceinline__ void row_over_keys(const PagedArgs& a, int s, int kv_head, const float* q, int j0, int j1,
                                              float* acc, float* m_out, float* l_out) {
    const int lane = threadIdx.x % kWave, d_all = a.c.head_dim;
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) acc[c] = 0.f;
    float m = -1e30f, l = 0.f;
    for (int j = j0; j < j1; j += kWave) {
        const KvSlot own = j + lane < j1 ? kv_slot(a.b, a.c.pages, a.c.page_div, s, j + lane) : KvSlot{-1, 0};
        const bool has = own.page >= 0;
        const int64_t at = (static_cast<int64_t>(has ? own.page : 0) * a.c.kv_heads + kv_head) * a.c.page_size + own.slot;
        float score = 0.f;
#pragma unroll 4
        for (int d = 0; d < d_all; d += 4) {
            const f4 k = elements<DT>(a.c.k, at, a.c.stride, d);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < d_all) score += q[d + e] * a.qscale * k[e];
        }
        if constexpr (DT == MIMIR_KV_I8) score *= a.c.k_scale[at];
        if (!has) score = -INFINITY;
        const float m_new = fmaxf(m, wave_max(score));
        const float alpha = __builtin_amdgcn_exp2f(m - m_new);
        const float p = has ? __builtin_amdgcn_exp2f(score - m_new) : 0.f;
        m = m_new;
        l = l * alpha + wave_sum(p);
        const float weight = DT == MIMIR_KV_I8 ? p * a.c.v_scale[at] : p;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) acc[c] *= alpha;
        uint64_t left = __ballot(has);
        while (left) {
            constexpr int kAhead = 8;
            float w[kAhead], v[kAhead][kRowChunks];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const bool any = left != 0;
                const int i = any ? __builtin_ctzll(left) : 0;
                const auto row = static_cast<int64_t>(lane_of(static_cast<uint64_t>(at), i));
                w[u] = __builtin_bit_cast(float, lane_of(__builtin_bit_cast(uint32_t, weight), i));
#pragma unroll
                for (int c = 0; c < kRowChunks; ++c) {
                    const int d = lane + c * kWave;
                    v[u][c] = any && d < d_all ? element<DT>(a.c.v, row, a.c.stride, d) : 0.f;
                }
                if (!any) w[u] = 0.f;
                left &= left - 1;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int c = 0; c < kRowChunks; ++c) acc[c] += w[u] * v[u][c];
        }
        // What is NaN stays NaN: a row that is all NaN is done.
        bool nan = true;
#pragma unroll
        for (int c = 0; c < kRowChunks; ++c) {
            if (l != l) acc[c] = l;
            nan = nan && (acc[c] != acc[c] || lane + c * kWave >= d_all);
        }
        if (__all(nan)) break;
    }
    *m_out = m;
    *l_out = l;
}

// The host's side (attention_paged_stream.hip, attention_paged_block.hip): sequences
// of up to `most_rows` query rows a key / value head, and of `least_rows` on.
// What is left to join is in `left` (no runs: nothing).  beside: another launch follows.
int paged_stream_launch(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t most_rows, bool beside, PagedRuns* left);
int paged_block_launch(mimir_ctx* ctx, const PagedArgs& p, int dtype, int64_t least_rows, PagedRuns* left);

// Contexts that the block kernel has whole, by workgroups of four waves: one prompt of
// 250 tokens, 32 heads of 128, bf16: 32 us cut and joined, 29 whole by eight waves, 24 by
// four; 64 of up to 102 57, 37 and 35.  (Up to 512: 12 prompts of 400, heads of 64, 78 and
// 63, but 49 sequences of 315 or single tokens 64 and 79.)
constexpr int kWholeLen = 256;

// Sets up `a` for at most `runs` workgroups in the workspace, or for one per block
// (`blocks` of them) where that is not to be had or `split` says not to, which it may not
// where so many do not fit a launch (of `threads` each): most are then of rows that max_new
// allows and no sequence has.  The grid.
int64_t paged_runs(mimir_ctx* ctx, const PagedArgs& p, PagedRuns* a, int64_t runs, int64_t blocks, int threads, bool split,
                   bool beside);

}  // namespace mimir
