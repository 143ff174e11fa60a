// Where a batch's tokens stand in a paged cache (kvindex.hpp), against plain
// arithmetic for arrays that say what they may, and, for arrays of any contents,
// that no row, table entry or slot lies outside its buffer.
#include <cstdio>
#include <random>
#include <vector>

#include "../../mimir-framework_amd/csrc/kvindex.hpp"

using namespace mimir;

static long failures = 0;
#define CHECK(c)                                                 \
    do {                                                         \
        if (!(c) && ++failures < 20) std::printf("line %d: %s\n", __LINE__, #c); \
    } while (0)

int main() {
    std::mt19937 rng(1);
    const auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
    for (int round = 0; round < 20000; ++round) {
        const bool wild = round % 2;
        const int32_t n = static_cast<int32_t>(pick(1, 6)), page = static_cast<int32_t>(16 * pick(1, 6));
        const int64_t pages = pick(1, 40);
        std::vector<int32_t> start(n + 1), len(n);
        int32_t longest = 0, most = 0;
        for (int s = 0; s < n; ++s) {
            const int32_t add = static_cast<int32_t>(pick(0, 30));
            start[s + 1] = start[s] + add;
            len[s] = static_cast<int32_t>(pick(0, 200));
            longest = len[s] > longest ? len[s] : longest;
            most = add > most ? add : most;
        }
        const int64_t ld = (longest + page - 1) / page + pick(0, 2);
        std::vector<int32_t> table(static_cast<size_t>(n * ld) + 1);
        for (auto& x : table) x = static_cast<int32_t>(wild ? pick(-(int64_t{1} << 31), (int64_t{1} << 31) - 1) : pick(0, pages - 1));
        KvBatch b{start.data(), len.data(), table.data(), ld, n, start[n], most, longest};
        if (wild) {
            for (auto& x : start) x = static_cast<int32_t>(pick(-(int64_t{1} << 31), (int64_t{1} << 31) - 1));
            for (auto& x : len) x = static_cast<int32_t>(pick(-(int64_t{1} << 31), (int64_t{1} << 31) - 1));
        }
        const FastDiv div = make_fastdiv(static_cast<uint32_t>(page));
        for (int s = 0; s < n; ++s) {
            const KvSequence q = kv_sequence(b, s);
            CHECK(q.first >= 0 && q.n >= 0 && int64_t{q.first} + q.n <= b.tokens && q.n <= b.max_new);
            CHECK(q.len >= 0 && q.len <= b.max_len);
            if (!wild) CHECK(q.first == start[s] && q.n == start[s + 1] - start[s] && q.len == len[s]);
            for (int32_t p = q.len - q.n; p < q.len; ++p) {
                if (p >= 0) CHECK(s * ld + p / page < n * ld);
                const KvSlot at = kv_slot(b, pages, div, s, p);
                CHECK(at.page >= -1 && at.page < pages && at.slot >= 0 && at.slot < page);
                if (p < 0) CHECK(at.page == -1);
                else if (!wild) CHECK(at.page == table[s * ld + p / page] && at.slot == p % page);
            }
        }
    }
    std::printf("kvindex: %ld failures\n", failures);
    return failures != 0;
}
