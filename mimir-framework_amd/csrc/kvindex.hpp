// kvindex.hpp -- where a batch's tokens stand in a paged cache (mimir_hip.h
// mimir_kv_batch), inside the host's bounds whatever the device arrays hold.  Plain
// C++ (no HIP types), so host tests compile it with g++.
#pragma once

#include <stdint.h>

#include "fastdiv.hpp"

namespace mimir {

struct KvBatch {
    const int32_t* token_start;
    const int32_t* kv_len;
    const int32_t* page_table;
    int64_t ld_pages;
    int32_t sequences, tokens, max_new, max_len;
};

// A sequence's part of a batch: its first row, its new tokens, its cached ones.
struct KvSequence {
    int32_t first, n, len;
};

MIMIR_HD inline int32_t kv_clamp(int32_t x, int32_t lo, int32_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// For 0 <= s < sequences: rows first .. first + n - 1 lie in [0, tokens).
MIMIR_HD inline KvSequence kv_sequence(const KvBatch& b, int32_t s) {
    KvSequence q;
    q.first = kv_clamp(b.token_start[s], 0, b.tokens);
    const int32_t end = kv_clamp(b.token_start[s + 1], q.first, b.tokens);
    q.n = end - q.first < b.max_new ? end - q.first : b.max_new;
    q.len = kv_clamp(b.kv_len[s], 0, b.max_len);
    return q;
}

// The page of sequence s's entry, -1 where it is none of the cache's `pages`.
// entry * page_size < max_len <= ld_pages * page_size keeps the read in the table.
MIMIR_HD inline int32_t kv_page(const KvBatch& b, int64_t pages, int32_t s, int32_t entry) {
    const int32_t page = b.page_table[s * b.ld_pages + entry];
    return page >= 0 && page < pages ? page : -1;
}

// Page (-1: none) and slot of a position below max_len; positions below 0 have none.
struct KvSlot {
    int32_t page, slot;
};

MIMIR_HD inline KvSlot kv_slot(const KvBatch& b, int64_t pages, const FastDiv& page_size, int32_t s, int32_t position) {
    if (position < 0) return KvSlot{-1, 0};
    const uint32_t entry = fastdiv(static_cast<uint32_t>(position), page_size);
    return KvSlot{kv_page(b, pages, s, static_cast<int32_t>(entry)),
                  position - static_cast<int32_t>(entry * page_size.d)};
}

}  // namespace mimir
