// matdeal.hpp -- how the contraction of a product (matrix.hpp) is dealt to workgroups
// where its tiles alone leave CUs idle, and the fp32 slices that the shares' sums take:
// arithmetic alone, the same on the host, which makes room for the slices, and in the
// kernels, which decide on the splits where the product's n is known on the device only.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace mimir {

constexpr int64_t mat_round(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// How many ways a contraction is split: as many as leave the tiles' workgroups at
// `fill`, at most `splits`.  fill 0: once.
constexpr int32_t mat_splits(int32_t fill, int32_t splits, int64_t tiles) {
    if (fill == 0) return 1;
    const int64_t s = fill / (tiles > 0 ? tiles : 1);
    return s < 1 ? 1 : s < splits ? static_cast<int32_t>(s) : splits;
}

// Rows of the slices of a product with m columns of C.  Of this product's m, not of a
// larger one's that the room was made for: a narrower product has fewer tiles and so more
// splits, and `fill` bounds their number times the tile, no wider rows.
constexpr int64_t mat_slice_ld(int64_t m) { return mat_round(m, 4); }

struct MatTileSize {
    int32_t m, n;
};

// Workgroups of a contraction's share.
constexpr int64_t mat_tiles_of(MatTileSize t, int64_t m, int64_t n, int64_t batches) {
    return (m + t.m - 1) / t.m * ((n + t.n - 1) / t.n) * batches;
}

// A product into MatOut: its shape, and how its contraction is dealt to workgroups where
// the tiles of C alone leave CUs idle.
struct MatDeal {
    bool big, thin;
    int32_t fill, splits;
    size_t partial;  // bytes of the slices
};

// Bytes that the slices of m x n of C take with deal `d` in tiles of `t`.
constexpr size_t mat_slice_bytes(const MatDeal& d, MatTileSize t, int64_t m, int64_t n, int64_t batches) {
    return sizeof(float) * static_cast<size_t>(mat_splits(d.fill, d.splits, mat_tiles_of(t, m, n, batches)) * batches * n * mat_slice_ld(m));
}

// The larger tiles where they fill the GPU, or, the contraction split, come to 1 for
// each CU; else the smaller ones, split to 2 for each CU.  A split has at least 512 of
// the contraction.  Measured, both gradients of a call, us, splits of at least 256 / 512 /
// 1024 / none: cross entropy 512 x 2048 x 4000 bf16 113 / 81 / 83 / 109, 256 x 1024 x 8000 fp32
// 141 / 132 / 145 / 341; gated 1024 x 512 x 1376 fp32 88 / 87 / 121 / 162.  Twice as many
// workgroups / these: 1024 x 512 x 32000 bf16 267 / 199, gated 4096 x 512 x 1376 fp32 226 /
// 178, most others the same.  `more`: the sums go through fp32 slices whether split or not.  The
// room holds for this m and n and any smaller ones.
struct MatDealRule {
    MatTileSize big, small;
    bool has_big, has_thin;
    int64_t big_tiles, thin_k;
    int32_t tuned;  // Tuning::mat_big
};
inline MatDeal mat_deal_of(const MatDealRule& r, int64_t m, int64_t n, int64_t k, int64_t batches, bool more) {
    constexpr int32_t kBigFill = 256, kSmallFill = 512;
    constexpr int64_t kLeastK = 512;
    const int64_t big = mat_tiles_of(r.big, m, n, batches), most = std::max<int64_t>(1, k / kLeastK);
    const int64_t big_most = std::max<int64_t>(1, kBigFill / std::max<int64_t>(big, 1));
    MatDeal d{};
    d.thin = r.has_thin && k <= r.thin_k && r.tuned != 1;
    d.big = r.has_big && !d.thin && (r.tuned >= 0 ? r.tuned == 1 : big * std::min(most, big_most) >= r.big_tiles);
    d.fill = d.big ? kBigFill : kSmallFill;
    d.splits = static_cast<int32_t>(std::min<int64_t>(most, 64));
    const MatTileSize t = d.big ? r.big : r.small;
    // n on the device may be smaller than here: then there are more splits, but no more
    // tiles' worth of sums than `fill`.
    if (d.splits == 1 || mat_tiles_of(t, m, n, batches) >= d.fill) d.splits = 1, d.fill = 0;
    if (d.splits > 1) d.partial = sizeof(float) * static_cast<size_t>(int64_t{d.fill} * t.m * t.n);
    if (more || d.splits > 1) d.partial = std::max(d.partial, sizeof(float) * static_cast<size_t>(n * mat_slice_ld(m) * batches));
    return d;
}

}  // namespace mimir
