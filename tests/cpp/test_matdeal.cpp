// The arithmetic of split contractions (csrc/matdeal.hpp) on the host: the room made
// for the fp32 slices of a product's sums holds those of the same product with any
// smaller n or m, whose splits are decided from its own tiles.
#include <cmath>
#include <cstdio>
#include <random>

#include "../../mimir-framework_amd/csrc/matdeal.hpp"

using namespace mimir;

static int failures = 0;

static void fits(const MatDealRule& r, const MatDeal& d, int64_t m, int64_t n, int64_t batches, const char* what) {
    const MatTileSize t = d.big ? r.big : r.small;
    if (mat_slice_bytes(d, t, m, n, batches) <= d.partial) return;
    if (++failures < 10)
        std::printf("%s: %lld x %lld x %lld needs %zu of %zu bytes\n", what, (long long)m, (long long)n, (long long)batches,
                    mat_slice_bytes(d, t, m, n, batches), d.partial);
}

// Weights' gradients of a gated block: m hidden columns in pieces, n = dim, both weights
// as batches, the contraction over the tokens.
static void pieces(const MatDealRule& r, int64_t tokens, int64_t dim, int64_t hidden, int64_t piece, const char* what) {
    const MatDeal d = mat_deal_of(r, std::min(piece, hidden), dim, tokens, 2, false);
    if (d.splits == 1) return;
    for (int64_t first = 0; first < hidden; first += piece) fits(r, d, std::min(piece, hidden - first), dim, 2, what);
}

int main() {
    // The rules of the shapes in matrix.hpp: fp32, bf16, two planes beside one.
    MatDealRule rules[] = {{{256, 128}, {128, 64}, true, false, 129, 256, -1},
                           {{256, 256}, {128, 128}, true, true, 129, 256, -1},
                           {{128, 128}, {128, 128}, false, true, 129, 256, -1}};
    // A short last piece behind a full one: 24 tiles where the room was made for 320.
    pieces(rules[0], 8192, 256, 5400, 5120, "fp32 8192 x 256 x 5400");
    pieces(rules[1], 131072, 1024, 1280, 1024, "bf16 131072 x 1024 x 1280");
    {
        // In rows of the full piece's width the same sums pass the end.
        const MatDeal d = mat_deal_of(rules[0], 5120, 256, 8192, 2, false);
        const int64_t splits = mat_splits(d.fill, d.splits, mat_tiles_of(d.big ? rules[0].big : rules[0].small, 280, 256, 2));
        if (sizeof(float) * splits * 2 * 256 * 5120 <= d.partial) std::printf("the short piece is no case of it\n"), ++failures;
    }
    std::mt19937_64 rng(1);
    const auto span = [&](double lo, double hi) {
        return static_cast<int64_t>(std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi + 1))(rng)));
    };
    for (int i = 0; i < 300000; ++i) {
        MatDealRule r = rules[i % 3];
        r.tuned = i % 5 == 0 ? static_cast<int32_t>(rng() % 2) : -1;
        const int64_t m = span(1, 1 << 18), n = span(1, 1 << 15), k = span(1, 1 << 18), batches = 1 + rng() % 2;
        const bool more = rng() % 2;
        const MatDeal d = mat_deal_of(r, m, n, k, batches, more);
        if (d.partial == 0 && d.splits == 1) continue;
        fits(r, d, m, n, batches, "whole");
        // Fewer rows (a count known on the device), a shorter last piece.
        fits(r, d, m, span(1, n), batches, "fewer n");
        fits(r, d, span(1, m), n, batches, "fewer m");
        if (i % 100 == 0)
            for (int64_t few = 0; few <= std::min<int64_t>(n, 600); ++few) fits(r, d, m, few, batches, "few n");
        pieces(r, k, n, span(1, 1 << 17), 8 * span(1, 1 << 13), "pieces");
    }
    std::printf("slices: %d failures\n", failures);
    return failures != 0;
}
