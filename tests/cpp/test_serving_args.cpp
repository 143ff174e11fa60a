// The serving entry points' refusals, without a GPU: a context of a device that is
// not there, so that a call whose arguments are in order ends with EDEVICE before
// anything is enqueued, and every other one with EINVAL and a message before that.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <limits>

#include "../../mimir-framework_amd/csrc/internal.hpp"

static int failures = 0;
static mimir_ctx* ctx = nullptr;

static void expect(int line, int want, int got) {
    if (got != want) std::printf("line %d: status %d, %d expected (%s)\n", line, got, want, mimir_last_error(ctx)), ++failures;
    else if (want == MIMIR_EINVAL && !*mimir_last_error(ctx)) std::printf("line %d: no message\n", line), ++failures;
    ctx->last_error.clear();
}
#define OK(x) expect(__LINE__, MIMIR_OK, (x))
#define BAD(x) expect(__LINE__, MIMIR_EINVAL, (x))
#define FINE(x) expect(__LINE__, MIMIR_EDEVICE, (x))

int main() {
    mimir_ctx fake;
    fake.device = 9999;
    ctx = &fake;
    alignas(16) static float f[64];
    static int32_t ids[64];
    float* odd = f + 1;
    const int64_t big = int64_t{1} << 40;

    // --- rope rows
    mimir_rope r{f, f, 10, 8, 0};
    const auto rows = [&](const mimir_rope* rope, int64_t t, int64_t d, int64_t qh, int64_t kh, int64_t ld, const int32_t* pos,
                          float* out, int64_t ld_out) {
        return mimir_rope_rows_fwd(ctx, f, ld, out, ld_out, qh, f + 32, ld, f + 48, ld, kh, t, d, pos, rope);
    };
    FINE(rows(&r, 2, 8, 2, 1, 16, ids, odd, 16));
    FINE(rows(&r, 2, 8, 2, 1, 16, ids, f, 16));      // in place
    BAD(rows(&r, 2, 8, 2, 1, 16, ids, f, 17));       // in place, other stride
    BAD(rows(&r, 2, 8, 2, 1, 15, ids, odd, 16));
    BAD(rows(&r, 2, 8, 2, 1, 16, ids, odd, 15));
    BAD(rows(&r, -1, 8, 2, 1, 16, ids, odd, 16));
    BAD(rows(&r, big, 8, 2, 1, 16, ids, odd, 16));
    BAD(rows(&r, 2, 0, 2, 1, 16, ids, odd, 16));
    BAD(rows(&r, 2, 8, -2, 1, 16, ids, odd, 16));
    BAD(rows(&r, 2, 8, 2, 1, 16, nullptr, odd, 16));
    BAD(rows(&r, 2, 8, 2, 1, 16, ids, nullptr, 16));
    BAD(rows(nullptr, 2, 8, 2, 1, 16, ids, odd, 16));
    OK(rows(&r, 0, 8, 2, 1, 16, nullptr, nullptr, 16));
    for (int rot : {0, -2, 7, 10}) {
        mimir_rope x = r;
        x.rot_dim = rot;
        BAD(rows(&x, 2, 8, 2, 1, 16, ids, odd, 16));
    }
    mimir_rope untabled{nullptr, f, 10, 8, 0};
    BAD(rows(&untabled, 2, 8, 2, 1, 16, ids, odd, 16));
    untabled.table_rows = -1;
    BAD(rows(&untabled, 2, 8, 2, 1, 16, ids, odd, 16));
    untabled.table_rows = 0;
    FINE(rows(&untabled, 2, 8, 2, 1, 16, ids, odd, 16));  // every position is outside
    FINE(mimir_rope_rows_bwd(ctx, f, 16, odd, 16, 2, nullptr, 0, nullptr, 0, 0, 2, 8, ids, &r, 1));
    BAD(mimir_rope_rows_bwd(ctx, f, 16, f, 16, 2, nullptr, 0, nullptr, 0, 0, 2, 8, ids, &r, 1));  // in place, accumulating
    FINE(mimir_rope_rows_bwd(ctx, f, 16, f, 16, 2, nullptr, 0, nullptr, 0, 0, 2, 8, ids, &r, 0));
    OK(mimir_rope_rows_fwd(ctx, nullptr, 0, nullptr, 0, 3, nullptr, 0, nullptr, 0, 4, 5, 8, ids, &r));

    // --- tables
    float c[8], s[8];
    mimir_rope_scaling z{MIMIR_ROPE_SCALE_BY_PARTS, 4, 100, 1, 32, 1};
    const auto table = [&](int64_t first, int64_t n, int64_t rot, double theta, const mimir_rope_scaling* how) {
        ctx->last_error = "a table has no context";
        return mimir_rope_table_scaled(first, n, rot, theta, how, c, s);
    };
    OK(table(0, 2, 8, 1e4, nullptr));
    OK(table(7, 2, 8, 1e4, &z));
    BAD(table(-1, 2, 8, 1e4, nullptr));
    BAD(table(0, -2, 8, 1e4, nullptr));
    BAD(table(0, 2, 7, 1e4, nullptr));
    BAD(table(0, 2, 0, 1e4, nullptr));
    BAD(table(0, 2, 8, 0, nullptr));
    BAD(table(0, 2, 8, NAN, nullptr));
    BAD(mimir_rope_table_scaled(0, 2, 8, 1e4, nullptr, nullptr, (ctx->last_error = "-", s)));
    const auto with = [&](const std::function<void(mimir_rope_scaling&)>& set) {
        mimir_rope_scaling x = z;
        set(x);
        return table(0, 2, 8, 1e4, &x);
    };
    BAD(with([](auto& x) { x.kind = 4; }));
    BAD(with([](auto& x) { x.kind = -1; }));
    BAD(with([](auto& x) { x.factor = 0; }));
    BAD(with([](auto& x) { x.factor = INFINITY; }));
    BAD(with([](auto& x) { x.low = 32; }));
    BAD(with([](auto& x) { x.original_len = 0; }));
    BAD(with([](auto& x) { x.magnitude = NAN; }));
    mimir_rope_scaling base{MIMIR_ROPE_SCALE_BASE, 4, 0, 0, 0, 1};
    OK(table(0, 2, 4, 1e4, &base));
    BAD(table(0, 2, 2, 1e4, &base));

    // --- cache, batch
    const mimir_kv_cache good{MIMIR_KV_I8, 16, 4, 2, 8, f, f, f, f};
    const mimir_kv_batch many{2, 3, ids, ids, ids, 4, 2, 64};
    const auto append = [&](const mimir_kv_cache& cache, const mimir_kv_batch& b) {
        return mimir_kv_append(ctx, &cache, &b, f, f, 16, nullptr, nullptr, 0, nullptr, 0, 0);
    };
    const auto all = [&](int line, int want, const mimir_kv_cache& cache, const mimir_kv_batch& b) {
        expect(line, want, append(cache, b));
        expect(line, want, mimir_kv_read(ctx, &cache, &b, f, f, 16));
        expect(line, want, mimir_attention_paged_fwd(ctx, &cache, &b, f, 16, f + 32, 16, 2, 1.f, 1));
    };
    all(__LINE__, MIMIR_EDEVICE, good, many);
    const auto cache_with = [&](int line, int want, const std::function<void(mimir_kv_cache&)>& set) {
        mimir_kv_cache x = good;
        set(x);
        all(line, want, x, many);
    };
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.dtype = 3; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.dtype = -1; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.page_size = 24; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.page_size = 0; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.page_size = -16; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.page_size = 1 << 21; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.kv_heads = 0; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.head_dim = 0; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.head_dim = 257; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.pages = -1; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.pages = int64_t{1} << 31; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.k = nullptr; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.v_scale = nullptr; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.v = f + 1; });
    cache_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.k_scale = f + 1; });
    cache_with(__LINE__, MIMIR_EDEVICE, [](auto& x) { x.dtype = MIMIR_KV_BF16, x.k_scale = x.v_scale = nullptr; });
    cache_with(__LINE__, MIMIR_EDEVICE, [](auto& x) { x.pages = 0, x.k = x.v = x.k_scale = x.v_scale = nullptr; });
    const auto batch_with = [&](int line, int want, const std::function<void(mimir_kv_batch&)>& set) {
        mimir_kv_batch x = many;
        set(x);
        all(line, want, good, x);
    };
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.sequences = -1; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.tokens = -1; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.tokens = int64_t{1} << 30; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.max_new = -1; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.max_len = 65; });  // 5 pages of 16, 4 entries
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.ld_pages = -1; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.token_start = nullptr; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.kv_len = nullptr; });
    batch_with(__LINE__, MIMIR_EINVAL, [](auto& x) { x.page_table = nullptr; });
    batch_with(__LINE__, MIMIR_EDEVICE, [](auto& x) { x.page_table = nullptr, x.max_len = 0, x.ld_pages = 0; });
    batch_with(__LINE__, MIMIR_OK, [](auto& x) { x.tokens = 0; });
    batch_with(__LINE__, MIMIR_OK, [](auto& x) { x.sequences = 0, x.token_start = x.kv_len = x.page_table = nullptr; });

    // --- append
    const mimir_rope rope{f, f, 64, 8, 0};
    const auto rotated = [&](const mimir_rope* how, const float* q, int64_t ld_q, float* out, int64_t ld_out, int64_t heads,
                             int64_t ld_kv, const float* k) {
        return mimir_kv_append(ctx, &good, &many, k, f, ld_kv, how, q, ld_q, out, ld_out, heads);
    };
    FINE(rotated(&rope, f, 32, f + 1, 32, 4, 16, f));
    FINE(rotated(&rope, f, 32, const_cast<float*>(f), 32, 4, 16, f));
    FINE(rotated(&rope, nullptr, 0, nullptr, 0, 0, 16, f));
    BAD(rotated(nullptr, f, 32, f + 1, 32, 4, 16, f));
    BAD(rotated(&rope, f, 31, f + 1, 32, 4, 16, f));
    BAD(rotated(&rope, f, 32, f + 1, 31, 4, 16, f));
    BAD(rotated(&rope, f, 32, const_cast<float*>(f), 33, 4, 16, f));
    BAD(rotated(&rope, f, 32, nullptr, 32, 4, 16, f));
    BAD(rotated(&rope, f, 32, f + 1, 32, 0, 16, f));
    BAD(rotated(&rope, f, 32, f + 1, 32, 4, 15, f));
    BAD(rotated(&rope, f, 32, f + 1, 32, 4, 16, nullptr));
    mimir_rope short_table = rope;
    short_table.table_rows = 63;
    BAD(rotated(&short_table, f, 32, f + 1, 32, 4, 16, f));
    mimir_rope wide = rope;
    wide.rot_dim = 10;
    BAD(rotated(&wide, f, 32, f + 1, 32, 4, 16, f));
    BAD(mimir_kv_append(ctx, nullptr, &many, f, f, 16, nullptr, nullptr, 0, nullptr, 0, 0));
    BAD(mimir_kv_append(ctx, &good, nullptr, f, f, 16, nullptr, nullptr, 0, nullptr, 0, 0));

    // --- read
    BAD(mimir_kv_read(ctx, &good, &many, f, f, 15));
    OK(mimir_kv_read(ctx, &good, &many, nullptr, nullptr, 16));

    // --- attention
    const auto attend = [&](const float* q, int64_t ld_q, float* out, int64_t ld_out, int64_t heads, float scale) {
        return mimir_attention_paged_fwd(ctx, &good, &many, q, ld_q, out, ld_out, heads, scale, 0);
    };
    FINE(attend(f, 32, f + 1, 32, 4, 1.f));
    BAD(attend(f, 31, f + 1, 32, 4, 1.f));
    BAD(attend(f, 32, f + 1, 31, 4, 1.f));
    BAD(attend(f, 32, f + 1, 32, 3, 1.f));
    BAD(attend(f, 32, f + 1, 32, 0, 1.f));
    BAD(attend(f, 32, f + 1, 32, 4, NAN));
    BAD(attend(f, 32, f + 1, 32, 4, INFINITY));
    BAD(attend(f, 32, f, 32, 4, 1.f));  // in place
    BAD(attend(nullptr, 32, f + 1, 32, 4, 1.f));
    BAD(attend(f, 32, nullptr, 32, 4, 1.f));

    size_t a = 0, b = 0;
    ctx->last_error = "-";
    OK(mimir_kv_cache_bytes(&good, &a, &b));
    if (a != 4 * 2 * 16 * 16 || b != 4 * 2 * 16 * 4) std::printf("cache bytes %zu %zu\n", a, b), ++failures;
    mimir_kv_cache huge = good;
    huge.pages = (int64_t{1} << 31) - 1;
    huge.page_size = 1 << 20;
    huge.kv_heads = 1 << 16;
    ctx->last_error = "-";
    BAD(mimir_kv_cache_bytes(&huge, &a, &b));

    std::printf("serving arguments: %d failures\n", failures);
    return failures != 0;
}
