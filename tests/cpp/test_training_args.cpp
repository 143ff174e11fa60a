// The training entry points' refusals, without a GPU: a context of a device that is
// not there, so that a call whose arguments are in order ends with EDEVICE before
// anything is enqueued, and every other one with EINVAL and a message before that.
// The adapter's calls are compiled as a program makes them.
#include <cmath>
#include <cstdio>
#include <limits>

#include "../../mimir-framework_amd/csrc/internal.hpp"
#include "../../mimir-framework_amd/host/mimir_layerops_hip.hpp"

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
    alignas(16) static float a[64], b[64], c[64], d[64], e[64], f[64];
    static int32_t ids[64];
    const int64_t big = int64_t{1} << 40;

    // --- cross entropy
    struct Ce {
        int type = MIMIR_NUM_F32;
        const void *x = a, *w = b;
        int64_t ld_x = 4, ld_w = 4, tokens = 2, dim = 4, vocab = 3;
        const int32_t* t = ids;
        float *loss = c, *lse = c + 8, *mean = c + 16;
        void *dx = d, *dw = e;
        int64_t ld_dx = 4, ld_dw = 4;
        int fwd() const { return mimir_linear_cross_entropy_fwd(ctx, type, x, ld_x, w, ld_w, t, tokens, dim, vocab, loss, lse, mean); }
        int bwd() const {
            return mimir_linear_cross_entropy_bwd(ctx, type, x, ld_x, w, ld_w, t, tokens, dim, vocab, lse, nullptr, mean, 1.0f, dx, ld_dx, 0,
                                                  dw, ld_dw, 0);
        }
    };
    const auto both = [&](auto change, bool fwd_bad, bool bwd_bad, int line) {
        Ce k;
        change(k);
        expect(line, fwd_bad ? MIMIR_EINVAL : MIMIR_EDEVICE, k.fwd());
        expect(line, bwd_bad ? MIMIR_EINVAL : MIMIR_EDEVICE, k.bwd());
    };
    both([](Ce&) {}, false, false, __LINE__);
    both([](Ce& k) { k.type = MIMIR_NUM_BF16; }, false, false, __LINE__);
    both([](Ce& k) { k.type = 2; }, true, true, __LINE__);
    both([](Ce& k) { k.type = -1; }, true, true, __LINE__);
    both([](Ce& k) { k.tokens = -1; }, true, true, __LINE__);
    both([&](Ce& k) { k.tokens = big; }, true, true, __LINE__);
    both([](Ce& k) { k.dim = 0; }, true, true, __LINE__);
    both([&](Ce& k) { k.dim = k.ld_x = k.ld_w = k.ld_dx = k.ld_dw = big; }, true, true, __LINE__);
    both([](Ce& k) { k.vocab = 0; }, true, true, __LINE__);
    both([&](Ce& k) { k.vocab = big; }, true, true, __LINE__);
    both([](Ce& k) { k.ld_x = 3; }, true, true, __LINE__);
    both([](Ce& k) { k.ld_w = 3; }, true, true, __LINE__);
    both([](Ce& k) { k.ld_dx = 3; }, false, true, __LINE__);
    both([](Ce& k) { k.ld_dw = 3; }, false, true, __LINE__);
    both([](Ce& k) { k.x = nullptr; }, true, true, __LINE__);
    both([](Ce& k) { k.w = nullptr; }, true, true, __LINE__);
    both([](Ce& k) { k.t = nullptr; }, true, true, __LINE__);
    both([](Ce& k) { k.lse = nullptr; }, true, true, __LINE__);
    both([](Ce& k) { k.loss = nullptr; }, true, false, __LINE__);
    both([](Ce& k) { k.mean = nullptr; }, false, false, __LINE__);
    both([](Ce& k) { k.dx = nullptr; }, false, false, __LINE__);
    both([](Ce& k) { k.dw = nullptr; }, false, false, __LINE__);
    both([](Ce& k) { k.dw = const_cast<void*>(k.w); }, false, true, __LINE__);
    both([](Ce& k) { k.dx = const_cast<void*>(k.x); }, false, false, __LINE__);
    both([](Ce& k) { k.dx = const_cast<void*>(k.x), k.ld_dx = 5; }, false, true, __LINE__);
    {
        Ce k;
        k.dx = k.dw = nullptr;
        OK(k.bwd());
        k = Ce{};
        k.tokens = 0;
        k.mean = nullptr;
        OK(k.fwd());
        k.dw = nullptr;
        FINE(k.bwd());
        k = Ce{};
        k.tokens = 0;
        k.x = k.dx = nullptr;  // no buffer in place of another
        k.ld_dx = 9;
        FINE(k.bwd());
    }

    // --- gated products
    struct Gated {
        int type = MIMIR_NUM_F32, act = MIMIR_ACT_SILU;
        const void *x = a, *wg = b, *wu = b + 32, *dy = c;
        int64_t ld_x = 4, ld_w = 5, tokens = 2, dim = 4, hidden = 5, ld_y = 5;
        void *y = d, *dx = e, *dg = f, *du = f + 32;
        float* gu = d + 32;
        int64_t ld_dx = 4, ld_dw = 5;
        int fwd() const { return mimir_gated_linear_fwd(ctx, type, act, x, ld_x, wg, wu, ld_w, tokens, dim, hidden, y, ld_y, gu); }
        int bwd() const {
            return mimir_gated_linear_bwd(ctx, type, act, x, ld_x, wg, wu, ld_w, tokens, dim, hidden, gu, dy, ld_y, dx, ld_dx, 0, dg, du, ld_dw,
                                          0);
        }
    };
    const auto gated = [&](auto change, bool fwd_bad, bool bwd_bad, int line) {
        Gated k;
        change(k);
        expect(line, fwd_bad ? MIMIR_EINVAL : MIMIR_EDEVICE, k.fwd());
        expect(line, bwd_bad ? MIMIR_EINVAL : MIMIR_EDEVICE, k.bwd());
    };
    gated([](Gated&) {}, false, false, __LINE__);
    gated([](Gated& k) { k.type = MIMIR_NUM_BF16, k.act = MIMIR_ACT_GELU; }, false, false, __LINE__);
    gated([](Gated& k) { k.type = 7; }, true, true, __LINE__);
    gated([](Gated& k) { k.act = 2; }, true, true, __LINE__);
    gated([](Gated& k) { k.act = -1; }, true, true, __LINE__);
    gated([](Gated& k) { k.tokens = -1; }, true, true, __LINE__);
    gated([&](Gated& k) { k.tokens = big; }, true, true, __LINE__);
    gated([](Gated& k) { k.dim = 0; }, true, true, __LINE__);
    gated([&](Gated& k) { k.dim = k.ld_x = k.ld_dx = big; }, true, true, __LINE__);
    gated([](Gated& k) { k.hidden = 0; }, true, true, __LINE__);
    gated([&](Gated& k) { k.hidden = k.ld_w = k.ld_y = k.ld_dw = big; }, true, true, __LINE__);
    gated([](Gated& k) { k.ld_x = 3; }, true, true, __LINE__);
    gated([](Gated& k) { k.ld_w = 4; }, true, true, __LINE__);
    gated([](Gated& k) { k.ld_y = 4; }, true, true, __LINE__);
    gated([](Gated& k) { k.ld_dx = 3; }, false, true, __LINE__);
    gated([](Gated& k) { k.ld_dw = 4; }, false, true, __LINE__);
    gated([](Gated& k) { k.x = nullptr; }, true, true, __LINE__);
    gated([](Gated& k) { k.wg = nullptr; }, true, true, __LINE__);
    gated([](Gated& k) { k.wu = nullptr; }, true, true, __LINE__);
    gated([](Gated& k) { k.y = nullptr; }, true, false, __LINE__);
    gated([](Gated& k) { k.gu = nullptr; }, false, true, __LINE__);
    gated([](Gated& k) { k.dy = nullptr; }, false, true, __LINE__);
    gated([](Gated& k) { k.y = const_cast<void*>(k.x); }, true, false, __LINE__);
    gated([](Gated& k) { k.dx = nullptr; }, false, false, __LINE__);
    gated([](Gated& k) { k.dg = nullptr; }, false, true, __LINE__);
    gated([](Gated& k) { k.dg = k.du = nullptr; }, false, false, __LINE__);
    gated([](Gated& k) { k.du = k.dg; }, false, true, __LINE__);
    gated([](Gated& k) { k.dg = const_cast<void*>(k.wg); }, false, true, __LINE__);
    gated([](Gated& k) { k.dx = const_cast<void*>(k.x); }, false, true, __LINE__);
    gated([](Gated& k) { k.dx = const_cast<void*>(k.dy); }, false, true, __LINE__);
    {
        Gated k;
        k.dx = k.dg = k.du = nullptr;
        OK(k.bwd());
        k = Gated{};
        k.tokens = 0;
        OK(k.fwd());
        FINE(k.bwd());
        k.dg = k.du = nullptr;
        OK(k.bwd());
    }

    // --- norm and clipping
    mimir_tensor t[2] = {{a, b, 5, MIMIR_NUM_F32}, {c, c, 7, MIMIR_NUM_BF16}};
    const auto norm = [&](int64_t n = 2) { return mimir_grad_norm(ctx, t, n, d); };
    const auto clip = [&](float most = 1.0f) { return mimir_grad_clip(ctx, t, 2, most, d); };
    FINE(norm());
    FINE(clip());
    FINE(clip(0.0f));
    FINE(clip(std::numeric_limits<float>::infinity()));
    BAD(clip(-1.0f));
    BAD(clip(std::nanf("")));
    BAD(norm(-1));
    BAD(norm(big));
    BAD(mimir_grad_norm(ctx, nullptr, 1, d));
    FINE(mimir_grad_norm(ctx, nullptr, 0, d));
    BAD(mimir_grad_norm(ctx, t, 2, nullptr));
    t[1].type = 3;
    BAD(norm());
    t[1].type = MIMIR_NUM_BF16;
    t[1].n = -1;
    BAD(clip());
    t[1].n = big * 2;
    BAD(clip());
    t[1].n = 7;
    t[0].out = nullptr;
    FINE(norm());
    BAD(clip());
    t[0].n = 0;
    FINE(clip());
    t[1].data = reinterpret_cast<char*>(c) + 1;
    BAD(norm());
    t[1].data = reinterpret_cast<char*>(c) + 2;
    FINE(norm());
    t[1].data = nullptr;
    BAD(norm());

    // The adapter's forms.
    (void)&mimir_hip::device::linear_cross_entropy;
    (void)&mimir_hip::device::linear_cross_entropy_bwd;
    (void)&mimir_hip::device::gated_linear;
    (void)&mimir_hip::device::gated_linear_bwd;
    (void)&mimir_hip::device::grad_norm;
    (void)&mimir_hip::device::grad_clip;
    std::printf("training args: %d failures\n", failures);
    return failures != 0;
}
