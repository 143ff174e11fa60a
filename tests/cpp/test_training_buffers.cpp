// Training entry points refuse outputs that are one of their inputs or another output,
// without a GPU: a context of a device that is not there, so that a call whose arguments
// are in order ends with EDEVICE before anything is enqueued.
#include <cstdio>

#include "../../mimir-framework_amd/csrc/internal.hpp"

static int failures = 0;

int main() {
    mimir_ctx fake;
    fake.device = 9999;
    mimir_ctx* ctx = &fake;
    alignas(16) static float m[16][64];
    const auto expect = [&](int line, bool bad, int got) {
        if (got != (bad ? MIMIR_EINVAL : MIMIR_EDEVICE)) std::printf("line %d: status %d (%s)\n", line, got, mimir_last_error(ctx)), ++failures;
    };
    const auto ids = reinterpret_cast<const int32_t*>(m[0]);
    // Cross entropy: buffers x 1, w 2, loss 3, lse 4, mean 5; gradients dloss 6, dx 7, dw 8.
    const auto ce = [&](int loss, int lse, int mean) {
        return mimir_linear_cross_entropy_fwd(ctx, MIMIR_NUM_F32, m[1], 4, m[2], 4, ids, 2, 4, 3, m[loss], m[lse], m[mean]);
    };
    const auto ce_bwd = [&](int dx, int dw) {
        return mimir_linear_cross_entropy_bwd(ctx, MIMIR_NUM_F32, m[1], 4, m[2], 4, ids, 2, 4, 3, m[4], m[6], m[5], 1.0f, m[dx], 4, 0, m[dw],
                                              4, 0);
    };
    expect(__LINE__, false, ce(3, 4, 5));
    for (int in : {0, 1, 2}) expect(__LINE__, true, ce(in, 4, 5)), expect(__LINE__, true, ce(3, in, 5)), expect(__LINE__, true, ce(3, 4, in));
    expect(__LINE__, true, ce(3, 3, 5));
    expect(__LINE__, true, ce(3, 4, 4));
    expect(__LINE__, false, ce_bwd(7, 8));
    expect(__LINE__, false, ce_bwd(1, 8));  // dx in place of x
    for (int in : {0, 2, 4, 5, 6, 8}) expect(__LINE__, true, ce_bwd(in, 8));
    for (int in : {0, 1, 2, 4, 5, 6, 7}) expect(__LINE__, true, ce_bwd(7, in));
    // Gated products: x 1, w_gate 2, w_up 3, y 4, gate_up 5, dy 6, dx 7, dw_gate 8, dw_up 9.
    const auto gated = [&](int y, int gate_up) {
        return mimir_gated_linear_fwd(ctx, MIMIR_NUM_BF16, MIMIR_ACT_SILU, m[1], 4, m[2], m[3], 5, 2, 4, 5, m[y], 5,
                                      gate_up < 0 ? nullptr : m[gate_up]);
    };
    const auto gated_bwd = [&](int dx, int dg, int du) {
        return mimir_gated_linear_bwd(ctx, MIMIR_NUM_F32, MIMIR_ACT_GELU, m[1], 4, m[2], m[3], 5, 2, 4, 5, m[5], m[6], 5, m[dx], 4, 0, m[dg],
                                      m[du], 5, 0);
    };
    expect(__LINE__, false, gated(4, 5));
    expect(__LINE__, false, gated(4, -1));
    for (int in : {1, 2, 3}) expect(__LINE__, true, gated(in, 5)), expect(__LINE__, true, gated(4, in));
    expect(__LINE__, true, gated(4, 4));
    expect(__LINE__, false, gated_bwd(7, 8, 9));
    for (int in : {1, 2, 3, 5, 6, 8, 9}) expect(__LINE__, true, gated_bwd(in, 8, 9));
    for (int in : {1, 2, 3, 5, 6, 7, 9}) expect(__LINE__, true, gated_bwd(7, in, 9)), expect(__LINE__, true, gated_bwd(7, 8, in == 9 ? 8 : in));
    // Two terms: with bf16 in a gradient's type alone.
    for (int type : {MIMIR_NUM_F32, MIMIR_NUM_BF16, 2})
        for (int with : {0, MIMIR_NUM_TWO_TERMS}) {
            const bool grad = type == 2 || (with && type != MIMIR_NUM_BF16), fwd = type == 2 || with;
            expect(__LINE__, fwd, mimir_linear_cross_entropy_fwd(ctx, type | with, m[1], 4, m[2], 4, ids, 2, 4, 3, m[3], m[4], m[5]));
            expect(__LINE__, grad, mimir_linear_cross_entropy_bwd(ctx, type | with, m[1], 4, m[2], 4, ids, 2, 4, 3, m[4], nullptr, nullptr,
                                                                  1.0f, m[7], 4, 0, m[8], 4, 0));
            expect(__LINE__, fwd, mimir_gated_linear_fwd(ctx, type | with, 0, m[1], 4, m[2], m[3], 5, 2, 4, 5, m[4], 5, m[5]));
            expect(__LINE__, grad, mimir_gated_linear_bwd(ctx, type | with, 0, m[1], 4, m[2], m[3], 5, 2, 4, 5, m[5], m[6], 5, m[7], 4, 0,
                                                          m[8], m[9], 5, 0));
        }
    std::printf("training buffers: %d failures\n", failures);
    return failures != 0;
}
