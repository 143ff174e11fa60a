// The serving calls of the C++ adapter (mimir_hip::device): one sequence's prompt, then
// a token, appended with rotated keys, read back and attended, against double; and the
// exception of a refused call.
#include <cmath>
#include <cstdio>
#include <vector>

#include "../../mimir-framework_amd/host/mimir_layerops_hip.hpp"

static int failures = 0;
#define CHECK(x) \
    if (!(x)) std::printf("line %d: %s\n", __LINE__, #x), ++failures

int main() {
    using namespace mimir_hip;
    constexpr int kTokens = 21, kHeads = 4, kKv = 2, kDim = 16, kPage = 16, kPages = 4;
    constexpr float kScale = 0.25f;
    Context c;
    const auto value = [](int i) { return std::sin(0.37f * static_cast<float>(i)) + 0.1f * static_cast<float>(i % 5); };
    std::vector<float> q(kTokens * kHeads * kDim), k(kTokens * kKv * kDim), v(k.size()), cos(32 * kDim / 2), sin(cos.size());
    for (size_t i = 0; i < q.size(); ++i) q[i] = value(static_cast<int>(i));
    for (size_t i = 0; i < k.size(); ++i) k[i] = value(static_cast<int>(3 * i + 1)), v[i] = value(static_cast<int>(5 * i + 2));
    CHECK(mimir_rope_table_scaled(0, 32, kDim, 10000.0, nullptr, cos.data(), sin.data()) == MIMIR_OK);

    DeviceBuffer<float> dq(c, q), dk(c, k), dv(c, v), dcos(c, cos), dsin(c, sin), turned(c, q.size()), again(c, q.size());
    DeviceBuffer<float> cache_k(c, kPages * kKv * kPage * kDim), cache_v(c, cache_k.size()), out(c, q.size());
    DeviceBuffer<float> k_back(c, k.size()), v_back(c, v.size());
    const mimir_rope rope{dcos.data(), dsin.data(), 32, kDim, 0};
    const mimir_kv_cache cache{MIMIR_KV_F32, kPage, kPages, kKv, kDim, cache_k.data(), cache_v.data(), nullptr, nullptr};
    DeviceBuffer<int32_t> table(c, std::vector<int32_t>{3, 1});
    int done = 0;
    for (int n : {kTokens - 1, 1}) {
        DeviceBuffer<int32_t> start(c, std::vector<int32_t>{0, n}), len(c, std::vector<int32_t>{done + n});
        const mimir_kv_batch batch{1, n, start.data(), len.data(), table.data(), 2, n, 2 * kPage};
        device::kv_append(c, cache, batch, dk.data() + done * kKv * kDim, dv.data() + done * kKv * kDim, kKv * kDim, &rope,
                          dq.data() + done * kHeads * kDim, kHeads * kDim, turned.data() + done * kHeads * kDim, kHeads * kDim,
                          kHeads);
        device::attention_paged(c, cache, batch, turned.data() + done * kHeads * kDim, kHeads * kDim,
                                out.data() + done * kHeads * kDim, kHeads * kDim, kHeads, kScale, true);
        done += n;
        c.sync();
    }
    DeviceBuffer<int32_t> start(c, std::vector<int32_t>{0, kTokens}), len(c, std::vector<int32_t>{kTokens});
    const mimir_kv_batch whole{1, kTokens, start.data(), len.data(), table.data(), 2, kTokens, 2 * kPage};
    device::kv_read(c, cache, whole, k_back.data(), v_back.data(), kKv * kDim);
    std::vector<int32_t> at(kTokens);
    for (int t = 0; t < kTokens; ++t) at[t] = t;
    DeviceBuffer<int32_t> positions(c, at);
    device::rope_rows(c, dq.data(), kHeads * kDim, again.data(), kHeads * kDim, kHeads, nullptr, 0, nullptr, 0, 0, kTokens, kDim,
                      positions.data(), rope);

    const std::vector<float> tq = turned.download(), bk = k_back.download(), bv = v_back.download(), o = out.download();
    CHECK(again.download() == tq);
    CHECK(bv == v);
    for (int t = 0; t < kTokens; ++t)
        for (int h = 0; h < kHeads; ++h) {
            const int g = h / (kHeads / kKv);
            double most = -1e30, sum = 0, acc[kDim] = {}, mag = 0;
            std::vector<double> s(t + 1);
            for (int j = 0; j <= t; ++j) {
                for (int d = 0; d < kDim; ++d) s[j] += double(tq[(t * kHeads + h) * kDim + d]) * bk[(j * kKv + g) * kDim + d] * kScale;
                most = std::max(most, s[j]);
            }
            for (int j = 0; j <= t; ++j) {
                const double e = std::exp(s[j] - most);
                sum += e;
                for (int d = 0; d < kDim; ++d) acc[d] += e * bv[(j * kKv + g) * kDim + d];
            }
            for (double x : acc) mag = std::max(mag, std::fabs(x) / sum);
            // Scores of up to 16 x 2 x 2 x 1/4 in products and sums of 2^-24 steps: 16 of them,
            // off by 16 x 16 steps at most; twice that and 21 x 2 steps of the sums on the result.
            for (int d = 0; d < kDim; ++d)
                CHECK(std::fabs(o[(t * kHeads + h) * kDim + d] - acc[d] / (sum + 1e-9)) <= (2 * 256 + 64) * 0x1p-24 * (mag + 2));
        }
    bool thrown = false;
    try {
        device::attention_paged(c, cache, whole, turned.data(), kHeads * kDim, turned.data(), kHeads * kDim, kHeads, kScale, true);
    } catch (const std::runtime_error&) {
        thrown = true;
    }
    CHECK(thrown);
    std::printf("%d failures\n", failures);
    return failures != 0;
}
