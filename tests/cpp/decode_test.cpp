// The decode-step operators through the C++ types.  `decode_test host` needs no GPU; `decode_test gpu` writes tokens, attends
// to them and runs an expert layer, each against sums made here in double.  Exit code 0 and a last line "ok".
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "vortx_b200.hpp"

using namespace vortx;

#define EXPECT(cond)                                                      \
    do {                                                                  \
        if (!(cond)) {                                                    \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            return 1;                                                     \
        }                                                                 \
    } while (0)

static std::vector<float> random_vec(size_t n, unsigned seed, float scale = 1.0f) {
    std::mt19937 g(seed);
    std::normal_distribution<float> d(0.0f, scale);
    std::vector<float> v(n);
    for (auto& x : v) x = d(g);
    return v;
}
// The values that the codes of `v` (rows of `cols`) stand for.
static std::vector<float> through_codes(vx_qtype t, const std::vector<float>& v, size_t cols) {
    std::vector<uint8_t> blocks(v.size() / 32 * vx_qblock_bytes(t));
    std::vector<float> out(v.size());
    check(vx_quantize(t, v.data(), v.size() / cols, cols, blocks.data()));
    check(vx_dequantize_host(t, blocks.data(), v.size() / cols, cols, out.data()));
    return out;
}

static int host() {
    const auto m = tree_mask({-1, 0, 0, 2});
    EXPECT((m == std::vector<uint32_t>{1, 3, 5, 13}));
    std::vector<int32_t> chain(40);
    for (int i = 0; i < 40; ++i) chain[i] = i - 1;
    const auto c = tree_mask(chain);
    EXPECT(c.size() == 80 && c[2 * 31] == 0xffffffffu && c[2 * 31 + 1] == 0 && c[2 * 39 + 1] == 0xff);
    bool refused = false;
    try {
        tree_mask({-1, 1});
    } catch (const Error& e) {
        refused = e.status == VX_ERR_INVALID_ARGUMENT;
    }
    EXPECT(refused);
    return 0;
}

static int gpu() {
    GpuBackend b(0);
    // ---- cache and attention: 40 tokens of context, then a tree of four
    const size_t heads = 4, kv = 2, dim = 64, context = 40, n = 4, width = kv * dim;
    QuantizedCache cache(b, VX_Q8_0, VX_Q4_0, kv, dim, 3, 32);
    CacheAttention attention(b, cache, heads, 1);
    auto i32 = [&](std::vector<int32_t> v) { return GpuBuffer<int32_t>(b, v.data(), v.size()); };
    const auto k = random_vec((context + n) * width, 1), v = random_vec((context + n) * width, 2), q = random_vec(n * heads * dim, 3);
    auto part = [&](const std::vector<float>& a, size_t from, size_t to) {
        return Tensor<float>::vector(b, std::vector<float>(a.begin() + from * width, a.begin() + to * width));
    };
    const auto table = i32({2, 0}), zero = i32({0}), at = i32({(int32_t)context}), upto_c = i32({0, (int32_t)context}), upto_n = i32({0, (int32_t)n});
    const CacheRows before(table, upto_c, zero, context), drafted(table, upto_n, at, n);
    const auto kc = part(k, 0, context), vc = part(v, 0, context), kn = part(k, context, context + n), vn = part(v, context, context + n);
    cache.append(b, kc.as_view(), vc.as_view(), before);
    cache.append(b, kn.as_view(), vn.as_view(), drafted);
    const auto kq = through_codes(VX_Q8_0, k, width), vq = through_codes(VX_Q4_0, v, width);
    auto ko = Tensor<float>::vector_uninit(b, n * width), vo = Tensor<float>::vector_uninit(b, n * width);
    cache.read(b, ko.as_view_mut(), vo.as_view_mut(), drafted);
    b.synchronize();
    EXPECT(std::memcmp(ko.read().data(), kq.data() + context * width, n * width * sizeof(float)) == 0);
    EXPECT(std::memcmp(vo.read().data(), vq.data() + context * width, n * width * sizeof(float)) == 0);
    const auto words = tree_mask({-1, 0, 0, 2});
    const GpuBuffer<uint32_t> mask(b, words.data(), words.size());
    const auto gq = Tensor<float>::vector(b, q);
    auto out = Tensor<float>::vector_uninit(b, q.size());
    attention.dispatch(b, out.as_view_mut(), gq.as_view(), drafted, 0.125f, &mask);
    b.synchronize();
    const auto got = out.read();
    for (size_t r = 0; r < n; ++r)
        for (size_t h = 0; h < heads; ++h) {
            std::vector<double> p(context + n, 0.0), want(dim, 0.0);
            double top = -1e300, sum = 0.0;
            auto may = [&](size_t t) { return t < context || (words[r] >> (t - context) & 1); };
            for (size_t t = 0; t < context + n; ++t) {
                for (size_t d = 0; d < dim; ++d) p[t] += 0.125 * q[(r * heads + h) * dim + d] * kq[(t * kv + h / 2) * dim + d];
                if (may(t)) top = std::max(top, p[t]);
            }
            for (size_t t = 0; t < context + n; ++t) sum += p[t] = may(t) ? std::exp(p[t] - top) : 0.0;
            for (size_t t = 0; t < context + n; ++t)
                for (size_t d = 0; d < dim; ++d) want[d] += p[t] / sum * vq[(t * kv + h / 2) * dim + d];
            for (size_t d = 0; d < dim; ++d) EXPECT(std::fabs(got[(r * heads + h) * dim + d] - want[d]) < 2e-5);
        }
    bool refused = false;
    try {
        attention.dispatch(b, out.as_view_mut(), kn.as_view(), drafted, 1.0f);
    } catch (const ShapeMismatch&) {
        refused = true;
    }
    EXPECT(refused);
    // ---- experts: the router's rows are unit vectors, so that x itself says who is chosen
    const size_t experts = 4, hidden = 64, inner = 32, tokens = 2;
    const auto g = random_vec(experts * inner * hidden, 4, 0.1f), u = random_vec(experts * inner * hidden, 5, 0.1f), dn = random_vec(experts * hidden * inner, 6, 0.1f);
    std::vector<float> router(experts * hidden, 0.0f), x = random_vec(tokens * hidden, 7);
    for (size_t e = 0; e < experts; ++e) router[e * hidden + e] = 1.0f;
    const float first[8] = {0.1f, 2.0f, -1.0f, 1.5f, 3.0f, 0.0f, 1.0f, -2.0f};
    for (size_t t = 0; t < tokens; ++t)
        for (size_t e = 0; e < experts; ++e) x[t * hidden + e] = first[t * 4 + e];
    QuantizedMatrix gate(b, VX_Q4_0, g, experts * inner, hidden), up(b, VX_Q4_0, u, experts * inner, hidden), down(b, VX_Q8_0, dn, experts * hidden, inner);
    const auto gr = Tensor<float>::vector(b, router), gx = Tensor<float>::vector(b, x);
    MoeLayer layer(b, gr.as_view(), gate, up, down, experts, 2, true, tokens);
    auto y = Tensor<float>::vector_uninit(b, tokens * hidden);
    GpuBuffer<int32_t> ids(b, tokens * 2);
    layer.dispatch(b, y.as_view_mut(), gx.as_view(), tokens, &ids);
    b.synchronize();
    EXPECT((ids.read() == std::vector<int32_t>{1, 3, 0, 2}));
    const auto gc = through_codes(VX_Q4_0, g, hidden), uc = through_codes(VX_Q4_0, u, hidden), dc = through_codes(VX_Q8_0, dn, inner), yr = y.read();
    for (size_t t = 0; t < tokens; ++t) {
        const auto id = ids.read();
        const double a = x[t * hidden + id[2 * t]], c = x[t * hidden + id[2 * t + 1]], w[2] = {1.0 / (1.0 + std::exp(c - a)), 1.0 / (1.0 + std::exp(a - c))};
        std::vector<double> want(hidden, 0.0);
        for (size_t j = 0; j < 2; ++j) {
            const size_t e = (size_t)id[2 * t + j];
            for (size_t i = 0; i < inner; ++i) {
                double s = 0.0, z = 0.0;
                for (size_t d = 0; d < hidden; ++d) {
                    s += gc[(e * inner + i) * hidden + d] * (double)x[t * hidden + d];
                    z += uc[(e * inner + i) * hidden + d] * (double)x[t * hidden + d];
                }
                for (size_t d = 0; d < hidden; ++d) want[d] += w[j] * dc[(e * hidden + d) * inner + i] * (s / (1.0 + std::exp(-s)) * z);
            }
        }
        for (size_t d = 0; d < hidden; ++d) EXPECT(std::fabs(yr[t * hidden + d] - want[d]) < 2e-5);
    }
    return 0;
}

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    const int rc = what == "host" ? host() : what == "gpu" ? gpu() : 2;
    if (rc == 0) std::printf("ok\n");
    return rc;
}
