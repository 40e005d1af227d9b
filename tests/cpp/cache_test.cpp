// A cache that drafts, appends, weighs and evicts, through TransformerRuntime (attention_tree, cache_append, cache_weights,
// cache_evict), against plain double arithmetic on the host: two sequences, 4 query heads over 2 kv heads of 128, trees of
// 5 drafts, f16 tiles and f32 rows. Tolerance: outputs within 2e-3 + 1e-2 |ref| (as the other attention tests), LSE within
// 1e-3, gathered weights within 1e-4; the cache's rows, positions and counts are equal.
//   cache_test
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "attn_oracle.h"
#include "transformer_runtime.hpp"

namespace {

class Harness final : public mako::models::TransformerRuntime {
public:
    Harness() : TransformerRuntime(mako::gpu::Telemetry::kernels) {}
    using TransformerRuntime::attention_tree;
    using TransformerRuntime::cache_append;
    using TransformerRuntime::cache_evict;
    using TransformerRuntime::cache_weights;
    using TransformerRuntime::encoder;
    using TransformerRuntime::finish;
    using TransformerRuntime::scratch;
};

int failures = 0;
void check(bool ok, const std::string& what)
{
    std::printf("  %s  %s\n", ok ? "ok  " : "FAIL", what.c_str());
    failures += !ok;
}

std::mt19937 rng(7);

std::vector<uint16_t> tile(size_t n)
{
    std::normal_distribution<float> d;
    std::vector<uint16_t> v(n);
    for (auto& x : v)
        x = oracle_f32_to_f16(d(rng));
    return v;
}

template <class T>
mako::gpu::Buffer* put(Harness& h, const char* name, const std::vector<T>& v)
{
    auto* b = h.scratch(name, v.size() * sizeof(T));
    if (hipMemcpy(b->ptr, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess)
        throw std::runtime_error("hipMemcpy");
    return b;
}

template <class T>
std::vector<T> get(const mako::gpu::Buffer* b, size_t n)
{
    std::vector<T> v(n);
    if (hipMemcpy(v.data(), b->ptr, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess)
        throw std::runtime_error("hipMemcpy");
    return v;
}

}  // namespace

int main()
{
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    constexpr uint32_t B = 2, H = 4, KV = 2, G = H / KV, D = 128, N = 5, CAP = 120, BUDGET = 90, RECENT = 10, SINKS = 2;
    const std::vector<uint32_t> ctx{97, 33}, seen{97, 33}, nodes{5, 4}, n_path{3, 2};
    const std::vector<uint32_t> path{0, 2, 4, 0, 0, 0, 3, 0, 0, 0};
    // sequence 0: 0 -> 1, 0 -> 2 -> {3, 4}; sequence 1: 0 -> {1, 2}, 0 -> 3
    const std::vector<uint64_t> mask{1, 3, 5, 13, 21, 1, 3, 5, 9, 0};
    const auto q = tile(size_t(H) * B * N * D), k = tile(size_t(B) * KV * CAP * D), v = tile(size_t(B) * KV * CAP * D),
               kd = tile(size_t(KV) * B * N * D), vd = tile(size_t(KV) * B * N * D);
    std::vector<float> w(size_t(B) * KV * CAP);
    std::vector<uint32_t> pos(w.size());
    for (size_t i = 0; i < w.size(); ++i) {
        w[i] = std::uniform_real_distribution<float>(0, 2)(rng);
        pos[i] = uint32_t(i % CAP);
    }
    Harness h;
    auto *qb = put(h, "q", q), *kb = put(h, "k", k), *vb = put(h, "v", v), *kdb = put(h, "kd", kd), *vdb = put(h, "vd", vd);
    auto *cb = put(h, "ctx", ctx), *sb = put(h, "seen", seen), *nb = put(h, "nodes", nodes), *mb = put(h, "mask", mask);
    auto *pb = put(h, "path", path), *npb = put(h, "n_path", n_path), *wb = put(h, "w", w), *posb = put(h, "pos", pos);
    auto* ob = h.scratch("o", size_t(B) * N * H * D * 4);
    auto* lb = h.scratch("lse", size_t(H) * B * N * 4);
    mako::models::AttnOptions opt;
    opt.lse = lb;
    auto* enc = h.encoder();
    h.attention_tree(enc, qb, kb, vb, kdb, vdb, cb, nb, mb, ob, B, N, H, KV, CAP, CAP, D, opt);
    h.cache_append(enc, kdb, vdb, pb, npb, cb, sb, wb, posb, kb, vb, B, N, KV, CAP);
    h.cache_weights(enc, qb, lb, kb, cb, pb, npb, wb, B, N, H, KV, CAP, CAP, 0.5f);
    h.finish(enc);

    const auto at = [&](const std::vector<uint16_t>& t, size_t row, uint32_t d) { return double(oracle_f16_to_f32(t[row * D + d])); };
    const auto o = get<float>(ob, size_t(B) * N * H * D), lse = get<float>(lb, size_t(H) * B * N);
    double worst = 0, worst_l = 0;
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t r = 0; r < nodes[b]; ++r)
            for (uint32_t hh = 0; hh < H; ++hh) {
                const uint32_t g = hh / G;
                std::vector<double> s;
                std::vector<std::pair<bool, size_t>> rows;  // in the cache, row
                for (uint32_t j = 0; j < ctx[b]; ++j)
                    rows.push_back({true, (size_t(b) * KV + g) * CAP + j});
                for (uint32_t j = 0; j < nodes[b]; ++j)
                    if (mask[b * N + r] >> j & 1)
                        rows.push_back({false, size_t(g) * B * N + b * N + j});
                double mx = -INFINITY, sum = 0;
                for (const auto& [cached, row] : rows) {
                    double x = 0;
                    for (uint32_t d = 0; d < D; ++d)
                        x += at(q, size_t(hh) * B * N + b * N + r, d) * at(cached ? k : kd, row, d);
                    s.push_back(x / std::sqrt(double(D)));
                    mx = std::max(mx, s.back());
                }
                for (auto& x : s)
                    sum += x = std::exp(x - mx);
                for (uint32_t d = 0; d < D; ++d) {
                    double x = 0;
                    for (size_t j = 0; j < s.size(); ++j)
                        x += s[j] / sum * at(rows[j].first ? v : vd, rows[j].second, d);
                    worst = std::max(worst, std::fabs(o[(size_t(b) * N + r) * H * D + hh * D + d] - x) / (2e-3 + 1e-2 * std::fabs(x)));
                }
                worst_l = std::max(worst_l, std::fabs(lse[size_t(hh) * B * N + b * N + r] - (mx + std::log(sum))));
            }
    check(worst <= 1 && worst_l <= 1e-3, "attention_tree: " + std::to_string(worst) + " of the tolerance, LSE error " + std::to_string(worst_l));

    // The cache after the append.
    auto k2 = k, v2 = v;
    auto pos2 = pos;
    auto w2 = std::vector<double>(w.begin(), w.end());
    std::vector<uint32_t> ctx2{100, 35}, seen2{100, 35};
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t g = 0; g < KV; ++g)
            for (uint32_t i = 0; i < n_path[b]; ++i) {
                const size_t to = (size_t(b) * KV + g) * CAP + ctx[b] + i, from = size_t(g) * B * N + b * N + path[b * N + i];
                std::copy_n(&kd[from * D], D, &k2[to * D]);
                std::copy_n(&vd[from * D], D, &v2[to * D]);
                pos2[to] = seen[b] + i;
                w2[to] = 0;
            }
    check(get<uint16_t>(kb, k2.size()) == k2 && get<uint16_t>(vb, v2.size()) == v2 && get<uint32_t>(posb, pos2.size()) == pos2 &&
              get<uint32_t>(cb, B) == ctx2 && get<uint32_t>(sb, B) == seen2,
          "cache_append: rows, positions and counts");

    // The accepted paths' weights, over the LSE that attention_tree wrote.
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t g = 0; g < KV; ++g)
            for (uint32_t j = 0; j < ctx2[b]; ++j) {
                const size_t row = (size_t(b) * KV + g) * CAP + j;
                double x = 0;
                for (uint32_t i = 0; i < n_path[b]; ++i)
                    for (uint32_t hh = g * G; hh < (g + 1) * G && j <= ctx[b] + i; ++hh) {
                        const size_t qr = size_t(hh) * B * N + b * N + path[b * N + i];
                        double s = 0;
                        for (uint32_t d = 0; d < D; ++d)
                            s += at(q, qr, d) * at(k2, row, d);
                        x += std::exp(s / std::sqrt(double(D)) - lse[qr]);
                    }
                w2[row] = 0.5 * w2[row] + x;
            }
    const auto w_got = get<float>(wb, w.size());
    double ww = 0;
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t g = 0; g < KV; ++g)
            for (uint32_t j = 0; j < ctx2[b]; ++j) {
                const size_t row = (size_t(b) * KV + g) * CAP + j;
                ww = std::max(ww, std::fabs(w_got[row] - w2[row]));
            }
    check(ww <= 1e-4, "cache_weights: off by " + std::to_string(ww));

    // Eviction: sequence 0 down to the budget, sequence 1 as it is.
    enc = h.encoder();
    h.cache_evict(enc, kb, vb, wb, posb, sb, cb, B, KV, CAP, CAP, BUDGET, RECENT, SINKS);
    h.finish(enc);
    const auto k3 = get<uint16_t>(kb, k.size()), v3 = get<uint16_t>(vb, v.size());
    const auto pos3 = get<uint32_t>(posb, pos.size());
    const auto w3 = get<float>(wb, w.size());
    bool same = get<uint32_t>(cb, B) == std::vector<uint32_t>{BUDGET, 35};
    for (uint32_t g = 0; g < KV; ++g) {
        const size_t base = size_t(g) * CAP;
        std::vector<uint32_t> order(100);
        for (uint32_t j = 0; j < 100; ++j)
            order[j] = j;
        const auto safe = [&](uint32_t j) { return pos2[base + j] < SINKS || pos2[base + j] >= seen2[0] - RECENT; };
        std::stable_sort(order.begin(), order.end(), [&](uint32_t x, uint32_t y) {
            return safe(x) != safe(y) ? safe(x) : !safe(x) && w_got[base + x] > w_got[base + y];
        });
        order.resize(BUDGET);
        std::sort(order.begin(), order.end());
        std::vector<uint32_t> left(BUDGET), sources;
        std::vector<bool> kept(100);
        for (auto j : order)
            kept[j] = true;
        for (auto j : order)
            if (j >= BUDGET)
                sources.push_back(j);
        for (uint32_t j = 0, i = 0; j < BUDGET; ++j)
            left[j] = kept[j] ? j : sources[i++];
        for (uint32_t j = 0; j < BUDGET; ++j) {
            same = same && std::equal(&k3[(base + j) * D], &k3[(base + j) * D] + D, &k2[(base + left[j]) * D]) &&
                   std::equal(&v3[(base + j) * D], &v3[(base + j) * D] + D, &v2[(base + left[j]) * D]);
            same = same && pos3[base + j] == pos2[base + left[j]] && w3[base + j] == w_got[base + left[j]];
        }
    }
    check(same, "cache_evict: rows, weights, positions and counts");

    bool refused = false;
    try {
        enc = h.encoder();
        h.cache_evict(enc, kb, vb, wb, posb, sb, cb, B, KV, CAP, CAP, 4, RECENT, SINKS);
    } catch (const std::runtime_error& e) {
        refused = std::string(e.what()).find("over the budget") != std::string::npos;
    }
    h.finish(enc);
    check(refused, "cache_evict refuses more protected rows than the budget");

    std::printf("%s\n", failures ? "FAILED" : "all passed");
    return failures != 0;
}
