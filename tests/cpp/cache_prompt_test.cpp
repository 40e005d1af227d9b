// A prompt enters a cache through TransformerRuntime by the tiles of attention(), whose heads are padded to a multiple of 64
// rows: heads, attention with its LSE, cache_append, cache_weights, for a prompt of 100 tokens in tiles of 128 rows, then a
// tree of 5 drafts in tiles of 64. f16 tiles, 4 query heads over 2 kv heads of 128. The rows that the cache gets and their
// counts are equal to the tiles'; the gathered weights within 1e-4 of double arithmetic over the tiles and the LSE; the
// tree's output the bits of the same call on tiles without padding.
//   cache_prompt_test
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
    Harness() : TransformerRuntime(mako::gpu::Telemetry::off) {}
    using TransformerRuntime::attention;
    using TransformerRuntime::attention_tree;
    using TransformerRuntime::cache_append;
    using TransformerRuntime::cache_weights;
    using TransformerRuntime::encoder;
    using TransformerRuntime::finish;
    using TransformerRuntime::heads;
    using TransformerRuntime::scratch;
};

int failures = 0;
void check(bool ok, const std::string& what)
{
    std::printf("  %s  %s\n", ok ? "ok  " : "FAIL", what.c_str());
    failures += !ok;
}

std::mt19937 rng(11);

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

std::vector<float> rows_of(uint32_t n)
{
    std::normal_distribution<float> d;
    std::vector<float> v(n);
    for (auto& x : v)
        x = d(rng);
    return v;
}

// The first `rows` of each head of a tile of `pad` rows.
std::vector<uint16_t> packed(const std::vector<uint16_t>& t, uint32_t heads, uint32_t rows, uint32_t pad, uint32_t D)
{
    std::vector<uint16_t> p(size_t(heads) * rows * D);
    for (uint32_t h = 0; h < heads; ++h)
        std::copy_n(&t[size_t(h) * pad * D], size_t(rows) * D, &p[size_t(h) * rows * D]);
    return p;
}

}  // namespace

int main()
{
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    constexpr uint32_t T = 100, PAD = 128, N = 5, NPAD = 64, H = 4, KV = 2, D = 128, CAP = 120;
    Harness h;
    auto* enc = h.encoder();
    auto* q = h.scratch("q", size_t(H) * PAD * D * 2);
    auto* k = h.scratch("kt", size_t(KV) * PAD * D * 2);
    auto* v = h.scratch("vt", size_t(KV) * PAD * D * 2);
    auto *xq = put(h, "xq", rows_of(T * H * D)), *xk = put(h, "xk", rows_of(T * KV * D)), *xv = put(h, "xv", rows_of(T * KV * D));
    h.heads(enc, xq, H * D, 0, H, T, PAD, nullptr, 0, q);
    h.heads(enc, xk, KV * D, 0, KV, T, PAD, nullptr, 0, k);
    h.heads(enc, xv, KV * D, 0, KV, T, PAD, nullptr, 0, v);
    auto *att = h.scratch("att", size_t(T) * H * D * 4), *lse = h.scratch("lse", size_t(H) * T * 4);
    mako::models::AttnOptions opt;
    opt.lse = lse;
    h.attention(enc, q, k, v, att, T, PAD, T, PAD, H, KV, 0, 0xffffffffu, D, opt);
    const std::vector<uint16_t> blank(size_t(KV) * CAP * D, 0x3c00);
    auto *kc = put(h, "kc", blank), *vc = put(h, "vc", blank);
    auto *ctx = put(h, "ctx", std::vector<uint32_t>{0}), *seen = put(h, "seen", std::vector<uint32_t>{0});
    auto* w = put(h, "w", std::vector<float>(KV * CAP, 5.0f));
    auto* pos = put(h, "pos", std::vector<uint32_t>(KV * CAP, 9u));
    h.cache_append(enc, k, v, nullptr, nullptr, ctx, seen, w, pos, kc, vc, 1, T, KV, CAP, D, MAKO_F16, PAD);
    h.cache_weights(enc, q, lse, kc, ctx, nullptr, nullptr, w, 1, T, H, KV, CAP, CAP, 1.0f, false, D, MAKO_F16, PAD);
    h.finish(enc);

    const auto qt = get<uint16_t>(q, size_t(H) * PAD * D), kt = get<uint16_t>(k, size_t(KV) * PAD * D),
               vt = get<uint16_t>(v, size_t(KV) * PAD * D);
    auto want_k = blank, want_v = blank;
    std::vector<uint32_t> want_pos(KV * CAP, 9u);
    for (uint32_t g = 0; g < KV; ++g) {
        std::copy_n(&kt[size_t(g) * PAD * D], size_t(T) * D, &want_k[size_t(g) * CAP * D]);
        std::copy_n(&vt[size_t(g) * PAD * D], size_t(T) * D, &want_v[size_t(g) * CAP * D]);
        for (uint32_t j = 0; j < T; ++j)
            want_pos[g * CAP + j] = j;
    }
    check(get<uint16_t>(kc, want_k.size()) == want_k && get<uint16_t>(vc, want_v.size()) == want_v &&
              get<uint32_t>(pos, want_pos.size()) == want_pos && get<uint32_t>(ctx, 1)[0] == T && get<uint32_t>(seen, 1)[0] == T,
          "cache_append of padded tiles: rows, positions and counts");
    const auto l = get<float>(lse, size_t(H) * T), got = get<float>(w, KV * CAP);
    double worst = 0;
    for (uint32_t g = 0; g < KV; ++g)
        for (uint32_t j = 0; j < CAP; ++j) {
            double x = j < T ? 0.0 : 5.0;
            for (uint32_t hh = g * H / KV; j < T && hh < (g + 1) * H / KV; ++hh)
                for (uint32_t i = j; i < T; ++i) {
                    double s = 0;
                    for (uint32_t d = 0; d < D; ++d)
                        s += double(oracle_f16_to_f32(qt[(size_t(hh) * PAD + i) * D + d])) *
                             double(oracle_f16_to_f32(kt[(size_t(g) * PAD + j) * D + d]));
                    x += std::exp(s / std::sqrt(double(D)) - l[size_t(hh) * T + i]);
                }
            worst = std::max(worst, std::fabs(got[g * CAP + j] - x));
        }
    check(worst <= 1e-4, "cache_weights of padded tiles: off by " + std::to_string(worst));

    enc = h.encoder();
    auto* dq = h.scratch("dq", size_t(H) * NPAD * D * 2);
    auto *dk = h.scratch("dk", size_t(KV) * NPAD * D * 2), *dv = h.scratch("dv", size_t(KV) * NPAD * D * 2);
    h.heads(enc, put(h, "xdq", rows_of(N * H * D)), H * D, 0, H, N, NPAD, nullptr, 0, dq);
    h.heads(enc, put(h, "xdk", rows_of(N * KV * D)), KV * D, 0, KV, N, NPAD, nullptr, 0, dk);
    h.heads(enc, put(h, "xdv", rows_of(N * KV * D)), KV * D, 0, KV, N, NPAD, nullptr, 0, dv);
    auto *o1 = h.scratch("o1", size_t(N) * H * D * 4), *o2 = h.scratch("o2", size_t(N) * H * D * 4);
    h.attention_tree(enc, dq, kc, vc, dk, dv, ctx, nullptr, nullptr, o1, 1, N, H, KV, CAP, CAP, D, {}, NPAD, NPAD);
    h.finish(enc);
    auto* pq = put(h, "pq", packed(get<uint16_t>(dq, size_t(H) * NPAD * D), H, N, NPAD, D));
    auto* pk = put(h, "pk", packed(get<uint16_t>(dk, size_t(KV) * NPAD * D), KV, N, NPAD, D));
    auto* pv = put(h, "pv", packed(get<uint16_t>(dv, size_t(KV) * NPAD * D), KV, N, NPAD, D));
    enc = h.encoder();
    h.attention_tree(enc, pq, kc, vc, pk, pv, ctx, nullptr, nullptr, o2, 1, N, H, KV, CAP, CAP, D);
    h.finish(enc);
    check(get<uint32_t>(o1, size_t(N) * H * D) == get<uint32_t>(o2, size_t(N) * H * D),
          "attention_tree of padded tiles: the bits of the call without padding");

    std::printf("%s\n", failures ? "FAILED" : "all passed");
    return failures != 0;
}
