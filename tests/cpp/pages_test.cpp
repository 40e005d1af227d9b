// A cache kept in pages through TransformerRuntime (pages_reserve, pages_write, attention_paged, pages_fork, pages_compact),
// against a host that keeps every sequence's rows: prompts, steps of one token, chunks among them, sequences that fork, end and
// start again, compaction, in two layers of 8 query heads over 2 kv heads of 128, f16 tiles and f32 rows. Tolerance: outputs
// within 2e-3 + 1e-2 |ref| (as the other attention tests), LSE within 1e-3; counts and the number of used pages are equal.
//   pages_test
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "attn_oracle.h"
#include "transformer_runtime.hpp"

namespace {

class Harness final : public mako::models::TransformerRuntime {
public:
    Harness() : TransformerRuntime(mako::gpu::Telemetry::kernels) {}
    using TransformerRuntime::attention_paged;
    using TransformerRuntime::encoder;
    using TransformerRuntime::finish;
    using TransformerRuntime::pages_compact;
    using TransformerRuntime::pages_fork;
    using TransformerRuntime::pages_reserve;
    using TransformerRuntime::pages_write;
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
mako::gpu::Buffer* put(Harness& h, const std::string& name, const std::vector<T>& v)
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

constexpr uint32_t B = 4, H = 8, KV = 2, D = 128, L = 2, PAGE = 64, PAGES = 40, MAX_PAGES = 8;
using Row = std::vector<double>;  // [L][2][KV][D]
std::vector<std::vector<Row>> seqs(B);

struct Step {
    Harness& h;
    mako::models::PagedCache c;
    mako::gpu::Buffer* end;

    void operator()(const std::vector<uint32_t>& n, const std::string& what)
    {
        std::vector<uint32_t> starts{0};
        for (uint32_t x : n)
            starts.push_back(starts.back() + x);
        const uint32_t rows = starts[B];
        std::normal_distribution<float> dist;
        const auto tile = [&](size_t size) {
            std::vector<uint16_t> v(size);
            for (auto& x : v)
                x = oracle_f32_to_f16(dist(rng));
            return v;
        };
        const auto at = [](const std::vector<uint16_t>& t, size_t i) { return double(oracle_f16_to_f32(t[i])); };
        std::vector<std::vector<uint16_t>> q, kd, vd;
        std::vector<mako::gpu::Buffer*> o, lse;
        auto* st = put(h, "starts", starts);
        uint32_t max_ctx = 0;
        for (uint32_t b = 0; b < B; ++b)
            max_ctx = std::max(max_ctx, uint32_t(seqs[b].size()) + n[b]);
        auto* enc = h.encoder();
        h.pages_reserve(enc, c, st, end, rows);
        for (uint32_t l = 0; l < L; ++l) {
            const std::string s = std::to_string(l);
            q.push_back(tile(size_t(H) * rows * D)), kd.push_back(tile(size_t(KV) * rows * D)), vd.push_back(tile(size_t(KV) * rows * D));
            auto *qb = put(h, "q" + s, q[l]), *kb = put(h, "kd" + s, kd[l]), *vb = put(h, "vd" + s, vd[l]);
            o.push_back(h.scratch("o" + s, size_t(rows) * H * D * 4));
            lse.push_back(h.scratch("lse" + s, size_t(H) * rows * 4));
            mako::models::AttnOptions opt;
            opt.lse = lse[l];
            h.pages_write(enc, kb, vb, c, l, st, end, rows);
            h.attention_paged(enc, qb, c, l, st, o[l], rows, H, *std::max_element(n.begin(), n.end()), max_ctx, opt);
        }
        h.finish(enc);
        std::swap(c.ctx_len, end);

        for (uint32_t b = 0; b < B; ++b)
            for (uint32_t i = starts[b]; i < starts[b + 1]; ++i) {
                Row row;
                for (uint32_t l = 0; l < L; ++l)
                    for (const auto* t : {&kd[l], &vd[l]})
                        for (uint32_t g = 0; g < KV; ++g)
                            for (uint32_t d = 0; d < D; ++d)
                                row.push_back(at(*t, (size_t(g) * rows + i) * D + d));
                seqs[b].push_back(row);
            }
        double worst = 0, worst_l = 0;
        for (uint32_t l = 0; l < L; ++l) {
            const auto got = get<float>(o[l], size_t(rows) * H * D), got_l = get<float>(lse[l], size_t(H) * rows);
            for (uint32_t b = 0; b < B; ++b)
                for (uint32_t i = 0; i < n[b]; ++i)
                    for (uint32_t hh = 0; hh < H; ++hh) {
                        const uint32_t g = hh * KV / H, r = starts[b] + i;
                        const size_t seen = seqs[b].size() - n[b] + i + 1;
                        std::vector<double> s(seen);
                        double mx = -INFINITY, sum = 0;
                        for (size_t j = 0; j < seen; ++j) {
                            double x = 0;
                            for (uint32_t d = 0; d < D; ++d)
                                x += at(q[l], (size_t(hh) * rows + r) * D + d) * seqs[b][j][((l * 2) * KV + g) * D + d];
                            s[j] = x / std::sqrt(double(D));
                            mx = std::max(mx, s[j]);
                        }
                        for (auto& x : s)
                            sum += x = std::exp(x - mx);
                        for (uint32_t d = 0; d < D; ++d) {
                            double x = 0;
                            for (size_t j = 0; j < seen; ++j)
                                x += s[j] / sum * seqs[b][j][((l * 2 + 1) * KV + g) * D + d];
                            worst = std::max(worst, std::fabs(got[size_t(r) * H * D + hh * D + d] - x) / (2e-3 + 1e-2 * std::fabs(x)));
                        }
                        worst_l = std::max(worst_l, std::fabs(got_l[size_t(hh) * rows + r] - (mx + std::log(sum))));
                    }
        }
        const auto ctx = get<uint32_t>(c.ctx_len, B);
        bool same = true;
        for (uint32_t b = 0; b < B; ++b)
            same = same && ctx[b] == seqs[b].size();
        check(worst <= 1 && worst_l <= 1e-3 && same,
              what + ": " + std::to_string(worst) + " of the tolerance, LSE error " + std::to_string(worst_l));
    }

    void fork(const std::vector<uint32_t>& parent, const std::vector<uint32_t>& keep, const std::string& what)
    {
        auto *p = put(h, "parent", parent), *k = put(h, "keep", keep);
        auto* enc = h.encoder();
        h.pages_fork(enc, c, p, k);
        h.finish(enc);
        auto next = seqs;
        for (uint32_t b = 0; b < B; ++b) {
            next[b] = parent[b] < B ? seqs[parent[b]] : std::vector<Row>{};
            next[b].resize(std::min<size_t>(next[b].size(), keep[b]));
        }
        seqs = next;
        check(holders(), what + ": holders");
    }

    // Every page has as many holders as the table names it, and the sequences' rows have pages.
    bool holders()
    {
        const auto table = get<uint32_t>(c.table, B * MAX_PAGES), refs = get<uint32_t>(c.refs, PAGES);
        std::vector<uint32_t> n(PAGES);
        bool ok = true;
        for (uint32_t b = 0; b < B; ++b)
            for (uint32_t j = 0; j < MAX_PAGES; ++j) {
                const uint32_t e = table[b * MAX_PAGES + j];
                ok = ok && (e < PAGES) == (j * PAGE < seqs[b].size());
                if (e < PAGES)
                    ++n[e];
            }
        return ok && n == refs;
    }
};

}  // namespace

int main()
{
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    Harness h;
    const size_t pool = size_t(L) * PAGES * KV * PAGE * D;
    const std::vector<uint16_t> nan(pool, 0x7e00);
    Step step{h,
              {put(h, "k", nan), put(h, "v", nan), put(h, "table", std::vector<uint32_t>(B * MAX_PAGES, ~0u)),
               put(h, "refs", std::vector<uint32_t>(PAGES, 0)), put(h, "ctx", std::vector<uint32_t>(B, 0)), B, PAGES, PAGE,
               MAX_PAGES, KV, D, L},
              h.scratch("end", B * 4)};
    step({150, 70, 1, 0}, "prompts");
    step({1, 1, 1, 1}, "one token each");
    step({1, 60, 1, 130}, "chunks among single tokens");
    step.fork({0, 0, 2, B}, {~0u, ~0u, ~0u, 0}, "a fork, an end");
    step({1, 1, 1, 90}, "forks go their own ways, a new prompt");
    step({1, 1, 80, 1}, "a later chunk");
    step.fork({0, 1, 3, 0}, {64, 100, ~0u, 130}, "cut back and forked");
    step({2, 3, 1, 1}, "drafted tokens");

    auto* used = h.scratch("used", 4);
    auto* map = h.scratch("map", PAGES * 4);
    auto* enc = h.encoder();
    h.pages_compact(enc, step.c, used, map);
    h.finish(enc);
    const auto refs = get<uint32_t>(step.c.refs, PAGES);
    const uint32_t n = get<uint32_t>(used, 1)[0];
    bool low = true;
    for (uint32_t i = 0; i < PAGES; ++i)
        low = low && (refs[i] > 0) == (i < n);
    check(low && step.holders(), "compaction: the used pages are the lowest");
    step({1, 1, 33, 1}, "after compaction");

    bool refused = false;
    try {
        enc = h.encoder();
        h.pages_reserve(enc, step.c, nullptr, step.c.ctx_len, B);
    } catch (const std::runtime_error& e) {
        refused = std::string(e.what()).find("ctx_len") != std::string::npos;
    }
    h.finish(enc);
    check(refused, "pages_reserve refuses ctx_len for end");
    refused = false;
    try {
        enc = h.encoder();
        h.pages_write(enc, used, used, step.c, L, nullptr, nullptr, B);
    } catch (const std::runtime_error& e) {
        refused = std::string(e.what()).find("layer 2") != std::string::npos;
    }
    h.finish(enc);
    check(refused, "pages_write refuses a layer that the pool does not have");

    std::printf("%s\n", failures ? "FAILED" : "all passed");
    return failures != 0;
}
