// The kernels of csrc/cache_rows.hip on the CPU (cpu_hip/hip/hip_runtime.h), called through mako_cache_evict, against a
// sort on the host: rows, weights, positions and counts equal, and the words around the workspace and each output as they
// were. Lists of one, two and three LDS blocks (32768 rows), budgets at and around the blocks' ends.
//   cache_rows_cpu
#include "../../mako-common_amd/csrc/cache_rows.hip"

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <numeric>
#include <random>
#include <string>

namespace mako {
static std::string last;
int fail(int code, const char* f, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, f);
    std::vsnprintf(buf, sizeof(buf), f, ap);
    va_end(ap);
    last = buf;
    return code;
}
int ok() { return MAKO_OK; }
int check_launch(const char*) { return MAKO_OK; }
uint32_t device_cus() { return 256; }
}  // namespace mako

namespace {

constexpr size_t kGuard = 40000;  // words on either side of the workspace and behind each output
constexpr uint32_t kMark = 0xa5a5a5a5u;

struct Case {
    std::vector<uint32_t> ctx;
    uint32_t budget, recent = 0, sinks = 0;
    int weights = 0;  // 0: distinct, 1: three values, 2: all equal, 3: few distinct, a tie at the cut
    bool moved = false;
    uint32_t max_ctx = 0;
};

std::mt19937 rng(5);

bool run(const Case& c, bool in_place)
{
    const uint32_t B = c.ctx.size(), D = 64, cap = *std::max_element(c.ctx.begin(), c.ctx.end()) + 2;
    std::vector<uint16_t> k(size_t(B) * cap * D), v(k.size());
    for (size_t i = 0; i < k.size(); ++i)
        k[i] = uint16_t(i * 40503u >> 3), v[i] = uint16_t(i * 30011u >> 5);
    std::vector<float> w(size_t(B) * cap);
    std::vector<uint32_t> pos(w.size()), ctx = c.ctx, seen(B);
    for (uint32_t b = 0; b < B; ++b) {
        std::vector<uint32_t> order(cap);
        std::iota(order.begin(), order.end(), 0u);
        std::shuffle(order.begin(), order.end(), rng);
        for (uint32_t j = 0; j < cap; ++j) {
            w[b * cap + j] = c.weights == 0 ? float(order[j]) * 0.25f : c.weights == 1 ? float(rng() % 3)
                             : c.weights == 2 ? 1.0f : float(order[j] / 50);
            pos[b * cap + j] = c.moved ? order[(j * 7 + 3) % cap] : j;
        }
        seen[b] = c.moved ? cap + 5 : ctx[b];
    }
    const mako_evict_args a{B, 1, D, cap, c.max_ctx ? c.max_ctx : cap, c.budget, c.recent, c.sinks};
    const size_t bytes = mako_cache_evict_workspace(&a);
    std::vector<uint32_t> space(2 * kGuard + (bytes + 3) / 4 + 64, kMark);
    uint32_t* ws = space.data() + kGuard;
    while (reinterpret_cast<uintptr_t>(ws) % 16)
        ++ws;
    auto k2 = k, v2 = v;
    std::vector<float> w2(w.size() + kGuard, 7.0f), w_in = w;
    std::vector<uint32_t> pos2(w2.size(), 7u), pos_in = pos, ctx2(B, 9u);
    if (in_place) {
        std::copy(w.begin(), w.end(), w2.begin());
        std::copy(pos.begin(), pos.end(), pos2.begin());
        ctx2 = ctx;
    }
    const bool given = c.moved || in_place;
    const int rc = mako_cache_evict(&a, MAKO_F16, k2.data(), v2.data(), in_place ? w2.data() : w_in.data(),
                                    !given ? nullptr : in_place ? pos2.data() : pos_in.data(), given ? seen.data() : nullptr,
                                    in_place ? ctx2.data() : ctx.data(), w2.data(), pos2.data(), ctx2.data(), ws, bytes,
                                    nullptr);
    if (rc != MAKO_OK) {
        std::printf("%s\n", mako::last.c_str());
        return false;
    }
    bool same = true;
    for (size_t i = 0; i < space.size(); ++i)
        if (&space[i] < ws || &space[i] >= ws + (bytes + 3) / 4)
            same = same && space[i] == kMark;
    if (!same)
        std::printf("    a word outside the workspace was written\n");
    auto want_k = k, want_v = v;
    std::vector<float> want_w = in_place ? w : std::vector<float>(w.size(), 7.0f);
    std::vector<uint32_t> want_pos = in_place ? pos : std::vector<uint32_t>(w.size(), 7u);
    for (uint32_t b = 0; b < B; ++b) {
        const uint32_t n = std::min(c.ctx[b], a.max_ctx), m = std::min(n, c.budget);
        const uint32_t tokens = given ? seen[b] : n;
        std::vector<uint32_t> order(n), left(m), sources;
        std::iota(order.begin(), order.end(), 0u);
        const auto safe = [&](uint32_t j) { return pos[b * cap + j] < c.sinks || pos[b * cap + j] + c.recent >= tokens; };
        std::stable_sort(order.begin(), order.end(), [&](uint32_t x, uint32_t y) {
            return safe(x) != safe(y) ? safe(x) : !safe(x) && w[b * cap + x] > w[b * cap + y];
        });
        order.resize(m);
        std::sort(order.begin(), order.end());
        std::vector<bool> kept(n);
        for (uint32_t j : order)
            kept[j] = true;
        for (uint32_t j : order)
            if (j >= m)
                sources.push_back(j);
        for (uint32_t j = 0, i = 0; j < m; ++j) {
            const size_t from = b * size_t(cap) + (left[j] = kept[j] ? j : sources[i++]), to = b * size_t(cap) + j;
            std::copy_n(&k[from * D], D, &want_k[to * D]);
            std::copy_n(&v[from * D], D, &want_v[to * D]);
            want_w[to] = w[from];
            want_pos[to] = pos[from];
        }
        same = same && ctx2[b] == m;
    }
    same = same && k2 == want_k && v2 == want_v;
    for (size_t i = 0; i < w2.size(); ++i)
        same = same && w2[i] == (i < want_w.size() ? want_w[i] : 7.0f) && pos2[i] == (i < want_pos.size() ? want_pos[i] : 7u);
    return same;
}

}  // namespace

int main()
{
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    std::vector<Case> cases{
        {{300, 3, 64, 0}, 64},
        {{4096, 4097}, 1000, 30, 4},
        {{4000, 513}, 512, 100, 0, 1, true},
        {{32768}, 32767},
        {{32769, 100}, 32768},
        {{33000}, 4096, 512, 4, 0, true},
        {{40000}, 32767},
        {{40000}, 32768},
        {{40000}, 32769},
        {{40000}, 33000},
        {{40000}, 33000, 400, 3, 0, true},
        {{40000, 36000}, 33000, 0, 0, 1},
        {{40000}, 33000, 0, 0, 2},
        {{40000}, 33333, 0, 0, 3},
        {{40000}, 39990, 0, 0, 0, true},
        {{70001}, 40000},
        {{70001}, 65535},
        {{70001}, 65536},
        {{70001}, 65537, 999, 2},
        {{70001}, 69000, 500, 4, 3, true},
        {{98305}, 98304},
        {{131072}, 65536},
        {{50000, 70001}, 34000, 0, 0, 0, false, 41000},
    };
    int failures = 0;
    for (const auto& c : cases)
        for (bool in_place : {false, true}) {
            std::printf("  list of %u rows to %u, weights %d%s%s\n", c.ctx[0], c.budget, c.weights, c.moved ? ", moved" : "",
                        in_place ? ", in place" : "");
            if (!run(c, in_place)) {
                std::printf("FAIL\n");
                ++failures;
            }
        }
    std::printf("%s\n", failures ? "FAILED" : "all passed");
    return failures != 0;
}
