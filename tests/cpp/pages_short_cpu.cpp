// Serving from a pool that runs out, by the kernels of csrc/pages.hip on the CPU (cpu_hip/hip/hip_runtime.h): sequences of
// unlike lengths that share pages reserve, write, fork, end and are cut back, with too few free pages as a rule. After each
// step every sequence's rows, through its table, are those that it was given and no others, the pages' holders are those that
// the tables name, and who got room is as defined.
//   pages_short_cpu
#include <hip/hip_runtime.h>

inline int __popcll(uint64_t x) { return __builtin_popcountll(x); }
inline uint32_t atomicSub(uint32_t* p, uint32_t x)
{
    const uint32_t old = *p;
    *p = old - x;
    return old;
}
inline uint32_t atomicMax(uint32_t* p, uint32_t x)
{
    const uint32_t old = *p;
    *p = old > x ? old : x;
    return old;
}
inline uint32_t atomicCAS(uint32_t* p, uint32_t expect, uint32_t x)
{
    const uint32_t old = *p;
    if (old == expect)
        *p = x;
    return old;
}

#include "../../mako-common_amd/csrc/pages.hip"

#include <cstdio>
#include <map>
#include <random>

namespace mako {
int fail(int code, const char*, ...) { return code; }
int ok() { return MAKO_OK; }
int check_launch(const char*) { return MAKO_OK; }
uint32_t device_cus() { return 256; }
}  // namespace mako

namespace {

using U32s = std::vector<uint32_t>;
constexpr uint32_t kNone = 0xffffffffu, kPage = 64, kRow = 32;  // a row of a head of 64: 32 words
std::mt19937 rng(11);
uint32_t upto(uint32_t n) { return rng() % (n + 1); }

struct Aligned {  // words at a 16-byte boundary
    U32s all;
    size_t off = 0;
    explicit Aligned(size_t n, uint32_t x = 0) : all(n + 4, x)
    {
        while (reinterpret_cast<uintptr_t>(all.data() + off) % 16)
            ++off;
    }
    uint32_t* data() { return all.data() + off; }
};

// Who gets room: sequences in order, free pages in order; of those that append to one partly filled page that nobody else holds
// the last keeps it, unless another got no page for its copy and has rows where the last one's new rows would go.
U32s room(U32s table, U32s refs, const U32s& ctx, const U32s& n, uint32_t max_pages)
{
    const uint32_t batch = (uint32_t)ctx.size();
    std::map<uint32_t, U32s> appends;
    for (uint32_t b = 0; b < batch; ++b)
        if (n[b] && ctx[b] % kPage && ctx[b] < max_pages * kPage)
            appends[table[b * max_pages + ctx[b] / kPage]].push_back(b);
    U32s out(batch);
    std::map<uint32_t, uint32_t> left;  // rows of those whose copy of a page failed
    size_t free = std::count(refs.begin(), refs.end(), 0u);
    for (uint32_t b = 0; b < batch; ++b) {
        const uint32_t end = std::min(ctx[b] + n[b], max_pages * kPage);
        uint32_t at = ctx[b];
        while (at < end) {
            const uint32_t e = table[b * max_pages + at / kPage], part = at % kPage;
            bool needs = e == kNone;
            if (e != kNone && part && refs[e] > 1) {
                const U32s& a = appends[e];
                if (refs[e] > a.size() || a.back() != b)
                    needs = true;
                else if (left[e] > part)
                    break;
                if (needs && !free)
                    left[e] = std::max(left[e], part);
            }
            if (needs && !free)
                break;
            free -= needs;
            at = std::min(end, (at / kPage + 1) * kPage);
        }
        out[b] = at;
    }
    return out;
}

struct Server {
    uint32_t batch, pages, max_pages;
    Aligned k, v;
    U32s table, refs, ctx;
    std::vector<U32s> rows;  // each sequence's rows, as what k holds in them (v: its complement)
    uint32_t next = 1;

    Server(uint32_t b, uint32_t p, uint32_t m)
        : batch(b), pages(p), max_pages(m), k((size_t)p * kPage * kRow), v((size_t)p * kPage * kRow), table(b * m, kNone),
          refs(p, 0), ctx(b, 0), rows(b)
    {
    }
    mako_pages_args args(uint32_t n = 0) const { return {batch, n, n, pages, kPage, max_pages, 1, 64, 1}; }

    bool step(const U32s& n, const char* what)
    {
        U32s starts(batch + 1, 0), end(batch);
        for (uint32_t b = 0; b < batch; ++b)
            starts[b + 1] = starts[b] + n[b];
        const uint32_t total = starts[batch];
        const mako_pages_args a = args(total);
        const U32s want = room(table, refs, ctx, n, max_pages);
        Aligned ws(mako_pages_reserve_workspace(&a) / 4 + 4), kd((size_t)total * kRow), vd((size_t)total * kRow);
        for (uint32_t r = 0; r < total; ++r)
            for (uint32_t d = 0; d < kRow; ++d) {
                kd.data()[r * kRow + d] = next + r;
                vd.data()[r * kRow + d] = ~(next + r);
            }
        if (mako_pages_reserve(&a, table.data(), refs.data(), starts.data(), ctx.data(), table.data(), refs.data(), end.data(),
                               k.data(), v.data(), ws.data(), mako_pages_reserve_workspace(&a), nullptr) ||
            mako_pages_write(&a, kd.data(), vd.data(), table.data(), starts.data(), ctx.data(), end.data(), k.data(), v.data(),
                             nullptr)) {
            std::printf("FAILED %s: refused\n", what);
            return false;
        }
        for (uint32_t b = 0; b < batch; ++b)
            for (uint32_t i = 0; ctx[b] + i < end[b]; ++i)
                rows[b].push_back(next + starts[b] + i);
        next += total;
        if (end != want) {
            for (uint32_t b = 0; b < batch; ++b)
                if (end[b] != want[b]) {
                    std::printf("FAILED %s: sequence %u has room for %u rows, not %u\n", what, b, end[b], want[b]);
                    break;
                }
            return false;
        }
        ctx = end;
        return check(what);
    }

    bool fork(const U32s& parent, const U32s& keep, const char* what)
    {
        const mako_pages_args a = args();
        Aligned ws(mako_pages_fork_workspace(&a) / 4 + 4);
        if (mako_pages_fork(&a, parent.data(), keep.data(), table.data(), refs.data(), ctx.data(), table.data(), refs.data(),
                            ctx.data(), ws.data(), mako_pages_fork_workspace(&a), nullptr))
            return false;
        std::vector<U32s> old = rows;
        for (uint32_t b = 0; b < batch; ++b) {
            rows[b] = parent[b] < batch ? old[parent[b]] : U32s{};
            rows[b].resize(std::min<size_t>(rows[b].size(), keep[b]));
        }
        return check(what);
    }

    bool check(const char* what)
    {
        U32s holders(pages, 0);
        for (uint32_t b = 0; b < batch; ++b) {
            for (uint32_t j = 0; j < max_pages; ++j)
                if (const uint32_t e = table[b * max_pages + j]; e < pages)
                    ++holders[e];
            if (ctx[b] != rows[b].size()) {
                std::printf("FAILED %s: sequence %u of %u rows, not %zu\n", what, b, ctx[b], rows[b].size());
                return false;
            }
            for (uint32_t i = 0; i < ctx[b]; ++i) {
                const uint32_t e = table[b * max_pages + i / kPage];
                const size_t at = ((size_t)e * kPage + i % kPage) * kRow;
                if (e >= pages || k.data()[at] != rows[b][i] || k.data()[at + kRow - 1] != rows[b][i] ||
                    v.data()[at] != ~rows[b][i]) {
                    std::printf("FAILED %s: row %u of sequence %u (of %u) is not its own\n", what, i, b, ctx[b]);
                    return false;
                }
            }
        }
        if (holders != refs) {
            std::printf("FAILED %s: holders\n", what);
            return false;
        }
        return true;
    }
};

// Two sequences that share the first rows of one; a row each.
bool two(uint32_t first, uint32_t second, uint32_t pages, U32s want)
{
    Server s(2, pages, 2);
    const bool good = s.step({std::max(first, second), 0}, "two: prompt") && s.fork({0, 0}, {first, second}, "two: fork") &&
                      s.step({1, 1}, "two: a row each");
    if (good && s.ctx != want)
        std::printf("FAILED two: %u and %u rows of %u pages\n", s.ctx[0], s.ctx[1], pages);
    return good && s.ctx == want;
}

bool loop(uint32_t batch, uint32_t pages, uint32_t rounds, uint32_t most)
{
    char what[64];
    Server s(batch, pages, 6);
    for (uint32_t i = 0; i < rounds; ++i) {
        std::snprintf(what, sizeof(what), "batch %u, %u pages, round %u", batch, pages, i);
        U32s n(batch), parent(batch), keep(batch);
        for (uint32_t b = 0; b < batch; ++b)
            n[b] = upto(5) == 0 ? 0 : upto(3) == 0 ? upto(most) : 1;
        if (!s.step(n, what))
            return false;
        if (i % 3 != 2)
            continue;
        // some go on from a neighbour, cut inside a page as a rule, some end
        for (uint32_t b = 0; b < batch; ++b) {
            const uint32_t x = upto(5);
            parent[b] = x == 0 ? kNone : x < 4 ? b - b % 4 + std::min(upto(3), batch - 1 - (b - b % 4)) : b;
            const uint32_t c = parent[b] == kNone ? 0 : s.ctx[parent[b]];
            keep[b] = x < 3 && c ? c - upto(std::min(c, kPage - 1)) : c;
        }
        if (!s.fork(parent, keep, what))
            return false;
    }
    return true;
}

}  // namespace

int main()
{
    bool good = two(50, 30, 1, {50, 30}) && two(50, 30, 2, {51, 31}) && two(50, 50, 1, {50, 51}) && two(50, 49, 1, {50, 49}) &&
                two(30, 50, 1, {30, 51}) && two(64, 30, 1, {64, 30}) && two(64, 30, 2, {65, 30}) && two(64, 30, 3, {65, 31});
    for (uint32_t round = 0; good && round < 3; ++round) {
        const uint32_t batch = 2 + upto(38);
        good &= loop(batch, batch / 2 + upto(2 * batch), 9, round % 2 ? 3 : 90);
    }
    good = good && loop(1030, 700, 4, 4);
    std::puts(good ? "all passed" : "FAILED");
    return good ? 0 : 1;
}
