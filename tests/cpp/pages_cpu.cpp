// The kernels of csrc/pages.hip on the CPU (cpu_hip/hip/hip_runtime.h), called through their entry points, against plain
// host code: pools, tables, holders and counts equal, in place and not, and the words around every output and workspace as
// they were, also where starts, tables and holders are not what they should be.
//   pages_cpu
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

#include <cstdarg>
#include <cstdio>
#include <cstring>
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

using U32s = std::vector<uint32_t>;
constexpr uint32_t kNone = 0xffffffffu, kMark = 0xa5a5a5a5u;
constexpr size_t kGuard = 4096;
std::mt19937 rng(7);
uint32_t upto(uint32_t n) { return rng() % (n + 1); }

// Words between guards, 16-byte aligned.
struct Guarded {
    U32s all;
    size_t n, off = kGuard;
    explicit Guarded(const U32s& x) : all(x.size() + 2 * kGuard + 4, kMark), n(x.size())
    {
        while (reinterpret_cast<uintptr_t>(all.data() + off) % 16)
            ++off;
        std::copy(x.begin(), x.end(), all.begin() + off);
    }
    uint32_t* data() { return all.data() + off; }
    U32s value() const { return U32s(all.begin() + off, all.begin() + off + n); }
    bool whole() const
    {
        for (size_t i = 0; i < all.size(); ++i)
            if ((i < off || i >= off + n) && all[i] != kMark)
                return false;
        return true;
    }
};
U32s numbers(size_t n, uint32_t seed)
{
    U32s x(n);
    for (size_t i = 0; i < n; ++i)
        x[i] = (uint32_t)i * 2654435761u + seed;
    return x;
}

struct State {
    uint32_t batch, pages, page, max_pages;
    U32s table, refs, ctx;
};
// Sequences of `low` to `high` rows over pages anywhere in the pool, in sets that hold the same pages.
State state(uint32_t batch, uint32_t page, uint32_t max_pages, uint32_t spare, uint32_t high, uint32_t beams)
{
    State s{batch, 0, page, max_pages, U32s(batch * max_pages, kNone), {}, U32s(batch)};
    U32s order;
    uint32_t held = 0;
    for (uint32_t b = 0; b < batch; ++b)
        s.ctx[b] = b % beams ? s.ctx[b - 1] : upto(high);
    for (uint32_t b = 0; b < batch; b += beams)
        held += (s.ctx[b] + page - 1) / page;
    s.pages = held + spare;
    for (uint32_t i = 0; i < s.pages; ++i)
        order.push_back(i);
    std::shuffle(order.begin(), order.end(), rng);
    s.refs.assign(s.pages, 0);
    uint32_t next = 0;
    for (uint32_t b = 0; b < batch; ++b)
        for (uint32_t j = 0; j < (s.ctx[b] + page - 1) / page; ++j) {
            const uint32_t e = b % beams ? s.table[(b - 1) * max_pages + j] : order[next++];
            s.table[b * max_pages + j] = e;
            ++s.refs[e];
        }
    return s;
}

bool report(bool same, const char* what, const State& s, const char* how)
{
    if (!same)
        std::printf("FAILED %s (%s): batch %u, pages %u of %u, max_pages %u\n", what, how, s.batch, s.pages, s.page, s.max_pages);
    return same;
}

U32s starts_for(uint32_t batch, uint32_t most, uint32_t behind, uint32_t& rows)
{
    U32s st(batch + 1, 0);
    for (uint32_t b = 0; b < batch; ++b)
        st[b + 1] = st[b] + upto(most);
    rows = st[batch] + behind;
    return st;
}

// A pool's row words: dim 64 is 32 words.
bool reserve(const State& s, uint32_t most, bool in_place, bool bad, uint32_t layers)
{
    const uint32_t kv = 2, dim = 64, row = dim / 2;
    uint32_t rows = s.batch;
    U32s st = starts_for(s.batch, most, 3, rows);
    State x = s;
    if (bad) {
        for (auto& y : st)
            y = upto(3) ? y : rng();
        for (auto& y : x.table)
            y = upto(9) ? y : rng();
        for (auto& y : x.refs)
            y = upto(9) ? y : upto(5);
        for (auto& y : x.ctx)
            y = upto(9) ? y : rng();
    }
    const mako_pages_args a{s.batch, rows, rows, s.pages, s.page, s.max_pages, kv, dim, layers};
    const size_t pool = (size_t)std::max(1u, layers) * s.pages * kv * s.page * row;
    Guarded k(numbers(pool, 1)), v(numbers(pool, 2)), table(x.table), refs(x.refs), ctx(x.ctx), sts(st);
    Guarded table_out(U32s(x.table.size(), 5u)), refs_out(U32s(x.refs.size(), 5u)), ctx_out(U32s(s.batch, 5u));
    Guarded ws(U32s((mako_pages_reserve_workspace(&a) + 3) / 4, 9u));
    Guarded &to = in_place ? table : table_out, &ro = in_place ? refs : refs_out, &co = in_place ? ctx : ctx_out;
    const bool data = layers != 0;
    const int rc = mako_pages_reserve(&a, table.data(), refs.data(), sts.data(), ctx.data(), to.data(), ro.data(), co.data(),
                                      data ? k.data() : nullptr, data ? v.data() : nullptr, ws.data(),
                                      mako_pages_reserve_workspace(&a), nullptr);
    bool same = rc == MAKO_OK && k.whole() && v.whole() && table.whole() && refs.whole() && ctx.whole() && ws.whole() &&
                table_out.whole() && refs_out.whole() && ctx_out.whole();
    if (bad)
        return report(same, "reserve, bad input", s, in_place ? "in place" : "out of place");
    U32s want_k = numbers(pool, 1), want_v = numbers(pool, 2), want_c(s.batch);
    U32s free;
    for (uint32_t p = s.pages; p-- > 0;)
        if (!x.refs[p])
            free.push_back(p);
    // who appends to which partly filled page: the last one keeps it where it has no other holder
    std::vector<std::vector<uint32_t>> appends(s.pages);
    for (uint32_t b = 0; b < s.batch; ++b)
        if (st[b + 1] > st[b] && x.ctx[b] % s.page && x.ctx[b] < s.max_pages * s.page)
            appends[x.table[b * s.max_pages + x.ctx[b] / s.page]].push_back(b);
    const U32s held = x.refs;
    for (uint32_t b = 0; b < s.batch; ++b) {
        uint32_t at = x.ctx[b];
        const uint32_t end = std::min(at + st[b + 1] - st[b], s.max_pages * s.page);
        while (at < end) {
            uint32_t& e = x.table[b * s.max_pages + at / s.page];
            const uint32_t part = at % s.page;
            const bool shared = e < s.pages && part && (held[e] > appends[e].size() || appends[e].back() != b);
            if (e >= s.pages || shared) {
                if (free.empty())
                    break;
                const uint32_t to_page = free.back();
                free.pop_back();
                x.refs[to_page] = 1;
                if (shared) {
                    --x.refs[e];
                    for (uint32_t l = 0; l < layers; ++l)
                        for (uint32_t h = 0; h < kv; ++h)
                            for (uint32_t i = 0; i < part * row; ++i) {
                                const size_t src = (((size_t)l * s.pages + e) * kv + h) * s.page * row + i;
                                const size_t dst = (((size_t)l * s.pages + to_page) * kv + h) * s.page * row + i;
                                want_k[dst] = want_k[src];
                                want_v[dst] = want_v[src];
                            }
                }
                e = to_page;
            }
            at = std::min(end, (at / s.page + 1) * s.page);
        }
        want_c[b] = at;
    }
    same = same && to.value() == x.table && ro.value() == x.refs && co.value() == want_c &&
           (!data || (k.value() == want_k && v.value() == want_v));
    if (!in_place)
        same = same && table.value() == s.table && refs.value() == s.refs && ctx.value() == s.ctx;
    return report(same, "reserve", s, in_place ? "in place" : "out of place");
}

bool fork(const State& s, bool in_place, bool refs_in_place, bool bad, int form)
{
    const mako_pages_args a{s.batch, 0, 0, s.pages, s.page, s.max_pages, 0, 0, 0};
    U32s parent(s.batch), keep(s.batch);
    for (uint32_t i = 0; i < s.batch; ++i) {
        parent[i] = upto(4) == 0 ? s.batch + upto(3) : upto(2) ? i : upto(s.batch - 1);
        keep[i] = upto(1) ? kNone : upto(300);
    }
    State x = s;
    if (bad) {
        for (auto& y : x.table)
            y = upto(9) ? y : rng();
        for (auto& y : x.ctx)
            y = upto(9) ? y : rng();
        for (auto& y : parent)
            y = upto(9) ? y : rng();
    }
    Guarded table(x.table), refs(x.refs), ctx(x.ctx), par(parent), kp(keep);
    Guarded table_out(U32s(x.table.size(), 5u)), refs_out(U32s(x.refs.size(), 5u)), ctx_out(U32s(s.batch, 5u));
    Guarded ws(U32s((mako_pages_fork_workspace(&a) + 3) / 4, 9u));
    Guarded &to = in_place ? table : table_out, &ro = refs_in_place ? refs : refs_out, &co = in_place ? ctx : ctx_out;
    const int rc = mako_pages_fork(&a, form & 1 ? nullptr : par.data(), form & 2 ? nullptr : kp.data(), table.data(),
                                   refs.data(), ctx.data(), to.data(), ro.data(), co.data(), in_place ? ws.data() : nullptr,
                                   in_place ? mako_pages_fork_workspace(&a) : 0, nullptr);
    bool same = rc == MAKO_OK && table.whole() && refs.whole() && ctx.whole() && ws.whole() && table_out.whole() &&
                refs_out.whole() && ctx_out.whole();
    if (!bad) {
        U32s want(x.table.size(), kNone), want_c(s.batch);
        for (uint32_t i = 0; i < s.batch; ++i) {
            const uint32_t p = form & 1 ? i : parent[i];
            const uint32_t c = p < s.batch ? std::min(form & 2 ? kNone : keep[i], s.ctx[p]) : 0;
            want_c[i] = c;
            for (uint32_t j = 0; j < (c + s.page - 1) / s.page; ++j)
                ++x.refs[want[i * s.max_pages + j] = s.table[p * s.max_pages + j]];
        }
        for (uint32_t e : s.table)
            if (e < s.pages)
                --x.refs[e];
        same = same && to.value() == want && ro.value() == x.refs && co.value() == want_c;
    }
    return report(same, bad ? "fork, bad input" : "fork", s, in_place ? "in place" : "out of place");
}

bool compact(const State& s, bool in_place, bool bad, uint32_t layers, bool map)
{
    const uint32_t kv = 2, dim = 64, row = dim / 2;
    const mako_pages_args a{s.batch, 0, 0, s.pages, s.page, s.max_pages, kv, dim, layers};
    State x = s;
    if (bad) {
        for (auto& y : x.table)
            y = upto(9) ? y : rng();
        for (auto& y : x.refs)
            y = upto(9) ? y : upto(5);
    }
    const size_t per = (size_t)kv * s.page * row, pool = (size_t)std::max(1u, layers) * s.pages * per;
    Guarded k(numbers(pool, 1)), v(numbers(pool, 2)), table(x.table), refs(x.refs), used(U32s(1, 5u)), names(U32s(s.pages, 5u));
    Guarded table_out(U32s(x.table.size(), 5u)), refs_out(U32s(x.refs.size(), 5u));
    Guarded ws(U32s((mako_pages_compact_workspace(&a) + 3) / 4, 9u));
    Guarded &to = in_place ? table : table_out, &ro = in_place ? refs : refs_out;
    const int rc = mako_pages_compact(&a, table.data(), refs.data(), to.data(), ro.data(), used.data(),
                                      map ? names.data() : nullptr, layers ? k.data() : nullptr, layers ? v.data() : nullptr,
                                      ws.data(), mako_pages_compact_workspace(&a), nullptr);
    bool same = rc == MAKO_OK && k.whole() && v.whole() && table.whole() && refs.whole() && ws.whole() && used.whole() &&
                table_out.whole() && refs_out.whole() && names.whole();
    U32s want_k = numbers(pool, 1), want_v = numbers(pool, 2), want_names(s.pages, kNone), want_refs = x.refs;
    uint32_t n = 0, hole = 0;
    for (uint32_t r : x.refs)
        n += r > 0;
    for (uint32_t p = 0; p < s.pages; ++p) {
        if (!x.refs[p])
            continue;
        want_names[p] = p;
        if (p < n)
            continue;
        while (want_refs[hole])
            ++hole;
        want_names[p] = hole;
        want_refs[hole] = x.refs[p];
        want_refs[p] = 0;
        for (uint32_t l = 0; l < layers; ++l)
            for (size_t i = 0; i < per; ++i) {
                want_k[(l * s.pages + hole) * per + i] = want_k[(l * s.pages + p) * per + i];
                want_v[(l * s.pages + hole) * per + i] = want_v[(l * s.pages + p) * per + i];
            }
    }
    for (auto& e : x.table)
        e = e < s.pages ? want_names[e] : kNone;
    same = same && to.value() == x.table && ro.value() == want_refs && used.value()[0] == n &&
           (!layers || (k.value() == want_k && v.value() == want_v)) && (!map || names.value() == want_names);
    return report(same, bad ? "compact, bad input" : "compact", s, in_place ? "in place" : "out of place");
}

bool write(const State& s, uint32_t most, bool bad, int form, uint32_t kv, uint32_t dim)
{
    const uint32_t row = dim / 2;
    uint32_t rows = s.batch;
    U32s st = starts_for(s.batch, most, 3, rows);
    if (form & 1)
        rows = s.batch + 2;
    State x = s;
    U32s end(s.batch);
    for (auto& y : end)
        y = upto(400);
    if (bad) {
        for (auto& y : st)
            y = upto(3) ? y : rng();
        for (auto& y : x.table)
            y = upto(9) ? y : rng();
        for (auto& y : x.ctx)
            y = upto(9) ? y : rng();
    }
    const mako_pages_args a{s.batch, rows, rows + 1, s.pages, s.page, s.max_pages, kv, dim, 1};
    const size_t pool = (size_t)s.pages * kv * s.page * row;
    Guarded k(numbers(pool, 1)), v(numbers(pool, 2)), kd(numbers((size_t)kv * (rows + 1) * row, 3)),
        vd(numbers((size_t)kv * (rows + 1) * row, 4)), table(x.table), ctx(x.ctx), sts(st), ends(end);
    const int rc = mako_pages_write(&a, kd.data(), vd.data(), table.data(), form & 1 ? nullptr : sts.data(), ctx.data(),
                                    form & 2 ? ends.data() : nullptr, k.data(), v.data(), nullptr);
    bool same = rc == MAKO_OK && k.whole() && v.whole();
    if (!bad) {
        U32s want_k = numbers(pool, 1), want_v = numbers(pool, 2), of_k = kd.value(), of_v = vd.value();
        for (uint32_t b = 0; b < s.batch; ++b) {
            const uint32_t s0 = form & 1 ? b : st[b], n = form & 1 ? 1 : st[b + 1] - st[b];
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t at = s.ctx[b] + i;
                if (at / s.page >= s.max_pages || (form & 2 && at >= end[b]))
                    continue;
                const uint32_t e = s.table[b * s.max_pages + at / s.page];
                if (e >= s.pages)
                    continue;
                for (uint32_t h = 0; h < kv; ++h)
                    for (uint32_t d = 0; d < row; ++d) {
                        const size_t to = (((size_t)e * kv + h) * s.page + at % s.page) * row + d;
                        const size_t of = ((size_t)h * (rows + 1) + s0 + i) * row + d;
                        want_k[to] = of_k[of];
                        want_v[to] = of_v[of];
                    }
            }
        }
        same = same && k.value() == want_k && v.value() == want_v;
    }
    return report(same, bad ? "write, bad input" : "write", s, "");
}

}  // namespace

int main()
{
    bool good = true;
    for (int round = 0; round < 6; ++round) {
        const uint32_t batch = round == 0 ? 1 : round == 1 ? 130 : round == 5 ? 1500 : 1 + upto(70);
        const uint32_t page = 64u << upto(1), beams = 1 + upto(3), most = round % 3 == 0 ? 1 : round % 3 == 1 ? 150 : 900;
        const uint32_t high = round == 5 ? 100 : 500, max_pages = high / page + 1 + upto(20);
        // spare pages: none, some, enough, and a pool that the look for free pages takes several rounds over
        const uint32_t spare = round % 4 == 0 ? upto(3) : round % 4 == 1 ? batch * 3 : round % 4 == 2 ? batch * 40 : 9000;
        const State s = state(batch, page, max_pages, spare, high, beams);
        const uint32_t layers = s.pages * page > 60000 ? 0 : 1 + upto(1);
        for (int bad = 0; bad < 2; ++bad)
            for (int in_place = 0; in_place < 2; ++in_place) {
                good &= reserve(s, most, in_place, bad, layers);
                good &= fork(s, in_place, upto(1), bad, (int)upto(3));
                good &= compact(s, in_place, bad, layers, upto(1));
            }
        if (s.pages * page <= 60000)
            for (int form = 0; form < 4; ++form)
                good &= write(s, most, false, form, 1 + upto(4), form == 1 ? 256 : 64) && write(s, most, true, form, 2, 64);
    }
    std::puts(good ? "all passed" : "FAILED");
    return good ? 0 : 1;
}
