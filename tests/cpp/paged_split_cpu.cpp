// The split of csrc/paged_split.hpp on the CPU (cpu_hip/hip/hip_runtime.h): over batches of all kinds, the ranges' pieces are
// each item's tiles once and in order, no piece starts behind the keys of a row, a range has at most one piece of each kind,
// and the range that ends an item names the one that starts it, between which its other pieces lie.
//   paged_split_cpu
#include <hip/hip_runtime.h>

#include "../../mako-common_amd/csrc/paged_split.hpp"

#include <cstdio>
#include <map>
#include <random>
#include <tuple>

namespace mako {
int fail(int code, const char*, ...) { return code; }
}  // namespace mako

namespace {

std::mt19937 rng(3);
uint32_t upto(uint32_t n) { return rng() % (n + 1); }

struct Got {
    uint32_t range;
    mako::PagedPiece x;
};
std::vector<Got> got;

void record(const mako::PagedSplit& p)
{
    const uint32_t range = blockIdx.x;
    const bool items = p.how == mako::kItems;
    mako::walk_range(p, items ? range % p.batch : range, items ? range / p.batch : 0, threadIdx.x, [&](const mako::PagedPiece& x) {
        if (threadIdx.x == 0)
            got.push_back({range, x});
    });
}

#define CHECK(...)                                                                                            \
    do {                                                                                                     \
        if (!(__VA_ARGS__)) {                                                                                       \
            std::printf("FAILED %s: batch %u kv %u rshift %u ranges %u how %u max_ctx %u\n", #__VA_ARGS__, p.batch, p.kv_heads, \
                        p.rshift, p.n_ranges, p.how, p.max_ctx);                                           \
            return false;                                                                                    \
        }                                                                                                    \
    } while (0)

bool run(mako::PagedSplit p, bool good)
{
    got.clear();
    cpu_hip::launch(dim3(p.how == mako::kItems ? p.batch * p.kv_heads : p.n_ranges), dim3(64), [&] { record(p); });
    std::map<std::tuple<uint32_t, uint32_t, uint32_t>, uint32_t> next;  // the tile that an item's next piece starts with
    std::map<std::tuple<uint32_t, uint32_t, uint32_t>, std::vector<Got>> parts;
    std::map<std::pair<uint32_t, uint32_t>, int> slots;
    const uint32_t R = 1u << p.rshift;
    double most = 0, all = 0;
    std::map<uint32_t, double> cost;
    for (const Got& g : got) {
        const auto& x = g.x;
        CHECK(x.b < p.batch && x.kvh < p.kv_heads && x.rows >= 1 && x.rows <= R && x.row0 + x.rows <= p.rows);
        CHECK(x.ta < x.tb && x.keys <= p.max_ctx && x.seen <= p.max_ctx && 64 * (x.tb - 1) < x.keys);
        CHECK(64 * x.ta < std::min(x.p0 + 1, x.seen));  // the first row sees a key of the piece's first tile
        CHECK(p.how == mako::kRanges || !x.part);
        const double few = x.rows <= p.few && x.seen - x.p0 <= p.few ? mako::kTileFew : mako::kTile;
        cost[g.range] += (x.tb - x.ta) * few + mako::kLead;
        all += (x.tb - x.ta) * few + mako::kLead;
        if (x.part)
            CHECK(slots[{g.range, x.kind}]++ == 0);
        if (!good)
            continue;
        const auto item = std::make_tuple(x.b, x.kvh, x.row0);
        CHECK(next[item] == x.ta);
        next[item] = x.tb;
        const uint32_t nt = (x.keys + 63) / 64;
        CHECK(x.part == (x.ta != 0 || x.tb != nt));
        if (x.part)
            parts[item].push_back(g);
        CHECK((x.first != mako::kNoPage) == (x.part && x.tb == nt));
        if (x.first != mako::kNoPage)  // what the merge joins: kind 1 of the first range, kind 0 of the others up to this
            for (const Got& y : parts[item])
                CHECK(y.range >= x.first && y.x.kind == (y.range == x.first ? 1u : 0u));
    }
    if (!good)
        return true;
    size_t items = 0;
    for (uint32_t b = 0; b < p.batch; ++b) {
        const auto s = mako::seq_of(p, b);
        for (uint32_t i = 0; i < s.n; i += R)
            for (uint32_t h = 0; h < p.kv_heads; ++h, ++items) {
                const uint32_t keys = std::min(s.c + std::min(s.n, i + R), s.keys);
                CHECK(next[std::make_tuple(b, h, s.s0 + i)] == (keys + 63) / 64);
            }
    }
    CHECK(items == next.size());
    for (const auto& c : cost)
        most = std::max(most, c.second);
    // no range has more than its share and a little
    CHECK(p.how != mako::kRanges || most <= all / p.n_ranges + mako::kTile * (3 * R / 64 + 8) + mako::kLead * (items / p.n_ranges + 3));
    return true;
}

}  // namespace

int main()
{
    bool good = true;
    for (int round = 0; round < 120; ++round) {
        const uint32_t batch = round < 4 ? 1 : round % 9 == 0 ? 60 + upto(80) : 1 + upto(12);
        const uint32_t most = round % 3 == 0 ? 1 : round % 3 == 1 ? 40 : 900, high = round % 5 == 0 ? 20 : round % 5 == 1 ? 300 : 9000;
        std::vector<uint32_t> starts(batch + 1, 0), ctx(batch);
        uint32_t top = 1;
        for (uint32_t b = 0; b < batch; ++b) {
            starts[b + 1] = starts[b] + (most == 1 ? 1 : upto(most));
            ctx[b] = upto(high);
            top = std::max(top, ctx[b] + starts[b + 1] - starts[b]);
        }
        mako::PagedSplit p{most == 1 ? nullptr : starts.data(), ctx.data(), batch, starts[batch] + upto(3), 1 + upto(8), most,
                           top + upto(1) * upto(500), 5 + upto(3), round % 2 ? 256 : 1 + upto(100), mako::kRanges, 0};
        if (upto(4) == 0)
            p.how = most <= 1u << p.rshift ? mako::kItems : mako::kWhole;
        p.few = upto(2) ? 1u << p.rshift >> 1 : 0;
        if (p.starts == nullptr)
            p.rows = batch;
        good &= run(p, true);
        if (round % 4 == 0) {  // bounds that cut, starts and contexts that are not what they should be
            p.max_ctx = 1 + upto(top);
            p.max_new = 1 + upto(most);
            good &= run(p, true);
            for (auto& x : starts)
                x = upto(2) ? x : rng();
            for (auto& x : ctx)
                x = upto(2) ? x : rng();
            good &= run(p, false);
        }
    }
    std::puts(good ? "all passed" : "FAILED");
    return good ? 0 : 1;
}
