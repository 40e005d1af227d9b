// The split of attention over a cache in pages: which tiles of which items a workgroup takes. Lengths are known on the device
// only, so every workgroup works it out.
//
// An item is a block of R = 1 << rshift rows of a sequence and a kv head; its tiles are the 64 keys each up to its last row's.
// Its cost is kTile units a tile (kTileFew in a sequence of at most `few` rows) and kLead (kLeadFew) for what it costs beside
// them. The items of all (kv head, sequence) segments lie end to end, a kv head's sequences together, and are cut into
// equal ranges, one a workgroup: ranges side by side on an XCD share keys, and every XCD has its part of each sequence. (With
// a sequence's kv heads together a batch's single tokens met on one XCD, whose reads then bound the call: a mixed batch took
// 225 us, 208 so.) Within a segment the row blocks go heavy and light in turn (the last, the first, the last but one, the
// second, ...), so two neighbours cost the same everywhere, and the ranges of a whole prompt fall on items' ends.
// A cut inside an item leaves kLeast tiles on either side, and no row without keys in a piece's first tile, which the
// attention's streams rely on; with kWhole, items are not cut: the range of an item's middle has it.
#pragma once

#include "pages_common.hpp"
#include "split_ranges.hpp"

namespace mako {

// The streams' tiles and pieces side by side in a mixed batch, in units of 0.14 us: 64 rows a wave 1.7 us a tile and 8 a piece,
// 32 rows 1.1 and 5 (a tile of these alone on a full chip: 1.6 and 0.9). With a tile of 32 rows at half of one of 64 the
// workgroups that met single tokens ended at 220 us, the others at 175.
constexpr uint32_t kTile = 12, kTileFew = 8, kLead = 60, kLeadFew = 36;
constexpr uint32_t kLeast = 3;  // tiles of a piece

// How a call is split: by equal ranges; by equal ranges that whole items fall to; or, where no sequence has more rows than an
// item, by sequence and kv head.
enum : uint32_t { kRanges, kWhole, kItems };

struct PagedSplit {
    const uint32_t *starts, *ctx;
    uint32_t batch, rows, kv_heads, max_new, max_ctx, rshift, n_ranges, how, few;
};

// A piece of an item: tiles [ta, tb) of sequence b for its rows row0 .. of o, the first at position p0.
struct PagedPiece {
    uint32_t b, kvh, row0, rows, p0;
    uint32_t keys, seen;  // of the item's last row; of the sequence's
    uint32_t ta, tb;
    uint32_t part, kind;  // part: not the whole item; kind: 1 if the item starts in this range
    uint32_t first;       // where it is an item's last piece of several: the range that the item starts in (else kNoPage)
};

// A sequence's new rows n, from row s0, behind c cache rows, keys with them, in nqb blocks. Block qb's item is lead + (qb + 1)
// step units.
struct PagedSeq {
    uint32_t c, n, s0, keys, nqb, lead, step, few;
};
__device__ __forceinline__ PagedSeq seq_of(const PagedSplit& p, uint32_t b)
{
    const NewRows nr = new_rows(p.starts, p.rows, b);
    PagedSeq s;
    s.n = min(nr.n, p.max_new);
    s.s0 = nr.s0;
    s.c = min(p.ctx[b], p.max_ctx);
    s.keys = s.c + min(s.n, p.max_ctx - s.c);
    s.nqb = (s.n + (1u << p.rshift) - 1) >> p.rshift;
    s.few = s.n <= p.few ? 1 : 0;
    const uint32_t tiles = (s.c + 63) / 64;
    s.lead = s.few ? kLeadFew + tiles * kTileFew : kLead + tiles * kTile;
    s.step = ((1u << p.rshift) * (s.few ? kTileFew : kTile)) / 64;
    return s;
}
// Sequence b, from the lane that holds it (lane b % 64).
__device__ __forceinline__ PagedSeq of_lane(const PagedSeq& s, uint32_t b)
{
    const uint32_t l = b % 64;
    const auto at = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane(x, l); };
    return {at(s.c), at(s.n), at(s.s0), at(s.keys), at(s.nqb), at(s.lead), at(s.step), at(s.few)};
}
__device__ __forceinline__ uint32_t item_units(const PagedSeq& s, uint32_t qb) { return s.lead + (qb + 1) * s.step; }
__device__ __forceinline__ uint32_t segment_units(const PagedSeq& s)
{
    return s.nqb * s.lead + s.nqb * (s.nqb + 1) / 2 * s.step;
}

// The tile that unit u of an item of nt tiles falls to (those from tmax on stay together).
__device__ __forceinline__ uint32_t cut_of(const PagedSplit& p, uint32_t u, uint32_t few, uint32_t nt, uint32_t tmax)
{
    const uint32_t t = few ? (max(u, kLeadFew) - kLeadFew) / kTileFew : (max(u, kLead) - kLead) / kTile;
    if (p.how == kWhole)
        return 2 * t < nt ? 0u : nt;
    return t < kLeast ? 0u : t + kLeast > nt ? nt : min(t, tmax);
}

// Calls piece(PagedPiece) for the pieces of a range, in order (kItems: for the item of sequence `range` and kv head kvh); all
// lanes of a wave do so together.
template <class F>
__device__ __forceinline__ void walk_range(const PagedSplit& p, uint32_t range, uint32_t kvh, uint32_t lane, F piece)
{
    uint32_t b = range, u0 = 0, item = 0, start = 0, left = 1;
    Ranges rg{};
    PagedSeq mine{}, s{};
    // The units of all segments; a lane holds a sequence, so up to 64 are looked up once.
    uint32_t units = 0, inc = 0;
    const auto look_up = [&](uint32_t i0) __attribute__((always_inline)) {
        mine = seq_of(p, min(i0 + lane, p.batch - 1));
        units = i0 + lane < p.batch ? segment_units(mine) : 0u;
        inc = scan_lanes(units);
    };
    if (p.how == kItems) {
        s = of_lane(seq_of(p, b), 0);
        if (s.n == 0)
            return;
    } else {
        uint32_t total = 0;
        for (uint32_t i0 = 0; i0 < p.batch; i0 += 64) {
            look_up(i0);
            total += (uint32_t)__builtin_amdgcn_readlane(inc, 63);
        }
        const uint32_t n = min(p.n_ranges, total * p.kv_heads);
        if (range >= n)
            return;
        rg = Ranges(total * p.kv_heads, n);
        const uint32_t x0 = rg.start(range);
        left = rg.start(range + 1) - x0;
        // Of kv head kvh, the sequence b whose segment holds x0, u0 units into it.
        kvh = x0 / total, u0 = x0 % total, b = 0;
        for (uint32_t i0 = 0; i0 < p.batch; i0 += 64) {
            if (p.batch > 64)
                look_up(i0);
            if (const uint64_t hit = __ballot(u0 < inc)) {
                const uint32_t l = (uint32_t)__builtin_ctzll(hit);
                b = i0 + l;
                u0 -= (uint32_t)__builtin_amdgcn_readlane(inc - units, l);
                break;
            }
            u0 -= (uint32_t)__builtin_amdgcn_readlane(inc, 63);
        }
        s = of_lane(mine, b);
        // item 2 i is block nqb - 1 - i, item 2 i + 1 block i: a pair's units do not depend on i
        const uint32_t pair = 2 * s.lead + (s.nqb + 1) * s.step, i = u0 / pair;
        u0 -= i * pair;
        item = 2 * i;
        const uint32_t heavy = item_units(s, s.nqb - 1 - i);
        if (u0 >= heavy) {
            u0 -= heavy;
            ++item;
        }
        start = x0 - u0;  // the item's first unit
    }
    for (;;) {
        const uint32_t qb = item & 1 ? item / 2 : s.nqb - 1 - item / 2, i0 = qb << p.rshift;
        const uint32_t cost = p.how == kItems ? 1 : item_units(s, qb), u1 = min(cost, u0 + left);
        PagedPiece x;
        x.b = b, x.kvh = kvh, x.row0 = s.s0 + i0, x.rows = min(1u << p.rshift, s.n - i0), x.p0 = s.c + i0;
        x.seen = s.keys, x.keys = min(x.p0 + x.rows, s.keys);
        const uint32_t nt = (x.keys + 63) / 64, tmax = (min(x.p0 + 1, s.keys) - 1) / 64;
        x.ta = u0 == 0 ? 0 : cut_of(p, u0, s.few, nt, tmax);
        x.tb = u1 == cost ? nt : cut_of(p, u1, s.few, nt, tmax);
        if (x.ta < x.tb) {
            x.part = x.ta != 0 || x.tb != nt;
            x.kind = u0 == 0 ? 1 : 0;
            x.first = kNoPage;
            if (x.part && x.tb == nt) {
                uint32_t lo = 0, hi = range;  // the last range that starts at or before the item
                while (lo < hi) {
                    const uint32_t mid = (lo + hi + 1) / 2;
                    if (rg.start(mid) <= start)
                        lo = mid;
                    else
                        hi = mid - 1;
                }
                x.first = lo;
            }
            piece(x);
        }
        left -= u1 - u0;
        if (left == 0)
            return;
        start += cost;
        u0 = 0;
        if (++item == s.nqb) {
            item = 0;
            do {
                if (++b == p.batch) {
                    b = 0;
                    if (++kvh == p.kv_heads)
                        return;  // (not where the lengths are as they were when the units were summed)
                }
                if (b % 64 == 0 && p.batch > 64)
                    look_up(b);
                s = of_lane(mine, b);
            } while (s.nqb == 0);
        }
    }
}

}  // namespace mako
