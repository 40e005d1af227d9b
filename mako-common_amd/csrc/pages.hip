// The calls that keep a cache's pages: the write of a step's rows, the reservation of pages for them, the fork of sequences
// and the compaction of the pool. All counts are on the device; what a launch is sized by are the arguments' bounds.
//
// Figures: us of kernel on one MI355X. What bounds the small calls is their chain of dependent loads and the launch; a pass of
// the smallest kernel takes 5.7 to 6.4 us with its host call (2.2 in a graph).
//
// * pages_write: a wave a new row. Its sequence is found by counting the starts up to it (64 at a time, a ballot), its page
//   by one load of the table; the row's 16-byte chunks of all kv heads, k and v, are loaded before either has come. 64 single
//   rows of 8 heads of 128 2.9-3.3 us; a long prompt's (12.6 MB read, and written) 7.0-7.5.
// * reserve_plan, one workgroup: the entries that need a page are counted a sequence (a thread each, a wave where a sequence
//   brings many), summed over the sequences, and the free pages looked for from the lowest number on until there are enough,
//   so the look ends early in a pool that is kept compact. Sequences that append to one shared page meet in a hash table in
//   LDS, by counts and maxima, which the order of the threads does not change. copy_pages then copies the shared pages' rows.
//   64 sequences' step 4.8-5.1 us; 64 beams of 16 prompts 5.9-6.1, and 3.7-4.6 for the copies. Where the pages run out, the
//   sequences that did not get the copy of a shared page are looked at once more: nobody writes where one of them has rows.
// * fork_rows: a workgroup a new sequence; the holders' counts change by integer atomics, only where old and new entry differ.
//   1024 sequences of up to 128 pages 3.1-3.6 us after the copies' 2.2-2.5; fork_small 4.0-4.2 for 64 beams.
// * compact_plan, one workgroup: used pages counted, then holes and sources ranked by one pass of sums over the threads; a
//   source meets its hole by rank, as the holes all lie before it. compact_move copies the pages and renumbers the tables:
//   4096 pages of two layers 7.8-8.2 us, then 202-209 (1.07 GB at 5.1 TB/s, a large copy's rate); 512 pages 5.4-5.7 and 9-11.
#include <algorithm>

#include "pages_common.hpp"
#include "split_ranges.hpp"

namespace mako {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kPlan = 1024;           // threads of the planning workgroups
constexpr uint32_t kMaxSeqs = 4096;   // sequences that reserve_plan takes
constexpr uint32_t kSlots = 2 * kMaxSeqs;
constexpr uint32_t kListHere = 2048;  // free pages that reserve_plan lists in LDS
constexpr uint32_t kLook = 8;         // refs a thread looks at a round
constexpr uint64_t kForkSmall = 4096; // table entries that one workgroup forks alone (64 x 32: 6.4 us a pass, by rows 9.0)
constexpr uint32_t kFew = 2;          // entries of a sequence that one thread goes through alone

// ---- write ---------------------------------------------------------------------------------------------------------

struct WriteParams {
    const u32x4 *kd, *vd;
    const uint32_t *table, *starts, *ctx, *end;
    u32x4 *k, *v;
    uint32_t batch, rows, d_pad, pages, shift, max_pages, kv_heads, cpr;  // cpr: 16-byte chunks of a row of a kv head
};

__global__ __launch_bounds__(256) void pages_write(const WriteParams p)
{
    const uint32_t lane = threadIdx.x & 63u, r = blockIdx.x * 4 + uniform(threadIdx.x >> 6);
    if (r >= p.rows)
        return;
    const uint32_t total = p.kv_heads * p.cpr;
    constexpr int U = 2;
    u32x4 a[U], b[U];
    const auto load = [&](uint32_t x0) __attribute__((always_inline)) {
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t x = x0 + 64 * u + lane;
            if (x < total) {
                const size_t at = ((size_t)(x / p.cpr) * p.d_pad + r) * p.cpr + x % p.cpr;
                a[u] = p.kd[at];
                b[u] = p.vd[at];
            }
        }
    };
    load(0);
    uint32_t seq = r;
    if (p.starts) {
        seq = 0;  // of the starts behind the first, those up to r
        for (uint32_t i = 0; i < p.batch; i += 64)
            seq += __popcll(__ballot(i + lane < p.batch && p.starts[i + lane + 1] <= r));
    }
    if (seq >= p.batch)
        return;
    const NewRows nr = new_rows(p.starts, p.rows, seq);
    if (r < nr.s0 || r - nr.s0 >= nr.n)
        return;
    const uint64_t at = (uint64_t)p.ctx[seq] + (r - nr.s0);
    if (at >> p.shift >= p.max_pages || (p.end && at >= p.end[seq]))
        return;
    const uint32_t page = p.table[(size_t)seq * p.max_pages + (uint32_t)(at >> p.shift)];
    if (page >= p.pages)
        return;
    const size_t base = ((size_t)page * p.kv_heads << p.shift) + ((uint32_t)at & ((1u << p.shift) - 1));
    for (uint32_t x0 = 0;;) {
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t x = x0 + 64 * u + lane;
            if (x < total) {
                const size_t to = (base + ((size_t)(x / p.cpr) << p.shift)) * p.cpr + x % p.cpr;
                p.k[to] = a[u];
                p.v[to] = b[u];
            }
        }
        x0 += 64 * U;
        if (x0 >= total)
            return;
        load(x0);
    }
}

// ---- shared pieces -------------------------------------------------------------------------------------------------

// The sum of x over the workgroup's threads before this one; total: over all. s: a word a wave. (Ends with every thread
// having read s only after a barrier of the caller's or of the next call.)
__device__ __forceinline__ uint32_t scan_threads(uint32_t x, uint32_t* s, uint32_t& total)
{
    const uint32_t inc = scan_lanes(x), lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 63)
        s[w] = inc;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    #pragma unroll
    for (uint32_t i = 0; i < kPlan / 64; ++i) {
        const uint32_t y = s[i];
        before += i < w ? y : 0u;
        total += y;
    }
    return before + inc - x;
}

// kLook refs from page p on, pages past the last counted as used.
__device__ __forceinline__ void load_refs(const uint32_t* refs, uint32_t p, uint32_t pages, uint32_t (&x)[kLook])
{
    if (p + kLook <= pages) {
        #pragma unroll
        for (uint32_t i = 0; i < kLook; i += 4) {
            const u32x4_any y = *reinterpret_cast<const u32x4_any*>(refs + p + i);
            x[i] = y[0], x[i + 1] = y[1], x[i + 2] = y[2], x[i + 3] = y[3];
        }
    } else {
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i)
            x[i] = p + i < pages ? refs[p + i] : 1u;
    }
}

// Arrays that a call copies before it changes the copies: by the planning workgroup itself where they are short
// (kCopyInPlan words; with a launch 64 sequences' reservation among 4096 pages takes 2.3 us more), else by copy_words.
struct CopyWords {
    const uint32_t* from[3];
    uint32_t* to[3];
    uint64_t n[3];
    uint32_t groups;
};
constexpr uint64_t kCopyInPlan = 16384;
__device__ __forceinline__ void copy_share(const CopyWords& p, uint64_t thread, uint64_t all)
{
    #pragma unroll
    for (int a = 0; a < 3; ++a)
        #pragma unroll 4
        for (uint64_t i = thread; i < p.n[a]; i += all)
            p.to[a][i] = p.from[a][i];
}
__global__ __launch_bounds__(256) void copy_words(const CopyWords p)
{
    copy_share(p, (uint64_t)blockIdx.x * 256 + threadIdx.x, (uint64_t)p.groups * 256);
}

// Rows [0, rows) of page src over page dst, in every layer and kv head.
struct Move {
    uint32_t src, dst, rows, pad;
};
struct MoveParams {
    const Move* moves;
    const uint32_t* count;
    u32x4 *k, *v;
    uint32_t layers, kv_heads, pages, shift, cpr, groups;
};
__device__ __forceinline__ void move_rows(const MoveParams& p, uint64_t item)
{
    const uint32_t h = (uint32_t)(item % p.kv_heads);
    const uint64_t rest = item / p.kv_heads;
    const Move m = p.moves[rest / p.layers];
    const uint64_t layer = rest % p.layers;
    const uint32_t n = m.rows * p.cpr;
    const size_t src = (((layer * p.pages + m.src) * p.kv_heads + h) << p.shift) * p.cpr;
    const size_t dst = (((layer * p.pages + m.dst) * p.kv_heads + h) << p.shift) * p.cpr;
    constexpr int U = 8;
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 256 * U) {
        u32x4 a[U], b[U];
        #pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < n) {
                a[u] = p.k[src + i0 + 256 * u];
                b[u] = p.v[src + i0 + 256 * u];
            }
        #pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < n) {  // (streaming stores: 4096 pages 212 us a pass, plain ones 217)
                __builtin_nontemporal_store(a[u], p.k + dst + i0 + 256 * u);
                __builtin_nontemporal_store(b[u], p.v + dst + i0 + 256 * u);
            }
    }
}
__global__ __launch_bounds__(256) void copy_pages(const MoveParams p)
{
    const uint64_t items = (uint64_t)p.count[0] * p.layers * p.kv_heads;
    for (uint64_t i = blockIdx.x; i < items; i += p.groups)
        move_rows(p, i);
}

// ---- reserve -------------------------------------------------------------------------------------------------------

struct ReserveParams {
    const uint32_t *table, *refs, *starts, *ctx;
    uint32_t *table_out, *refs_out, *ctx_out;
    uint32_t* count;  // moves
    Move* moves;      // [batch]
    uint32_t* list;   // free pages, in order
    uint32_t batch, rows, pages, shift, max_pages, list_max;
    CopyWords copy;   // (done before any entry is given)
};

__global__ __launch_bounds__(kPlan) void reserve_plan(const ReserveParams p)
{
    __shared__ uint32_t s_key[kSlots], s_cnt[kSlots], s_last[kSlots];  // pages that are appended to and shared
    // a sequence's entries, then the sum before it; kCopies: it copies its last page; kKeeps: it keeps one that others copy
    __shared__ uint32_t s_need[kMaxSeqs];
    constexpr uint32_t kCopies = 1u << 31, kKeeps = 1u << 30;
    __shared__ uint32_t s_list[kListHere];  // the list's first entries
    __shared__ uint32_t s_wave[kPlan / 64];
    __shared__ uint32_t s_any, s_moves;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, cap = p.max_pages << p.shift, in_page = (1u << p.shift) - 1;
    if (tid == 0)
        s_any = s_moves = 0;

    // The entries [first, last) that the new rows [c, end) of sequence b fall into.
    struct Window {
        uint32_t c, end, first, last;
    };
    const auto window = [&](uint32_t b) __attribute__((always_inline)) {
        Window w{0, 0, 0, 0};
        if (b < p.batch) {
            w.c = min(p.ctx[b], cap);
            w.end = w.c + min(new_rows(p.starts, p.rows, b).n, cap - w.c);
            w.first = w.c >> p.shift;
            w.last = w.end > w.c ? (w.end + in_page) >> p.shift : w.first;
        }
        return w;
    };
    const auto entry = [&](uint32_t b, uint32_t j) { return p.table[(size_t)b * p.max_pages + j]; };
    // Sequence b: its window, the first kFew entries of it, and the partly filled page that it appends to and others hold
    // (kNoPage: none) with its holders.
    struct Seq {
        Window w;
        uint32_t e[kFew], page, held;
    };
    const auto look = [&](uint32_t b, const Window& w) __attribute__((always_inline)) {
        Seq s{w, {}, kNoPage, 0};
        #pragma unroll
        for (uint32_t i = 0; i < kFew; ++i)
            s.e[i] = w.first + i < w.last ? entry(b, w.first + i) : 0u;
        if (w.end != w.c && (w.c & in_page) && s.e[0] < p.pages) {
            s.held = p.refs[s.e[0]];
            s.page = s.held > 1 ? s.e[0] : kNoPage;
        }
        return s;
    };
    // Most calls have a sequence a thread at most and few pages to look through: what those need is loaded once, all of it before
    // the first use (64 sequences' step 4.8 us of kernel, 5.5 with a load in front of each use).
    const Window mine_w = window(tid);
    uint32_t refs0[kLook];
    load_refs(p.refs, tid * kLook, p.pages, refs0);
    copy_share(p.copy, tid, kPlan);
    const Seq mine = look(tid, mine_w);
    const auto seq = [&](uint32_t b) __attribute__((always_inline)) { return b == tid ? mine : look(b, window(b)); };
    __syncthreads();

    const auto slot_of = [](uint32_t e) { return (e * 2654435761u) >> (32 - 13); };
    static_assert(kSlots == 1u << 13, "slot_of takes 13 bits");

    for (uint32_t b = tid; b < p.batch; b += kPlan)
        if (seq(b).page != kNoPage)
            s_any = 1;
    __syncthreads();
    const bool any = s_any != 0;
    if (any) {
        for (uint32_t i = tid; i < kSlots; i += kPlan) {
            s_key[i] = kNoPage;
            s_cnt[i] = s_last[i] = 0;
        }
        __syncthreads();
        for (uint32_t b = tid; b < p.batch; b += kPlan) {
            const uint32_t e = seq(b).page;
            if (e == kNoPage)
                continue;
            uint32_t i = slot_of(e);
            for (;;) {  // (at most kMaxSeqs of the kSlots are ever taken)
                const uint32_t old = atomicCAS(&s_key[i], kNoPage, e);
                if (old == kNoPage || old == e)
                    break;
                i = (i + 1) % kSlots;
            }
            atomicAdd(&s_cnt[i], 1u);
            atomicMax(&s_last[i], b);
        }
        __syncthreads();
    }
    const auto slot_with = [&](uint32_t e) __attribute__((always_inline)) {
        uint32_t i = slot_of(e);
        while (s_key[i] != e && s_key[i] != kNoPage)  // (e is there; were it not, a slot is free)
            i = (i + 1) % kSlots;
        return i;
    };
    // What sequence b does with a last page that is shared: it copies it, unless all of its holders append to it and b is the
    // last of them, who keeps it.
    const auto shared = [&](uint32_t b, const Seq& s) __attribute__((always_inline)) {
        if (s.page == kNoPage)
            return 0u;
        const uint32_t i = slot_with(s.page);
        return s.held > s_cnt[i] || s_last[i] != b ? kCopies : kKeeps;
    };

    // A sequence's entries without a page, in the order of their rows: few by its thread, many by its wave.
    uint32_t carry = 0;
    for (uint32_t b0 = 0; b0 < p.batch; b0 += kPlan) {
        const uint32_t b = b0 + tid;
        const Seq s = seq(b);
        const Window& w = s.w;
        const uint32_t how = shared(b, s);
        const bool few = w.last - w.first <= kFew;
        uint32_t need = how == kCopies ? 1u : 0u;
        #pragma unroll
        for (uint32_t i = 0; i < kFew; ++i)
            need += few && w.first + i < w.last && s.e[i] >= p.pages ? 1u : 0u;
        for (uint64_t m = __ballot(!few); m; m &= m - 1) {
            const uint32_t l = (uint32_t)__builtin_ctzll(m), bl = b - lane + l;
            const uint32_t first = (uint32_t)__builtin_amdgcn_readlane(w.first, l);
            const uint32_t last = (uint32_t)__builtin_amdgcn_readlane(w.last, l);
            uint32_t x = 0;
            for (uint32_t j = first; j < last; j += 64)
                x += __popcll(__ballot(j + lane < last && entry(bl, j + lane) >= p.pages));
            need += lane == l ? x : 0u;
        }
        uint32_t total;
        const uint32_t before = scan_threads(need, s_wave, total);
        if (b < p.batch)
            s_need[b] = ((carry + before) & (kKeeps - 1)) | how;
        carry += total;
    }
    const uint32_t want = min(carry, p.list_max);

    // The free pages of the lowest numbers.
    uint32_t found = 0;
    for (uint32_t p0 = 0; p0 < p.pages && found < want; p0 += kPlan * kLook) {
        uint32_t x[kLook], n = 0, total;
        const uint32_t at = p0 + tid * kLook;
        if (p0 != 0)
            load_refs(p.refs, at, p.pages, x);
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i) {
            x[i] = p0 == 0 ? refs0[i] : x[i];
            n += x[i] == 0 ? 1u : 0u;
        }
        uint32_t to = found + scan_threads(n, s_wave, total);
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i)
            if (x[i] == 0 && to < want) {
                (to < kListHere ? s_list[to] : p.list[to]) = at + i;
                ++to;
            }
        found += total;
    }
    found = min(found, want);
    // Where the free pages run out, a sequence may stay on a shared page that another one, whose new rows would go where it has
    // rows of its own, was to keep: s_cnt becomes the rows of those whose copy of a page fails.
    const bool runs_out = any && found < carry;
    if (runs_out)
        for (uint32_t i = tid; i < kSlots; i += kPlan)
            s_cnt[i] = 0;
    __syncthreads();  // the list, s_cnt, and every read of refs, before their writes

    for (uint32_t b0 = 0; b0 < p.batch; b0 += kPlan) {
        const uint32_t b = b0 + tid;
        // (refs, and so what `look` says of shared pages, may have changed by now: the sequence copies if s_need says so)
        const Seq s = seq(b);
        const Window& w = s.w;
        const bool few = w.last - w.first <= kFew;
        const uint32_t need = b < p.batch ? s_need[b] : 0u, prefix = need & (kKeeps - 1);
        const bool copy = need & kCopies;
        uint32_t fail = kNoPage;  // the first entry that gets none
        if (runs_out) {  // (those that copy a page come before the one that keeps it: in this round of sequences, or an earlier one)
            if (copy && prefix >= found)
                atomicMax(&s_cnt[slot_with(s.e[0])], w.c & in_page);
            __syncthreads();
            if ((need & kKeeps) && s_cnt[slot_with(s.e[0])] > (w.c & in_page))
                fail = w.first;
        }
        // entry j of sequence x, now old, takes the idx-th page; cp: in place of its shared page of rows [0, part)
        const auto give = [&](uint32_t x, uint32_t j, uint32_t idx, uint32_t old, bool cp, uint32_t part) __attribute__((always_inline)) {
            const uint32_t page = idx < kListHere ? s_list[idx] : p.list[idx];
            if (cp) {
                atomicSub(&p.refs_out[old], 1u);
                p.moves[atomicAdd(&s_moves, 1u)] = Move{old, page, part, 0u};
            }
            p.refs_out[page] = 1;
            p.table_out[(size_t)x * p.max_pages + j] = page;
        };
        if (few) {
            uint32_t idx = prefix;
            #pragma unroll
            for (uint32_t i = 0; i < kFew; ++i) {
                const uint32_t j = w.first + i;
                const bool cp = copy && i == 0;
                if (j >= w.last || (!cp && s.e[i] < p.pages))
                    continue;
                if (idx < found)
                    give(b, j, idx, s.e[i], cp, w.c & in_page);
                else
                    fail = min(fail, j);
                ++idx;
            }
        }
        for (uint64_t m = __ballot(!few); m; m &= m - 1) {
            const uint32_t l = (uint32_t)__builtin_ctzll(m), bl = b - lane + l;
            const uint32_t first = (uint32_t)__builtin_amdgcn_readlane(w.first, l);
            const uint32_t last = (uint32_t)__builtin_amdgcn_readlane(w.last, l);
            const uint32_t c = (uint32_t)__builtin_amdgcn_readlane(w.c, l);
            const bool cpl = __builtin_amdgcn_readlane(copy ? 1u : 0u, l) != 0;
            uint32_t idx = (uint32_t)__builtin_amdgcn_readlane(prefix, l), none = kNoPage;
            for (uint32_t j0 = first; j0 < last; j0 += 64) {
                const uint32_t j = j0 + lane;
                const bool cp = cpl && j == first;
                const uint32_t old = j < last ? entry(bl, j) : 0u;
                const bool needs = j < last && (cp || old >= p.pages);
                const uint64_t all = __ballot(needs);
                const uint32_t rank = idx + (uint32_t)__popcll(all & ((1ull << lane) - 1));
                if (needs && rank < found)
                    give(bl, j, rank, old, cp, c & in_page);
                const uint64_t lack = __ballot(needs && rank >= found);
                if (lack && none == kNoPage)
                    none = j0 + (uint32_t)__builtin_ctzll(lack);
                idx += (uint32_t)__popcll(all);
            }
            fail = lane == l ? min(fail, none) : fail;
        }
        if (b < p.batch)
            p.ctx_out[b] = fail == kNoPage ? w.end : max(w.c, fail << p.shift);
    }
    __syncthreads();
    if (tid == 0)
        p.count[0] = s_moves;
}

// ---- fork ----------------------------------------------------------------------------------------------------------

struct ForkParams {
    const uint32_t *parent, *keep, *table, *ctx;
    uint32_t *table_out, *refs_out, *ctx_out;
    uint32_t batch, pages, shift, max_pages;
    CopyWords copy;
};

// New sequence i, by `threads` threads.
__device__ __forceinline__ void fork_row(const ForkParams& p, uint32_t i, uint32_t thread, uint32_t threads)
{
    const uint32_t* old = p.table + (size_t)i * p.max_pages;
    const uint32_t was0 = thread < p.max_pages ? old[thread] : kNoPage;  // (beside the parent's load)
    const uint32_t cap = p.max_pages << p.shift;
    const uint32_t src = p.parent ? p.parent[i] : i;
    uint32_t c = 0;
    if (src < p.batch)
        c = min(min(p.keep ? p.keep[i] : ~0u, p.ctx[src]), cap);
    const uint32_t kept = (c + (1u << p.shift) - 1) >> p.shift;
    if (thread == 0)
        p.ctx_out[i] = c;
    const uint32_t* from = p.table + (size_t)(src < p.batch ? src : i) * p.max_pages;
    for (uint32_t j = thread; j < p.max_pages; j += threads) {
        const uint32_t was = j == thread ? was0 : old[j];
        uint32_t e = j < kept ? src == i ? was : from[j] : kNoPage;
        if (e >= p.pages)
            e = kNoPage;
        p.table_out[(size_t)i * p.max_pages + j] = e;
        if (e == was)
            continue;
        if (e != kNoPage)
            atomicAdd(&p.refs_out[e], 1u);
        if (was < p.pages)
            atomicSub(&p.refs_out[was], 1u);
    }
}
__global__ __launch_bounds__(256) void fork_rows(const ForkParams p) { fork_row(p, blockIdx.x, threadIdx.x, 256); }

// A small call whole, by one workgroup: the copies, then a wave a sequence.
__global__ __launch_bounds__(kPlan) void fork_small(const ForkParams p)
{
    copy_share(p.copy, threadIdx.x, kPlan);
    __syncthreads();
    for (uint32_t i = threadIdx.x >> 6; i < p.batch; i += kPlan / 64)
        fork_row(p, i, threadIdx.x & 63u, 64);
}

// ---- compact -------------------------------------------------------------------------------------------------------

struct CompactParams {
    const uint32_t *table, *refs;
    uint32_t *table_out, *refs_out, *used_out;
    uint32_t* map;    // [pages]
    uint32_t* count;  // moves
    Move* moves;      // [most]
    uint32_t* hole;   // [most]
    uint32_t batch, pages, shift, max_pages, most;
};

// Holes that are listed in LDS (4096 pages 212.2 us a pass, by memory 213.3; 512 15.9 and 16.1).
constexpr uint32_t kHolesHere = 16384;
__global__ __launch_bounds__(kPlan) void compact_plan(const CompactParams p)
{
    __shared__ uint32_t s_wave[kPlan / 64], s_hole[kHolesHere];
    const uint32_t tid = threadIdx.x;
    uint32_t mine = 0, used;
    for (uint32_t at = tid * kLook; at < p.pages; at += kPlan * kLook) {
        uint32_t x[kLook];
        load_refs(p.refs, at, p.pages, x);
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i)
            mine += at + i < p.pages && x[i] != 0 ? 1u : 0u;
    }
    scan_threads(mine, s_wave, used);
    // Holes [0, used), then sources [used, pages): a round's holes are listed before its sources look for theirs.
    uint32_t holes = 0, sources = 0;
    for (uint32_t p0 = 0; p0 < p.pages; p0 += kPlan * kLook) {
        uint32_t x[kLook], nh = 0, ns = 0, th = 0, ts = 0, h = 0, s = 0;
        const uint32_t at = p0 + tid * kLook;
        load_refs(p.refs, at, p.pages, x);
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i) {
            nh += at + i < used && x[i] == 0 ? 1u : 0u;
            ns += at + i >= used && at + i < p.pages && x[i] != 0 ? 1u : 0u;
        }
        if (p0 < used)
            h = holes + scan_threads(nh, s_wave, th);
        if (p0 + kPlan * kLook > used)
            s = sources + scan_threads(ns, s_wave, ts);
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i) {
            const uint32_t page = at + i;
            if (page >= used)
                continue;
            if (x[i] == 0) {
                if (h < kHolesHere)
                    s_hole[h] = page;
                else
                    p.hole[h] = page;
                ++h;
            } else {
                p.refs_out[page] = x[i];
            }
            p.map[page] = x[i] ? page : kNoPage;
        }
        __syncthreads();
        #pragma unroll
        for (uint32_t i = 0; i < kLook; ++i) {
            const uint32_t page = at + i;
            if (page < used || page >= p.pages)
                continue;
            uint32_t to = kNoPage;
            if (x[i] != 0) {
                to = s < kHolesHere ? s_hole[s] : p.hole[s];
                p.moves[s++] = Move{page, to, 1u << p.shift, 0u};
                p.refs_out[to] = x[i];
            }
            p.refs_out[page] = 0;
            p.map[page] = to;
        }
        holes += th;
        sources += ts;
    }
    if (tid == 0) {
        p.count[0] = sources;
        p.used_out[0] = used;
    }
}

// The pages' data, a (page, layer, kv head) a workgroup at a time, then the tables.
__global__ __launch_bounds__(256) void compact_move(const MoveParams p, const CompactParams c)
{
    if (p.k) {
        const uint64_t items = (uint64_t)p.count[0] * p.layers * p.kv_heads;
        for (uint64_t i = blockIdx.x; i < items; i += p.groups)
            move_rows(p, i);
    }
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)c.batch * c.max_pages;
         i += (uint64_t)p.groups * 256) {
        const uint32_t e = c.table[i];
        c.table_out[i] = e < c.pages ? c.map[e] : kNoPage;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------

size_t round16(size_t x) { return (x + 15) / 16 * 16; }

int check_sizes(const char* what, const mako_pages_args* a, bool data)
{
    if (!page_size_ok(a->page))
        return fail(MAKO_EINVAL, "%s: pages of %u rows (a power of two, 64 to 4096)", what, a->page);
    if ((uint64_t)a->max_pages * a->page >= (1ull << 31))
        return fail(MAKO_EINVAL, "%s: %u pages of %u rows a sequence (below 2^31 rows)", what, a->max_pages, a->page);
    if ((uint64_t)a->batch * a->max_pages >= (1ull << 32) || a->pages >= (1u << 31) || a->rows >= (1u << 31))
        return fail(MAKO_EINVAL, "%s: %u x %u table entries, %u pages or %u rows are too many", what, a->batch, a->max_pages,
                    a->pages, a->rows);
    if (data && a->dim != 64 && a->dim != 128 && a->dim != 256)
        return fail(MAKO_EUNSUPPORTED, "%s: heads of %u (64, 128 or 256)", what, a->dim);
    if (data && (!a->kv_heads || a->kv_heads > (1u << 16)))
        return fail(MAKO_EINVAL, "%s: %u kv heads", what, a->kv_heads);
    return MAKO_OK;
}

int check_pools(const char* what, const mako_pages_args* a, const void* k, const void* v)
{
    if (!k != !v)
        return fail(MAKO_EINVAL, "%s: k and v go together", what);
    if (k && !a->layers)
        return fail(MAKO_EINVAL, "%s: pools of no layers", what);
    if (!aligned16(k) || !aligned16(v))
        return fail(MAKO_EINVAL, "%s: k and v must be 16-byte aligned", what);
    return MAKO_OK;
}

int check_workspace(const char* what, const void* ws, size_t bytes, size_t need)
{
    if (bytes < need || (need && !ws) || !aligned16(ws))
        return fail(MAKO_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, bytes, need);
    return MAKO_OK;
}

// Entries that a step's rows can need: each sequence's first, one a page from there on, and a copy.
uint64_t reserve_most(const mako_pages_args* a)
{
    return std::min<uint64_t>((uint64_t)a->rows / a->page + 2ull * a->batch, a->pages);
}
// Pages that compaction can move.
uint64_t compact_most(const mako_pages_args* a) { return a->pages / 2; }

uint32_t groups_for(uint64_t items) { return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(items, 2048)); }

CopyWords copies_of(const uint32_t* const (&from)[3], uint32_t* const (&to)[3], const uint64_t (&n)[3])
{
    CopyWords c{};
    for (int i = 0; i < 3; ++i)
        if (to[i] && from[i] != to[i])
            c.from[i] = from[i], c.to[i] = to[i], c.n[i] = n[i];
    return c;
}
// Copies more than `most` words by a launch, and leaves c empty then.
void launch_long(CopyWords& c, uint64_t most, hipStream_t s)
{
    if (c.n[0] + c.n[1] + c.n[2] <= most)
        return;
    c.groups = groups_for((std::max({c.n[0], c.n[1], c.n[2]}) + 1023) / 1024);
    hipLaunchKernelGGL(copy_words, dim3(c.groups), dim3(256), 0, s, c);
    c = CopyWords{};
}

}  // namespace
}  // namespace mako

using namespace mako;

extern "C" int mako_pages_write(const mako_pages_args* a, const void* kd, const void* vd, const uint32_t* table,
                                const uint32_t* starts, const uint32_t* ctx_len, const uint32_t* end, void* k, void* v,
                                void* stream)
{
    const char* what = "pages_write";
    if (!a || !kd || !vd || !table || !ctx_len || !k || !v)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (const int rc = check_sizes(what, a, true))
        return rc;
    if (!starts && a->batch > a->rows)
        return fail(MAKO_EINVAL, "%s: a row each of %u sequences in %u rows", what, a->batch, a->rows);
    if (a->rows > a->d_pad)
        return fail(MAKO_EINVAL, "%s: %u rows in kv heads of %u", what, a->rows, a->d_pad);
    if (!aligned16(kd) || !aligned16(vd) || !aligned16(k) || !aligned16(v))
        return fail(MAKO_EINVAL, "%s: kd, vd, k and v must be 16-byte aligned", what);
    if (!a->batch || !a->rows || !a->pages || !a->max_pages)
        return ok();
    const uint32_t rows = starts ? a->rows : a->batch;
    if (!grid_fits((rows + 3) / 4, 256))
        return fail(MAKO_EINVAL, "%s: %u rows exceed the grid", what, rows);
    const WriteParams p{static_cast<const u32x4*>(kd), static_cast<const u32x4*>(vd), table, starts, ctx_len, end,
                        static_cast<u32x4*>(k), static_cast<u32x4*>(v), a->batch, rows, a->d_pad, a->pages,
                        log2_of(a->page), a->max_pages, a->kv_heads, a->dim / 8};
    hipLaunchKernelGGL(pages_write, dim3((rows + 3) / 4), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return check_launch(what);
}

extern "C" size_t mako_pages_reserve_workspace(const mako_pages_args* a)
{
    return a && page_size_ok(a->page) ? 16 + (size_t)a->batch * sizeof(Move) + round16(reserve_most(a) * 4) : 0;
}

extern "C" int mako_pages_reserve(const mako_pages_args* a, const uint32_t* table, const uint32_t* refs,
                                  const uint32_t* starts, const uint32_t* ctx_len, uint32_t* table_out,
                                  uint32_t* refs_out, uint32_t* ctx_out, void* k, void* v, void* workspace,
                                  size_t workspace_bytes, void* stream)
{
    const char* what = "pages_reserve";
    if (!a || !table || !refs || !ctx_len || !table_out || !refs_out || !ctx_out)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (const int rc = check_sizes(what, a, k != nullptr))
        return rc;
    if (a->batch > kMaxSeqs)
        return fail(MAKO_EINVAL, "%s: %u sequences (at most %u)", what, a->batch, kMaxSeqs);
    if (!starts && a->batch > a->rows)
        return fail(MAKO_EINVAL, "%s: a row each of %u sequences in %u rows", what, a->batch, a->rows);
    if (const int rc = check_pools(what, a, k, v))
        return rc;
    if (const int rc = check_workspace(what, workspace, workspace_bytes, mako_pages_reserve_workspace(a)))
        return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    CopyWords copy = copies_of({table, refs, nullptr}, {table_out, refs_out, nullptr},
                               {(uint64_t)a->batch * a->max_pages, a->pages, 0});
    launch_long(copy, kCopyInPlan, s);
    char* ws = static_cast<char*>(workspace);
    uint32_t* count = reinterpret_cast<uint32_t*>(ws);
    Move* moves = reinterpret_cast<Move*>(ws + 16);
    const ReserveParams p{table, refs, starts, ctx_len, table_out, refs_out, ctx_out, count, moves,
                          reinterpret_cast<uint32_t*>(ws + 16 + (size_t)a->batch * sizeof(Move)), a->batch, a->rows,
                          a->pages, log2_of(a->page), a->max_pages, (uint32_t)reserve_most(a), copy};
    hipLaunchKernelGGL(reserve_plan, dim3(1), dim3(kPlan), 0, s, p);
    if (k) {
        const uint32_t groups = groups_for((uint64_t)a->batch * a->layers * a->kv_heads);
        const MoveParams m{moves, count, static_cast<u32x4*>(k), static_cast<u32x4*>(v), a->layers, a->kv_heads, a->pages,
                           log2_of(a->page), a->dim / 8, groups};
        hipLaunchKernelGGL(copy_pages, dim3(groups), dim3(256), 0, s, m);
    }
    return check_launch(what);
}

extern "C" size_t mako_pages_fork_workspace(const mako_pages_args* a)
{
    return a ? round16((size_t)a->batch * a->max_pages * 4) + (size_t)a->batch * 4 : 0;
}

extern "C" int mako_pages_fork(const mako_pages_args* a, const uint32_t* parent, const uint32_t* keep,
                               const uint32_t* table, const uint32_t* refs, const uint32_t* ctx_len, uint32_t* table_out,
                               uint32_t* refs_out, uint32_t* ctx_out, void* workspace, size_t workspace_bytes,
                               void* stream)
{
    const char* what = "pages_fork";
    if (!a || !table || !refs || !ctx_len || !table_out || !refs_out || !ctx_out)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (const int rc = check_sizes(what, a, false))
        return rc;
    if ((table_out == table) != (ctx_out == ctx_len))
        return fail(MAKO_EINVAL, "%s: table and ctx_len are both updated in place, or neither", what);
    if (!grid_fits(a->batch, 256))
        return fail(MAKO_EINVAL, "%s: %u sequences exceed the grid", what, a->batch);
    const bool in_place = table_out == table;
    if (in_place)
        if (const int rc = check_workspace(what, workspace, workspace_bytes, mako_pages_fork_workspace(a)))
            return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint64_t entries = (uint64_t)a->batch * a->max_pages;
    uint32_t* table_ws = static_cast<uint32_t*>(workspace);
    uint32_t* ctx_ws = in_place ? table_ws + round16(entries * 4) / 4 : nullptr;
    CopyWords copy = copies_of({in_place ? table : nullptr, refs, in_place ? ctx_len : nullptr},
                               {in_place ? table_ws : nullptr, refs_out, ctx_ws}, {entries, a->pages, a->batch});
    const bool small = entries <= kForkSmall;
    launch_long(copy, small ? kCopyInPlan : 0, s);
    const ForkParams p{parent, keep, in_place ? table_ws : table, in_place ? ctx_ws : ctx_len, table_out, refs_out,
                       ctx_out, a->batch, a->pages, log2_of(a->page), a->max_pages, copy};
    if (small)
        hipLaunchKernelGGL(fork_small, dim3(1), dim3(kPlan), 0, s, p);
    else
        hipLaunchKernelGGL(fork_rows, dim3(a->batch), dim3(256), 0, s, p);
    return check_launch(what);
}

extern "C" size_t mako_pages_compact_workspace(const mako_pages_args* a)
{
    return a ? 16 + compact_most(a) * sizeof(Move) + round16(compact_most(a) * 4) + (size_t)a->pages * 4 : 0;
}

extern "C" int mako_pages_compact(const mako_pages_args* a, const uint32_t* table, const uint32_t* refs,
                                  uint32_t* table_out, uint32_t* refs_out, uint32_t* used_out, uint32_t* map_out, void* k,
                                  void* v, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* what = "pages_compact";
    if (!a || !table || !refs || !table_out || !refs_out || !used_out)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (const int rc = check_sizes(what, a, k != nullptr))
        return rc;
    if (const int rc = check_pools(what, a, k, v))
        return rc;
    if (const int rc = check_workspace(what, workspace, workspace_bytes, mako_pages_compact_workspace(a)))
        return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint64_t most = compact_most(a), entries = (uint64_t)a->batch * a->max_pages;
    char* ws = static_cast<char*>(workspace);
    uint32_t* count = reinterpret_cast<uint32_t*>(ws);
    Move* moves = reinterpret_cast<Move*>(ws + 16);
    uint32_t* hole = reinterpret_cast<uint32_t*>(ws + 16 + most * sizeof(Move));
    uint32_t* map = map_out ? map_out : reinterpret_cast<uint32_t*>(ws + 16 + most * sizeof(Move) + round16(most * 4));
    const CompactParams c{table, refs, table_out, refs_out, used_out, map, count, moves, hole, a->batch, a->pages,
                          log2_of(a->page), a->max_pages, (uint32_t)most};
    hipLaunchKernelGGL(compact_plan, dim3(1), dim3(kPlan), 0, s, c);
    const uint64_t items = std::max(k ? most * a->layers * a->kv_heads : 0, (entries + 1023) / 1024);
    if (items) {
        const uint32_t groups = groups_for(items);
        const MoveParams m{moves, count, static_cast<u32x4*>(k), static_cast<u32x4*>(v), a->layers, a->kv_heads, a->pages,
                           log2_of(a->page), a->dim / 8, groups};
        hipLaunchKernelGGL(compact_move, dim3(groups), dim3(256), 0, s, m, c);
    }
    return check_launch(what);
}
