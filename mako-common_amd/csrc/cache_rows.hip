// The rows of a key / value cache: the append of accepted drafts, and the eviction down to a budget by gathered weight.
//
// cache_append: one workgroup a sequence copies its path's rows, 16 bytes a thread at a time, for every kv head. One
// workgroup reads ctx and seen and writes them after its barrier, so they can be updated in place. For accepted paths bound
// by the latency of a launch and a few dependent loads (ctx and the path, then the rows): 1.9 us for one sequence of 8 kv
// heads of 128, 3.5 for 64. Many rows a sequence, a prompt's, are bound by its one CU: 512 rows 56 us, 4096 rows 424.
//
// Eviction, per list (sequence, kv head) of n > budget rows, in two launches:
// * evict_select, one workgroup a list. A row's key is its weight as an integer in the same order (protected rows the
//   largest key, NaN that of -inf, -0 that of 0), held in LDS. The budget-th largest key T comes from histograms of 11 bits
//   of the unprotected keys' range, the highest first, until the rows of a digit all stay (two digits mostly: weights share
//   their leading bits, a digit of the range spreads them); rows above T stay, of those at T the first `need` do. A sum
//   over the threads of their rows' counts gives every row its rank among the kept, and from ranks follow the rows' places:
//   a row j below the budget that is given up is hole j - (kept before j), a kept row past the budget source (kept before
//   it) - (kept below the budget). The lists of holes and sources go into the workspace.
// * evict_move copies source i over hole i, K, V, weight and position. Sources lie past the budget and holes below it,
//   so no row is read and written.
#include <algorithm>

#include "device.hpp"
#include "split_ranges.hpp"

namespace mako {
namespace {

constexpr int kThreads = 1024;  // of append_rows

struct AppendParams {
    const void *kd, *vd;
    const uint32_t *path, *n_path;
    const uint32_t* ctx;   // (may be ctx_out)
    uint32_t* ctx_out;
    const uint32_t* seen;  // (may be seen_out)
    uint32_t* seen_out;
    float* w;
    uint32_t* pos;
    void *k, *v;
    uint32_t batch, n_draft, d_pad, kv_heads, dim, cap;
};

__global__ __launch_bounds__(kThreads) void append_rows(const AppendParams p)
{
    const uint32_t b = blockIdx.x, tid = threadIdx.x;
    const uint32_t ctx = min(p.ctx[b], p.cap), seen = p.seen ? p.seen[b] : 0u;
    const uint32_t n = min(p.n_path ? min(p.n_path[b], p.n_draft) : p.n_draft, p.cap - ctx);
    __syncthreads();  // every read of ctx and seen before their writes
    if (tid == 0) {
        p.ctx_out[b] = ctx + n;
        if (p.seen_out)
            p.seen_out[b] = seen + n;
    }
    const uint32_t cpr = p.dim / 8, per = n * cpr;  // 16-byte chunks of a row, of a kv head's rows
    const u32x4 *kd = static_cast<const u32x4*>(p.kd), *vd = static_cast<const u32x4*>(p.vd);
    u32x4 *k = static_cast<u32x4*>(p.k), *v = static_cast<u32x4*>(p.v);
    for (uint32_t x = tid; x < p.kv_heads * per; x += kThreads) {
        const uint32_t kvh = x / per, i = x % per / cpr, c = x % cpr;
        const uint32_t r = p.path ? p.path[(size_t)b * p.n_draft + i] : i;
        const size_t row = ((size_t)b * p.kv_heads + kvh) * p.cap + ctx + i;
        const size_t src = ((size_t)kvh * p.d_pad + (size_t)b * p.n_draft + r) * cpr + c;
        const bool has = r < p.n_draft;
        k[row * cpr + c] = has ? kd[src] : u32x4{};
        v[row * cpr + c] = has ? vd[src] : u32x4{};
        if (c == 0) {
            if (p.w)
                p.w[row] = 0.0f;
            if (p.pos)
                p.pos[row] = seen + i;
        }
    }
}

struct EvictParams {
    void *k, *v;
    const float* w;        // (may be w_out)
    const uint32_t* pos;   // (may be pos_out)
    const uint32_t *seen, *ctx;
    float* w_out;
    uint32_t *pos_out, *ctx_out;
    uint32_t* count;       // [lists] rows that move
    uint32_t *hole, *src;  // [lists][most]
    uint32_t kv_heads, dim, cap, max_ctx, budget, recent, sinks, most;
};

// Weights as integers in the same order: below 2^31 the negative ones, above the others; 0xffffffff (a NaN's) is free
// for protected rows.
__device__ __forceinline__ uint32_t order_of(float x)
{
    const uint32_t u = as_u32(fmaxf(x, -INFINITY) + 0.0f);  // (NaN gives the other; -0 + 0 = 0)
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

constexpr int kDigitBits = 11, kDigits = 1 << kDigitBits;

// The largest x of a wave's lanes, in lane 63.
__device__ __forceinline__ uint32_t max_lanes(uint32_t x)
{
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, false));  // row_shr 1
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false));  // lane 15 of rows 0 and 2 to rows 1 and 3
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false));  // lane 31 to rows 2 and 3
    return x;
}

// The inclusive sum of x over the workgroup's threads up to this one; total: over all of them (s: a word a wave; two barriers).
template <int W>
__device__ __forceinline__ uint32_t scan_threads(uint32_t x, u32x4 (&s)[W / 4], uint32_t lane, uint32_t wv, uint32_t& total)
{
    x = scan_lanes(x);
    if (lane == 63)
        reinterpret_cast<uint32_t*>(s)[wv] = x;
    __syncthreads();
    total = 0;
    #pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const u32x4 y = s[i];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            x += 4 * i + j < (int)wv ? y[j] : 0u;
            total += y[j];
        }
    }
    __syncthreads();
    return x;
}

// A workgroup of TH threads; the keys of ROWS rows in LDS (registers would hold them too, but unrolled over them the code
// outgrows the instruction cache, and each line of it runs once). Thread t has R consecutive rows, its first at t R, in
// LDS rows of R + 4 words (R a power of two from 8 on: 16-byte reads without bank conflicts). A longer list goes through in
// blocks of ROWS, read again in each pass. Bound by the passes of one CU: 8 lists of 32768 rows take 20 us, of them loads 5,
// two digits 6, ranks 1.5, lists 3.5; 128 lists of 2112 rows 9, of them 5 after the launch and the first loads.
template <int TH, int ROWS>
__global__ __launch_bounds__(TH) void evict_select(const EvictParams p)
{
    constexpr int W = TH / 64, kPer = kDigits / TH;  // digits a thread sums
    static_assert(ROWS <= 32768 && ROWS / TH % 8 == 0, "counts of a block fit 16 bits, rows go eight at a time");
    __shared__ u32x4 keys[(ROWS + 4 * TH) / 4];
    __shared__ u32x4 hist[kDigits / 4], s_scan[W / 4], s_lo[W / 4], s_hi[W / 4];
    __shared__ uint32_t s_digit, s_above, s_count;
    const uint32_t list = blockIdx.x, b = list / p.kv_heads, tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
    const uint32_t n = min(p.ctx[b], p.max_ctx), seen = p.seen ? p.seen[b] : n, budget = p.budget;
    const size_t base = (size_t)list * p.cap;
    const char* w_in = reinterpret_cast<const char*>(p.w + base);  // (byte offsets of 32 bits: scalar base addressing)
    const char* pos_in = p.pos ? reinterpret_cast<const char*>(p.pos + base) : nullptr;
    const bool copies = p.w_out != p.w || p.pos_out != p.pos;
    if (n <= budget || budget == 0) {
        if (copies && budget)
            for (uint32_t j = tid; j < n; j += TH) {
                p.w_out[base + j] = p.w[base + j];
                p.pos_out[base + j] = p.pos ? p.pos[base + j] : j;
            }
        if (tid == 0)
            p.count[list] = 0;
        return;
    }
    const uint32_t late = seen > p.recent ? seen - p.recent : 0u;  // positions from here on, and below sinks, are protected
    const uint32_t blocks = (n + ROWS - 1) / ROWS;
    const uint32_t lg = blocks > 1 ? 31 - __builtin_clz(ROWS / TH) : max(3, 32 - __builtin_clz((n - 1) / TH | 1)), R = 1u << lg;
    // The unprotected rows' smallest and largest key of what this thread has loaded; and how many rows are protected.
    uint32_t low = 0xffffffffu, high = 0, safe = 0;
    const uint32_t lds_step = TH + 4 * (TH >> lg);  // words between a thread's places: rows TH apart
    // Block blk's keys (rows past the list: key 0, below every row's), eight rows a thread at a time, loaded ahead; `copy`:
    // with the copies below the budget (the rows that are given up get theirs from evict_move); `count`: with the above.
    auto load = [&](uint32_t blk, bool copy, bool count) __attribute__((always_inline)) {
        float next_w[8];
        uint32_t next_pos[8];
        auto fetch = [&](uint32_t e) __attribute__((always_inline)) {
            const uint32_t f = blk * ROWS + e * TH;
            if (f + 8 * TH <= n) {
                #pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    next_w[i] = *reinterpret_cast<const float*>(w_in + 4 * (f + i * TH) + 4 * tid);
                if (pos_in)
                    #pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        next_pos[i] = *reinterpret_cast<const uint32_t*>(pos_in + 4 * (f + i * TH) + 4 * tid);
            } else {
                #pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    next_w[i] = *reinterpret_cast<const float*>(w_in + 4 * min(f + i * TH + tid, n - 1));
                if (pos_in)
                    #pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        next_pos[i] = *reinterpret_cast<const uint32_t*>(pos_in + 4 * min(f + i * TH + tid, n - 1));
            }
        };
        fetch(0);
        uint32_t* to = reinterpret_cast<uint32_t*>(keys) + tid + 4 * (tid >> lg);
        #pragma unroll 1
        for (uint32_t e = 0; e < R; e += 8) {
            const uint32_t f = blk * ROWS + e * TH, end = f + 8 * TH;  // the rows of all threads
            float w[8];
            uint32_t at[8], key[8];
            #pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                w[i] = next_w[i];
                at[i] = pos_in ? next_pos[i] : f + i * TH + tid;
            }
            if (e + 8 < R)
                fetch(e + 8);
            #pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                key[i] = order_of(w[i]);
            if (pos_in || f < p.sinks || end > late || end > n) {
                #pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const bool in = f + i * TH + tid < n, kept = at[i] < p.sinks || at[i] >= late;
                    if (count) {
                        low = in && !kept ? min(low, key[i]) : low;
                        high = in && !kept ? max(high, key[i]) : high;
                        safe += in && kept;
                    }
                    key[i] = !in ? 0u : kept ? 0xffffffffu : key[i];
                }
            } else if (count) {
                #pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    low = min(low, key[i]), high = max(high, key[i]);
            }
            #pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                to[(e + i) * lds_step] = key[i];
            if (copy && copies && f < budget)
                #pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t j = f + i * TH + tid;
                    if (j < budget) {
                        p.w_out[base + j] = w[i];
                        p.pos_out[base + j] = at[i];
                    }
                }
        }
    };
    load(0, true, true);
    for (uint32_t blk = 1; blk < blocks; ++blk)
        load(blk, true, true);  // (a thread writes the same places of LDS each time)
    low = max_lanes(~low);
    high = max_lanes(high);
    if (lane == 63) {
        reinterpret_cast<uint32_t*>(s_lo)[wv] = low;
        reinterpret_cast<uint32_t*>(s_hi)[wv] = high;
    }
    uint32_t total;
    scan_threads<W>(safe, s_scan, lane, wv, total);
    low = high = 0;
    #pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const u32x4 x = s_lo[i], y = s_hi[i];
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            low = max(low, x[j]), high = max(high, y[j]);
    }
    // The budget-th largest key T, a digit of the unprotected keys' range at a time: it is among [lo, lo + span], and `need`
    // of the rows there stay. Where the protected rows alone reach the budget, theirs is the key.
    uint32_t lo = ~uniform(low), span = uniform(high) - lo, need = budget;
    const u32x4* mine = keys + tid * (R / 4 + 1);  // this thread's keys
    uint32_t T = 0xffffffffu;
    if (uniform(total) < budget) {
        need -= uniform(total);
        #pragma unroll 1
        for (;;) {
            T = lo;
            if (span == 0)
                break;
            const uint32_t bits = 32 - __builtin_clz(span), shift = max(bits, (uint32_t)kDigitBits) - kDigitBits;
            for (uint32_t i = tid; i < kDigits / 4; i += TH)
                hist[i] = u32x4{};
            for (uint32_t blk = 0; blk < blocks; ++blk) {
                if (blocks > 1) {
                    __syncthreads();
                    load(blk, false, false);
                }
                __syncthreads();
                #pragma unroll 1
                for (uint32_t e = 0; e < R / 4; e += 2) {
                    const u32x4 key[2] = {mine[e], mine[e + 1]};
                    #pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const uint32_t x = key[i / 4][i % 4] - lo;  // (past the span: key 0 and protected rows too)
                        if (x <= span)
                            atomicAdd(reinterpret_cast<uint32_t*>(hist) + (x >> shift), 1u);
                    }
                }
            }
            __syncthreads();
            // Thread t: kPer digits from the largest down.
            uint32_t c[kPer], sum = 0;
            #pragma unroll
            for (int i = 0; i < kPer; ++i) {
                c[i] = reinterpret_cast<const uint32_t*>(hist)[kDigits - 1 - (kPer * tid + i)];
                sum += c[i];
            }
            uint32_t above = scan_threads<W>(sum, s_scan, lane, wv, total) - sum;
            #pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (above < need && above + c[i] >= need) {
                    s_digit = kDigits - 1 - (kPer * tid + i);
                    s_above = above;
                    s_count = c[i];
                }
                above += c[i];
            }
            __syncthreads();
            lo += uniform(s_digit) << shift;
            span = (1u << shift) - 1;
            need -= uniform(s_above);
            if (uniform(s_count) == need) {  // all of the digit's rows stay, those below do not
                T = lo - 1;
                need = 0;
                break;
            }
        }
    }
    // The kept rows before each, in row order: of the blocks before, of the threads before (the counts above T in the low
    // half, at T in the high), and the thread's own.
    uint32_t* hole = p.hole + (size_t)list * p.most;
    uint32_t* src = p.src + (size_t)list * p.most;
    uint32_t gt0 = 0, eq0 = 0;
    for (uint32_t blk = 0; blk < blocks; ++blk) {
        if (blocks > 1) {
            __syncthreads();
            load(blk, false, false);
            __syncthreads();
        }
        uint32_t c = 0;
        #pragma unroll 1
        for (uint32_t e = 0; e < R / 4; e += 2) {
            const u32x4 key[2] = {mine[e], mine[e + 1]};
            #pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                c += key[i / 4][i % 4] > T;
                c += key[i / 4][i % 4] == T ? 0x10000u : 0u;
            }
        }
        const uint32_t before = scan_threads<W>(c, s_scan, lane, wv, total) - c;
        uint32_t* bases = reinterpret_cast<uint32_t*>(hist);  // the threads' counts, for whoever takes their rows
        bases[tid] = before;
        __syncthreads();
        // Up to the budget, where rows may be holes, and wherever ties at T count, the waves take 64 rows at a time (a lane a
        // row); behind, a row that stays is a source, and its thread lists it. (Of this block: the budget may lie past it.)
        const uint32_t first = blk * ROWS, per_wave = 64 * R;
        uint32_t by_lane = first > budget ? 0u : min((uint32_t)ROWS, (budget - first) / per_wave * per_wave + per_wave);
        if (need)
            by_lane = ROWS;
        for (uint32_t x0 = 64 * wv; x0 < min(by_lane, n - first); x0 += TH) {
            const uint32_t x = first + x0 + lane, k = reinterpret_cast<const uint32_t*>(keys)[x0 + lane + 4 * ((x0 + lane) >> lg)];
            const uint64_t more = __ballot(k > T), tie = __ballot(k == T);
            const uint32_t counts = bases[x0 >> lg];
            const uint32_t gt = __builtin_amdgcn_mbcnt_hi((uint32_t)(more >> 32),
                                                          __builtin_amdgcn_mbcnt_lo((uint32_t)more, gt0 + (counts & 0xffffu)));
            const uint32_t eq = __builtin_amdgcn_mbcnt_hi((uint32_t)(tie >> 32),
                                                          __builtin_amdgcn_mbcnt_lo((uint32_t)tie, eq0 + (counts >> 16)));
            const uint32_t kept_before = gt + min(eq, need);
            const bool kept = k > T || (k == T && eq < need);
            if (x == budget)
                p.count[list] = budget - kept_before;
            if (x < budget && !kept)
                hole[x - kept_before] = x;
            if (x >= budget && kept)
                src[budget - 1 - kept_before] = x;  // from the end: the first source comes last
        }
        if (wv * per_wave >= by_lane) {
            uint32_t at = budget - 1 - gt0 - (before & 0xffffu);  // (need is 0)
            #pragma unroll 1
            for (uint32_t e = 0; e < R / 4; e += 2) {
                const u32x4 key[2] = {mine[e], mine[e + 1]};
                #pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    if (key[i / 4][i % 4] > T)
                        src[at--] = first + tid * R + 4 * e + i;
            }
        }
        gt0 += total & 0xffffu;
        eq0 += total >> 16;
    }
}

constexpr int kMoveRows = 16;  // rows of K and V a workgroup of evict_move

// Bound by the copy. Streaming loads: a call that moves 4096 rows of 128 lists of 16384 takes 87 us with them, 102 without
// (93 with streaming stores too); one that moves 152 rows of lists of 2200, 13.8 and 13.5.
__global__ __launch_bounds__(256) void evict_move(const EvictParams p)
{
    const uint32_t chunks = (p.most + kMoveRows - 1) / kMoveRows;
    const uint32_t list = chunks ? blockIdx.x / chunks : blockIdx.x, chunk = chunks ? blockIdx.x % chunks : 0u;
    const uint32_t b = list / p.kv_heads;
    if (chunk == 0 && list % p.kv_heads == 0 && threadIdx.x == 0)
        p.ctx_out[b] = min(min(p.ctx[b], p.max_ctx), p.budget);
    const uint32_t count = p.count[list], i0 = chunk * kMoveRows, i1 = min(count, i0 + kMoveRows);
    if (i0 >= i1)
        return;
    const size_t base = (size_t)list * p.cap;
    const uint32_t *hole = p.hole + (size_t)list * p.most, *src = p.src + (size_t)list * p.most;
    const uint32_t cpr = p.dim / 8;
    u32x4 *k = static_cast<u32x4*>(p.k) + base * cpr, *v = static_cast<u32x4*>(p.v) + base * cpr;
    for (uint32_t x = threadIdx.x; x < (i1 - i0) * cpr; x += 256) {
        const uint32_t i = i0 + x / cpr, c = x % cpr;
        const size_t to = (size_t)hole[i] * cpr + c, from = (size_t)src[count - 1 - i] * cpr + c;
        const u32x4 kk = __builtin_nontemporal_load(k + from), vv = __builtin_nontemporal_load(v + from);
        k[to] = kk;
        v[to] = vv;
    }
    if (threadIdx.x < i1 - i0) {
        const uint32_t i = i0 + threadIdx.x, to = hole[i], from = src[count - 1 - i];
        p.w_out[base + to] = p.w[base + from];
        p.pos_out[base + to] = p.pos ? p.pos[base + from] : from;
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool dim_ok(uint32_t dim) { return dim == 64 || dim == 128 || dim == 256; }

// Most rows of a list that can move: as many as are kept, and as lie past the budget.
uint32_t most_of(const mako_evict_args* a)
{
    return a->max_ctx > a->budget ? std::min(a->budget, a->max_ctx - a->budget) : 0u;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace
}  // namespace mako

using namespace mako;

extern "C" int mako_cache_append(const mako_append_args* a, mako_dtype in, const void* kd, const void* vd,
                                 const uint32_t* path, const uint32_t* n_path, const uint32_t* ctx_len,
                                 uint32_t* ctx_out, const uint32_t* seen, uint32_t* seen_out, float* w, uint32_t* pos,
                                 void* k, void* v, void* stream)
{
    const char* what = "cache_append";
    if (!a || !kd || !vd || !ctx_len || !ctx_out || !k || !v)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if ((pos || seen_out) && !seen)
        return fail(MAKO_EINVAL, "%s: pos and seen_out need seen", what);
    if (!dim_ok(a->dim))
        return fail(MAKO_EUNSUPPORTED, "%s: heads of %u (64, 128 or 256)", what, a->dim);
    if (in != MAKO_F16 && in != MAKO_BF16)
        return fail(MAKO_EUNSUPPORTED, "%s: input type %d (f16 or bf16)", what, (int)in);
    if (!a->kv_heads)
        return fail(MAKO_EINVAL, "%s: no kv heads", what);
    if ((uint64_t)a->batch * a->n_draft > a->d_pad)
        return fail(MAKO_EINVAL, "%s: %u x %u draft rows in kv heads of %u rows", what, a->batch, a->n_draft, a->d_pad);
    if ((uint64_t)a->kv_heads * a->n_draft * (a->dim / 8) > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %u draft rows of %u kv heads exceed 2^31 chunks", what, a->n_draft, a->kv_heads);
    if ((uint64_t)a->cap * a->dim * 2 > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %u cache rows exceed 2 GiB a head", what, a->cap);
    if (!grid_fits(a->batch, kThreads))
        return fail(MAKO_EINVAL, "%s: %u sequences exceed the grid", what, a->batch);
    if (!aligned16(kd) || !aligned16(vd) || !aligned16(k) || !aligned16(v))
        return fail(MAKO_EINVAL, "%s: kd, vd, k and v must be 16-byte aligned", what);
    if (a->batch == 0)
        return ok();
    const AppendParams p{kd, vd, path, n_path, ctx_len, ctx_out, seen, seen_out, w, pos, k, v, a->batch, a->n_draft,
                         a->d_pad, a->kv_heads, a->dim, a->cap};
    hipLaunchKernelGGL(append_rows, dim3(a->batch), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
    return check_launch(what);
}

extern "C" size_t mako_cache_evict_workspace(const mako_evict_args* a)
{
    if (!a)
        return 0;
    const size_t lists = (size_t)a->batch * a->kv_heads;
    return round256(lists * 4) + 2 * round256(lists * most_of(a) * 4);
}

extern "C" int mako_cache_evict(const mako_evict_args* a, mako_dtype in, void* k, void* v, const float* w,
                                const uint32_t* pos, const uint32_t* seen, const uint32_t* ctx_len, float* w_out,
                                uint32_t* pos_out, uint32_t* ctx_out, void* workspace, size_t workspace_bytes,
                                void* stream)
{
    const char* what = "cache_evict";
    if (!a || !k || !v || !w || !ctx_len || !w_out || !pos_out || !ctx_out)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (!pos != !seen)
        return fail(MAKO_EINVAL, "%s: pos and seen go together", what);
    if (!dim_ok(a->dim))
        return fail(MAKO_EUNSUPPORTED, "%s: heads of %u (64, 128 or 256)", what, a->dim);
    if (in != MAKO_F16 && in != MAKO_BF16)
        return fail(MAKO_EUNSUPPORTED, "%s: input type %d (f16 or bf16)", what, (int)in);
    if (!a->kv_heads)
        return fail(MAKO_EINVAL, "%s: no kv heads", what);
    if (a->max_ctx > a->cap)
        return fail(MAKO_EINVAL, "%s: max_ctx %u over the cache's %u rows", what, a->max_ctx, a->cap);
    if ((uint64_t)a->cap * a->dim * 2 > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %u cache rows exceed 2 GiB a head", what, a->cap);
    if ((uint64_t)a->recent + a->sinks > a->budget)
        return fail(MAKO_EINVAL, "%s: %u recent rows and %u sinks over the budget of %u", what, a->recent, a->sinks,
                    a->budget);
    const uint32_t most = most_of(a), chunks = std::max(1u, (most + kMoveRows - 1) / kMoveRows);
    const uint64_t lists = (uint64_t)a->batch * a->kv_heads;
    const uint32_t threads = a->max_ctx <= 4096 ? 512 : 1024;
    if (!grid_fits(lists, threads) || !grid_fits(lists * chunks, 256))
        return fail(MAKO_EINVAL, "%s: %llu lists of %u rows exceed the grid", what, (unsigned long long)lists, most);
    if (!aligned16(k) || !aligned16(v))
        return fail(MAKO_EINVAL, "%s: k and v must be 16-byte aligned", what);
    const size_t need = mako_cache_evict_workspace(a);
    if (workspace_bytes < need || (need && !workspace) || !aligned16(workspace))
        return fail(MAKO_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, workspace_bytes,
                    need);
    if (lists == 0)
        return ok();
    char* ws = static_cast<char*>(workspace);
    const size_t at = round256(lists * 4), bytes = round256(lists * most * 4);
    const EvictParams p{k, v, w, pos, seen, ctx_len, w_out, pos_out, ctx_out, reinterpret_cast<uint32_t*>(ws),
                        reinterpret_cast<uint32_t*>(ws + at), reinterpret_cast<uint32_t*>(ws + at + bytes), a->kv_heads,
                        a->dim, a->cap, a->max_ctx, a->budget, a->recent, a->sinks, most};
    hipStream_t s = static_cast<hipStream_t>(stream);
    // The call's us with 512 threads for blocks of 4096 rows, and with 1024 for 32768: 8 lists of 1024 10.7, 13.0, of 4096
    // 11.1, 13.4, of 6000 21, 14, of 16384 34, 20; 512 lists of 4096 39, 48, of 8192 87, 89, of 16384 162, 159.
    if (threads == 512)
        hipLaunchKernelGGL((evict_select<512, 4096>), dim3((uint32_t)lists), dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((evict_select<1024, 32768>), dim3((uint32_t)lists), dim3(1024), 0, s, p);
    hipLaunchKernelGGL(evict_move, dim3((uint32_t)(lists * chunks)), dim3(256), 0, s, p);
    return check_launch(what);
}
