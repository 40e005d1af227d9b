// The rows of a key / value cache: the append of accepted drafts, and the eviction down to a budget by gathered weight.
//
// cache_append: one workgroup a sequence copies its path's rows, 16 bytes a thread at a time, for every kv head. One
// workgroup reads ctx and seen and writes them after its barrier, so they can be updated in place. Bound by the latency of
// a launch and a few dependent loads (ctx and the path, then the rows).
//
// Eviction, per list (sequence, kv head) of n > budget rows, in two launches:
// * evict_select, one workgroup a list. A row's key is its weight as an integer in the same order (protected rows the
//   largest key, NaN that of -inf, -0 that of 0). The budget-th largest key T comes from four histograms of 8 bits, the
//   highest first; rows above T stay, of those at T the first `need` do. Each wave then counts its run of rows, the
//   counts before it give every row its rank among the kept, and from ranks follow the rows' places: a row j below the
//   budget that is given up is hole j - (kept before j), a kept row past the budget source (kept before it) - (kept
//   below the budget). The lists of holes and sources go into the workspace.
// * evict_move copies source i over hole i, K, V, weight and position. Sources lie past the budget and holes below it,
//   so no row is read and written.
#include <algorithm>

#include "device.hpp"

namespace mako {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

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
    if (x != x)
        x = -INFINITY;
    const uint32_t u = as_u32(x + 0.0f);  // -0 + 0 = 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictList {
    const float* w;
    const uint32_t* pos;
    uint32_t sinks, late;  // positions below sinks, and from late on, are protected
    __device__ __forceinline__ uint32_t key(uint32_t j) const
    {
        const uint32_t at = pos ? pos[j] : j;
        return at < sinks || at >= late ? 0xffffffffu : order_of(w[j]);
    }
};

__global__ __launch_bounds__(kThreads) void evict_select(const EvictParams p)
{
    __shared__ uint32_t hist[kWaves][256], s_digit, s_above, s_gt[kWaves], s_eq[kWaves];
    const uint32_t list = blockIdx.x, b = list / p.kv_heads, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint32_t n = min(p.ctx[b], p.max_ctx), seen = p.seen ? p.seen[b] : n;
    const size_t base = (size_t)list * p.cap;
    const EvictList a{p.w + base, p.pos ? p.pos + base : nullptr, p.sinks, seen > p.recent ? seen - p.recent : 0u};
    float* w_out = p.w_out + base;
    uint32_t* pos_out = p.pos_out + base;
    if (n <= p.budget) {
        for (uint32_t j = tid; j < n; j += kThreads) {
            w_out[j] = a.w[j];
            pos_out[j] = a.pos ? a.pos[j] : j;
        }
        if (tid == 0)
            p.count[list] = 0;
        return;
    }
    // The budget-th largest key, 8 bits at a time: `need` rows are still to be found among those with the prefix.
    uint32_t prefix = 0, need = p.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (uint32_t i = tid; i < kWaves * 256; i += kThreads)
            hist[i / 256][i % 256] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < n; j += kThreads) {
            const uint32_t key = a.key(j);
            if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8))
                atomicAdd(&hist[wv][key >> shift & 255], 1u);
        }
        __syncthreads();
        if (wv == 0) {  // lane l: digits 255 - 4 l down to 252 - 4 l
            uint32_t c[4], sum = 0;
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = 0;
                for (int x = 0; x < kWaves; ++x)
                    c[i] += hist[x][255 - 4 * lane - i];
                sum += c[i];
            }
            uint32_t inc = sum;
            #pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                const uint32_t t = __shfl_up(inc, x);
                inc += lane >= (uint32_t)x ? t : 0u;
            }
            uint32_t above = inc - sum;
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < need && above + c[i] >= need) {
                    s_digit = 255 - 4 * lane - i;
                    s_above = above;
                }
                above += c[i];
            }
        }
        __syncthreads();
        if (need) {  // (a budget of 0 keeps nothing)
            prefix |= s_digit << shift;
            need -= s_above;
        }
        __syncthreads();
    }
    const uint32_t T = p.budget ? prefix : 0xffffffffu;
    const bool none = p.budget == 0;
    // Each wave's run of rows: how many above T, and at T, in it.
    const uint32_t run = (n + kWaves * 64 - 1) / (kWaves * 64) * 64, j0 = wv * run, j1 = min(n, j0 + run);
    uint32_t gt = 0, eq = 0;
    for (uint32_t j = j0; j < j1; j += 64) {
        const uint32_t key = j + lane < n ? a.key(j + lane) : 0u;
        gt += __popcll(__ballot(j + lane < n && !none && key > T));
        eq += __popcll(__ballot(j + lane < n && !none && key == T));
    }
    if (lane == 0) {
        s_gt[wv] = gt;
        s_eq[wv] = eq;
    }
    __syncthreads();
    gt = eq = 0;
    for (uint32_t x = 0; x < wv; ++x) {
        gt += s_gt[x];
        eq += s_eq[x];
    }
    // The ranks: the rows below the budget first (their number sets the sources' ranks).
    uint32_t* hole = p.hole + (size_t)list * p.most;
    uint32_t* src = p.src + (size_t)list * p.most;
    __shared__ uint32_t s_low;
    for (uint32_t j = j0; j < j1; j += 64) {
        const uint32_t x = j + lane;
        const uint32_t key = x < n ? a.key(x) : 0u;
        const uint64_t g = __ballot(x < n && !none && key > T), e = __ballot(x < n && !none && key == T);
        const uint64_t below = (1ull << lane) - 1;
        const uint32_t eb = eq + __popcll(e & below);
        const uint32_t before = gt + __popcll(g & below) + min(eb, need);  // kept rows before x
        const bool kept = x < n && !none && (key > T || (key == T && eb < need));
        if (x == p.budget)
            s_low = before;
        if (x < p.budget && !kept)
            hole[x - before] = x;
        if (x < p.budget && kept) {
            w_out[x] = a.w[x];
            pos_out[x] = a.pos ? a.pos[x] : x;
        }
        if (x >= p.budget && kept)  // counted from the end: the last kept row is source 0 here
            src[p.budget - 1 - before] = x;
        gt += __popcll(g);
        eq += __popcll(e);
    }
    __syncthreads();
    if (tid == 0)
        p.count[list] = p.budget - s_low;
}

constexpr int kMoveRows = 16;  // rows of K and V a workgroup of evict_move

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
        const u32x4 kk = k[from], vv = v[from];
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
    if (a->batch > 0x7fffffffu)
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
    if (lists * chunks > 0x7fffffffu)
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
    hipLaunchKernelGGL(evict_select, dim3((uint32_t)lists), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL(evict_move, dim3((uint32_t)(lists * chunks)), dim3(256), 0, s, p);
    return check_launch(what);
}
