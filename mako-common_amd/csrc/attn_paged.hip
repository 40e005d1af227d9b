// Attention of the sequences' new tokens over a cache kept in pages.
//
// Mathematics: new row i of sequence b sits at position c + i, c = ctx_len[b], and sees the cache rows j <= c + i:
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j,  lse = m + ln(sum),  m any bound
// Row j is row j % page of page table[b][j / page].
//
// paged_simple: a workgroup a (row, head), 256 keys a round: a thread a key's score, the round's maximum and sum through
// LDS, then a thread a head dim (and part of the keys) for the outputs. Every row reads all of its keys.
#include <algorithm>

#include "pages_common.hpp"
#include "split_ranges.hpp"

namespace mako {
namespace {

struct PagedParams {
    const void *q, *k, *v;
    const uint32_t *table, *starts, *ctx;
    void* o;
    float* lse;
    uint32_t batch, rows, q_pad, heads, kv_heads, group, pages, shift, max_pages, max_new, max_ctx, width;
    float scale_log2;
};

template <class T, class TO, int D>
__global__ __launch_bounds__(256) void paged_simple(const PagedParams p)
{
    __shared__ float s_q[D], s_p[256], s_red[4], s_o[256];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, w = tid >> 6;
    const uint32_t r = blockIdx.x / p.heads, h = blockIdx.x % p.heads, kvh = h / p.group;
    uint32_t seq = r;
    if (p.starts) {
        seq = 0;
        for (uint32_t i = 0; i < p.batch; i += 64)
            seq += __popcll(__ballot(i + lane < p.batch && p.starts[i + lane + 1] <= r));
    }
    if (seq >= p.batch)
        return;
    const NewRows nr = new_rows(p.starts, p.rows, seq);
    if (r < nr.s0 || r - nr.s0 >= min(nr.n, p.max_new))
        return;
    const uint32_t n_k = min(min(p.ctx[seq], p.max_ctx) + (r - nr.s0) + 1, p.max_ctx);
    const uint32_t* table = p.table + (size_t)seq * p.max_pages;
    const auto row_of = [&](uint32_t j, bool& has) {
        const uint32_t page = table[j >> p.shift];
        has = page < p.pages;
        return ((((size_t)page * p.kv_heads + kvh) << p.shift) + (j & ((1u << p.shift) - 1))) * D;
    };
    if (tid < D)
        s_q[tid] = (float)static_cast<const T*>(p.q)[((size_t)h * p.q_pad + r) * D + tid];
    constexpr uint32_t kParts = 256 / D;
    const uint32_t d = tid % D, part = tid / D;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (uint32_t j0 = 0; j0 < n_k; j0 += 256) {
        __syncthreads();
        float x = -INFINITY;
        if (j0 + tid < n_k) {
            bool has;
            const size_t at = row_of(j0 + tid, has);
            x = 0.0f;
            if (has)
                for (int i = 0; i < D; ++i)
                    x += s_q[i] * (float)static_cast<const T*>(p.k)[at + i];
            x *= p.scale_log2;
        }
        float mx = x;
        for (int i = 32; i; i >>= 1)
            mx = fmaxf(mx, __shfl_xor(mx, i));
        if (lane == 0)
            s_red[w] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        const float nm = fmaxf(m, mx), mu = nm == -INFINITY ? 0.0f : nm, f = m == -INFINITY ? 0.0f : exp2_fast(m - mu);
        m = nm;
        const float e = exp2_fast(x - mu);
        s_p[tid] = e;
        float sum = e;
        for (int i = 32; i; i >>= 1)
            sum += __shfl_xor(sum, i);
        __syncthreads();
        if (lane == 0)
            s_red[w] = sum;
        __syncthreads();
        l = l * f + ((s_red[0] + s_red[1]) + (s_red[2] + s_red[3]));
        acc *= f;
        for (uint32_t j = part; j < 256 && j0 + j < n_k; j += kParts) {
            bool has;
            const size_t at = row_of(j0 + j, has);
            if (has)
                acc += s_p[j] * (float)static_cast<const T*>(p.v)[at + d];
        }
    }
    s_o[tid] = acc;
    __syncthreads();
    if (tid < D) {
        for (uint32_t i = 1; i < kParts; ++i)
            acc += s_o[i * D + tid];
        static_cast<TO*>(p.o)[(size_t)r * p.width + (size_t)h * D + tid] = (TO)(l == 0.0f ? 0.0f : acc / l);
        if (p.lse && tid == 0)
            p.lse[(size_t)h * p.rows + r] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
    }
}

template <class T, class TO>
void launch_dim(const PagedParams& p, uint32_t dim, uint32_t groups, hipStream_t s)
{
    const dim3 grid(groups), block(256);
    if (dim == 64)
        hipLaunchKernelGGL((paged_simple<T, TO, 64>), grid, block, 0, s, p);
    else if (dim == 128)
        hipLaunchKernelGGL((paged_simple<T, TO, 128>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((paged_simple<T, TO, 256>), grid, block, 0, s, p);
}

int check_args(const mako_paged_args* a, mako_dtype in, mako_dtype out, const void* q, const void* k, const void* v,
               const uint32_t* table, const uint32_t* starts, const uint32_t* ctx_len, const void* o)
{
    const char* what = "attention_paged";
    if (!a || !q || !k || !v || !table || !ctx_len || !o)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (a->dim != 64 && a->dim != 128 && a->dim != 256)
        return fail(MAKO_EUNSUPPORTED, "%s: heads of %u (64, 128 or 256)", what, a->dim);
    if (in != MAKO_F16 && in != MAKO_BF16)
        return fail(MAKO_EUNSUPPORTED, "%s: input type %d (f16 or bf16)", what, (int)in);
    if (out != MAKO_F32 && out != in)
        return fail(MAKO_EUNSUPPORTED, "%s: output type %d (f32 or the input's)", what, (int)out);
    if (!a->heads || !a->kv_heads || a->heads % a->kv_heads)
        return fail(MAKO_EINVAL, "%s: %u heads over %u kv heads", what, a->heads, a->kv_heads);
    if (!page_size_ok(a->page))
        return fail(MAKO_EINVAL, "%s: pages of %u rows (a power of two, 64 to 4096)", what, a->page);
    if (a->max_ctx >= (1u << 31) || (uint64_t)a->max_ctx > (uint64_t)a->max_pages * a->page)
        return fail(MAKO_EINVAL, "%s: max_ctx %u over a table of %u pages of %u rows", what, a->max_ctx, a->max_pages,
                    a->page);
    if ((uint64_t)a->kv_heads * a->page * a->dim * 2 >= (1ull << 32))
        return fail(MAKO_EINVAL, "%s: pages of %u kv heads exceed 4 GiB", what, a->kv_heads);
    if (a->rows > a->q_pad || a->max_new > a->rows)
        return fail(MAKO_EINVAL, "%s: %u rows (%u of a sequence) in query heads of %u", what, a->rows, a->max_new, a->q_pad);
    if (!starts && a->batch > a->rows)
        return fail(MAKO_EINVAL, "%s: a row each of %u sequences in %u rows", what, a->batch, a->rows);
    if ((uint64_t)a->heads * a->dim > a->width || a->width % 4 || a->width >= (1u << 20))
        return fail(MAKO_EINVAL, "%s: o rows of %u for %u heads of %u (a multiple of 4, at least their width, below 2^20)",
                    what, a->width, a->heads, a->dim);
    // what the split counts: 32 keys a unit, for every 32 rows of a sequence at least
    const uint64_t units = ((uint64_t)a->rows / 32 + a->batch) * ((uint64_t)a->max_ctx / 32 + 512) * a->kv_heads;
    if (units >= (1ull << 32) || (uint64_t)a->rows * a->heads >= (1u << 30))
        return fail(MAKO_EINVAL, "%s: %u rows of %u heads over %u keys are too many", what, a->rows, a->heads, a->max_ctx);
    if (!(a->scale > 0.0f) || a->scale == INFINITY)
        return fail(MAKO_EINVAL, "%s: scale %g (positive and finite)", what, (double)a->scale);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
        return fail(MAKO_EINVAL, "%s: q, k, v and o must be 16-byte aligned", what);
    return MAKO_OK;
}

}  // namespace
}  // namespace mako

using namespace mako;

extern "C" size_t mako_attn_paged_workspace(const mako_paged_args*) { return 0; }

extern "C" int mako_attn_paged(const mako_paged_args* a, mako_dtype in, mako_dtype out, const void* q, const void* k,
                               const void* v, const uint32_t* table, const uint32_t* starts, const uint32_t* ctx_len,
                               void* o, float* lse, void*, size_t, void* stream)
{
    const char* what = "attention_paged";
    if (const int rc = check_args(a, in, out, q, k, v, table, starts, ctx_len, o))
        return rc;
    if (!a->batch || !a->max_new)
        return ok();
    const uint32_t rows = starts ? a->rows : a->batch;
    if (!grid_fits((uint64_t)rows * a->heads, 256))
        return fail(MAKO_EINVAL, "%s: %u rows of %u heads exceed the grid", what, rows, a->heads);
    const PagedParams p{q, k, v, table, starts, ctx_len, o, lse, a->batch, a->rows, a->q_pad, a->heads, a->kv_heads,
                        a->heads / a->kv_heads, a->pages, log2_of(a->page), a->max_pages, a->max_new, a->max_ctx,
                        a->width, a->scale * kLog2e};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t groups = rows * a->heads;
    if (in == MAKO_BF16 && out == MAKO_F32)
        launch_dim<__bf16, float>(p, a->dim, groups, s);
    else if (in == MAKO_BF16)
        launch_dim<__bf16, __bf16>(p, a->dim, groups, s);
    else if (out == MAKO_F32)
        launch_dim<_Float16, float>(p, a->dim, groups, s);
    else
        launch_dim<_Float16, _Float16>(p, a->dim, groups, s);
    return check_launch(what);
}
