// Attention of drafted tokens over a cache: each sequence's n_draft rows, the nodes of a tree of drafts, attend its cache
// rows [0, ctx) and the drafts that their mask bits name, in one call for the whole batch.
//
// Mathematics: row r of sequence b, head h, with S the cache rows below ctx[b] and the drafts j < n_nodes[b] that r sees:
//   o = sum_{j in S} exp(s_j - m) v_j / sum_{j in S} exp(s_j - m),  s_j = scale q.k_j,  lse = m + ln(sum),  m any bound
//
// tree_rows: one workgroup a row and head. Each wave takes every fourth key, its lanes the head dims, with a running
// maximum; the waves meet in LDS. Every row reads its keys for itself.
#include "device.hpp"

namespace mako {
namespace {

struct TreeParams {
    const void *q, *k, *v, *kd, *vd;
    const uint32_t *ctx, *nodes;
    const uint64_t* mask;
    uint32_t batch, n_draft, q_pad, d_pad, heads, kv_heads, group, cap, max_ctx, width;
    float scale_log2;
};

constexpr int kRowWaves = 4;

template <class T, class TO, int D>
__global__ __launch_bounds__(kRowWaves * 64) void tree_rows(const TreeParams p, TO* __restrict__ o,
                                                             float* __restrict__ lse)
{
    constexpr int E = D / 64;  // head dims a lane
    __shared__ float s_m[kRowWaves], s_l[kRowWaves], s_o[kRowWaves][D];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t row = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
    const uint32_t b = row / p.n_draft, r = row % p.n_draft, kvh = h / p.group;
    const uint32_t nodes = p.nodes ? min(p.nodes[b], p.n_draft) : p.n_draft;
    if (r >= nodes)
        return;
    const uint32_t ctx = min(p.ctx[b], p.max_ctx);
    const uint64_t mask = p.mask ? p.mask[row] : (2ull << r) - 1;
    const T* q = static_cast<const T*>(p.q) + ((size_t)h * p.q_pad + row) * D;
    const size_t cache = ((size_t)b * p.kv_heads + kvh) * p.cap * D;
    const size_t draft = ((size_t)kvh * p.d_pad + (size_t)b * p.n_draft) * D;
    float qr[E], acc[E], m = -INFINITY, l = 0.0f;
    #pragma unroll
    for (int e = 0; e < E; ++e) {
        qr[e] = (float)q[lane + 64 * e];
        acc[e] = 0.0f;
    }
    for (uint32_t j = w; j < ctx + nodes; j += kRowWaves) {
        if (j >= ctx && !(mask >> (j - ctx) & 1))
            continue;
        const T* kr = j < ctx ? static_cast<const T*>(p.k) + cache + (size_t)j * D
                              : static_cast<const T*>(p.kd) + draft + (size_t)(j - ctx) * D;
        const T* vr = j < ctx ? static_cast<const T*>(p.v) + cache + (size_t)j * D
                              : static_cast<const T*>(p.vd) + draft + (size_t)(j - ctx) * D;
        float s = 0.0f;
        #pragma unroll
        for (int e = 0; e < E; ++e)
            s = fmaf(qr[e], (float)kr[lane + 64 * e], s);
        #pragma unroll
        for (int x = 32; x > 0; x >>= 1)
            s += __shfl_xor(s, x);
        s *= p.scale_log2;
        const float nm = fmaxf(m, s), f = m == -INFINITY ? 0.0f : exp2_fast(m - nm), e0 = exp2_fast(s - nm);
        l = l * f + e0;
        #pragma unroll
        for (int e = 0; e < E; ++e)
            acc[e] = acc[e] * f + e0 * (float)vr[lane + 64 * e];
        m = nm;
    }
    if (lane == 0) {
        s_m[w] = m;
        s_l[w] = l;
    }
    #pragma unroll
    for (int e = 0; e < E; ++e)
        s_o[w][lane + 64 * e] = acc[e];
    __syncthreads();
    if (w != 0)
        return;
    float mx = s_m[0];
    for (int i = 1; i < kRowWaves; ++i)
        mx = fmaxf(mx, s_m[i]);
    float sum = 0.0f, f[kRowWaves];
    for (int i = 0; i < kRowWaves; ++i) {
        f[i] = s_m[i] == -INFINITY ? 0.0f : exp2_fast(s_m[i] - mx);
        sum += s_l[i] * f[i];
    }
    TO* orow = o + (size_t)row * p.width + (size_t)h * D;
    #pragma unroll
    for (int e = 0; e < E; ++e) {
        float x = 0.0f;
        for (int i = 0; i < kRowWaves; ++i)
            x += s_o[i][lane + 64 * e] * f[i];
        orow[lane + 64 * e] = (TO)(sum == 0.0f ? 0.0f : x / sum);
    }
    if (lse && lane == 0)
        lse[(size_t)h * p.batch * p.n_draft + row] = sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * kLn2;
}

template <class T, int D>
void launch(const TreeParams& p, mako_dtype out, void* o, float* lse, hipStream_t s)
{
    const dim3 grid(p.batch * p.n_draft * p.heads), block(kRowWaves * 64);
    if (out == MAKO_F32)
        hipLaunchKernelGGL((tree_rows<T, float, D>), grid, block, 0, s, p, static_cast<float*>(o), lse);
    else
        hipLaunchKernelGGL((tree_rows<T, T, D>), grid, block, 0, s, p, static_cast<T*>(o), lse);
}

template <class T>
void launch_dim(const TreeParams& p, uint32_t dim, mako_dtype out, void* o, float* lse, hipStream_t s)
{
    if (dim == 64)
        launch<T, 64>(p, out, o, lse, s);
    else if (dim == 128)
        launch<T, 128>(p, out, o, lse, s);
    else
        launch<T, 256>(p, out, o, lse, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_args(const mako_tree_args* a, mako_dtype in, mako_dtype out, const void* q, const void* k, const void* v,
               const void* kd, const void* vd, const uint32_t* ctx_len, const uint64_t* mask, const void* o)
{
    const char* what = "attention_tree";
    if (!a || !q || !k || !v || !kd || !vd || !ctx_len || !o)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (a->dim != 64 && a->dim != 128 && a->dim != 256)
        return fail(MAKO_EUNSUPPORTED, "%s: heads of %u (64, 128 or 256)", what, a->dim);
    if (in != MAKO_F16 && in != MAKO_BF16)
        return fail(MAKO_EUNSUPPORTED, "%s: input type %d (f16 or bf16)", what, (int)in);
    if (out != MAKO_F32 && out != in)
        return fail(MAKO_EUNSUPPORTED, "%s: output type %d (f32 or the input's)", what, (int)out);
    if (!a->heads || !a->kv_heads || a->heads % a->kv_heads)
        return fail(MAKO_EINVAL, "%s: %u heads over %u kv heads", what, a->heads, a->kv_heads);
    if (a->n_draft > 64)
        return fail(MAKO_EINVAL, "%s: %u drafts a sequence (at most 64)", what, a->n_draft);
    const uint64_t rows = (uint64_t)a->batch * a->n_draft;
    if (rows > a->q_pad || rows > a->d_pad)
        return fail(MAKO_EINVAL, "%s: %u x %u draft rows in query heads of %u rows and kv heads of %u", what, a->batch,
                    a->n_draft, a->q_pad, a->d_pad);
    if (rows * a->heads > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %llu rows of %u heads exceed the grid", what, (unsigned long long)rows, a->heads);
    if (a->max_ctx > a->cap)
        return fail(MAKO_EINVAL, "%s: max_ctx %u over the cache's %u rows", what, a->max_ctx, a->cap);
    if ((uint64_t)a->cap * a->dim * 2 > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %u cache rows exceed 2 GiB a head", what, a->cap);
    if ((uint64_t)a->batch * a->kv_heads * (a->max_ctx + 64ull) >= (1ull << 32))
        return fail(MAKO_EINVAL, "%s: %u x %u x %u rows exceed 2^32", what, a->batch, a->kv_heads, a->max_ctx);
    if ((uint64_t)a->heads * a->dim > a->width || a->width % 4)
        return fail(MAKO_EINVAL, "%s: o rows of %u for %u heads of %u (a multiple of 4, at least their width)", what,
                    a->width, a->heads, a->dim);
    if (!(a->scale > 0.0f) || a->scale == INFINITY)
        return fail(MAKO_EINVAL, "%s: scale %g (positive and finite)", what, (double)a->scale);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(kd) || !aligned16(vd) || !aligned16(o))
        return fail(MAKO_EINVAL, "%s: q, k, v, kd, vd and o must be 16-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(mask) % 8)
        return fail(MAKO_EINVAL, "%s: mask must be 8-byte aligned", what);
    return MAKO_OK;
}

}  // namespace
}  // namespace mako

using namespace mako;

extern "C" size_t mako_attn_tree_workspace(const mako_tree_args*) { return 0; }

extern "C" int mako_attn_tree(const mako_tree_args* a, mako_dtype in, mako_dtype out, const void* q, const void* k,
                              const void* v, const void* kd, const void* vd, const uint32_t* ctx_len,
                              const uint32_t* n_nodes, const uint64_t* mask, void* o, float* lse, void*, size_t,
                              void* stream)
{
    if (const int rc = check_args(a, in, out, q, k, v, kd, vd, ctx_len, mask, o))
        return rc;
    if (a->batch == 0 || a->n_draft == 0)
        return ok();
    const TreeParams p{q, k, v, kd, vd, ctx_len, n_nodes, mask, a->batch, a->n_draft, a->q_pad, a->d_pad, a->heads,
                       a->kv_heads, a->heads / a->kv_heads, a->cap, a->max_ctx, a->width, a->scale * kLog2e};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (in == MAKO_BF16)
        launch_dim<__bf16>(p, a->dim, out, o, lse, s);
    else
        launch_dim<_Float16>(p, a->dim, out, o, lse, s);
    return check_launch("attention_tree");
}
