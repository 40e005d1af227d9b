// The attention weight that each cache row gathers from queries whose softmax statistics are known.
//
// Mathematics: w_out[j] = decay w[j] + sum over the group's heads h and the queries i that see row j of
//   exp(scale q_i.k_j - lse_i)
// No maximum is needed: lse bounds every score it was summed from.
//
// weights_keys: one thread a key, its row of K in registers eight head dims at a time, every query in turn.
#include "device.hpp"

namespace mako {
namespace {

struct WeightsParams {
    const void *q, *k;
    const float *lse, *w;
    float* w_out;
    const uint32_t *ctx, *path, *n_path;
    uint32_t batch, n_q, heads, kv_heads, group, dim, cap, max_ctx;
    uint64_t qs_b, qs_h;  // q strides (elements) of a sequence and a head
    uint64_t ls_b, ls_h;  // lse strides
    float scale_log2, decay;
};

template <class T>
__global__ __launch_bounds__(256) void weights_keys(const WeightsParams p)
{
    const uint32_t b = blockIdx.x / p.kv_heads, kvh = blockIdx.x % p.kv_heads;
    const uint32_t ctx = min(p.ctx[b], p.max_ctx), n = p.n_path ? min(p.n_path[b], p.n_q) : p.n_q;
    const size_t list = (size_t)b * p.kv_heads + kvh;
    for (uint32_t j = threadIdx.x; j < ctx; j += 256) {
        const T* kr = static_cast<const T*>(p.k) + (list * p.cap + j) * p.dim;
        float sum = 0.0f;
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t r = p.path ? p.path[(size_t)b * p.n_q + i] : i;
            if (r >= p.n_q || (uint64_t)j + n > (uint64_t)ctx + i)
                continue;
            for (uint32_t h = kvh * p.group; h < (kvh + 1) * p.group; ++h) {
                const float l = p.lse[b * p.ls_b + h * p.ls_h + r];
                if (l == -INFINITY)
                    continue;
                const T* qr = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h + (size_t)r * p.dim;
                float s = 0.0f;
                for (uint32_t d = 0; d < p.dim; ++d)
                    s = fmaf((float)qr[d], (float)kr[d], s);
                sum += exp2_fast(fmaf(s, p.scale_log2, -l * kLog2e));
            }
        }
        const size_t at = list * p.cap + j;
        p.w_out[at] = p.w ? fmaf(p.decay, p.w[at], sum) : sum;
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_args(const mako_weights_args* a, mako_dtype in, const void* q, const float* lse, const void* k,
               const uint32_t* ctx_len, const float* w_out)
{
    const char* what = "cache_weights";
    if (!a || !q || !lse || !k || !ctx_len || !w_out)
        return fail(MAKO_EINVAL, "%s: a null argument", what);
    if (a->dim != 64 && a->dim != 128 && a->dim != 256)
        return fail(MAKO_EUNSUPPORTED, "%s: heads of %u (64, 128 or 256)", what, a->dim);
    if (in != MAKO_F16 && in != MAKO_BF16)
        return fail(MAKO_EUNSUPPORTED, "%s: input type %d (f16 or bf16)", what, (int)in);
    if (!a->heads || !a->kv_heads || a->heads % a->kv_heads)
        return fail(MAKO_EINVAL, "%s: %u heads over %u kv heads", what, a->heads, a->kv_heads);
    if (a->q_pad && (uint64_t)a->batch * a->n_q > a->q_pad)
        return fail(MAKO_EINVAL, "%s: %u x %u queries in heads of %u rows", what, a->batch, a->n_q, a->q_pad);
    if (a->max_ctx > a->cap)
        return fail(MAKO_EINVAL, "%s: max_ctx %u over the cache's %u rows", what, a->max_ctx, a->cap);
    if ((uint64_t)a->cap * a->dim * 2 > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %u cache rows exceed 2 GiB a head", what, a->cap);
    if ((uint64_t)a->n_q * a->dim * 2 > 0x7fffffffu)
        return fail(MAKO_EINVAL, "%s: %u queries exceed 2 GiB a head", what, a->n_q);
    if ((uint64_t)a->batch * a->kv_heads * a->max_ctx >= (1ull << 32))
        return fail(MAKO_EINVAL, "%s: %u x %u x %u rows exceed 2^32", what, a->batch, a->kv_heads, a->max_ctx);
    if (!(a->scale > 0.0f) || a->scale == INFINITY)
        return fail(MAKO_EINVAL, "%s: scale %g (positive and finite)", what, (double)a->scale);
    if (!(a->decay >= 0.0f) || a->decay == INFINITY)
        return fail(MAKO_EINVAL, "%s: decay %g (at least 0 and finite)", what, (double)a->decay);
    if (!aligned16(q) || !aligned16(k))
        return fail(MAKO_EINVAL, "%s: q and k must be 16-byte aligned", what);
    return MAKO_OK;
}

}  // namespace
}  // namespace mako

using namespace mako;

extern "C" size_t mako_cache_weights_workspace(const mako_weights_args*) { return 0; }

extern "C" int mako_cache_weights(const mako_weights_args* a, mako_dtype in, const void* q, const float* lse,
                                  const void* k, const uint32_t* ctx_len, const uint32_t* path, const uint32_t* n_path,
                                  const float* w, float* w_out, void*, size_t, void* stream)
{
    if (const int rc = check_args(a, in, q, lse, k, ctx_len, w_out))
        return rc;
    if (a->batch == 0 || a->max_ctx == 0)
        return ok();
    WeightsParams p{q, k, lse, a->decay == 0.0f ? nullptr : w, w_out, ctx_len, path, n_path, a->batch, a->n_q, a->heads,
                    a->kv_heads, a->heads / a->kv_heads, a->dim, a->cap, a->max_ctx, 0, 0, 0, 0, a->scale * kLog2e,
                    a->decay};
    if (a->q_pad) {
        p.qs_b = (uint64_t)a->n_q * a->dim, p.qs_h = (uint64_t)a->q_pad * a->dim;
        p.ls_b = a->n_q, p.ls_h = (uint64_t)a->batch * a->n_q;
    } else {
        p.qs_b = (uint64_t)a->heads * a->n_q * a->dim, p.qs_h = (uint64_t)a->n_q * a->dim;
        p.ls_b = (uint64_t)a->heads * a->n_q, p.ls_h = a->n_q;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(a->batch * a->kv_heads);
    if (in == MAKO_BF16)
        hipLaunchKernelGGL(weights_keys<__bf16>, grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL(weights_keys<_Float16>, grid, dim3(256), 0, s, p);
    return check_launch("cache_weights");
}
