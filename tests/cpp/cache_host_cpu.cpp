// The cache calls of TransformerRuntime without a GPU: the C ABI's entry points and the HIP calls under them are this
// program's own (they come before the libraries'), record what they are given and run nothing. With MAKO_REPEAT set, the
// calls that change their own inputs run once; tiles with padded heads are passed on as such.
//   cache_host_cpu
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <string>
#include <vector>

#include "transformer_runtime.hpp"

namespace {
std::vector<mako_tree_args> trees;
std::vector<mako_append_args> appends;
std::vector<mako_weights_args> weighings;
std::vector<mako_evict_args> evictions;

int failures = 0;
void check(bool ok, const char* what)
{
    std::printf("  %s  %s\n", ok ? "ok  " : "FAIL", what);
    failures += !ok;
}
}  // namespace

extern "C" {
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevice(int* d)
{
    *d = 0;
    return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int)
{
    *v = 256;
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned)
{
    *s = nullptr;
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { return posix_memalign(p, 256, n) ? hipErrorOutOfMemory : hipSuccess; }
hipError_t hipFree(void* p)
{
    std::free(p);
    return hipSuccess;
}

int mako_attn_tree(const mako_tree_args* a, mako_dtype, mako_dtype, const void*, const void*, const void*, const void*,
                   const void*, const uint32_t*, const uint32_t*, const uint64_t*, void*, float*, void*, size_t, void*)
{
    trees.push_back(*a);
    return MAKO_OK;
}
int mako_cache_append(const mako_append_args* a, mako_dtype, const void*, const void*, const uint32_t*, const uint32_t*,
                      const uint32_t*, uint32_t*, const uint32_t*, uint32_t*, float*, uint32_t*, void*, void*, void*)
{
    appends.push_back(*a);
    return MAKO_OK;
}
int mako_cache_weights(const mako_weights_args* a, mako_dtype, const void*, const float*, const void*, const uint32_t*,
                       const uint32_t*, const uint32_t*, const float*, float*, void*, size_t, void*)
{
    weighings.push_back(*a);
    return MAKO_OK;
}
int mako_cache_evict(const mako_evict_args* a, mako_dtype, void*, void*, const float*, const uint32_t*, const uint32_t*,
                     const uint32_t*, float*, uint32_t*, uint32_t*, void*, size_t, void*)
{
    evictions.push_back(*a);
    return MAKO_OK;
}
}

namespace {

class Harness final : public mako::models::TransformerRuntime {
public:
    Harness() : TransformerRuntime(mako::gpu::Telemetry::off) {}
    using TransformerRuntime::attention_tree;
    using TransformerRuntime::cache_append;
    using TransformerRuntime::cache_evict;
    using TransformerRuntime::cache_weights;
    using TransformerRuntime::encoder;
    using TransformerRuntime::finish;
    using TransformerRuntime::scratch;
};

constexpr uint32_t B = 2, N = 5, H = 4, KV = 2, CAP = 9000;

void repeated()
{
    setenv("MAKO_REPEAT", "cache_,attn_tree:3", 1);
    Harness h;
    unsetenv("MAKO_REPEAT");
    auto* x = h.scratch("x", 64);
    auto* enc = h.encoder();
    h.attention_tree(enc, x, x, x, x, x, x, nullptr, nullptr, x, B, N, H, KV, CAP, CAP);
    h.cache_append(enc, x, x, nullptr, nullptr, x, x, x, x, x, x, B, N, KV, CAP);
    h.cache_weights(enc, x, x, x, x, nullptr, nullptr, x, B, N, H, KV, CAP, CAP);
    h.cache_evict(enc, x, x, x, x, x, x, B, KV, CAP, CAP, 100, 10, 2);
    h.finish(enc);
    check(trees.size() == 3, "MAKO_REPEAT: attention_tree three times");
    check(appends.size() == 1, "MAKO_REPEAT: cache_append once");
    check(weighings.size() == 1, "MAKO_REPEAT: cache_weights once");
    check(evictions.size() == 1, "MAKO_REPEAT: cache_evict once (a second call would find nothing over the budget)");
}

void padded()
{
    Harness h;
    auto* x = h.scratch("x", 64);
    auto* enc = h.encoder();
    trees.clear(), appends.clear(), weighings.clear();
    h.attention_tree(enc, x, x, x, x, x, x, nullptr, nullptr, x, B, N, H, KV, CAP, CAP, 128, {}, 64, 128);
    h.attention_tree(enc, x, x, x, x, x, x, nullptr, nullptr, x, B, N, H, KV, CAP, CAP);
    check(trees[0].q_pad == 64 && trees[0].d_pad == 128 && trees[1].q_pad == B * N && trees[1].d_pad == B * N,
          "attention_tree: the tiles' padding");
    h.cache_append(enc, x, x, nullptr, nullptr, x, x, x, x, x, x, 1, 100, KV, CAP, 128, MAKO_BF16, 128);
    h.cache_append(enc, x, x, nullptr, nullptr, x, x, x, x, x, x, B, N, KV, CAP);
    check(appends[0].d_pad == 128 && appends[1].d_pad == B * N, "cache_append: the tiles' padding");
    h.cache_weights(enc, x, x, x, x, nullptr, nullptr, x, 1, 100, H, KV, CAP, CAP, 1.0f, false, 128, MAKO_BF16, 128);
    h.cache_weights(enc, x, x, x, x, nullptr, nullptr, x, B, N, H, KV, CAP, CAP);
    h.cache_weights(enc, x, x, x, x, nullptr, nullptr, x, B, 1, H, KV, CAP, CAP, 1.0f, true);
    check(weighings[0].q_pad == 128 && weighings[1].q_pad == B * N && weighings[2].q_pad == 0,
          "cache_weights: the tiles' padding");
    bool refused = false;
    try {
        h.cache_weights(enc, x, x, x, x, nullptr, nullptr, x, B, 1, H, KV, CAP, CAP, 1.0f, true, 128, MAKO_F16, 64);
    } catch (const std::runtime_error&) {
        refused = true;
    }
    check(refused && weighings.size() == 3, "cache_weights refuses padding by sequence");
    h.finish(enc);
}

}  // namespace

int main()
{
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    repeated();
    padded();
    std::printf("%s\n", failures ? "FAILED" : "all passed");
    return failures != 0;
}
