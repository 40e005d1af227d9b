// The calls of TransformerRuntime on a cache kept in pages without a GPU: the C ABI's entry points and the HIP calls under them
// are this program's own (they come before the libraries'), record what they are given and run nothing. With MAKO_REPEAT set,
// the calls that change their own inputs run once; layers and padded tiles are passed on as such.
//   pages_host_cpu
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <string>
#include <vector>

#include "transformer_runtime.hpp"

namespace {
struct Call {
    std::string name;
    mako_pages_args p;
    mako_paged_args a;
    const void *k, *v, *in0, *in1, *in2, *out0, *out1, *out2;
    size_t bytes;
};
std::vector<Call> calls;

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

int mako_attn_paged(const mako_paged_args* a, mako_dtype, mako_dtype, const void* q, const void* k, const void* v,
                    const uint32_t* table, const uint32_t* starts, const uint32_t*, void* o, float* lse, void*, size_t n,
                    void*)
{
    calls.push_back({"attn", {}, *a, k, v, q, table, starts, o, lse, nullptr, n});
    return MAKO_OK;
}
int mako_pages_write(const mako_pages_args* a, const void* kd, const void*, const uint32_t* table, const uint32_t* starts,
                     const uint32_t*, const uint32_t* end, void* k, void* v, void*)
{
    calls.push_back({"write", *a, {}, k, v, kd, table, starts, end, nullptr, nullptr, 0});
    return MAKO_OK;
}
int mako_pages_reserve(const mako_pages_args* a, const uint32_t* table, const uint32_t* refs, const uint32_t*,
                       const uint32_t* ctx, uint32_t* table_out, uint32_t* refs_out, uint32_t* ctx_out, void* k, void* v,
                       void*, size_t n, void*)
{
    calls.push_back({"reserve", *a, {}, k, v, table, refs, ctx, table_out, refs_out, ctx_out, n});
    return MAKO_OK;
}
int mako_pages_fork(const mako_pages_args* a, const uint32_t*, const uint32_t*, const uint32_t* table, const uint32_t* refs,
                    const uint32_t* ctx, uint32_t* table_out, uint32_t* refs_out, uint32_t* ctx_out, void*, size_t n, void*)
{
    calls.push_back({"fork", *a, {}, nullptr, nullptr, table, refs, ctx, table_out, refs_out, ctx_out, n});
    return MAKO_OK;
}
int mako_pages_compact(const mako_pages_args* a, const uint32_t* table, const uint32_t* refs, uint32_t* table_out,
                       uint32_t* refs_out, uint32_t* used_out, uint32_t*, void* k, void* v, void*, size_t n, void*)
{
    calls.push_back({"compact", *a, {}, k, v, table, refs, nullptr, table_out, refs_out, used_out, n});
    return MAKO_OK;
}
}

namespace {

class Harness final : public mako::models::TransformerRuntime {
public:
    Harness() : TransformerRuntime(mako::gpu::Telemetry::off) {}
    using TransformerRuntime::attention_paged;
    using TransformerRuntime::encoder;
    using TransformerRuntime::finish;
    using TransformerRuntime::pages_compact;
    using TransformerRuntime::pages_fork;
    using TransformerRuntime::pages_reserve;
    using TransformerRuntime::pages_write;
    using TransformerRuntime::scratch;
};

template <class F>
bool throws(F f, const char* part)
{
    try {
        f();
    } catch (const std::runtime_error& e) {
        return std::string(e.what()).find(part) != std::string::npos;
    }
    return false;
}

}  // namespace

int main()
{
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    setenv("MAKO_REPEAT", "pages_,attn_paged:3", 1);
    Harness h;
    unsetenv("MAKO_REPEAT");
    constexpr uint32_t B = 3, KV = 2, H = 8, D = 64, L = 3, PAGES = 5, PAGE = 64, MAX = 4;
    constexpr uint64_t kLayer = 2ull * PAGES * KV * PAGE * D;
    auto *k = h.scratch("k", L * kLayer), *v = h.scratch("v", L * kLayer), *x = h.scratch("x", 4096);
    auto *table = h.scratch("table", 64), *refs = h.scratch("refs", 64), *ctx = h.scratch("ctx", 64), *end = h.scratch("end", 64);
    const mako::models::PagedCache c{k, v, table, refs, ctx, B, PAGES, PAGE, MAX, KV, D, L};
    auto* enc = h.encoder();
    h.pages_reserve(enc, c, nullptr, end, 7);
    h.pages_fork(enc, c, nullptr, x);
    h.pages_compact(enc, c, x);
    check(calls.size() == 3, "MAKO_REPEAT: reserve, fork and compact once");
    const auto in_place = [](const Call& r) { return r.in0 == r.out0 && r.in1 == r.out1; };
    check(in_place(calls[0]) && in_place(calls[1]) && in_place(calls[2]) && calls[1].in2 == calls[1].out2 &&
              calls[0].in2 == ctx->ptr && calls[0].out2 == end->ptr,
          "table and refs in place; reserve leaves ctx_len");
    bool enough = true;
    for (const auto& r : calls) {
        const auto query = r.name == "reserve" ? mako_pages_reserve_workspace : r.name == "fork" ? mako_pages_fork_workspace : mako_pages_compact_workspace;
        enough = enough && r.bytes >= query(&r.p) && r.p.layers == L && r.p.pages == PAGES && r.p.max_pages == MAX;
    }
    check(enough, "workspaces of the queries' sizes");

    calls.clear();
    h.pages_write(enc, x, x, c, 1, nullptr, end, 7);
    check(calls.size() == 3 && calls[0].k == static_cast<char*>(k->ptr) + kLayer && calls[2].v == static_cast<char*>(v->ptr) + kLayer &&
              calls[0].p.rows == 7 && calls[0].p.d_pad == 7 && calls[0].out0 == end->ptr,
          "MAKO_REPEAT: write three times, into its layer");
    calls.clear();
    mako::models::AttnOptions opt;
    opt.lse = end;
    h.attention_paged(enc, x, c, 2, table, x, 7, H, 4, 200, opt, 64);
    check(calls.size() == 3 && calls[1].k == static_cast<char*>(k->ptr) + 2 * kLayer && calls[1].a.q_pad == 64 && calls[1].a.rows == 7 &&
              calls[1].a.width == H * D && calls[1].a.max_new == 4 && calls[1].in2 == table->ptr && calls[1].out1 == end->ptr &&
              calls[1].bytes >= mako_attn_paged_workspace(&calls[1].a),
          "MAKO_REPEAT: attention three times, over its layer, with padded queries");
    calls.clear();
    h.pages_write(enc, x, x, c, 0, nullptr, nullptr, 7, 64);
    check(calls[0].p.d_pad == 64 && calls[0].out0 == nullptr, "write: the tiles' padding, no end");
    calls.clear();
    const mako::models::PagedCache small{k, x, table, refs, ctx, B, PAGES, PAGE, MAX, KV, D, L};
    check(throws([&] { h.pages_reserve(enc, c, nullptr, ctx, 7); }, "ctx_len") &&
              throws([&] { h.pages_write(enc, x, x, c, 3, nullptr, end, 7); }, "layer 3 of 3") &&
              throws([&] { h.attention_paged(enc, x, small, 0, nullptr, x, 7, H, 4, 200); }, "layer 0 of 3") &&
              throws([&] { h.pages_compact(enc, small, x); }, "layer 2 of 3") && calls.empty(),
          "refused: ctx_len for end, layers that the pools do not have");
    h.finish(enc);
    std::printf("%s\n", failures ? "FAILED" : "all passed");
    return failures != 0;
}
