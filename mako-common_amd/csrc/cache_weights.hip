// The attention weight that each cache row gathers from queries whose softmax statistics are known.
//
// Mathematics: w_out[j] = decay w[j] + sum over the group's heads h and the queries i that see row j of
//   exp(scale q_i.k_j - lse_i)
// No maximum is needed: lse bounds every score it was summed from. The scores come from v_mfma_f32_32x32x16; a query that
// adds nothing (past the sequence's, lse = -inf) is a row of zeros with an offset of -inf.
//
// weights_few, up to 64 (query, head of the group) rows a kv head. Bound: the read of K. The rows are the A operand, in
// registers, and 32 keys a tile the B operand: a lane holds one key's scores, so the sum over the rows is lane-local but
// for one exchange of halves. K comes raw by LDS DMA into a ring of each wave's own (chunks XORed by row), w beside it;
// the tiles of all (sequence, kv head) segments, end to end, are cut into equal ranges, one a wave. No wave waits for
// another, and every key's sum is its wave's alone. K by streaming loads: 256 lists of 8192 keys of 128 take 91 us, 5.9 TB/s
// (105 without them).
//
// weights_many, any number of rows. Bound: an exponential a pair beside 2 D operations of its product. A workgroup holds
// 4 x 32 KB keys in registers as the A operand, and the queries come in tiles of 32 through an LDS ring that the four
// waves share: a lane holds one query's scores, so its offset is one register, and the sums stay in registers, a lane's
// queries apart, until the end. Queries are cut into chunks where keys alone leave CUs idle; each chunk's sums go to the
// workspace and weights_join adds them in order. A causal prompt of 4096 tokens, 32 heads of 128 over 8: 87 us with
// the join, 790 TFLOP/s; without the exponentials it would take 79, without the products 68.
#include <algorithm>

#include "lds_tiles.hpp"
#include "split_ranges.hpp"

namespace mako {
namespace {

constexpr int kTK = 32;     // keys, or queries, a tile
// weights_few's most rows: two groups of them fill its registers. The call's us with weights_few and with weights_many, 32
// lists of 16384 keys, 64 rows: heads of 64 23, 37, of 128 32, 48, of 256 58, 81.
constexpr int kFewRows = 64;

struct WeightsParams {
    const void *q, *k;
    const float *lse, *w;
    float* w_out;
    const uint32_t *ctx, *path, *n_path;
    float* part;          // [range + block][keys]: sums of the ranges' share of a key block
    uint32_t* ends;       // [lists][n_blocks][2]: the first and the last range of each block
    uint32_t batch, n_q, heads, kv_heads, group, cap, max_ctx;
    uint32_t n_ranges;    // waves (weights_few), workgroups (weights_many)
    uint32_t n_blocks;    // weights_many: key blocks of max_ctx
    uint64_t qs_b, qs_h;  // q strides (elements) of a sequence and a head
    uint64_t ls_b, ls_h;  // lse strides
    float scale_log2, decay;
};

__device__ __forceinline__ uint32_t ctx_of(const WeightsParams& p, uint32_t b) { return min(p.ctx[b], p.max_ctx); }
__device__ __forceinline__ uint32_t n_of(const WeightsParams& p, uint32_t b)
{
    return p.n_path ? min(p.n_path[b], p.n_q) : p.n_q;
}
struct KeyTiles {
    const WeightsParams& p;
    __device__ __forceinline__ uint32_t operator()(uint32_t i) const { return (ctx_of(p, i) + kTK - 1) / kTK; }
};

// Query i of sequence b: its row of q (n_q: none) for head h, and its offset, lse in base 2 (inf: adds nothing).
__device__ __forceinline__ uint32_t query(const WeightsParams& p, uint32_t b, uint32_t h, uint32_t i, bool has, float& off)
{
    uint32_t r = has ? i : p.n_q;
    if (has && p.path)
        r = p.path[(size_t)b * p.n_q + i];
    off = INFINITY;
    if (r >= p.n_q)
        return p.n_q;
    const float l = p.lse[b * p.ls_b + h * p.ls_h + r];
    if (l == -INFINITY)
        return p.n_q;
    off = l * kLog2e;
    return r;
}

// Four bytes a lane from rsrc + voff to LDS m0 + 4 lane.
__device__ __forceinline__ void dma4_at(uint32_t m0, uint32_t voff, u32x4 rsrc)
{
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(m0), "v"(voff), "s"(rsrc)
                 : "memory", "m0");
#pragma clang diagnostic pop
}

template <int D>
struct Few {
    static constexpr int kWaves = 4;
    static constexpr int kRow = 2 * D, kTile = kTK * kRow, kPieces = kTile / 1024;
    static constexpr int kDepth = D == 64 ? 8 : D == 128 ? 4 : 2;
    static constexpr int kSlot = kTile + 256;  // K, and 64 lanes' weights
    static constexpr int kLds = kWaves * kDepth * kSlot;
};

template <class T, int D, int NCG>
__global__ __launch_bounds__(256, 1) void weights_few(const WeightsParams p)
{
    using S = Few<D>;
    using E = Elem<T>;
    using V8 = typename E::vec8;
    constexpr int NK = D / 16, kRow = S::kRow;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[S::kLds];
    __shared__ __attribute__((aligned(16))) float s_off[S::kWaves][32 * NCG];
    __shared__ __attribute__((aligned(16))) uint32_t s_lim[S::kWaves][32 * NCG];
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c32 = lane & 31, wl = uniform(tid >> 6);
    const Place at = place_of(p.batch, p.kv_heads, blockIdx.x * S::kWaves + wl, p.n_ranges, lane, KeyTiles{p});
    if (at.x0 == at.x1)
        return;
    uint32_t b = at.b, len = at.len, kvh = (at.x0 - at.first) / len, t0 = (at.x0 - at.first) % len, left = at.x1 - at.x0;

    uint32_t kd[S::kPieces];
    #pragma unroll
    for (int m = 0; m < S::kPieces; ++m) {
        const uint32_t at = 1024 * m + 16 * lane, r = at / kRow, pos = at % kRow;
        kd[m] = r * kRow + 16 * ((pos / 16) ^ k_xor<D>(r));
    }
    const uint32_t lbase = uniform((uint32_t)reinterpret_cast<uintptr_t>(lds)) + wl * S::kDepth * S::kSlot;
    unsigned char* ring = lds + wl * S::kDepth * S::kSlot;
    const uint32_t ka = c32 * kRow + 16 * (g ^ k_xor<D>(c32));

    for (;;) {
        const uint32_t ctx = uniform(ctx_of(p, b)), n = uniform(n_of(p, b)), t1 = min(len, t0 + left);
        const size_t list = (size_t)b * p.kv_heads + kvh;
        const u32x4 krs = tile_rsrc(static_cast<const T*>(p.k) + list * p.cap * D, ctx * kRow);
        const u32x4 wrs = tile_rsrc(p.w + list * p.cap, p.w ? ctx * 4 : 0u);
        auto stage = [&](uint32_t t) __attribute__((always_inline)) {
            const uint32_t dst = lbase + t % S::kDepth * S::kSlot;
            #pragma unroll
            for (int m = 0; m < S::kPieces; ++m)
                dma16_nt(dst + 1024 * m, kd[m] + t * S::kTile, krs);
            dma4_at(dst + S::kTile, (t * kTK + c32) * 4, wrs);
        };
        // The rows: lane l looks up row l's offset and how many keys it sees; the A operand holds row c32 of each group.
        V8 qreg[NCG][NK];
        #pragma unroll
        for (int cg = 0; cg < NCG; ++cg) {
            const uint32_t row = 32 * cg + c32, i = row / p.group, h = kvh * p.group + row % p.group;
            float off;
            const uint32_t r = query(p, b, h, i, i < n, off);
            const T* src = static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h + (size_t)r * D + 8 * g;
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                qreg[cg][kk] = r < p.n_q ? *reinterpret_cast<const V8*>(src + 16 * kk) : V8{};
            s_off[wl][row] = off;
            s_lim[wl][row] = r < p.n_q && ctx + i >= n ? ctx + i - n + 1 : 0u;
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                settle(qreg[cg][kk]);
        }
        for (uint32_t t = t0; t < min(t1, t0 + S::kDepth - 1); ++t)
            stage(t);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        f32x4 off[NCG][4];
        #pragma unroll
        for (int cg = 0; cg < NCG; ++cg)
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                off[cg][i] = *reinterpret_cast<const f32x4*>(&s_off[wl][32 * cg + 8 * i + 4 * g]);
        for (uint32_t t = t0; t < t1; ++t) {
            if (t + S::kDepth - 1 <= t1)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::kDepth - 2) * (S::kPieces + 1)) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            if (t + S::kDepth - 1 < t1)
                stage(t + S::kDepth - 1);
            const unsigned char* tile = ring + t % S::kDepth * S::kSlot;
            const uint32_t j = t * kTK + c32;
            bool masked = (t + 1) * kTK + n > ctx + 1;  // some row does not see all of the tile
            f32x16 x[NCG];
            #pragma unroll
            for (int cg = 0; cg < NCG; ++cg)
                x[cg] = f32x16{};
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                const V8 kf = *reinterpret_cast<const V8*>(tile + (ka ^ (32 * kk)));
                #pragma unroll
                for (int cg = 0; cg < NCG; ++cg)
                    x[cg] = E::mfma32(qreg[cg][kk], kf, x[cg]);
            }
            const float w = *reinterpret_cast<const float*>(tile + S::kTile + 4 * c32);
            // Register i: row 8 (i / 4) + 4 g + i % 4. A key that is not finite gives NaN against the rows that are no
            // query too: then those are masked.
            float sum;
            for (;;) {
                sum = 0.0f;
                #pragma unroll
                for (int cg = 0; cg < NCG; ++cg)
                    #pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        f32x4 e;
                        #pragma unroll
                        for (int i = 0; i < 4; ++i)
                            e[i] = exp2_fast(fmaf(x[cg][4 * i4 + i], p.scale_log2, -off[cg][i4][i]));
                        if (masked) {
                            const u32x4 lim = *reinterpret_cast<const u32x4*>(&s_lim[wl][32 * cg + 8 * i4 + 4 * g]);
                            #pragma unroll
                            for (int i = 0; i < 4; ++i)
                                e[i] = j < lim[i] ? e[i] : 0.0f;
                        }
                        sum += (e[0] + e[1]) + (e[2] + e[3]);
                    }
                if (masked || !__any(sum != sum))
                    break;
                masked = true;
            }
            sum = pair_sum(sum);
            if (g == 0 && j < ctx)
                p.w_out[list * p.cap + j] = p.w ? fmaf(p.decay, w, sum) : sum;
        }
        left -= t1 - t0;
        if (left == 0)
            return;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        t0 = 0;
        if (++kvh == p.kv_heads) {
            kvh = 0;
            do {
                if (++b >= p.batch)
                    return;
                len = uniform(KeyTiles{p}(b));
            } while (len == 0);
        }
    }
}

template <int D>
struct Many {
    static constexpr int kKB = D == 256 ? 1 : 2;             // blocks of 32 keys a wave
    static constexpr int kKeys = 4 * 32 * kKB;               // keys a workgroup
    static constexpr int kRow = 2 * D, kTile = kTK * kRow;   // a tile of queries
    static constexpr int kPieces = kTile / 1024 / 4;         // 1 KiB pieces of it a wave
    static constexpr int kStep = D == 256 ? 2 : 4;           // tiles a step: a barrier and a ring slot of two
    static constexpr int kTable = 1024;                      // rows of a path looked up at a time
};

// The query tiles of a list's key blocks. Block i's keys start at i keys; the first query that sees them is the (i keys -
// (ctx - n))-th, in tile i per - a, so block i has count - max(0, i per - a) tiles a head, at least one where n > 0.
struct BlockTiles {
    int per, a, count, group;  // 32-key tiles a block; ctx - n in tiles, rounded up; tiles of n; heads
    uint32_t blocks;
    __device__ __forceinline__ BlockTiles(const WeightsParams& p, uint32_t b, uint32_t keys)
    {
        const uint32_t ctx = ctx_of(p, b), n = n_of(p, b);
        per = keys / kTK;
        a = ctx >= n ? (int)((ctx - n + kTK - 1) / kTK) : -(int)((n - ctx) / kTK);
        count = (n + kTK - 1) / kTK;
        group = p.group;
        blocks = n ? (ctx + keys - 1) / keys : 0u;
    }
    __device__ __forceinline__ uint32_t first_tile(uint32_t i) const { return max(0, (int)i * per - a); }
    __device__ __forceinline__ uint32_t tiles(uint32_t i) const { return count - first_tile(i); }  // of a head
    // The tiles of blocks [0, i), over the heads.
    __device__ __forceinline__ uint32_t before(uint32_t i) const
    {
        const uint32_t i0 = a < 0 ? 0u : min(i, (uint32_t)(a / per) + 1);  // blocks below see every query's tile
        const uint32_t m = i - i0;
        // i0 per - a, then per more each
        return group * (i * count - m * (uint32_t)((int)i0 * per - a) - per * (m * (m - 1) / 2));
    }
    __device__ __forceinline__ uint32_t total() const { return before(blocks); }
    // The block that holds tile x of them.
    __device__ __forceinline__ uint32_t of(uint32_t x) const
    {
        uint32_t lo = 0, hi = blocks;  // before(lo) <= x < before(hi)
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            (before(mid) <= x ? lo : hi) = mid;
        }
        return lo;
    }
};
struct ListTiles {
    const WeightsParams& p;
    uint32_t keys;
    __device__ __forceinline__ uint32_t operator()(uint32_t i) const { return BlockTiles(p, i, keys).total(); }
};

template <class T, int D, bool PATH>
__global__ __launch_bounds__(256, 2) void weights_many(const WeightsParams p)
{
    using S = Many<D>;
    using E = Elem<T>;
    using V8 = typename E::vec8;
    constexpr int NK = D / 16, kRow = S::kRow, KB = S::kKB;
    constexpr int kKPieces = KB * 32 * kRow / 1024;  // 1 KiB pieces of a wave's keys
    static_assert(4 * kKPieces * 1024 <= 2 * S::kStep * S::kTile, "the keys pass through the ring");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * S::kStep * S::kTile];
    // lse of the ring's tiles (64 words each, the DMA's), or with a path the offsets and places of kTable rows
    __shared__ float s_off[PATH ? 2 * S::kTable : 2 * S::kStep * 64];
    uint32_t* const s_row = reinterpret_cast<uint32_t*>(s_off) + (PATH ? S::kTable : 0);
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c32 = lane & 31, wl = uniform(tid >> 6);
    // An XCD's workgroups take neighbouring ranges: they share queries and keys in its L2.
    const uint32_t per_xcd = (p.n_ranges + 7) / 8, range = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    const Place at = place_of(p.batch, p.kv_heads, range, p.n_ranges, lane, ListTiles{p, S::kKeys});
    if (at.x0 == at.x1)
        return;
    uint32_t left = at.x1 - at.x0, b = at.b, kvh = (at.x0 - at.first) / at.len, block, tb;  // tiles from tb of the block on
    {
        const BlockTiles bt(p, b, S::kKeys);
        const uint32_t x = (at.x0 - at.first) % at.len;
        block = uniform(bt.of(x));
        tb = x - uniform(bt.before(block));
    }

    uint32_t qr[S::kPieces], qc[S::kPieces];  // the row and byte of a tile that the lane's 16 LDS bytes hold
    #pragma unroll
    for (int m = 0; m < S::kPieces; ++m) {
        const uint32_t at = 1024 * (wl * S::kPieces + m) + 16 * lane, pos = at % kRow;
        qr[m] = at / kRow;
        qc[m] = 16 * ((pos / 16) ^ k_xor<D>(qr[m]));
    }
    const uint32_t lbase = uniform((uint32_t)reinterpret_cast<uintptr_t>(lds));
    const uint32_t obase = uniform((uint32_t)reinterpret_cast<uintptr_t>(s_off));
    const uint32_t qa = c32 * kRow + 16 * (g ^ k_xor<D>(c32));
    for (;;) {
        const BlockTiles bt(p, b, S::kKeys);
        const uint32_t ctx = uniform(ctx_of(p, b)), n = uniform(n_of(p, b)), list = b * p.kv_heads + kvh;
        const uint32_t nt = uniform(bt.tiles(block)), ia = uniform(bt.first_tile(block)) * kTK, all = nt * p.group;
        const uint32_t t_end = min(all, tb + left), kw = block * S::kKeys + wl * 32 * KB;  // the wave's first key
        const bool whole = tb == 0 && t_end == all;
        left -= t_end - tb;
        // The wave's keys, through its part of the ring.
        {
            const u32x4 rs = tile_rsrc(static_cast<const T*>(p.k) + (size_t)list * p.cap * D, ctx * kRow);
            #pragma unroll
            for (int m = 0; m < kKPieces; ++m) {
                const uint32_t at = 1024 * m + 16 * lane, r = at / kRow, pos = at % kRow;
                dma16_at(lbase + 1024 * (wl * kKPieces + m), (kw + r) * kRow + 16 * ((pos / 16) ^ k_xor<D>(r)), 0, rs);
            }
        }
        if (tid == 0) {
            uint32_t* ends = p.ends + 2 * ((size_t)list * p.n_blocks + block);
            if (tb == 0)
                ends[0] = range;
            if (t_end == all)
                ends[1] = range;
        }
        float acc[KB][16];  // (scalars: 16-register tuples would be copied where the loop's branches meet)
        #pragma unroll
        for (int i = 0; i < KB; ++i)
            #pragma unroll
            for (int y = 0; y < 16; ++y)
                acc[i][y] = 0.0f;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        V8 kreg[KB][NK];
        #pragma unroll
        for (int i = 0; i < KB; ++i)
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                kreg[i][kk] = *reinterpret_cast<const V8*>(lds + 1024 * wl * kKPieces + 32 * i * kRow + (qa ^ (32 * kk)));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        while (tb < t_end) {
            const uint32_t te = PATH ? min(t_end, tb + S::kTable / kTK) : t_end;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the ring and the tables are free
            if (PATH) {
                for (uint32_t x = tid; x < (te - tb) * kTK; x += 256) {
                    const uint32_t t = tb + x / kTK, h = kvh * p.group + t / nt, i = ia + t % nt * kTK + x % kTK;
                    float off;
                    const uint32_t r = query(p, b, h, i, i < n, off);
                    s_off[x] = off;
                    s_row[x] = r * kRow;  // (n_q: past the descriptor, zeros)
                }
                __syncthreads();
            }
            // Tile t's head and place in it, as t goes on.
            uint32_t sh = uniform(tb / nt), st = uniform(tb % nt), ct = st;
            u32x4 qrs, lrs;
            auto head = [&]() __attribute__((always_inline)) {
                const uint64_t h = kvh * p.group + sh;
                qrs = tile_rsrc(static_cast<const T*>(p.q) + b * p.qs_b + h * p.qs_h, p.n_q * kRow);
                lrs = tile_rsrc(p.lse + b * p.ls_b + h * p.ls_h, p.n_q * 4);
            };
            head();
            // The step from tile t on (the steps start at tb). Without a path, rows past the last query are another's, or past
            // the descriptor: masked.
            auto stage = [&](uint32_t t) __attribute__((always_inline)) {
                const uint32_t slot = ((t - tb) / S::kStep & 1) * S::kStep;
                #pragma unroll
                for (int i = 0; i < S::kStep; ++i) {
                    if (t + i >= te)
                        break;
                    const uint32_t dst = lbase + (slot + i) * S::kTile + 1024 * wl * S::kPieces;
                    #pragma unroll
                    for (int m = 0; m < S::kPieces; ++m) {
                        const uint32_t at = PATH ? s_row[(t + i - tb) * kTK + qr[m]] : (ia + st * kTK + qr[m]) * kRow;
                        dma16_at(dst + 1024 * m, at + qc[m], 0, qrs);
                    }
                    if (!PATH && wl == i % 4)
                        dma4_at(obase + (slot + i) * 256, (ia + st * kTK + c32) * 4, lrs);
                    if (++st == nt) {
                        st = 0;
                        ++sh;
                        head();
                    }
                }
            };
            stage(tb);
            for (uint32_t t0 = tb; t0 < te; t0 += S::kStep) {
                // The step has landed, and every wave is done with the one before, whose slot takes the next.
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (t0 + S::kStep < te)
                    stage(t0 + S::kStep);
                const uint32_t slot = ((t0 - tb) / S::kStep & 1) * S::kStep, t1 = min(te, t0 + S::kStep);
                // A tile's operands are read a tile ahead, beside the exponentials of the one before.
                V8 qf[NK];
                float off_next;
                auto read = [&](uint32_t t) __attribute__((always_inline)) {
                    off_next = PATH ? s_off[(t - tb) * kTK + c32] : s_off[(slot + t - t0) * 64 + c32];
                    #pragma unroll
                    for (int kk = 0; kk < NK; ++kk)
                        qf[kk] = *reinterpret_cast<const V8*>(lds + (slot + t - t0) * S::kTile + (qa ^ (32 * kk)));
                };
                read(t0);
                #pragma unroll 1
                for (uint32_t t = t0; t < t1; ++t) {
                    const uint32_t i0 = ia + ct * kTK;
                    if (++ct == nt)
                        ct = 0;
                    // No query: -inf as lse, or past the last. (With 0 for a row, against a key that is not finite, NaN: masked.)
                    const bool none = PATH ? off_next == INFINITY : off_next == -INFINITY || i0 + c32 >= n;
                    const float off = PATH ? off_next : off_next * kLog2e;
                    f32x16 x[KB];
                    #pragma unroll
                    for (int i = 0; i < KB; ++i)
                        x[i] = f32x16{};
                    #pragma unroll
                    for (int kk = 0; kk < NK; ++kk)
                        #pragma unroll
                        for (int i = 0; i < KB; ++i)
                            x[i] = E::mfma32(kreg[i][kk], qf[kk], x[i]);
                    __builtin_amdgcn_sched_barrier(0);
                    read(min(t + 1, t1 - 1));
                    __builtin_amdgcn_sched_barrier(0);
                    const bool some = __any(none);
                    #pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        // The first query sees `seen` of the block's keys, the last 31 more.
                        const int seen = (int)(ctx + i0 + 1) - (int)(n + kw + 32 * i);
                        if (seen + 31 <= 0)
                            continue;
                        if (seen >= 32 && !some) {
                            #pragma unroll
                            for (int y = 0; y < 16; ++y)
                                acc[i][y] += exp2_fast(fmaf(x[i][y], p.scale_log2, -off));
                        } else {
                            const int lim = none ? -1 : seen + (int)c32 - 4 * (int)g;
                            #pragma unroll
                            for (int y = 0; y < 16; ++y) {
                                const float e = exp2_fast(fmaf(x[i][y], p.scale_log2, -off));
                                acc[i][y] += 8 * (y >> 2) + (y & 3) < lim ? e : 0.0f;
                            }
                        }
                    }
                }
            }
            tb = te;
        }
        // A key's sum over the 32 lanes of its half: halving exchanges, 16 registers to 1. Lane bit s picks register bit s,
        // so lane (g, c32) ends with register c32 % 16 summed over all lanes but bit 4, which the last one adds.
        #pragma unroll
        for (int i = 0; i < KB; ++i) {
            #pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bool up = lane >> s & 1;
                #pragma unroll
                for (int y = 0; y < 8 >> s; ++y) {
                    const float keep = up ? acc[i][2 * y + 1] : acc[i][2 * y];
                    const float give = up ? acc[i][2 * y] : acc[i][2 * y + 1];
                    acc[i][y] = keep + __shfl_xor(give, 1 << s);
                }
            }
            const float sum = acc[i][0] + __shfl_xor(acc[i][0], 16);
            const uint32_t y = c32 & 15, j = kw + 32 * i + 8 * (y >> 2) + 4 * g + (y & 3);
            if (c32 < 16 && j < ctx) {
                const size_t at = (size_t)list * p.cap + j;
                if (whole)
                    p.w_out[at] = p.w ? fmaf(p.decay, p.w[at], sum) : sum;
                else
                    p.part[((size_t)range + (size_t)list * p.n_blocks + block) * S::kKeys + j % S::kKeys] = sum;
            }
        }
        if (left == 0)
            return;
        __syncthreads();  // the ring is free
        tb = 0;
        if (++block == bt.blocks) {
            block = 0;
            if (++kvh == p.kv_heads) {
                kvh = 0;
                do {
                    if (++b >= p.batch)
                        return;
                } while (uniform(BlockTiles(p, b, S::kKeys).blocks) == 0);
            }
        }
    }
}

// The blocks that more than one range met: their sums, in order (one range: weights_many wrote the result; no query at all:
// the old weights).
__global__ __launch_bounds__(256) void weights_join(const WeightsParams p, uint32_t keys, uint32_t per_list)
{
    const uint32_t list = blockIdx.x / per_list, b = list / p.kv_heads;
    const uint32_t ctx = ctx_of(p, b), j = blockIdx.x % per_list * 256 + threadIdx.x;
    if (j >= ctx)
        return;
    const size_t at = (size_t)list * p.cap + j, block = (size_t)list * p.n_blocks + j / keys;
    float sum = 0.0f;
    if (n_of(p, b)) {
        const uint32_t r0 = p.ends[2 * block], r1 = p.ends[2 * block + 1];
        if (r0 == r1)
            return;
        for (uint32_t r = r0; r <= r1; ++r)
            sum += p.part[(r + block) * keys + j % keys];
    }
    p.w_out[at] = p.w ? fmaf(p.decay, p.w[at], sum) : sum;
}

// A call's shape, from its sizes alone. Ranges: a wave each of one workgroup a CU (weights_few; twice as many waves: 108 for
// 107 us at 256 lists of 8192, 20.9 for 18.1 at 8 of 32768), two workgroups a CU (weights_many; us with one, two and four a
// CU: 120, 88, 92 for the prompt above; 38, 31, 33 for two of 1000 queries over 3000 keys of 64).
struct Plan {
    bool few;
    uint32_t keys, n_blocks, n_ranges;
};

Plan plan_of(const mako_weights_args* a, uint32_t cus)
{
    const uint64_t rows = (uint64_t)a->n_q * (a->heads / a->kv_heads);
    Plan pl{rows <= kFewRows, 0, 0, 4 * cus};
    if (pl.few)
        return pl;
    pl.keys = a->dim == 256 ? Many<256>::kKeys : Many<128>::kKeys;
    pl.n_blocks = (a->max_ctx + pl.keys - 1) / pl.keys;
    pl.n_ranges = 2 * cus;
    return pl;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// The ranges' ends of the blocks, then the shares.
size_t ends_bytes(const Plan& pl, const mako_weights_args* a)
{
    return round256((size_t)a->batch * a->kv_heads * pl.n_blocks * 2 * sizeof(uint32_t));
}
size_t workspace_for(const Plan& pl, const mako_weights_args* a)
{
    if (pl.few)
        return 0;
    return ends_bytes(pl, a) + (pl.n_ranges + (size_t)a->batch * a->kv_heads * pl.n_blocks) * pl.keys * sizeof(float);
}

template <class T, int D>
void launch(const WeightsParams& p, const Plan& pl, hipStream_t s)
{
    if (pl.few) {
        const dim3 grid(p.n_ranges / Few<D>::kWaves);
        if (p.n_q * p.group <= 32)
            hipLaunchKernelGGL((weights_few<T, D, 1>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((weights_few<T, D, 2>), grid, dim3(256), 0, s, p);
        return;
    }
    const dim3 grid((p.n_ranges + 7) / 8 * 8);
    if (p.path)
        hipLaunchKernelGGL((weights_many<T, D, true>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((weights_many<T, D, false>), grid, dim3(256), 0, s, p);
    const uint32_t per_list = (p.max_ctx + 255) / 256;
    hipLaunchKernelGGL(weights_join, dim3(p.batch * p.kv_heads * per_list), dim3(256), 0, s, p, pl.keys, per_list);
}

template <class T>
void launch_dim(const WeightsParams& p, uint32_t dim, const Plan& pl, hipStream_t s)
{
    if (dim == 64)
        launch<T, 64>(p, pl, s);
    else if (dim == 128)
        launch<T, 128>(p, pl, s);
    else
        launch<T, 256>(p, pl, s);
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

extern "C" size_t mako_cache_weights_workspace(const mako_weights_args* a)
{
    const uint32_t cus = device_cus();
    if (!a || !cus || !a->heads || !a->kv_heads || a->heads % a->kv_heads || !a->batch || !a->max_ctx)
        return 0;
    return workspace_for(plan_of(a, cus), a);
}

extern "C" int mako_cache_weights(const mako_weights_args* a, mako_dtype in, const void* q, const float* lse,
                                  const void* k, const uint32_t* ctx_len, const uint32_t* path, const uint32_t* n_path,
                                  const float* w, float* w_out, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* what = "cache_weights";
    if (const int rc = check_args(a, in, q, lse, k, ctx_len, w_out))
        return rc;
    if (a->batch == 0 || a->max_ctx == 0)
        return ok();
    const uint32_t cus = device_cus();
    if (!cus)
        return fail(MAKO_EHIP, "%s: no device to size the split for", what);
    const Plan pl = plan_of(a, cus);
    const size_t need = workspace_for(pl, a);
    if (workspace_bytes < need || (need && !workspace) || reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail(MAKO_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, workspace_bytes,
                    need);
    // (the query tiles of all key blocks, counted in 32 bits)
    if (!pl.few && (uint64_t)a->batch * a->heads * pl.n_blocks * ((a->n_q + kTK - 1) / kTK) >= (1ull << 32))
        return fail(MAKO_EINVAL, "%s: %u x %u heads of %u queries over %u rows exceed 2^32 tiles", what, a->batch, a->heads,
                    a->n_q, a->max_ctx);
    if (!pl.few && !grid_fits((uint64_t)a->batch * a->kv_heads * ((a->max_ctx + 255) / 256), 256))
        return fail(MAKO_EINVAL, "%s: %u x %u lists of %u rows exceed the grid", what, a->batch, a->kv_heads, a->max_ctx);
    WeightsParams p{q, k, lse, a->decay == 0.0f ? nullptr : w, w_out, ctx_len, path, n_path,
                    need ? reinterpret_cast<float*>(static_cast<char*>(workspace) + ends_bytes(pl, a)) : nullptr,
                    static_cast<uint32_t*>(workspace), a->batch, a->n_q, a->heads, a->kv_heads, a->heads / a->kv_heads,
                    a->cap, a->max_ctx, pl.n_ranges, pl.n_blocks, 0, 0, 0, 0, a->scale * kLog2e, a->decay};
    if (a->q_pad) {
        p.qs_b = (uint64_t)a->n_q * a->dim, p.qs_h = (uint64_t)a->q_pad * a->dim;
        p.ls_b = a->n_q, p.ls_h = (uint64_t)a->batch * a->n_q;
    } else {
        p.qs_b = (uint64_t)a->heads * a->n_q * a->dim, p.qs_h = (uint64_t)a->n_q * a->dim;
        p.ls_b = (uint64_t)a->heads * a->n_q, p.ls_h = a->n_q;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (in == MAKO_BF16)
        launch_dim<__bf16>(p, a->dim, pl, s);
    else
        launch_dim<_Float16>(p, a->dim, pl, s);
    return check_launch(what);
}
