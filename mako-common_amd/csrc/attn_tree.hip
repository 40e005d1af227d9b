// Attention of drafted tokens over a cache: each sequence's n_draft rows, the nodes of a tree of drafts, attend its cache
// rows [0, ctx) and the drafts that their mask bits name, in one call for the whole batch.
//
// Mathematics: row r of sequence b, head h, with S the cache rows below ctx[b] and the drafts j < n_nodes[b] that r sees:
//   o = sum_{j in S} exp(s_j - m) v_j / sum_{j in S} exp(s_j - m),  s_j = scale q.k_j,  lse = m + ln(sum),  m any bound
// Sums over parts of S join by their maxima, so the keys are split over workgroups.
//
// Bound: the read of K and V, once for all the rows and heads that share a kv head: the (row, head of the group) pairs
// are the columns of S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16, 32 a wave. Past a few hundred columns the
// matrix products bind.
//
// * A tile is 32 keys: of the cache, or of the drafts, whose tiles follow the cache's. A workgroup is NG column groups
//   times KW key ways: wave w takes columns 32 (w % NG) .. and every KW-th tile; the NG waves of a way share its tiles,
//   each staging 1 / NG of them. A step is KW tiles. More columns than 32 NG go to further workgroups (column blocks) on
//   the same keys, next to each other on an XCD so that the second read hits its L2.
// * Tiles come raw by LDS DMA into a ring of DEPTH steps, DEPTH - 1 of them in flight; one barrier a step (none with one
//   column group, whose waves share nothing). K rows lie in slot order (bits 2 and 3 of the row swapped: the
//   exponentiated scores are then the B operand of the P V product) with their 16-byte chunks XORed by the row, V rows
//   with their 32-byte units permuted; V^T comes from transpose reads. Rows past the context or the tree lie outside the
//   buffer descriptors and load zeros.
// * Each row's mask word masks the draft tiles alone. Infinities and NaN of a draft's V must not reach the rows that do
//   not see it (0 times them is NaN): a draft tile's are zeroed in LDS, and added to the rows that do at the end.
// * The steps of all (sequence, kv head) segments, end to end, are cut into equal ranges, one a workgroup. Each overlap of
//   a range and a segment is a piece; its ways join through LDS and leave one f32 partial a column at index range +
//   segment (unique: pieces are intervals between consecutive boundaries), which tree_merge joins. Short contexts take a
//   segment a workgroup and no merge.
#include <algorithm>
#include <type_traits>

#include "lds_tiles.hpp"
#include "split_ranges.hpp"

namespace mako {
namespace {

constexpr int kTK = 32;  // keys a tile
constexpr float kRescale = 8.0f;

struct TreeParams {
    const void *q, *k, *v, *kd, *vd;
    const uint32_t *ctx, *nodes;
    const uint64_t* mask;
    float* part_o;   // [pieces][nc][D]
    float* part_ml;  // [pieces][nc][2]: maximum (base 2), sum
    uint32_t* part_odd;  // [pieces]: a draft's V holds what is not finite
    uint32_t* seg_ends;  // [segments][2]: the first and the last range of each
    uint32_t batch, n_draft, q_pad, d_pad, heads, kv_heads, group, cap, max_ctx, width;
    uint32_t nc, ncb;   // columns (n_draft x group), column blocks
    uint32_t ways;      // tiles a step
    uint32_t n_ranges;  // 0: a segment a workgroup
    float scale_log2;
};

__device__ __forceinline__ uint32_t ctx_of(const TreeParams& p, uint32_t b) { return min(p.ctx[b], p.max_ctx); }
__device__ __forceinline__ uint32_t nodes_of(const TreeParams& p, uint32_t b)
{
    return p.nodes ? min(p.nodes[b], p.n_draft) : p.n_draft;
}
// The drafts that node r of a tree of `nodes` sees.
__device__ __forceinline__ uint64_t sees_of(const TreeParams& p, uint32_t b, uint32_t r, uint32_t nodes)
{
    return (p.mask ? p.mask[(size_t)b * p.n_draft + r] : (2ull << r) - 1) & (~0ull >> (64 - nodes));
}
__device__ __forceinline__ uint32_t steps_of(const TreeParams& p, uint32_t ctx, uint32_t nodes)
{
    return ((ctx + kTK - 1) / kTK + (nodes + kTK - 1) / kTK + p.ways - 1) / p.ways;
}

// The units of a segment of sequence i: its steps, and lead_of more in front of them for what a piece costs beside its
// steps, so that ranges that meet two segments get fewer (heads of 128, 256 lists of 4096 keys: 94 us with 0 of them, 90
// with 3, 89.6 with 6, 90 with 10; 40 lists of 5000: 37.1, 34.0, 33.2, 33.8. Heads of 256, 4 x 64 drafts, 16 heads over 2,
// 8700 to 13600 keys: 95 with 10, 90 with 13, as a piece writes 128 columns of 256; trees of fewer columns, whose pieces
// write less, have the same weight and were not timed with another).
constexpr uint32_t lead_of(int dim) { return dim == 256 ? 13 : 6; }
template <int D>
struct SegUnits {
    const TreeParams& p;
    __device__ __forceinline__ uint32_t operator()(uint32_t i) const
    {
        const uint32_t steps = steps_of(p, ctx_of(p, i), nodes_of(p, i));
        return steps ? steps + lead_of(D) : 0u;
    }
};

// The key in slot s of a tile's K image (its own inverse).
__device__ __forceinline__ uint32_t slot_of(uint32_t s) { return (s & ~12u) | ((s & 4u) << 1) | ((s & 8u) >> 1); }

// Where 32-byte unit u of V row k sits in its LDS row: the two units of the four rows that a transpose read's 32 lanes
// address cover the 64 banks once (a bijection of the units; its own inverse up to the parity term).
template <int D>
__device__ __forceinline__ uint32_t v_unit(uint32_t u, uint32_t k)
{
    return D == 64 ? u ^ (k & 2u) : u ^ (k & 3u) ^ (4u * (u & 1u));
}
template <int D>
__device__ __forceinline__ uint32_t v_unit_at(uint32_t pos, uint32_t k)
{
    if (D == 64)
        return pos ^ (k & 2u);
    const uint32_t x = pos ^ (k & 3u);
    return x ^ (4u * (x & 1u));
}

// The exponent bits of a value of T: all set in an infinity or NaN.
template <class T>
constexpr uint32_t kExp = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;

// What the drafts' infinities and NaN add to head dim d of row r: p v is v for p > 0.
template <class T, int D>
__device__ float odd_sum(const TreeParams& p, uint32_t b, uint32_t kvh, uint32_t r, uint32_t nodes, uint32_t d)
{
    const uint64_t sees = sees_of(p, b, r, nodes);
    const T* v = static_cast<const T*>(p.vd) + ((size_t)kvh * p.d_pad + (size_t)b * p.n_draft) * D + d;
    float x = 0.0f;
    for (uint32_t j = 0; j < nodes; ++j) {
        const T y = v[(size_t)j * D];
        if (sees >> j & 1 && (__builtin_bit_cast(uint16_t, y) & kExp<T>) == kExp<T>)
            x += (float)y;
    }
    return x;
}

// Waves, ways and ring depth by head dims and column groups: at most 128 KiB of tiles, one workgroup a CU.
template <int D, int NG>
struct Shape {
    static constexpr int kSlot = 2 * kTK * 2 * D;  // a tile's K and V
    static constexpr int kKW = D == 64 ? (NG == 1 ? 8 : NG == 2 ? 4 : 2) : D == 128 ? (NG == 4 ? 2 : 4) : NG == 4 ? 1 : 2;
    static constexpr int kDepth = 128 * 1024 / (kSlot * kKW);
    static constexpr int kWaves = NG * kKW;
    static constexpr int kLds = kDepth * kKW * kSlot;
    static_assert(kDepth >= 2 && kLds >= kWaves * 32 * D * 4, "a ring of two steps, and room for the waves' sums");
};

// Zeros the infinities and NaN of a V image of `bytes` in LDS (waves that share the tile may do so side by side: they
// write the same); whether the wave found one.
template <class T, int bytes>
__device__ __forceinline__ bool finite_only(unsigned char* v, uint32_t lane)
{
    constexpr uint32_t e = kExp<T>;
    bool found = false;
    #pragma unroll 1
    for (int i = 0; i < bytes; i += 1024) {
        u32x4* at = reinterpret_cast<u32x4*>(v + i + 16 * lane);
        u32x4 x = *at;
        bool hit = false;
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool lo = (x[j] & e) == e, hi = (x[j] & e << 16) == e << 16;
            hit = hit || lo || hi;
            x[j] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
        }
        if (hit)
            *at = x;
        found = found || hit;
    }
    return __any(found);
}

template <class T>
__device__ __forceinline__ float value_of(uint32_t x, int i)
{
    const uint16_t h = (uint16_t)(i ? x >> 16 : x);
    return (float)__builtin_bit_cast(T, h);
}

template <class T, class TO, int D, int NG>
__global__ __launch_bounds__((Shape<D, NG>::kWaves * 64), ((Shape<D, NG>::kWaves + 3) / 4)) void tree_split(
    const TreeParams p, TO* __restrict__ o, float* __restrict__ lse)
{
    using S = Shape<D, NG>;
    using E = Elem<T>;
    using V8 = typename E::vec8;
    // Heads of 256: one wave a SIMD, so nothing else hides the wave's LDS reads. Its registers hold K's operands of the next
    // tile beside V's of this one and Q (in accumulator registers); K's are read between the products with V, V's between
    // those of the scores (two chains of these: scores and V^T 860-890 clocks for 1030), loads issued between the last. 4 x
    // 64 drafts, 16 heads over 2: 113 us before, 96 so; a step 2700 clocks (softmax 450, products with V 1290), 1540 of products.
    constexpr bool kAhead = D == 256;
    constexpr int kChains = kAhead ? 2 : 1;
    constexpr int KW = S::kKW, ND = D / 32, NK = D / 16, W = S::kWaves;
    constexpr uint32_t kLead = lead_of(D);
    constexpr int kRow = 2 * D, kHalf = kTK * kRow, kPieces = kHalf / 1024 / NG;  // 1 KiB pieces of K (of V) a wave
    static_assert(kPieces >= 1, "every wave stages some");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[S::kLds];
    __shared__ float2 s_ml[W][32];
    __shared__ uint32_t s_odd;  // a draft's V holds what is not finite

    const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c32 = lane & 31;
    const uint32_t wl = uniform(tid >> 6), cg = wl % NG, kw = wl / NG;
    uint32_t range = blockIdx.x, cb = 0;
    if (p.ncb > 1) {  // the column blocks of a range 8 apart: one XCD
        const uint32_t in = blockIdx.x % (8 * p.ncb);
        range = blockIdx.x / (8 * p.ncb) * 8 + in % 8;
        cb = in / 8;
    }
    const uint32_t n_seg = p.batch * p.kv_heads;
    if (range >= (p.n_ranges ? p.n_ranges : n_seg))
        return;

    // This wave's DMA pieces: the bytes of the tile's rows that the lane's 16 LDS bytes hold.
    uint32_t kd[kPieces], vd[kPieces];
    #pragma unroll
    for (int m = 0; m < kPieces; ++m) {
        const uint32_t at = 1024 * (cg * kPieces + m) + 16 * lane, r = at / kRow, pos = at % kRow;
        kd[m] = slot_of(r) * kRow + 16 * ((pos / 16) ^ k_xor<D>(r));
        vd[m] = r * kRow + 32 * v_unit_at<D>(pos / 32, r) + (pos & 16);
    }
    const uint32_t lbase = uniform((uint32_t)reinterpret_cast<uintptr_t>(lds));
    // K operand: row c32, chunk (2 kk + g) at its place; V^T operand: see v_unit (lane 4 j + y of a group of 16: head
    // dims 16 (group % 2) + 4 y .. of key 8 g + j).
    const uint32_t ka = c32 * kRow + 16 * (g ^ k_xor<D>(c32));
    const uint32_t gj = (lane >> 2) & 3u, gy = lane & 3u, gg = (lane >> 4) & 1u;
    constexpr int NV = D == 64 ? 2 : 4;
    uint32_t va[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i)
        va[i] = kHalf + (8 * g + gj) * kRow + 32 * v_unit<D>(2 * i + gg, gj) + 8 * gy;

    // The first piece of the range (or the segment): steps [s0, s1) of the segment's len; units of the range behind them.
    uint32_t b, kvh, len, s0, s1, left = 0;
    if (p.n_ranges) {
        const Place at = place_of(p.batch, p.kv_heads, range, p.n_ranges, lane, SegUnits<D>{p});
        if (at.x0 == at.x1)
            return;
        b = at.b;
        len = at.len - kLead;
        kvh = (at.x0 - at.first) / at.len;
        const uint32_t u0 = (at.x0 - at.first) % at.len, u1 = min(at.len, u0 + (at.x1 - at.x0));
        s0 = max(u0, kLead) - kLead;
        s1 = max(u1, kLead) - kLead;
        left = at.x1 - at.x0 - (u1 - u0);
    } else {
        b = range / p.kv_heads, kvh = range % p.kv_heads, s0 = 0;
        s1 = len = uniform(steps_of(p, ctx_of(p, b), nodes_of(p, b)));
    }
    // On to the segment behind; whether the range has a piece of it.
    const auto next = [&]() __attribute__((always_inline)) {
        do {
            if (++kvh == p.kv_heads) {
                kvh = 0;
                ++b;
            }
            len = b < p.batch ? uniform(steps_of(p, ctx_of(p, b), nodes_of(p, b))) : 0u;
        } while (b < p.batch && len == 0);
        s0 = 0;
        s1 = max(min(len + kLead, left), kLead) - kLead;
        left -= min(len + kLead, left);
        return b < p.batch && s1 > 0;
    };
    if (p.n_ranges && s0 == s1 && !(left && next()))
        return;

    for (;;) {
        const uint32_t ctx = uniform(ctx_of(p, b)), nodes = uniform(nodes_of(p, b)), tc = (ctx + kTK - 1) / kTK;
        const size_t cache = ((size_t)b * p.kv_heads + kvh) * p.cap * D;
        const size_t draft = ((size_t)kvh * p.d_pad + (size_t)b * p.n_draft) * D;
        const u32x4 rs[4] = {tile_rsrc(static_cast<const T*>(p.k) + cache, ctx * kRow),
                             tile_rsrc(static_cast<const T*>(p.v) + cache, ctx * kRow),
                             tile_rsrc(static_cast<const T*>(p.kd) + draft, nodes * kRow),
                             tile_rsrc(static_cast<const T*>(p.vd) + draft, nodes * kRow)};
        // The wave's share of the tile of way kw in step s, into its ring slot, a piece of K or V at a time (past the segment's
        // tiles: rows past the tree, zeros; kAhead, past the range's steps: zeros too, so that as many are always in flight).
        // Streaming loads: 128 lists of 8192 keys of 128 take 88 us with them, 103 without (with column blocks, which read the
        // keys again from the L2, the same either way).
        struct Slot {
            uint32_t dst, off;
            u32x4 k, v;
        };
        auto slot_for = [&](uint32_t s) __attribute__((always_inline)) {
            const uint32_t t = s * KW + kw;
            Slot x{lbase + (s % S::kDepth * KW + kw) * S::kSlot + 1024 * cg * kPieces, (t < tc ? t : t - tc) * kHalf,
                   t < tc ? rs[0] : rs[2], t < tc ? rs[1] : rs[3]};
            if (kAhead && s >= s1)
                x.k[2] = x.v[2] = 0;
            return x;
        };
        auto stage_piece = [&](const Slot& x, int m) __attribute__((always_inline)) {
            if (m < kPieces)
                dma16_nt(x.dst + 1024 * m, kd[m] + x.off, x.k);
            else
                dma16_nt(x.dst + kHalf + 1024 * (m - kPieces), vd[m - kPieces] + x.off, x.v);
        };
        auto stage = [&](uint32_t s) __attribute__((always_inline)) {
            const Slot x = slot_for(s);
            #pragma unroll
            for (int m = 0; m < 2 * kPieces; ++m)
                stage_piece(x, m);
        };
        for (uint32_t s = s0; s < (kAhead ? s0 + S::kDepth - 1 : min(s1, s0 + S::kDepth - 1)); ++s)
            stage(s);
        // The lane's column: row r, head h; its mask, cut to the tree; Q, beside the first tiles' loads.
        const uint32_t col = 32 * (cb * NG + cg) + c32, r = col / p.group, h = kvh * p.group + col % p.group;
        const bool has = col < p.nc && r < nodes;
        uint64_t sees = has ? sees_of(p, b, r, nodes) : 0;
        V8 qreg[NK];
        {
            const T* src = static_cast<const T*>(p.q) + ((size_t)h * p.q_pad + (size_t)b * p.n_draft + r) * D + 8 * g;
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                qreg[kk] = has ? *reinterpret_cast<const V8*>(src + 16 * kk) : V8{};
        }
        asm volatile("" : "+v"(sees));
        // Q has come; kAhead: into accumulator registers, which the products read as well as the others.
        auto operand = [&](V8& x) __attribute__((always_inline)) {
            if constexpr (kAhead)
                asm volatile("" : "+a"(x));
            else
                settle(x);
        };
        f32x16 acc[ND];
        #pragma unroll
        for (int db = 0; db < ND; ++db)
            acc[db] = f32x16{};
        float m = -INFINITY, l = 0.0f;
        bool odd = false;
        const float c = p.scale_log2;
        if (tid == 0)
            s_odd = 0;
        #pragma unroll
        for (int kk = 0; kk < NK; ++kk)
            operand(qreg[kk]);
        // Step s has landed; every wave is done with step s - 1, whose slots take step s + DEPTH - 1.
        auto landed = [&](uint32_t s) __attribute__((always_inline)) {
            if (kAhead || s + S::kDepth - 1 <= s1)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::kDepth - 2) * 2 * kPieces) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            if (NG > 1)
                asm volatile("s_barrier" ::: "memory");
        };
        auto arrive = [&](uint32_t s) __attribute__((always_inline)) {
            landed(s);
            if (kAhead || s + S::kDepth - 1 < s1)
                stage(s + S::kDepth - 1);
        };
        // kAhead: K's operands are read a tile ahead, beside the products of the one before.
        V8 kf[NK];
        auto read_k = [&](uint32_t s) __attribute__((always_inline)) {
            const unsigned char* tile = lds + (s % S::kDepth * KW + kw) * S::kSlot;
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                kf[kk] = *reinterpret_cast<const V8*>(tile + (ka ^ (32 * kk)));
        };
        // The wave's tile of step s; CUT: one that not every column sees all of.
        auto tile_step = [&](auto cut, uint32_t s) __attribute__((always_inline)) {
            constexpr bool CUT = decltype(cut)::value;
            const uint32_t t = s * KW + kw;
            unsigned char* tile = lds + (s % S::kDepth * KW + kw) * S::kSlot;
            // V^T's operands come while the scores (kAhead) or the exponentials are made.
            V8 vf[2][ND];
            auto read_v = [&]() __attribute__((always_inline)) {
                if (CUT && t >= tc)
                    odd |= finite_only<T, kHalf>(tile + kHalf, lane);
                #pragma unroll
                for (int a = 0; a < 2; ++a)
                    #pragma unroll
                    for (int db = 0; db < ND; ++db) {
                        const unsigned char* at = tile + va[db % NV] + db / NV * 256 + 16 * a * kRow;
                        const s16x4 v0 = tr_read(at), v1 = tr_read(at + 4 * kRow);
                        vf[a][db] = __builtin_bit_cast(V8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                    }
            };
            if (kAhead) {
                #pragma unroll
                for (int kk = 0; kk < NK; ++kk)
                    settle(kf[kk]);
                read_v();
            } else {
                read_k(s);
            }
            f32x16 chain[kChains];
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                chain[kk % kChains] = E::mfma32(kf[kk], qreg[kk], kk < kChains ? f32x16{} : chain[kk % kChains]);
            f32x16 x = chain[0];
            if (kChains > 1)
                x += chain[kChains - 1];
            if (kAhead)
                #pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 4 * ND / NK, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
            if (!kAhead)
                read_v();
            __builtin_amdgcn_sched_barrier(0);
            // Register i holds key 16 (i / 8) + 8 g + i % 8 of the tile.
            #pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] *= c;
            if (CUT) {
                uint32_t word;
                if (t >= tc)
                    word = (uint32_t)(sees >> (32 * (t - tc)));
                else
                    word = (t + 1) * kTK <= ctx ? ~0u : (1u << (ctx - t * kTK)) - 1;
                word >>= 8 * g;
                #pragma unroll
                for (int i = 0; i < 16; ++i)
                    x[i] = word >> (16 * (i >> 3) + (i & 7)) & 1 ? x[i] : -INFINITY;
            }
            float mx = fmaxf(x[0], x[1]);
            #pragma unroll
            for (int i = 2; i < 16; i += 2)
                mx = fmaxf(fmaxf(mx, x[i]), x[i + 1]);
            mx = pair_max(mx);
            if (__any(mx > m + kRescale)) {
                float f = 1.0f;
                if (mx > m + kRescale) {
                    f = exp2_fast(m - mx);
                    m = mx;
                }
                l *= f;
                #pragma unroll
                for (int db = 0; db < ND; ++db)
                    #pragma unroll
                    for (int i = 0; i < 16; ++i)
                        acc[db][i] *= f;
            }
            const float mu = m == -INFINITY ? 0.0f : m;
            // 16 keys at a time: the second half's exponentials run beside the first half's products.
            u32x4 hi[2], lo[2];  // P as the sum of two values of T (bf16: 16 bits, f16: 22; one would show in the output)
            auto half = [&](int a) __attribute__((always_inline)) {
                #pragma unroll
                for (int i = 8 * a; i < 8 * a + 8; ++i)
                    x[i] = exp2_fast(x[i] - mu);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e0 = x[8 * a + 2 * i], e1 = x[8 * a + 2 * i + 1];
                    hi[a][i] = E::pack2(e0, e1);
                    lo[a][i] = E::pack2(e0 - value_of<T>(hi[a][i], 0), e1 - value_of<T>(hi[a][i], 1));
                }
                l += (x[8 * a] + x[8 * a + 1]) + (x[8 * a + 2] + x[8 * a + 3]) +
                     ((x[8 * a + 4] + x[8 * a + 5]) + (x[8 * a + 6] + x[8 * a + 7]));
            };
            auto product = [&](int a, int i) __attribute__((always_inline)) {
                acc[i % ND] = E::mfma32(vf[a][i % ND], __builtin_bit_cast(V8, i < ND ? hi[a] : lo[a]), acc[i % ND]);
            };
            constexpr int kMf = 2 * ND;  // products of a half
            half(0);
            __builtin_amdgcn_sched_barrier(0);
            if (kAhead) {
                landed(s + 1);
                read_k(s + 1);
            }
            #pragma unroll
            for (int i = 0; i < kMf; ++i)
                product(0, i);
            half(1);
            #pragma unroll
            for (int i = 0; i < kMf; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (kAhead)
                    __builtin_amdgcn_sched_group_barrier(0x100, NK / kMf, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 40 / kMf + 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 8 / kMf + 1, 0);
            }
            if (kAhead) {
                // the loads of a step to come between the products: issued together they would hold the wave up
                const Slot next = slot_for(s + S::kDepth);
                #pragma unroll
                for (int i = 0; i < kMf; ++i) {
                    product(1, i);
                    __builtin_amdgcn_sched_barrier(0);
                    #pragma unroll
                    for (int m = 2 * kPieces * i / kMf; m < 2 * kPieces * (i + 1) / kMf; ++m)
                        stage_piece(next, m);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                #pragma unroll
                for (int i = 0; i < kMf; ++i)
                    product(1, i);
            }
        };
        if (kAhead) {
            arrive(s0);
            read_k(s0);
        }
        uint32_t s = s0;
        for (const uint32_t whole = min(s1, ctx / kTK / KW); s < whole; ++s) {
            if (!kAhead)
                arrive(s);
            tile_step(std::false_type{}, s);
        }
        for (; s < s1; ++s) {
            if (!kAhead)
                arrive(s);
            if ((s * KW + kw) * kTK < tc * kTK + nodes) {
                tile_step(std::true_type{}, s);
            } else if (kAhead) {
                arrive(s + 1);
                read_k(s + 1);
            }
        }
        // The piece's ways join: every wave's columns into LDS (the ring is idle: nothing is in flight), column c32 a row of
        // D floats, its 16-byte chunks XORed by the column.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        {
            f32x4* row = reinterpret_cast<f32x4*>(lds) + (wl * 32 + c32) * (D / 4);
            #pragma unroll
            for (int q = 0; q < D / 8; ++q)
                row[(8 * (q / 4) + 2 * (q % 4) + g) ^ (c32 & 15)] =
                    f32x4{acc[q / 4][4 * (q % 4)], acc[q / 4][4 * (q % 4) + 1], acc[q / 4][4 * (q % 4) + 2],
                          acc[q / 4][4 * (q % 4) + 3]};
            const float lt = pair_sum(l);
            if (g == 0)
                s_ml[wl][c32] = float2{m, lt};
            if (odd)
                s_odd = 1;
        }
        __syncthreads();
        const size_t part = (size_t)range + (size_t)b * p.kv_heads + kvh;
        const bool any_odd = s_odd != 0;
        if (p.n_ranges && tid == 0 && cb == 0) {
            p.part_odd[part] = any_odd;
            if (s0 == 0)
                p.seg_ends[2 * (b * p.kv_heads + kvh)] = range;
            if (s1 == len)
                p.seg_ends[2 * (b * p.kv_heads + kvh) + 1] = range;
        }
        constexpr int kItems = NG * 32 * (D / 4) / (W * 64);  // quads of a column a thread
        constexpr int kUnroll = W > 4 && KW >= 4 ? 1 : 4;  // (as registers allow)
        #pragma unroll kUnroll
        for (int i = 0; i < kItems; ++i) {
            const uint32_t it = i * (W * 64) + tid, q = it % (D / 4), cc = it / (D / 4) % 32, gi = it / (D / 4) / 32;
            const uint32_t ccol = 32 * (cb * NG + gi) + cc, rr = ccol / p.group;
            float mx = -INFINITY, sum = 0.0f;
            f32x4 a = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float2 ml[KW];
            f32x4 v[KW];
            #pragma unroll
            for (int y = 0; y < KW; ++y) {
                const uint32_t w = gi + NG * y;
                ml[y] = s_ml[w][cc];
                v[y] = reinterpret_cast<const f32x4*>(lds)[(w * 32 + cc) * (D / 4) + (q ^ (cc & 15))];
                mx = fmaxf(mx, ml[y].x);
            }
            #pragma unroll
            for (int y = 0; y < KW; ++y) {
                const float f = ml[y].x == -INFINITY ? 0.0f : exp2_fast(ml[y].x - mx);
                sum += ml[y].y * f;
                a += v[y] * f;
            }
            const bool live = ccol < p.nc && rr < nodes;
            if (p.n_ranges) {
                if (live)
                    *reinterpret_cast<f32x4*>(p.part_o + (part * p.nc + ccol) * D + 4 * q) = a;
                if (live && q == 0)
                    *reinterpret_cast<float2*>(p.part_ml + (part * p.nc + ccol) * 2) = float2{mx, sum};
            } else if (live) {
                const uint32_t hh = kvh * p.group + ccol % p.group;
                const size_t row = (size_t)b * p.n_draft + rr;
                a *= sum == 0.0f ? 0.0f : 1.0f / sum;
                if (any_odd)
                    #pragma unroll
                    for (int y = 0; y < 4; ++y)
                        a[y] += odd_sum<T, D>(p, b, kvh, rr, nodes, 4 * q + y);
                store4<TO>(o + row * p.width + (size_t)hh * D + 4 * q, a[0], a[1], a[2], a[3]);
                if (lse && q == 0)
                    lse[(size_t)hh * p.batch * p.n_draft + row] = sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * kLn2;
            }
        }
        if (left == 0 || !next())
            return;
        __syncthreads();  // the ring is free again
    }
}

// NW waves a row and head, each every NW-th piece of its segment: a running maximum, 8 pieces' loads in flight, and with
// more than one wave a join in LDS.
template <class T, class TO, int D, int NW>
__global__ __launch_bounds__(256) void tree_merge(const TreeParams p, TO* __restrict__ o, float* __restrict__ lse)
{
    constexpr int E = D / 64, U = 8;
    typedef float fE __attribute__((ext_vector_type(E)));
    __shared__ float s_m[4], s_l[4];
    __shared__ fE s_o[4][64];
    const uint32_t lane = threadIdx.x & 63, wl = uniform(threadIdx.x >> 6), wv = wl % NW;
    const uint32_t item = blockIdx.x * (4 / NW) + wl / NW, row = item / p.heads, h = item % p.heads;
    const uint32_t b = row / p.n_draft, r = row % p.n_draft;
    if (row >= p.batch * p.n_draft)
        return;  // (with NW = 4 the whole workgroup)
    const uint32_t nodes = uniform(nodes_of(p, b));
    if (r >= nodes)
        return;
    const uint32_t kvh = h / p.group, col = r * p.group + h % p.group, seg = b * p.kv_heads + kvh;
    const uint32_t w0 = uniform(p.seg_ends[2 * seg]), w1 = uniform(p.seg_ends[2 * seg + 1]);
    bool odd = false;
    for (uint32_t x = w0 + lane; x <= w1; x += 64)
        odd = odd || p.part_odd[x + seg];
    float m = -INFINITY, l = 0.0f;
    fE acc = fE(0.0f);
    for (uint32_t x0 = w0 + wv; x0 <= w1; x0 += U * NW) {
        float2 ml[U];
        fE v[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t x = x0 + u * NW;
            const size_t at = ((size_t)min(x, w1) + seg) * p.nc + col;
            ml[u] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
            v[u] = *reinterpret_cast<const fE*>(p.part_o + at * D + E * lane);
            if (x > w1)
                ml[u].x = -INFINITY;
        }
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const float nm = fmaxf(m, ml[u].x);
            const float f = m == -INFINITY ? 0.0f : exp2_fast(m - nm);
            const float e = ml[u].x == -INFINITY ? 0.0f : exp2_fast(ml[u].x - nm);
            l = l * f + ml[u].y * e;
            acc = acc * f + v[u] * e;
            m = nm;
        }
    }
    if (NW > 1) {
        if (lane == 0) {
            s_m[wl] = m;
            s_l[wl] = l;
        }
        s_o[wl][lane] = acc;
        __syncthreads();
        if (wv != 0)
            return;
        #pragma unroll
        for (int i = 1; i < NW; ++i) {
            const float mi = s_m[i], nm = fmaxf(m, mi);
            const float f = m == -INFINITY ? 0.0f : exp2_fast(m - nm), e = mi == -INFINITY ? 0.0f : exp2_fast(mi - nm);
            l = l * f + s_l[i] * e;
            acc = acc * f + s_o[i][lane] * e;
            m = nm;
        }
    }
    acc *= l == 0.0f ? 0.0f : 1.0f / l;
    if (__any(odd))
        #pragma unroll
        for (int e = 0; e < E; ++e)
            acc[e] += odd_sum<T, D>(p, b, kvh, r, nodes, E * lane + e);
    TO* orow = o + (size_t)row * p.width + (size_t)h * D + E * lane;
    #pragma unroll
    for (int e = 0; e < E; ++e)
        orow[e] = (TO)acc[e];
    if (lse && lane == 0)
        lse[(size_t)h * p.batch * p.n_draft + row] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// A call's split, from its sizes alone (contexts are known on the device only).
struct Plan {
    uint32_t ng, ways, ncb, n_ranges;  // n_ranges 0: a segment a workgroup
    size_t pieces;
};

template <int D>
uint32_t ways_of(uint32_t ng)
{
    return ng == 1 ? Shape<D, 1>::kKW : ng == 2 ? Shape<D, 2>::kKW : Shape<D, 4>::kKW;
}

// A segment a workgroup, and no partials or second launch, up to this many steps: 5, and more the more segments there are to
// fill the CUs and the more columns a partial has. A workgroup takes its segment's steps one after the other, whatever the
// others' contexts, so the limit also bounds the loss where one is max_ctx long and the rest an eighth of it.
// us direct / split, heads of 128: 32 columns, 8 segments of 5 steps 12.8 / 13.3, of 6 14.2 / 13.7; 64 of 17 29 / 24; 128 of
// 9 21 / 25; 256 of 13 38 / 44. 128 columns: 64 of 9 23 / 27, of 17 32 / 31; 128 of 17 35 / 41; 256 of 25 57 / 78. One long
// among short ones, 128 columns: 128 of 17 33 / 33; 256 of 17 34 / 45, of 33 55 / 49.
uint32_t direct_steps(uint64_t segs, uint32_t nc, uint32_t cus)
{
    return 5 + (uint32_t)std::min<uint64_t>(28, segs * std::min(3u, (nc + 31) / 32) * 8 / cus);
}

Plan plan_of(const mako_tree_args* a, uint32_t cus)
{
    const uint32_t nc = a->n_draft * (a->heads / a->kv_heads);
    Plan pl{};
    // Column groups: as many as there are columns for. The other side, us at 64 lists (8 lists) of 8192 keys, heads of 128:
    // 64 columns in 2 groups 57 (23), in 1 and two column blocks 61 (20), in 4 68 (26); 96 columns in 4 71 (28), in 2 80
    // (24); 128 columns in 4 77 (30), in 2 81 (25); 32 columns, 32 lists, in 1 group 32, in 2 35, in 4 40; heads of 256 61, 58-60, 72.
    pl.ng = nc <= 32 && a->dim != 256 ? 1 : nc <= 64 ? 2 : 4;
    pl.ncb = (nc + 32 * pl.ng - 1) / (32 * pl.ng);
    pl.ways = a->dim == 64 ? ways_of<64>(pl.ng) : a->dim == 128 ? ways_of<128>(pl.ng) : ways_of<256>(pl.ng);
    const uint32_t tiles = (a->max_ctx + kTK - 1) / kTK + (a->n_draft + kTK - 1) / kTK;
    const uint32_t steps = (tiles + pl.ways - 1) / pl.ways;
    const uint64_t segs = (uint64_t)a->batch * a->kv_heads;
    if (steps > direct_steps(segs, nc, cus)) {
        pl.n_ranges = (uint32_t)std::min<uint64_t>(std::max(1u, cus / pl.ncb), segs * steps);
        pl.pieces = pl.n_ranges + segs;
    }
    return pl;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// The partials' parts: outputs, maxima and sums, flags.
size_t part_o_bytes(const Plan& pl, const mako_tree_args* a)
{
    return round256(pl.pieces * a->n_draft * (a->heads / a->kv_heads) * a->dim * sizeof(float));
}
size_t part_ml_bytes(const Plan& pl, const mako_tree_args* a)
{
    return round256(pl.pieces * a->n_draft * (a->heads / a->kv_heads) * 2 * sizeof(float));
}
size_t workspace_for(const Plan& pl, const mako_tree_args* a)
{
    return pl.pieces ? part_o_bytes(pl, a) + part_ml_bytes(pl, a) + round256(pl.pieces * sizeof(uint32_t)) +
                           (size_t)a->batch * a->kv_heads * 2 * sizeof(uint32_t)
                     : 0;
}

// Workgroups of tree_split, and of tree_merge: a wave an item where segments have few pieces (n_ranges of them over all, and
// a cut one more each). The call's us with a wave and with four, 16 drafts, heads of 128: 4 pieces 37.9, 43.1; 8 pieces 37.4,
// 38.9; 32 pieces 41.9, 41.5; 64 drafts, heads of 256, 128 pieces: 60.6, 58.3.
uint64_t split_groups(const Plan& pl, uint64_t segs)
{
    const uint64_t units = pl.n_ranges ? pl.n_ranges : segs;
    return pl.ncb > 1 ? (units + 7) / 8 * 8 * pl.ncb : units;
}
bool merge_by_wave(uint32_t n_ranges, uint64_t segs) { return n_ranges / segs < 16; }
uint64_t merge_groups(uint32_t n_ranges, uint64_t segs, uint64_t items)
{
    return n_ranges == 0 ? 0 : merge_by_wave(n_ranges, segs) ? (items + 3) / 4 : items;
}

template <class T, class TO, int D, int NG>
void launch_split(const TreeParams& p, const Plan& pl, void* o, float* lse, hipStream_t s)
{
    const dim3 grid((uint32_t)split_groups(pl, (uint64_t)p.batch * p.kv_heads)), block(Shape<D, NG>::kWaves * 64);
    hipLaunchKernelGGL((tree_split<T, TO, D, NG>), grid, block, 0, s, p, static_cast<TO*>(o), lse);
}

template <class T, class TO, int D>
void launch(const TreeParams& p, const Plan& pl, void* o, float* lse, hipStream_t s)
{
    if (D < 256 && pl.ng == 1)
        launch_split<T, TO, D, D < 256 ? 1 : 2>(p, pl, o, lse, s);
    else if (pl.ng == 2)
        launch_split<T, TO, D, 2>(p, pl, o, lse, s);
    else
        launch_split<T, TO, D, 4>(p, pl, o, lse, s);
    if (!pl.n_ranges)
        return;
    const uint64_t segs = (uint64_t)p.batch * p.kv_heads;
    const dim3 grid((uint32_t)merge_groups(pl.n_ranges, segs, (uint64_t)p.batch * p.n_draft * p.heads));
    if (merge_by_wave(pl.n_ranges, segs))
        hipLaunchKernelGGL((tree_merge<T, TO, D, 1>), grid, dim3(256), 0, s, p, static_cast<TO*>(o), lse);
    else
        hipLaunchKernelGGL((tree_merge<T, TO, D, 4>), grid, dim3(256), 0, s, p, static_cast<TO*>(o), lse);
}

template <class T, class TO>
void launch_dim(const TreeParams& p, uint32_t dim, const Plan& pl, void* o, float* lse, hipStream_t s)
{
    if (dim == 64)
        launch<T, TO, 64>(p, pl, o, lse, s);
    else if (dim == 128)
        launch<T, TO, 128>(p, pl, o, lse, s);
    else
        launch<T, TO, 256>(p, pl, o, lse, s);
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
    if ((uint64_t)a->batch * a->kv_heads * (a->max_ctx + 512ull) >= (1ull << 32))
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

extern "C" size_t mako_attn_tree_workspace(const mako_tree_args* a)
{
    const uint32_t cus = device_cus();
    if (!a || !cus || !a->heads || !a->kv_heads || a->heads % a->kv_heads || !a->batch || !a->n_draft || a->n_draft > 64 ||
        (a->dim != 64 && a->dim != 128 && a->dim != 256))
        return 0;
    return workspace_for(plan_of(a, cus), a);
}

extern "C" int mako_attn_tree(const mako_tree_args* a, mako_dtype in, mako_dtype out, const void* q, const void* k,
                              const void* v, const void* kd, const void* vd, const uint32_t* ctx_len,
                              const uint32_t* n_nodes, const uint64_t* mask, void* o, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream)
{
    const char* what = "attention_tree";
    if (const int rc = check_args(a, in, out, q, k, v, kd, vd, ctx_len, mask, o))
        return rc;
    if (a->batch == 0 || a->n_draft == 0)
        return ok();
    const uint32_t cus = device_cus();
    if (!cus)
        return fail(MAKO_EHIP, "%s: no device to size the split for", what);
    const Plan pl = plan_of(a, cus);
    const size_t need = workspace_for(pl, a);
    if (workspace_bytes < need || (need && !workspace) || !aligned16(workspace))
        return fail(MAKO_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, workspace_bytes,
                    need);
    const uint64_t segs = (uint64_t)a->batch * a->kv_heads;
    if (!grid_fits(split_groups(pl, segs), 64 * pl.ng * pl.ways) ||
        !grid_fits(merge_groups(pl.n_ranges, segs, (uint64_t)a->batch * a->n_draft * a->heads), 256))
        return fail(MAKO_EINVAL, "%s: %u x %u rows of %u heads exceed the grid", what, a->batch, a->n_draft, a->heads);
    const uint32_t group = a->heads / a->kv_heads;
    const auto at = [&](size_t off) { return need ? static_cast<char*>(workspace) + off : nullptr; };
    const size_t ob = part_o_bytes(pl, a), mb = part_ml_bytes(pl, a), fb = round256(pl.pieces * sizeof(uint32_t));
    const TreeParams p{q, k, v, kd, vd, ctx_len, n_nodes, mask, reinterpret_cast<float*>(at(0)),
                       reinterpret_cast<float*>(at(ob)), reinterpret_cast<uint32_t*>(at(ob + mb)),
                       reinterpret_cast<uint32_t*>(at(ob + mb + fb)),
                       a->batch, a->n_draft, a->q_pad, a->d_pad, a->heads, a->kv_heads, group, a->cap, a->max_ctx,
                       a->width, a->n_draft * group, pl.ncb, pl.ways, pl.n_ranges, a->scale * kLog2e};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (in == MAKO_BF16 && out == MAKO_F32)
        launch_dim<__bf16, float>(p, a->dim, pl, o, lse, s);
    else if (in == MAKO_BF16)
        launch_dim<__bf16, __bf16>(p, a->dim, pl, o, lse, s);
    else if (out == MAKO_F32)
        launch_dim<_Float16, float>(p, a->dim, pl, o, lse, s);
    else
        launch_dim<_Float16, _Float16>(p, a->dim, pl, o, lse, s);
    return check_launch(what);
}
