// Attention of the sequences' new tokens over a cache kept in pages.
//
// Mathematics: new row i of sequence b sits at position c + i, c = ctx_len[b], and sees the cache rows j <= c + i:
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j,  lse = m + ln(sum),  m any bound
// Row j is row j % page of page table[b][j / page]. Sums over parts of the keys join by their log-sums.
//
// Bound: the matrix unit for chunks, the read of K and V for single tokens (64 keys of a kv head are 32 KiB at heads of 128,
// 1.2 us of a CU's products for 64 rows of four heads: 7 TB/s over the chip, so the same stream serves both).
//
// * paged_rows runs the streams of flash_fwd_r64 (heads of 64 and 128) and flash_fwd_r32 (256) over pages
//   (gen_attn_paged.py): a tile is 64 keys, a run of memory within a page; its page's number is read by a scalar load an
//   iteration before the tile is staged.
// * An item is a block of R rows of a sequence and `hq` heads of a kv head (8, 4, 2 or 1, as they divide the group), R = 256 / hq
//   (heads of 256: 128 / hq): one workgroup's four waves, 64 (32) columns each. A wave has one head; of eight, two side by
//   side, since a second workgroup on the same keys costs their read again (16 heads of 256 over 2, a step of 16 sequences,
//   605 MB: 143 us with two workgroups of four heads, 103 us with one of eight; 32 heads of 128 over 4 149 and 103 us).
//   Larger groups, and those that 8, 4 or 2 do not divide, take further workgroups (column blocks), beside each other on an XCD.
//   Each reads the item's K and V again, which bounds single tokens: a step of 16 with 32 or 64 heads over 8 167-198 us, with
//   24 over 8 (three readings) 336-373, with 40 over 8 (five) 534-593; 28 over 4 (seven, of half the bytes) 401-443, 64 over 4
//   (two) 156-171.
// * Items of half the rows or fewer take a stream of 32 columns a wave with streaming loads (heads of 256, in calls of such
//   items alone: tiles of 32 keys, three of them in flight).
// * Lengths are known on the device only, so every workgroup works out its share of the work (paged_split.hpp): ranges of
//   equal cost over the items of all sequences, one a workgroup.
// * A piece of an item leaves normalised f32 rows and their log-sums at slot 2 range (+ 1 if the item starts in it): a range
//   has at most one of each kind. The range with an item's last piece names its first one, and paged_merge joins them.
//   Contexts that are too short for a second launch (max_ctx) take whole items and none.
// * A piece of several rows ends with a look at the v that some of its rows do not see (hidden_not_finite).
//
// P meets V in the input type, as in the prefill streams: a second product for what that leaves off would be half as many matrix
// instructions again. Outputs are off by 2.9e-4 (f16) and 2.3e-3 (bf16) of their size, where rounded ones are by 2.1e-4 and 1.7e-3.
//
// us a call on one MI355X, 32 heads of 128 over 8: one token over 391 rows (16 heads) 10.8 (with max_ctx past 832, and so a join,
// 15); 16 single tokens over 1.02 to 1.21 GB 159-187 (6.4 to 6.5 TB/s); 11 single tokens beside two chunks of up to 1333 rows,
// contexts up to 12001, 210-272 over four sets of lengths (800 to 870 TFLOP/s); 512 rows behind 32256 218-233 (1050 to 1110);
// a prompt of 4096 rows 112 (865), of 1531 25-28. 16 heads of 256 over 2: 16 single tokens over 605 MB 103 (5.9 TB/s), four
// chunks of up to 300 rows behind up to 16000 163-207 (930 to 960), a prompt of 4096 rows 113 (855). 16 heads of 64 over 16: 16
// single tokens over up to 640 MB 88-103 (6.0 to 6.2 TB/s). paged_merge: 14-18 us of kernel for 57 MB of pieces (heads of 256
// 12), 5 for the single tokens'.
#include <algorithm>

#include "attn_paged_asm.inc"
#include "fwd64_common.hpp"
#include "paged_split.hpp"

namespace mako {
namespace {

constexpr uint32_t kNone = 0xffffffffu;

struct PagedParams : PagedSplit {
    const void *q, *k, *v;
    const uint32_t* table;
    void* o;
    float* lse;
    float* part_o;    // [ranges][ncb][2][hq / hpw][slot_rows][hpw][D]: pieces' normalised rows
    float* part_l;    // [ranges][ncb][2][hq][slot_rows]: their log-sums
    uint32_t* whole;  // [ranges][2]: which of a range's pieces there are
    u32x4* last;      // [ranges]: the item whose last piece a range has: first range (kNone: no item), row of o, rows, kv head
    uint32_t q_pad, group, pages, page_bytes, shift, max_pages, width, hq, ncb, slot_rows;
    uint32_t hs, ws;  // log2 of hpw (heads a wave) and of hq / hpw
    float scale_log2;
};

__device__ __forceinline__ uint64_t uniform64(uint64_t x)
{
    return (uint64_t)uniform((uint32_t)(x >> 32)) << 32 | uniform((uint32_t)x);
}

// uniform(x), kept in a scalar register: the compiler takes a uniform value's readfirstlane away, and where it has the value in a
// vector register gives a stream that for a scalar operand. It adds wait states around its own instructions only, so these are
// here: between the write of x and its read by readfirstlane, and before a vector instruction reads the scalar.
__device__ __forceinline__ uint32_t scalar(uint32_t x)
{
    uint32_t y;
    asm("s_nop 1\n\tv_readfirstlane_b32 %0, %1\n\ts_nop 4" : "=s"(y) : "v"(x));
    return y;
}

// The kernel's parameters, read where they are named: held in scalar registers through the streams, which take most of those,
// they would be spilled and restored around each.
typedef const __attribute__((address_space(4))) PagedParams* ParamsAt;
__device__ __forceinline__ ParamsAt params_here(ParamsAt p)
{
    asm volatile("" : "+s"(p));
    return p;
}

// What a piece is to the streams: tiles [ta, tb) of a sequence, rows `rows` of its block from position p0 on.
struct Piece {
    const void *q, *k, *v;  // of the block's first row and the wave's first head; of the kv head in page 0
    void* o;                // of the block's first row and the wave's first head
    float* l;               // of the block's first row and the wave's first head
    uint64_t table;         // the sequence's row
    uint32_t ta, tb, rows, p0, keys;  // keys: those of the block's last row
    uint32_t seen;                    // keys of the sequence: no row sees more
    uint32_t o_row, o_head;           // bytes between rows of o and between the wave's heads
    uint32_t l_head;                  // floats between the wave's heads in l
    uint32_t items, first_pages;      // items: lane i of first_pages has the table row's entry i
};

// FEW: the stream of 32 rows a wave and streaming loads, at heads of 256 by tiles of 32 keys; else 64 rows a wave, at heads of
// 256 flash_fwd_r32's 32.
template <class T, class TO, int D, bool FEW>
__device__ __forceinline__ void run_piece(ParamsAt at_p, unsigned char* lds, const Piece& x)
{
    const auto& p = *params_here(at_p);
    constexpr bool kR32 = D == 256 && !FEW;
    constexpr uint32_t RW = FEW || kR32 ? 32 : 64, KT = D == 256 && FEW ? 32 : 64, NBUF = kR32 ? 2 : kNBuf;
    constexpr uint32_t kKRowB = 2 * D + 16, kKTileB = (KT * kKRowB + 1023) / 1024 * 1024, kVRowB = 2 * D, kVTileB = KT * kVRowB;
    constexpr uint32_t NKP = (kKTileB / 1024 - 1) / 4;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, g = lane >> 5, c32 = lane & 31u, w = uniform(tid >> 6);
    // A wave's RW columns are RW / hpw rows of hpw heads, a row's heads side by side: lane column c32 (block 1: c32 + 32) is row
    // q0 + cr (+ 32 / hpw), head ch.
    const uint32_t hs = p.hs, RR = RW >> hs;  // (0 or 1)
    const uint32_t q0 = (w >> p.ws) * RR, cr = c32 >> hs, ch = c32 & hs;
    const uint32_t ks = 64 * x.ta, n_keys = min(64 * x.tb, x.keys) - ks;
    const uint32_t lim_w = x.p0 + min(q0 + RR, x.rows);  // (position of the wave's last row) + 1
    const uint32_t w_keys = q0 < x.rows ? min(n_keys, min(lim_w, x.seen) - ks) : 0u;
    const uint32_t nt = (n_keys + KT - 1) / KT, ntw = (w_keys + KT - 1) / KT;
    // keys that a row sees, counted from the piece's first one: lmin the wave's first row, lim0 and lim1 the lane's
    const uint32_t r0 = x.p0 + q0;
    const uint32_t lmin = min(r0 + 1, x.seen) - ks;
    const uint32_t lim0 = min(r0 + cr + 1, x.seen) - ks - 8 * g;

    // LDS addresses, staging and epilogue: as flash_fwd_r64 and flash_fwd_r32 have them.
    const uint32_t lbase = (uint32_t)reinterpret_cast<uintptr_t>(lds), vbase = lbase + NBUF * kKTileB;
    uint32_t kr = lbase + c32 * kKRowB + 16 * g;
    const uint32_t th = (lane >> 4) & 1u, ti = lane & 15u;
    const uint32_t vrow = vbase + (8 * g + ti / 4) * kVRowB + 8 * (ti % 4);
    auto kd_of = [&](uint32_t i) {
        const uint32_t by = 1024 * i + 16 * lane, row = by / kKRowB, ch = by % kKRowB / 16;
        return row < KT ? slot_of(row) * (2 * D) + 16 * (ch < D / 8 ? ch : 0) : 0u;
    };
    const uint32_t skw = uniform(lbase), skww = uniform(lbase + 1024 * w), svww = uniform(vbase + (kVTileB / 4) * w);
    const uint32_t qo = ((ch * p.q_pad + q0 + cr) * D + 8 * g) * 2, qo1 = uniform((64u >> hs) * D);
    constexpr uint32_t so = sizeof(TO), orow = D * so, lpr = orow / 16;
    const uint32_t obase = lbase + w * RW * orow;
    const uint32_t ew = so == 4 ? obase + c32 * orow + 16 * ((c32 & 7u) ^ g)
                                : obase + c32 * orow + 8 * g + 16 * (c32 & 7u);
    const uint32_t er = obase + (lane / lpr) * orow + 16 * ((lane % lpr) ^ (lane / lpr));
    // stores of 64 / lpr columns each: one of both heads steps by rows, one of a single column by head and row in turn
    constexpr uint32_t cols = 64 / lpr;
    const uint32_t oc = lane / lpr, og = (q0 + (oc >> hs)) * x.o_row + (oc & hs) * x.o_head + 16 * (lane % lpr);
    const uint32_t ogs = uniform(cols > hs ? (cols >> hs) * x.o_row : x.o_head);
    const uint32_t ogs2 = uniform(cols > hs ? 2 * ogs : x.o_row);
    const uint32_t lo0 = q0 + cr < x.rows ? (ch * x.l_head + q0 + cr) * 4 : kNone;
    const uint32_t swp = (lane ^ 32) * 4;
    const u32x4 qrs = rsrc_of(x.q, (hs * p.q_pad + x.rows) * 2 * D);
    const u32x4 ors = rsrc_of(x.o, (x.rows - 1) * x.o_row + hs * x.o_head + orow);
    const u32x4 lrs = rsrc_of(x.l, x.l ? (hs * x.l_head + x.rows) * 4 : 0);
    const uint32_t has_lse = scalar(x.l ? 1u : 0u);
    const float c = __builtin_bit_cast(float, uniform(__builtin_bit_cast(uint32_t, p.scale_log2)));
    const uint32_t s_nt = uniform(nt), s_ntw = uniform(ntw), s_lmin = uniform(lmin);
    const uint32_t kn = uniform(n_keys * 2 * D);  // (mod 2^32: the streams take the last tile's bytes from it)
    const uint64_t kb = reinterpret_cast<uint64_t>(x.k), vb = reinterpret_cast<uint64_t>(x.v);
    const uint32_t kb0 = uniform((uint32_t)kb), kb1 = uniform((uint32_t)(kb >> 32) & 0xffffu);
    const uint32_t vb0 = uniform((uint32_t)vb), vb1 = uniform((uint32_t)(vb >> 32) & 0xffffu);
    const uint32_t pshift = p.shift - (KT == 64 ? 6 : 5);
    const uint32_t* row = reinterpret_cast<const uint32_t*>(x.table);
    const uint32_t t0 = uniform(ks / KT), tlast = uniform(t0 + nt - 1), npages = uniform(p.pages);
    uint32_t pg0, pg1, pg2, pg3;
    const auto entry_of = [&](uint32_t t) { return uniform(min(t0 + t, tlast) >> pshift); };
    if (x.items) {
        const auto page_of = [&](uint32_t t) { return (uint32_t)__builtin_amdgcn_readlane(x.first_pages, entry_of(t)); };
        pg0 = page_of(0), pg1 = page_of(1), pg2 = page_of(2), pg3 = page_of(3);
    } else {
        const auto page_of = [&](uint32_t t) { return uniform(row[entry_of(t)]); };
        pg0 = page_of(0), pg1 = page_of(1), pg2 = page_of(2), pg3 = page_of(3);
    }
    const uint64_t ent = uniform64(x.table);
    const uint32_t pstride = uniform(p.page_bytes), pmask = uniform((1u << pshift) - 1), s_pshift = uniform(pshift);

#define MAKO_PAGED_SCALARS                                                                                        \
    [qrs] "s"(qrs), [ors] "s"(ors), [lrs] "s"(lrs), [c] "s"(c), [nt] "s"(s_nt), [ntw] "s"(s_ntw), [lmin] "s"(s_lmin),  \
        [has_lse] "s"(has_lse), [ogs] "s"(ogs), [ogs2] "s"(ogs2), [kb0] "s"(kb0), [kb1] "s"(kb1), [kn] "s"(kn),    \
        [vb0] "s"(vb0), [vb1] "s"(vb1), [skw] "s"(skw), [skww] "s"(skww), [svww] "s"(svww), [ent] "s"(ent), [t0] "s"(t0), \
        [tlast] "s"(tlast), [npages] "s"(npages), [pstride] "s"(pstride), [pmask] "s"(pmask), [pshift] "s"(s_pshift), \
        [pg0] "s"(pg0), [pg1] "s"(pg1), [pg2] "s"(pg2)
#define MAKO_PAGED_STREAM(NAME, OPERANDS)                                                                         \
    do {                                                                                                          \
        if constexpr (__is_same(T, __bf16)) {                                                                     \
            if constexpr (__is_same(TO, float))                                                                   \
                asm volatile(NAME##_BF16_F32 OPERANDS);                                                           \
            else                                                                                                  \
                asm volatile(NAME##_BF16_BF16 OPERANDS);                                                          \
        } else {                                                                                                  \
            if constexpr (__is_same(TO, float))                                                                   \
                asm volatile(NAME##_F16_F32 OPERANDS);                                                            \
            else                                                                                                  \
                asm volatile(NAME##_F16_F16 OPERANDS);                                                            \
        }                                                                                                         \
    } while (0)

    if constexpr (kR32) {
        // r32's V image: the bytes a lane's slot holds, for pieces that start on a multiple of 4 rows and the others
        const auto vunit = [](uint32_t u, uint32_t k) { return u ^ (k & 3u) ^ (4u * (u & 1u)); };
        const auto vd_at = [&](uint32_t row0) {
            const uint32_t by = 16 * lane, r = by / kVRowB, pos = by % kVRowB;
            const uint32_t y = (pos / 32) ^ ((row0 + r) & 3u), u = y ^ (4u * (y & 1u));
            return r * kVRowB + 32 * u + 16 * ((pos / 16) & 1u);
        };
        uint32_t vr0 = vrow + 32 * vunit(th, ti / 4), vr1 = vrow + 32 * vunit(2 + th, ti / 4);
        uint32_t vr2 = vrow + 32 * vunit(4 + th, ti / 4), vr3 = vrow + 32 * vunit(6 + th, ti / 4);
        const uint32_t kd0 = kd_of(w), kd1 = kd_of(w + 4), kd2 = kd_of(w + 8), kd3 = kd_of(w + 12);
        const uint32_t kd4 = kd_of(w + 16), kd5 = kd_of(w + 20), kd6 = kd_of(w + 24), kd7 = kd_of(w + 28);
        const uint32_t kd8 = kd_of(4 * NKP);
        const uint32_t vd = (kVTileB / 4) * w + vd_at(0), vdo = (kVTileB / 4) * w + vd_at(2);
        const uint32_t vd2 = vd + 4096, vdo2 = vdo + 4096;
#define MAKO_PAGED_R32                                                                                            \
    : [kr] "+v"(kr), [vr0] "+v"(vr0), [vr1] "+v"(vr1), [vr2] "+v"(vr2), [vr3] "+v"(vr3)                           \
    : [kd0] "v"(kd0), [kd1] "v"(kd1), [kd2] "v"(kd2), [kd3] "v"(kd3), [kd4] "v"(kd4), [kd5] "v"(kd5),              \
      [kd6] "v"(kd6), [kd7] "v"(kd7), [kd8] "v"(kd8), [vd] "v"(vd), [vdo] "v"(vdo), [vd2] "v"(vd2),                  \
      [vdo2] "v"(vdo2), [lim0] "v"(lim0), [qo] "v"(qo), [lo0] "v"(lo0), [swp] "v"(swp), [ew] "v"(ew), [er] "v"(er),   \
      [og] "v"(og), MAKO_PAGED_SCALARS                                                                            \
    : MAKO_PAGED_R32_CLOBBERS, "vcc", "scc", "memory"
        MAKO_PAGED_STREAM(MAKO_PAGED_D256_MANY, MAKO_PAGED_R32);
    } else {
        uint32_t vr0 = vrow + 32 * v_unit(th, ti / 4), vr1 = vrow + 32 * v_unit(2 + th, ti / 4);
        const uint32_t kr0 = kr, lim1 = min(r0 + (32u >> hs) + cr + 1, x.seen) - ks - 8 * g;
        const uint32_t r1 = q0 + (32u >> hs) + cr, lo1 = r1 < x.rows ? (ch * x.l_head + r1) * 4 : kNone;
        const uint32_t kd0 = kd_of(w), kd1 = kd_of(w + 4);
        const uint32_t kd2 = NKP > 2 ? kd_of(w + 8) : 0u, kd3 = NKP > 3 ? kd_of(w + 12) : 0u, kd4 = kd_of(4 * NKP);
        // the bytes a lane's slot of a V piece holds (vd_of); a piece of heads of 256 is two rows, so every other one starts
        // two rows on
        const auto vd_at = [&](uint32_t row0) {
            const uint32_t by = 16 * lane, r = by / kVRowB, pos = by % kVRowB;
            return (kVTileB / 4) * w + r * kVRowB + 32 * v_unit(pos / 32, r + row0) + 16 * ((pos / 16) & 1u);
        };
        const uint32_t vd = vd_at(0), vdo = vd_at(2);
#define MAKO_PAGED_R64                                                                                            \
    : [kr] "+v"(kr), [vr0] "+v"(vr0), [vr1] "+v"(vr1)                                                             \
    : [kd0] "v"(kd0), [kd1] "v"(kd1), [kd2] "v"(kd2), [kd3] "v"(kd3), [kd4] "v"(kd4), [vd] "v"(vd),                \
      [vdo] "v"(vdo), [lim0] "v"(lim0), [lim1] "v"(lim1), [kr0] "v"(kr0), [qo] "v"(qo), [lo0] "v"(lo0),             \
      [lo1] "v"(lo1), [swp] "v"(swp), [ew] "v"(ew), [er] "v"(er), [og] "v"(og), [pg3] "s"(pg3), [qo1] "s"(qo1),   \
      MAKO_PAGED_SCALARS                                                                                          \
    : MAKO_PAGED_CLOBBERS, "vcc", "scc", "memory"
        if constexpr (D == 64 && FEW)
            MAKO_PAGED_STREAM(MAKO_PAGED_D64_FEW, MAKO_PAGED_R64);
        else if constexpr (D == 64)
            MAKO_PAGED_STREAM(MAKO_PAGED_D64_MANY, MAKO_PAGED_R64);
        else if constexpr (D == 128 && FEW)
            MAKO_PAGED_STREAM(MAKO_PAGED_D128_FEW, MAKO_PAGED_R64);
        else if constexpr (D == 128)
            MAKO_PAGED_STREAM(MAKO_PAGED_D128_MANY, MAKO_PAGED_R64);
        else
            MAKO_PAGED_STREAM(MAKO_PAGED_D256_FEW, MAKO_PAGED_R64);
    }
#undef MAKO_PAGED_R64
#undef MAKO_PAGED_R32
#undef MAKO_PAGED_STREAM
#undef MAKO_PAGED_SCALARS
    // every wave's stream has ended (its LDS reads landed) before the next piece's staging overwrites LDS
    asm volatile("s_barrier" ::: "memory");
}

template <int D>
constexpr uint32_t lds_bytes()
{
    return kNBuf * (D == 64 ? 9 + 8 : 17 + 16) * 1024;  // (heads of 256: four tiles of 32 keys; two of 64 take less)
}

// Whether some v that a piece's tiles hold and some of its rows do not see (positions past the first row's) is not finite. All
// threads of the workgroup; lds is between two streams.
template <class T, int D>
__device__ __forceinline__ bool hidden_not_finite(ParamsAt at_p, unsigned char* lds, const PagedPiece& at)
{
    const auto& p = *params_here(at_p);
    constexpr uint32_t kExp = __is_same(T, __bf16) ? 0x7f807f80u : 0x7c007c00u;
    const uint32_t lo = max(at.p0 + 1, 64 * at.ta), hi = min(at.keys, 64 * at.tb), n = (hi - lo) * (D / 8);
    if (hi <= lo)
        return false;
    const uint32_t* row = p.table + (size_t)at.b * p.max_pages;
    uint32_t finite = 0x80008000u;  // the upper bits of (the exponent's complement + 0x7fff) are 0 where that is 0
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        const uint32_t j = lo + i / (D / 8), page = row[j >> p.shift];
        if (page >= p.pages)
            continue;
        const size_t base = ((size_t)page * p.kv_heads + at.kvh) << p.shift;
        const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.v) +
                                                        (base + (j & ((1u << p.shift) - 1))) * D + i % (D / 8) * 8);
        #pragma unroll
        for (int u = 0; u < 4; ++u)
            finite &= (~v[u] & kExp) + 0x7fff7fffu;
    }
    uint32_t* flags = reinterpret_cast<uint32_t*>(lds);
    const bool bad = __ballot((finite & 0x80008000u) != 0x80008000u) != 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the piece's stores are done, where another wave is to write there again
    flags[threadIdx.x >> 6] = bad ? 1 : 0;
    __syncthreads();
    const uint32_t any = flags[0] | flags[1] | flags[2] | flags[3];
    __syncthreads();
    return uniform(any) != 0;
}

// FEW: every piece takes the stream of 32 rows a wave; else pieces of few rows do (heads of 256: none).
template <class T, class TO, int D, bool FEW>
__global__ __launch_bounds__(256, 1) void paged_rows(const PagedParams q)
{
    __shared__ __attribute__((aligned(1024))) unsigned char lds[lds_bytes<D>()];
    const uint32_t lane = threadIdx.x & 63u, w = uniform(threadIdx.x >> 6);
    // blockIdx.x is the XCD: ranges side by side on one, a range's column blocks too (kItems: the kv head)
    const uint32_t range = q.how == kItems ? blockIdx.z : blockIdx.x * gridDim.z + blockIdx.z, cb = blockIdx.y;

    // kItems: the tiles begin with the first page, whose number needs no length, so it is loaded beside the lengths (one token
    // over 391 rows 11.1 -> 10.7 us).
    uint32_t first_pages = 0;
    if (q.how == kItems)
        first_pages = q.table[(size_t)blockIdx.z * q.max_pages + min(lane, q.max_pages - 1)];
    uint32_t here[2] = {0, 0};
    u32x4 done = u32x4{kNone, 0, 0, 0};
    const ParamsAt at_p = (ParamsAt)__builtin_amdgcn_kernarg_segment_ptr();
    walk_range(q, range, blockIdx.x, lane, [&](const PagedPiece& at) __attribute__((always_inline)) {
        const auto& p = *params_here(at_p);
        const uint32_t hl = (w & ((1u << p.ws) - 1)) << p.hs, h = at.kvh * p.group + cb * p.hq + hl;
        Piece x;
        x.q = static_cast<const T*>(p.q) + ((size_t)h * p.q_pad + at.row0) * D;
        x.k = static_cast<const T*>(p.k) + ((size_t)at.kvh << p.shift) * D;
        x.v = static_cast<const T*>(p.v) + ((size_t)at.kvh << p.shift) * D;
        x.table = reinterpret_cast<uint64_t>(p.table + (size_t)at.b * p.max_pages);
        x.ta = at.ta, x.tb = at.tb, x.rows = at.rows, x.p0 = at.p0, x.keys = at.keys, x.seen = at.seen;
        x.items = p.how == kItems, x.first_pages = first_pages;
        x.o = static_cast<TO*>(p.o) + (size_t)at.row0 * p.width + (size_t)h * D;
        x.o_row = p.width * sizeof(TO), x.o_head = D * sizeof(TO), x.l_head = p.rows;
        x.l = p.lse ? p.lse + (size_t)h * p.rows + at.row0 : nullptr;
        if (at.part) {
            const size_t slot = ((size_t)range * p.ncb + cb) * 2 + at.kind;
            x.o = p.part_o + (slot * p.hq + hl) * p.slot_rows * D;
            x.o_row = (D * 4) << p.hs, x.o_head = D * 4, x.l_head = p.slot_rows;
            x.l = p.part_l + (slot * p.hq + hl) * p.slot_rows;
            here[at.kind] = 1;
            if (at.first != kNone)
                done = u32x4{at.first, at.row0, at.rows, at.kvh};
        }
        // A row's probability of 0 for a key that it does not see, times a v that is not finite, is NaN: where there is such a v
        // the piece is done again row by row, so that no row meets keys past its own.
        for (uint32_t n = at.rows, r = 0;;) {
            const uint32_t few_rows = params_here(at_p)->few;
            const bool few = FEW || (D != 256 && n <= few_rows);
            if (at.part || __is_same(TO, float)) {
                if (few)
                    run_piece<T, float, D, D != 256 || FEW>(at_p, lds, x);
                else
                    run_piece<T, float, D, FEW>(at_p, lds, x);
            } else if (few) {
                run_piece<T, TO, D, D != 256 || FEW>(at_p, lds, x);
            } else {
                run_piece<T, TO, D, FEW>(at_p, lds, x);
            }
            r += n;
            if (r == at.rows) {
                if (n == 1 || !hidden_not_finite<T, D>(at_p, lds, at))
                    break;
                n = 1, r = 0;
            } else {
                x.q = static_cast<const T*>(x.q) + D;
                x.o = static_cast<char*>(x.o) + x.o_row;
                x.l = x.l ? x.l + 1 : x.l;
            }
            x.rows = 1, x.p0 = at.p0 + r, x.keys = min(x.p0 + 1, at.seen), x.tb = min(at.tb, (x.keys + 63) / 64);
        }
    });
    const auto& p = *params_here(at_p);
    if (p.how == kRanges && cb == 0 && threadIdx.x == 0) {
        p.whole[2 * range] = here[0];
        p.whole[2 * range + 1] = here[1];
        p.last[range] = done;
    }
}

// The pieces of the item whose last one range r has: their normalised rows weighted by exp(their log-sum - the largest). D / 4
// lanes a (row, head), four head dims each; where rows are few, NW such sets take every NW-th piece and meet in LDS. A piece
// with a log-sum of -inf is added with weight 0, so that NaN reaches the result whichever piece it is in; a row that is NaN
// throughout in such a piece gives -inf, as in a call without pieces.
template <class TO, int D, int NW>
__global__ __launch_bounds__(256) void paged_merge(const PagedParams p, uint32_t per)
{
    constexpr uint32_t L = D / 4, U = 8 / (NW == 1 ? 2 : 1);  // U pieces' loads in flight together
    __shared__ float s_m[NW][256 / L], s_l[NW][256 / L];
    __shared__ f32x4 s_o[NW][256];
    const uint32_t r = blockIdx.x / per, sub = blockIdx.x % per;
    const u32x4 item = p.last[r];
    const uint32_t first = item[0];
    if (first == kNone)
        return;
    const uint32_t set = threadIdx.x / L, w = set % NW, t = (sub * (256 / L) + set) / NW, d = 4 * (threadIdx.x % L);
    const uint32_t hl = t & (p.hq - 1), at_cb = t >> (p.hs + p.ws), cb = at_cb % p.ncb, row = at_cb / p.ncb;
    const bool live = row < item[2];
    float mx = -INFINITY, sum = 0.0f;
    f32x4 acc = f32x4{};
    for (uint32_t i0 = first + w; live && i0 <= r; i0 += U * NW) {
        float l[U];
        f32x4 v[U];
        #pragma unroll
        for (uint32_t u = 0; u < U; ++u) {  // (slots that no piece is in are read too, and left out)
            const uint32_t i = min(i0 + u * NW, r), kind = i == first ? 1 : 0;
            const size_t slot = ((size_t)i * p.ncb + cb) * 2 + kind;
            const bool has = i0 + u * NW <= r && p.whole[2 * i + kind];
            const float y = p.part_l[(slot * p.hq + hl) * p.slot_rows + row];
            const size_t at = ((slot * p.hq + (hl >> p.hs << p.hs)) * p.slot_rows + (row << p.hs) + (hl & p.hs)) * D + d;
            const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + at);
            l[u] = has ? y * kLog2e : -INFINITY;
            v[u] = has ? x : f32x4{};
        }
        #pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            if (l[u] == -INFINITY) {  // (the same in a row's lanes)
                const uint64_t nan = __ballot(v[u][0] != v[u][0] && v[u][1] != v[u][1] && v[u][2] != v[u][2] && v[u][3] != v[u][3]);
                const uint64_t lanes = L == 64 ? ~0ull : ((1ull << (L % 64)) - 1) << (threadIdx.x & 63u & ~(L - 1));
                acc += v[u] * 0.0f;
                if ((nan & lanes) == lanes)
                    sum = NAN;
                continue;
            }
            const float m = fmaxf(mx, l[u]), a = exp2_fast(mx - m), b = exp2_fast(l[u] - m);
            sum = sum * a + b;
            acc = acc * a + v[u] * b;
            mx = m;
        }
    }
    if (NW > 1) {
        if (threadIdx.x % L == 0) {
            s_m[w][set / NW] = mx;
            s_l[w][set / NW] = sum;
        }
        s_o[w][set / NW * L + threadIdx.x % L] = acc;
        __syncthreads();
        if (w != 0)
            return;
        #pragma unroll
        for (uint32_t i = 1; i < NW; ++i) {
            const float mi = s_m[i][set / NW], m = fmaxf(mx, mi);
            const float a = mx == -INFINITY ? 1.0f : exp2_fast(mx - m), b = mi == -INFINITY ? 1.0f : exp2_fast(mi - m);
            sum = sum * a + s_l[i][set / NW] * b;  // (without a piece: zeros, or NaN)
            acc = acc * a + s_o[i][set / NW * L + threadIdx.x % L] * b;
            mx = m;
        }
    }
    if (!live)
        return;
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    const uint32_t h = item[3] * p.group + cb * p.hq + hl, at = item[1] + row;
    store4<TO>(static_cast<TO*>(p.o) + (size_t)at * p.width + (size_t)h * D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv,
               acc[3] * inv);
    if (p.lse && d == 0)
        p.lse[(size_t)h * p.rows + at] = sum > 0.0f ? (mx + __log2f(sum)) * kLn2 : -INFINITY;
}

// A call's split, from its sizes alone (lengths are known on the device only).
struct Plan {
    uint32_t hq, hpw, rshift, ncb, n_ranges, slot_rows, how, few;
};

constexpr uint32_t kFewMerged = 16;  // (row, head) pairs a range up to which paged_merge parts an item's pieces

// Whole items and no second launch up to this many tiles a sequence: 13, where a merge joins more rows 20, and more the
// nearer the items come to one a workgroup. us split / whole, sequences of one length. Single tokens, 32 heads of 128 over 8: 8
// items of 12 tiles 16.3 / 14.9, of 16 16.4 / 17.9; 64 of 12 15.9 / 15.6, of 16 17.7 / 18.7; 128 of 20 25.6 / 23.7, of 33 35.6 /
// 34.5; 512 of 33 93 / 91. 16 heads of 256 over 2: 8 of 12 21.4 / 20.1, of 16 21.8 / 24.3; 64 of 16 28.2 / 26.4. 64 rows of 32
// heads: 8 items of 16 32.2 / 28.5, of 24 36.0 / 37.7; 256 rows: 128 of 24 44 / 40. A workgroup takes its item's tiles one after
// the other whatever the others' lengths, so the limit also bounds what one long sequence among short ones costs.
// (A workgroup an item, where sequences are one item each: 0.4 to 0.6 us less a call than looking for its range; more items
// than workgroups are better spread by ranges.)
uint32_t direct_tiles(uint64_t items, uint32_t ranges, bool many)
{
    const uint64_t x = std::min<uint64_t>(items * 30 / ranges, 30);
    return (many ? 20 : 13) + (x > 7 ? (uint32_t)x - 7 : 0);
}

uint32_t item_heads(const mako_paged_args* a)
{
    const uint32_t group = a->heads / a->kv_heads;
    if (group % 8 == 0 && 4ull * a->dim * a->q_pad < (1ull << 32))  // (two heads' queries have 32-bit offsets)
        return 8;
    return group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
}
uint32_t item_rows(const mako_paged_args* a) { return (a->dim == 256 ? 128 : 256) / item_heads(a); }

Plan plan_of(const mako_paged_args* a, uint32_t cus)
{
    const uint32_t group = a->heads / a->kv_heads;
    Plan pl{};
    pl.hq = item_heads(a);
    pl.hpw = pl.hq == 8 ? 2 : 1;
    pl.rshift = log2_of(item_rows(a));
    pl.ncb = group / pl.hq;
    pl.n_ranges = std::max(1u, cus / pl.ncb);
    if (pl.n_ranges > 8)
        pl.n_ranges &= ~7u;
    pl.slot_rows = std::min(1u << pl.rshift, a->max_new);
    const uint64_t items = ((uint64_t)(a->rows >> pl.rshift) + a->batch) * a->kv_heads;
    if ((a->max_ctx + 63) / 64 <= direct_tiles(items, pl.n_ranges, pl.slot_rows * group > kFewMerged))
        pl.how = a->max_new <= item_rows(a) && (uint64_t)a->batch * a->kv_heads <= pl.n_ranges ? kItems : kWhole;
    // Heads of 256, tiles of 32 keys / of 64: a step of 16 sequences over up to 32767 rows 103 us / 116, 8 tokens each 110 / 121,
    // 16 tokens each 136 / 129; steps among chunks 267 / 225; one token over 391 rows in one launch 16.1 / 15.5.
    pl.few = (1u << pl.rshift) / 2;
    if (a->dim == 256 && (pl.how != kRanges || a->max_new > pl.few))
        pl.few = 0;
    return pl;
}
size_t round256(size_t x) { return (x + 255) / 256 * 256; }
size_t part_o_bytes(const Plan& pl, uint32_t dim)
{
    return round256((size_t)pl.n_ranges * pl.ncb * 2 * pl.slot_rows * pl.hq * dim * 4);
}
size_t part_l_bytes(const Plan& pl) { return round256((size_t)pl.n_ranges * pl.ncb * 2 * pl.slot_rows * pl.hq * 4); }
size_t workspace_for(const Plan& pl, uint32_t dim)
{
    return pl.how != kRanges ? 0 : part_o_bytes(pl, dim) + part_l_bytes(pl) + (size_t)pl.n_ranges * 24;
}

template <class T, class TO, int D>
void launch(const PagedParams& p, hipStream_t s)
{
    const uint32_t xcds = p.n_ranges % 8 == 0 ? 8 : 1;
    const dim3 grid = p.how == kItems ? dim3(p.kv_heads, p.ncb, p.batch) : dim3(xcds, p.ncb, p.n_ranges / xcds);
    if (p.max_new <= p.few)
        hipLaunchKernelGGL((paged_rows<T, TO, D, true>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((paged_rows<T, TO, D, false>), grid, dim3(256), 0, s, p);
    if (p.how != kRanges)
        return;
    const uint32_t nw = p.slot_rows * p.group <= kFewMerged ? 4 : 1, per = (p.slot_rows * p.group * nw * D + 1023) / 1024;
    if (nw == 4)
        hipLaunchKernelGGL((paged_merge<TO, D, 4>), dim3(p.n_ranges * per), dim3(256), 0, s, p, per);
    else
        hipLaunchKernelGGL((paged_merge<TO, D, 1>), dim3(p.n_ranges * per), dim3(256), 0, s, p, per);
}

template <class T, class TO>
void launch_dim(const PagedParams& p, uint32_t dim, hipStream_t s)
{
    if (dim == 64)
        launch<T, TO, 64>(p, s);
    else if (dim == 128)
        launch<T, TO, 128>(p, s);
    else
        launch<T, TO, 256>(p, s);
}

bool valid(const mako_paged_args* a)
{
    return a && a->heads && a->kv_heads && a->heads % a->kv_heads == 0 && a->batch && a->max_new &&
           (a->dim == 64 || a->dim == 128 || a->dim == 256);
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
    // What the split counts: the items, kLead and kTile a tile each (tiles of new rows past max_ctx too).
    const uint32_t R = item_rows(a);
    const uint64_t units = ((uint64_t)a->rows / R + a->batch) * a->kv_heads *
                           (kLead + kTile * (((uint64_t)a->max_ctx + a->max_new + R) / 64 + 2));
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

extern "C" size_t mako_attn_paged_workspace(const mako_paged_args* a)
{
    const uint32_t cus = device_cus();
    return valid(a) && cus ? workspace_for(plan_of(a, cus), a->dim) : 0;
}

extern "C" int mako_attn_paged(const mako_paged_args* a, mako_dtype in, mako_dtype out, const void* q, const void* k,
                               const void* v, const uint32_t* table, const uint32_t* starts, const uint32_t* ctx_len,
                               void* o, float* lse, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* what = "attention_paged";
    if (const int rc = check_args(a, in, out, q, k, v, table, starts, ctx_len, o))
        return rc;
    if (!a->batch || !a->max_new || !a->max_ctx)
        return ok();
    const uint32_t cus = device_cus();
    if (!cus)
        return fail(MAKO_EHIP, "%s: no device to size the split for", what);
    const Plan pl = plan_of(a, cus);
    const size_t need = workspace_for(pl, a->dim);
    if (workspace_bytes < need || (need && !workspace) || !aligned16(workspace))
        return fail(MAKO_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, workspace_bytes,
                    need);
    char* ws = need ? static_cast<char*>(workspace) : nullptr;
    const size_t ob = part_o_bytes(pl, a->dim), lb = part_l_bytes(pl), wb = (size_t)pl.n_ranges * 8;
    const auto at = [&](size_t off) { return ws ? ws + off : nullptr; };
    const PagedParams p{{starts, ctx_len, a->batch, a->rows, a->kv_heads, a->max_new, a->max_ctx, pl.rshift, pl.n_ranges,
                         pl.how, pl.few},
                        q, k, v, table, o, lse, reinterpret_cast<float*>(at(0)), reinterpret_cast<float*>(at(ob)),
                        reinterpret_cast<uint32_t*>(at(ob + lb + 2 * wb)), reinterpret_cast<u32x4*>(at(ob + lb)), a->q_pad,
                        a->heads / a->kv_heads, a->pages, a->kv_heads * a->page * a->dim * 2, log2_of(a->page),
                        a->max_pages, a->width, pl.hq, pl.ncb, pl.slot_rows, pl.hpw - 1,
                        log2_of(pl.hq / pl.hpw), a->scale * kLog2e};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (in == MAKO_BF16 && out == MAKO_F32)
        launch_dim<__bf16, float>(p, a->dim, s);
    else if (in == MAKO_BF16)
        launch_dim<__bf16, __bf16>(p, a->dim, s);
    else if (out == MAKO_F32)
        launch_dim<_Float16, float>(p, a->dim, s);
    else
        launch_dim<_Float16, _Float16>(p, a->dim, s);
    return check_launch(what);
}
