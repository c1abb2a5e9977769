// A paged cache of keys and values and the attention of one new row per sequence over it.
//
// Layout: k and v each [pages][kv_heads][page_size][128], a head's rows of a page behind one another, so that what one
// (sequence, kv head) pair reads of a page is contiguous.  Stored as bf16, or as fp8 (e4m3) or int8 codes with one fp32 scale for each token
// and head in arrays [pages][kv_heads][page_size]: x ~ code * scale.  No counterpart in o1.c, which keeps no keys or values
// from one forward to the next.
#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "../../include/o1_b200.h"


#include <math.h>

namespace o1 {

enum { KV_BF16 = O1_KV_BF16, KV_FP8 = O1_KV_FP8, KV_INT8 = O1_KV_INT8 };
static constexpr int KV_D = 128;
// Codes of the device's table word: what a kernel found in a table on the device.  Nothing is read or written for such an entry, and nothing else stops for it.
static constexpr int ERR_KV_PLACE = 70;    // a slot or page outside the cache
static constexpr int ERR_KV_LENGTH = 71;   // a length that is negative or does not fit its row of the page table

struct KvView {
    uint8_t *k, *v;
    float *ks, *vs;
    int pages, page_shift, page_size, heads;   // page_shift < 0: page_size is no power of two
};

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
__device__ __forceinline__ uint32_t f32_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// To the nearest integers, ties to even, in bytes: the sum with 1.5 * 2^23 has them in its low bits.  (Conversions to and from integers go through a pipe of a
// quarter of the rate.)
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
    constexpr float M = 12582912.0f;
    auto bits = [](float x) { return __float_as_uint(__fadd_rn(x, M)); };      // (x, a product, is rounded by itself)
    return __byte_perm(__byte_perm(bits(a), bits(b), 0x0040), __byte_perm(bits(c), bits(d), 0x0040), 0x5410);
}

// Quantising a row of 128, eight values to each of 16 lanes.  The scale is the row's largest magnitude over the
// largest code (127, or e4m3's 448), so no code saturates and one row's outlier costs no other row anything; codes are x times the
// reciprocal, rounded to nearest even (as are scale and reciprocal, in fp32).  A maximum below 2^-100 counts as 2^-100: its reciprocal stays finite and a
// row of zeros gets codes of zero.  A row with an Inf or NaN gets a NaN scale: it reads as NaN, as its bf16 form would
// carry it into the attention, where int8 has no code for either.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Magnitudes of eight values as bits, the largest in each half of a word.
__device__ __forceinline__ uint32_t magnitudes(const uint4& x) {
    constexpr uint32_t M = 0x7FFF7FFFu;
    return max_u16x2(max_u16x2(x.x & M, x.y & M), max_u16x2(x.z & M, x.w & M));
}
// Of a row's largest magnitude (either half of a word): scale and reciprocal, 0 where there are no codes.
__device__ __forceinline__ float scale_of(uint32_t top, int type, float& inv) {
    top = max(top & 0xFFFFu, top >> 16);
    const bool finite = top < 0x7F80u;
    const float a = fmaxf(__uint_as_float(top << 16), 7.888609052210118e-31f), q = type == KV_INT8 ? 127.0f : 448.0f;
    inv = finite ? __fdiv_rn(q, a) : 0.0f;
    return finite ? __fdiv_rn(a, q) : __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint2 codes_of(const uint4& x, int type, float inv) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    float f[8];
    if (inv == 0.0f) return make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf16lo(w[i]) * inv; f[2 * i + 1] = bf16hi(w[i]) * inv; }
    if (type == KV_INT8) return make_uint2(int8x4(f[0], f[1], f[2], f[3]), int8x4(f[4], f[5], f[6], f[7]));
    return make_uint2(f32_to_e4m3x2(f[0], f[1]) | (f32_to_e4m3x2(f[2], f[3]) << 16), f32_to_e4m3x2(f[4], f[5]) | (f32_to_e4m3x2(f[6], f[7]) << 16));
}
__device__ __forceinline__ uint2 quantise8(const uint4& x, int type, float& scale) {
    uint32_t top = magnitudes(x);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
    float inv;
    scale = scale_of(top, type, inv);
    return codes_of(x, type, inv);
}
__device__ __forceinline__ uint4 dequantise8(const uint2& c, int type, float scale) {
    float f[8];
    const uint32_t w[2] = {c.x, c.y};
    if (type == KV_INT8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)      // (c ^ 0x80) + 2^23 as bits
            f[i] = (__uint_as_float(__byte_perm(w[i >> 2] ^ 0x80808080u, 0x4B000000u, 0x7540 + (i & 3))) - 8388736.0f) * scale;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = f16x2_to_f32(e4m3x2_to_f16x2((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu));
            f[2 * i] = p.x * scale;
            f[2 * i + 1] = p.y * scale;
        }
    }
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    if (VEC) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v) {
    if (VEC) { *reinterpret_cast<uint4*>(p) = v; return; }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { p[2 * i] = (uint16_t)w[i]; p[2 * i + 1] = (uint16_t)(w[i] >> 16); }
}

// A unit is a row's head; a warp has EACH of them, behind one another: keys in the lower 16 lanes, values in the others, eight columns to a lane.  HBM bound for
// many rows: 2 bytes in, 1 (or 2) and the scale out a value.  What the units need is asked for together (a warp of eight has 4 KB on its way), a lane has one
// unit's place and scale, and the maxima are found for all units at once: with four exchanges for each and divisions in every lane the write's instructions
// (135 a unit, now 100) took longer than its bytes, 22.8 us.  Written and read, us: 16640 rows of 8 heads of int8 18.9 + 18.7 (5.5 TB/s), 100000 rows of one head
// 15.2 + 15.1; a row to a warp 23.5 + 19.5 and 43 + 39, a head to a half warp 34 + 35 for the former.  Few rows have more warps with two units: 1800 rows of
// 8 heads 3.5 + 3.7, with eight 5.3 + 4.0; 2600 rows 4.5 + 4.7 and 4.3 + 4.3; 4111 rows 6.9 + 7.5 and 5.8 + 6.2.
// Launches overlap at any size (the next one is let in once the rows have been asked for: its blocks, placed earlier, leave these unevenly spread, 1000 rows 5.1 us, so
// 4.1): written and read through a stream, 4111 rows 14.4 us without, 12.4 with; 16640 42.7 and 38.
static constexpr int KV_EACH = 8, KV_EACH_OF_FEW = 2, KV_FEW_UNITS = 19200;
// A unit's place in a [pages][heads][page_size] array, -1: none.
__device__ __forceinline__ int64_t place(int64_t slot, int head, const KvView& c, int* bad) {
    if (slot < 0) return -1;
    if (slot >= (int64_t)c.pages * c.page_size) { atomicExch(bad, ERR_KV_PLACE); return -1; }
    const int64_t page = c.page_shift >= 0 ? slot >> c.page_shift : slot / c.page_size;
    return (page * c.heads + head) * c.page_size + slot - page * c.page_size;
}
template <bool VEC, int EACH>
__global__ void __launch_bounds__(128, EACH == 8 ? 9 : 12)
kv_write_kernel(KvView c, int type, const uint16_t* __restrict__ k, int64_t ldk, const uint16_t* __restrict__ v, int64_t ldv,
                const int64_t* __restrict__ slots, unsigned units, const int* err, int* bad) {
    grid_dep_wait();
    const unsigned from = (blockIdx.x * 4 + (threadIdx.x >> 5)) * EACH;
    if (from >= units) return;
    const int lane = threadIdx.x & 15, count = min((unsigned)EACH, units - from);
    const bool is_v = threadIdx.x & 16;
    const int mine = lane / (16 / EACH);       // the unit whose place and scale are this lane's
    const unsigned row = from / (unsigned)c.heads, my_row = (from + mine) / (unsigned)c.heads;
    const int64_t slot = mine < count ? slots[my_row] : -1, ld = is_v ? ldv : ldk;
    const int failed = error_word(err);        // rows that a failed kernel should have made stay out of the cache
    int head = from - row * c.heads;
    const uint16_t* src = (is_v ? v : k) + row * ld + lane * 8;
    uint8_t* const base = is_v ? c.v : c.k;
    float* const scales = is_v ? c.vs : c.ks;
    uint4 x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        x[i] = make_uint4(0, 0, 0, 0);
        if (i < count) x[i] = load8<VEC>(src + head * KV_D);
        if (++head == c.heads) { head = 0; src += ld; }
    }
    const int64_t places = place(failed ? -1 : slot, from + mine - my_row * c.heads, c, bad);
    grid_dep_launch();
    float inv = 0.f;
    if (type != KV_BF16) {
        // maxima: a step halves the lanes that a unit is spread over, and, until a lane has one, its units
        uint32_t top[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) top[i] = magnitudes(x[i]);
#pragma unroll
        for (int o = 8, n = EACH / 2; o > 0; o >>= 1, n >>= 1) {
            if (n == 0) top[0] = max_u16x2(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const uint32_t keep = lane & o ? top[n + i] : top[i], give = lane & o ? top[i] : top[n + i];
                top[i] = max_u16x2(keep, __shfl_xor_sync(0xffffffffu, give, o));
            }
        }
        const float scale = scale_of(top[0], type, inv);
        if (places >= 0 && lane % (16 / EACH) == 0) scales[places] = scale;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, places, i * (16 / EACH), 16);
        const float f = __shfl_sync(0xffffffffu, inv, i * (16 / EACH), 16);
        if (at < 0) continue;
        if (type == KV_BF16) reinterpret_cast<uint4*>(base)[at * 16 + lane] = x[i];
        else reinterpret_cast<uint2*>(base)[at * 16 + lane] = codes_of(x[i], type, f);
    }
}

template <bool VEC, int EACH>
__global__ void __launch_bounds__(128, EACH == 8 ? 7 : 12)
kv_read_kernel(KvView c, int type, uint16_t* __restrict__ k, int64_t ldk, uint16_t* __restrict__ v, int64_t ldv,
               const int64_t* __restrict__ slots, unsigned units, int* bad) {
    grid_dep_wait();
    const unsigned from = (blockIdx.x * 4 + (threadIdx.x >> 5)) * EACH;
    if (from >= units) return;
    const int lane = threadIdx.x & 15, count = min((unsigned)EACH, units - from);
    const bool is_v = threadIdx.x & 16;
    const int mine = lane / (16 / EACH);       // the unit whose place and scale are this lane's
    const unsigned row = from / (unsigned)c.heads, my_row = (from + mine) / (unsigned)c.heads;
    const int64_t slot = mine < count ? slots[my_row] : -1, ld = is_v ? ldv : ldk;
    int head = from - row * c.heads;
    uint16_t* dst = (is_v ? v : k) + row * ld + lane * 8;
    const uint8_t* const base = is_v ? c.v : c.k;
    const float* const scales = is_v ? c.vs : c.ks;
    const int64_t places = place(slot, from + mine - my_row * c.heads, c, bad);
    const float scale = type != KV_BF16 && places >= 0 ? scales[places] : 0.f;
    uint4 x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, places, i * (16 / EACH), 16);
        x[i] = make_uint4(0, 0, 0, 0);
        if (at < 0) continue;
        if (type == KV_BF16) { x[i] = reinterpret_cast<const uint4*>(base)[at * 16 + lane]; continue; }
        const uint2 codes = reinterpret_cast<const uint2*>(base)[at * 16 + lane];
        x[i].x = codes.x;
        x[i].y = codes.y;
    }
    grid_dep_launch();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (i >= count) break;
        const float s = __shfl_sync(0xffffffffu, scale, i * (16 / EACH), 16);
        store8<VEC>(dst + head * KV_D, type == KV_BF16 ? x[i] : dequantise8(make_uint2(x[i].x, x[i].y), type, s));
        if (++head == c.heads) { head = 0; dst += ld; }
    }
}

// ------------------------------------------------------------------ attention of a new row
// out = sum_t p_t v_t / sum_t p_t, p_t = exp(scale q . k_t - max): one pass over the keys with a running maximum and sum (in base 2).  HBM bound: every cached
// value is read once and used by the G = heads / kv_heads queries that share it, 2 G multiply-adds for its one or two bytes, so all that counts is that
// enough bytes are on their way at all times, on all SMs, whatever the lengths are.  Measured: 582 MB of fp8 rows (96 sequences of 300 to 5400 tokens, 8 kv heads) in
// 98 us of the GPU, 5.9 TB/s, 91 % of a copy's rate (101 to 109 through the Python call; without a pause 1000 W allow 1620 MHz); 211 MB of int8 (one sequence of 100003) in
// 45.5 us, 4.6 TB/s; 100 MB of bf16 (24 sequences of 1 to 2100) in 25.
// With few bytes the chain of steps counts: 2.3 us until the first loads are asked for (lengths, their sums, parts, pages), 2 for them, 1.3 for the
// warps' join, 3 for that of the teams: 85 tokens of one sequence take 6.0 us, 600 take 8.5.
//
//  * The work is one stream of chunks (16 tokens, 32 of a quantised cache: 8 KB of keys and values) over sequences, kv heads and length.  A block is one SM's; its
//    consumer warps form teams of four, and every team takes a contiguous part of the stream, of equal cost.  How long that is follows from the lengths, which only the
//    device knows: each block sums them up.  (Parts of an equal number of chunks, whatever they hold, kept SMs busy for between 24 and 49 us with the 211 MB.)
//  * A fifth warp of each team does its loading: lane w walks the chunks of consumer warp w (every fourth one of the team's part), looks their pages up a round ahead,
//    and one thread asks for them by TMA, into a ring that each consumer warp has of its own.  So loads run ahead over the ends of sequences, and a consumer
//    does nothing but arithmetic: with loads of its own (cp.async) a chunk of codes was 920 instructions, of which an SM issued 2.3 a clock.  One loading warp
//    for an SM was not enough: 145 us where one for each team took 107.
//  * Products on the tensor cores (mma.sync: at most 16 rows of queries, tcgen05's tiles have 64 at least).  Scores: A = queries (rows = heads), B = keys.
//    Their accumulators are, packed in pairs, the B operand of the second product, A = values transposed (rows = columns of a head).  The operands' k and row
//    indices are permuted so that a thread's part of a key or value row is 16 contiguous bytes, and so that the eight threads which a step of a shared-memory
//    load serves meet eight different sets of banks in TMA's 128-byte swizzle.  The arithmetic alone takes 91 us for the 582 MB, the loads alone 101 (then).
//  * A team's warps join in shared memory.  Where teams share an item - a (sequence, kv head, up to 16 of its query heads) - each leaves its maximum, sum and weighted
//    sum, and the last team to come adds them up (of many: the last of each group, then the last group), always in the order of the teams: the result does not
//    depend on which came when.  Which teams share an item is found while the first rows load, and a warp's heads are joined at once: a head after the
//    other, 16 heads on one kv head took 45 us for 50000 bf16 rows, now 21.  An item costs a team 3.8 us however short it is, so where the table is short and items
//    are many, each goes to one warp, which needs no join (200 sequences of 30 rows of fp8, 8 kv heads: 20 us, now 7.7).
//  * Rounding: scores and sums in fp32.  Probabilities (times v's scale) enter the second product as two parts of bf16, value and rest, 16 bits of significand; codes
//    of a byte are exact in f16 and bf16.  Keys' codes go through f16, which takes fewer instructions, with queries scaled to f16's top by a power of two for each head (those
//    below 2^-29 of its largest lose bits); values' codes through bf16, whose range a probability needs.  The result is rounded once.
// Times below: "batch" 24 sequences of 1 to 2100 rows of bf16, "shared" 32 sequences of 1000 to 3000, 16 query heads on one kv head; us.
static constexpr int KV_STAGE_BYTES = 8192;            // keys and values of a chunk
static constexpr int KV_SEQS = 256;                    // sequences of a launch
static constexpr int KV_TEAM = 4;                      // warps
static constexpr int KV_TEAMS_MAX = 160 * 3;           // what the workspace has room for
// Up to so many teams' parts of an item are joined at once (a part to a lane), more in groups of so many: 100003 tokens, 55 parts to an item, in two steps 48.1 us, at once 50.8 (then).
static constexpr int KV_FLAT = 32, KV_FAN = 16;
// What an item costs a team beside its chunks (the warps' join, the next queries), in chunks: 4, 7, 10, 12: batch 26.1, 25.5, 24.9, 24.5, shared 22.5, 20.0, 18.1, 17.8,
// 582 MB 97.4, 97.1, 96.9, 97.6.
static constexpr int KV_ITEM_COST = 10;
// Items of so few chunks are not cut: 9 sequences of up to 1999 rows of fp8, 16 kv heads: 16 or 24 18, 48 26; 60 of 100 to 900 rows of int8: 16 18.3, 24 19.8.
// Nor are those of a quarter of a team's part (half: 582 MB 104), and, where there are no more items than teams, of up to half more cost than a team has on average:
// 51 sequences of 304 rows of bf16, 8 kv heads, 16.0, cut 20.6; 54 of 1000 of fp8 24.7 and 30.5; 55 of 100 to 700 of bf16 23.0 and 24.3.
static constexpr int KV_KEEP = 16;
static constexpr int KV_SOLO = 16;                     // chunks of an item that a warp can have for itself (no item of KV_KEEP chunks is cut)
static_assert(KV_SOLO <= KV_KEEP, "an item of a warp is whole");
static constexpr int KV_JOIN_BYTES = 8192;             // of a team
static constexpr int KV_JOIN_STEP = 4;                 // parts that a join has under way (of all a warp's heads; two take 1 us longer for 16 heads; eight spill registers of all types, four of bf16 only)
static constexpr int ERR_KV_WAIT = 72;                 // a wait of the attention kernel ran out
static constexpr float KV_LIFT = 20.0f;                // probabilities are relative to 2^-20 of the largest: those that fp32 has no value for are 2^-146 and less of it

struct KvAttn {
    KvView c;
    const uint16_t *q, *kn, *vn;
    int64_t ldq, ldk, ldv, ldp, ldo;
    const int32_t *pages, *lens;
    uint16_t* out;
    float* lse;
    unsigned* arrived;     // [2][team][2] teams that have come, of a group whose first part that is; groups that have come
    float2* stats;         // [team][2][heads of an item] maximum and sum of a team's first and last part of an item
    float* parts;          // [team][2][heads of an item][128] weighted sum
    int batch, heads, group, chunks_of_heads, per_item, width, flags;    // flags: 1 = queries in 16-byte pieces, 2 = results, 4 = new rows; 8 = a box of the maps is a whole chunk's rows
    float scale;
    int *err, *bad;        // the device's error and table words
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int TYPE>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (TYPE == KV_BF16) mma_bf16(d, a0, a1, a2, a3, b0, b1);
    else mma_f16(d, a0, a1, a2, a3, b0, b1);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two values as bf16, and what is left of them as another two.
__device__ __forceinline__ void two_parts(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_bf16x2(a, b);
    lo = pack_bf16x2(a - bf16lo(hi), b - bf16hi(hi));
}
template <int SEL>
__device__ __forceinline__ uint32_t prmt(uint32_t x, uint32_t y) {      // (a selector's top bit: the byte's sign, eight times)
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "n"(SEL));
    return r;
}
// Codes J of two words as a pair of bf16, exactly.  e4m3: sign and the seven bits behind it in a bf16's places are the value
// times 2^-120, subnormal codes too.  int8: behind the exponent of 128, a code's seven low bits are 128 + bits and its top bit is 128 or 256.
template <int TYPE, int J>
__device__ __forceinline__ uint32_t pair_to_bf16(uint32_t x, uint32_t y) {
    uint32_t r;
    if (TYPE == KV_FP8) {
        const uint32_t s = (prmt<J | (8 | J) << 4 | (4 | J) << 8 | (12 | J) << 12>(x, y) << 4) & 0x87F087F0u;
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(s), "r"(0x7B807B80u));
    } else {
        const uint32_t z = prmt<(J < 2 ? 0x5140 : 0x7362)>(x, y), s = prmt<(J & 1) ? 0x4342 : 0x4140>(z, 0x43434343u);
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(s & 0xFF7FFF7Fu), "r"(s & 0xFF80FF80u));
    }
    return r;
}
// Four codes of a byte as two pairs of f16, exactly.  int8: c ^ 0x80 behind the exponent of 1024 is 1024 + 128 + c.
template <int TYPE>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (TYPE == KV_FP8) {
        lo = e4m3x2_to_f16x2(w & 0xFFFFu);
        hi = e4m3x2_to_f16x2(w >> 16);
    } else {
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        asm("add.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0xE480E480u));   // - 1152
        asm("add.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0xE480E480u));
    }
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void team_sync(int team) { asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(KV_TEAM * 32) : "memory"); }
// Of eight: 0 2 4 6 1 3 5 7's inverse.  Rows kv_perm(2m) and kv_perm(2m + 1) lie four apart, as the swizzle wants them.
__device__ __forceinline__ int kv_perm(int i) { return (i >> 1) | (i & 1) << 2; }

template <int TYPE, int HG>
struct KvKernel {
    static constexpr int KEYS = TYPE == KV_BF16 ? 16 : 32, ROWB = TYPE == KV_BF16 ? 256 : 128, TILES = KEYS / 8;
    static constexpr int TEAMS = HG == 1 ? 3 : 2, WARPS = KV_TEAM * TEAMS, STAGES = HG == 1 ? 2 : 3, THREADS = (WARPS + TEAMS) * 32;
    // (HG == 1: 128 registers and 24 slots of 8 KB; HG == 2 holds twice the queries and sums: 168 registers, two teams, again 24 slots)
    // shared memory: the rings, their scales, the teams' join buffers, then Shared
    static constexpr int SCALES = WARPS * STAGES * KV_STAGE_BYTES, JOIN = SCALES + (TYPE == KV_BF16 ? 0 : WARPS * STAGES * 256), SHARED = JOIN + TEAMS * KV_JOIN_BYTES;
    struct Share { int first, here, fan, item, groups, b, head0, heads; };        // a part's group begins at part `first` and has `here` (0: no part), its item at part `item`
    struct Segment { int b, item, first, begin, end, n; };        // first: the item's first chunk; begin ... end - 1: the team's
    struct Shared {
        uint64_t full[WARPS][STAGES], empty[WARPS][STAGES];
        Segment seg[TEAMS][2];
        Share share[TEAMS][2];
        int prefix[KV_SEQS + 1], cost[KV_SEQS], len[KV_SEQS], last[TEAMS][2];      // chunks and costs before a sequence
        int rows[WARPS][STAGES][2];       // where the cache has a chunk's rows, 16 at a time, if new ones may go there, else negative
        int2 scan[WARPS + TEAMS];
        float m[TEAMS][KV_TEAM][8 * HG], l[TEAMS][KV_TEAM][8 * HG];
    };
    static constexpr int SMEM = SHARED + (int)sizeof(Shared);
};

// Position in the stream: chunk c of n of item `item` of sequence b.  Items are (kv head, up to 16 of its query heads) pairs.
struct KvWalk {
    int b, item, c, n;
    // the chunk f
    __device__ __forceinline__ void seek(int f, const int* prefix, int batch, int items) {
        int lo = 0, hi = batch - 1;       // the last sequence that begins at or before f; it is no empty one: the next one begins behind it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] * items <= f) lo = mid; else hi = mid - 1;
        }
        b = lo;
        n = prefix[lo + 1] - prefix[lo];
        item = (f - prefix[lo] * items) / n;
        c = f - prefix[lo] * items - item * n;
    }
    __device__ __forceinline__ void step(int by, const int* prefix, int items) {       // not past the stream's end
        c += by;
        while (c >= n) {
            c -= n;
            if (++item < items) continue;
            item = 0;
            do { ++b; n = prefix[b + 1] - prefix[b]; } while (n == 0);
        }
    }
};

// Sums of v over the block's threads before this one, and over all, of both components.
template <int WARPS>
__device__ __forceinline__ int2 block_scan(int2 v, int2& all, int2* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
        if (lane >= o) { sum.x += x; sum.y += y; }
    }
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    int2 before = make_int2(sum.x - v.x, sum.y - v.y);
    all = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const int2 p = part[w];
        if (w < warp) { before.x += p.x; before.y += p.y; }
        all.x += p.x;
        all.y += p.y;
    }
    return before;
}

__device__ __forceinline__ void store_row4(uint16_t* dst, const float4& v, float f, bool vec) {
    const uint2 r = make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
    if (vec) { *reinterpret_cast<uint2*>(dst) = r; return; }
    dst[0] = (uint16_t)r.x; dst[1] = (uint16_t)(r.x >> 16); dst[2] = (uint16_t)r.y; dst[3] = (uint16_t)(r.y >> 16);
}

// Whether this thread is the last of `wanted` to come, each with what its team has written before a barrier; the counter is then as it was.
__device__ __forceinline__ bool all_came(unsigned* counter, int wanted) {
    unsigned seen;
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    asm volatile("atom.relaxed.gpu.global.add.u32 %0, [%1], 1;" : "=r"(seen) : "l"(counter) : "memory");
    if (seen != (unsigned)(wanted - 1)) return false;
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    *counter = 0;
    return true;
}

// The sums of `count` parts of HEADS heads (head, head + KV_TEAM, ... below `heads`), by a warp: the first part is `first`, the others in slot 0 of every `stride`-th
// team behind it.  Into the result, or (to_out false) into the first one's place.  A lane has a part's weights; the first parts' rows are under way while the
// weights are, and all heads' at once.
template <int HEADS>
__device__ __forceinline__ void kv_join(const KvAttn& a, int first, int stride, int count, int b, int head, int heads, int head0, bool to_out) {
    static_assert(KV_FLAT <= 32 && KV_FAN <= 32 && (KV_TEAMS_MAX + KV_FAN - 1) / KV_FAN <= 32, "a part to a lane");
    const int lane = threadIdx.x & 31;
    const int64_t step = (int64_t)2 * stride * a.per_item, at0 = (int64_t)first * a.per_item + head, at1 = (int64_t)(first & ~1) * a.per_item + head;
    float4* const mine = reinterpret_cast<float4*>(a.parts) + at0 * (KV_D / 4) + lane;
    const float4* src = reinterpret_cast<const float4*>(a.parts) + at1 * (KV_D / 4) + lane;
    float2 s[HEADS];
    const float2* const stats = a.stats + (lane == 0 ? at0 : at1 + lane * step);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        s[h] = make_float2(-INFINITY, 0.f);
        if (lane < count && head + h * KV_TEAM < heads) s[h] = __ldcg(stats + h * KV_TEAM);
    }
    float top[HEADS], sum[HEADS], w[HEADS];
    float4 r[HEADS];
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += KV_JOIN_STEP, src += KV_JOIN_STEP * step * (KV_D / 4)) {
        float4 x[KV_JOIN_STEP][HEADS];
#pragma unroll
        for (int i = 0; i < KV_JOIN_STEP; ++i) {
            const float4* const from = i0 + i == 0 ? mine : src + i * step * (KV_D / 4);
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                x[i][h] = make_float4(0, 0, 0, 0);
                if (i0 + i < count && head + h * KV_TEAM < heads) x[i][h] = __ldcg(from + h * (KV_TEAM * KV_D / 4));
            }
        }
        if (i0 == 0) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                r[h] = make_float4(0, 0, 0, 0);
                top[h] = s[h].x;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
                w[h] = exp2_fast(s[h].x - (top[h] == -INFINITY ? 0.f : top[h]));
                sum[h] = s[h].y * w[h];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
            }
        }
#pragma unroll
        for (int i = 0; i < KV_JOIN_STEP; ++i) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                const float f = __shfl_sync(0xffffffffu, w[h], i0 + i);
                if (i0 + i < count) { r[h].x += x[i][h].x * f; r[h].y += x[i][h].y * f; r[h].z += x[i][h].z * f; r[h].w += x[i][h].w * f; }
            }
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        const int at = head + h * KV_TEAM;
        if (at >= heads) break;
        if (to_out) {
            store_row4(a.out + b * a.ldo + (head0 + at) * KV_D + lane * 4, r[h], 1.0f / sum[h], a.flags & 2);
            if (a.lse && lane == 0) a.lse[(int64_t)b * a.heads + head0 + at] = (top[h] - KV_LIFT + log2f(sum[h])) * 0.6931471805599453f;
        } else {
            mine[h * (KV_TEAM * KV_D / 4)] = r[h];
            if (lane == 0) a.stats[at0 + h * KV_TEAM] = make_float2(top[h], sum[h]);
        }
    }
}

// solo: items of at most KV_SOLO chunks, each to one warp; "teams" are then warps.
template <int TYPE, int HG, bool solo>
__global__ void __launch_bounds__(KvKernel<TYPE, HG>::THREADS, 1)
kv_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ KvAttn a) {
    using K = KvKernel<TYPE, HG>;
    constexpr int KEYS = K::KEYS, TILES = K::TILES, WARPS = K::WARPS, STAGES = K::STAGES;
    extern __shared__ __align__(1024) uint8_t smem[];
    auto& sh = *reinterpret_cast<typename K::Shared*>(smem + K::SHARED);
    const int warp = warp_index(), lane = threadIdx.x & 31, tid = threadIdx.x;
    if (tid < WARPS * STAGES) {
        mbar_init(&sh.full[0][0] + tid, 1);
        mbar_init(&sh.empty[0][0] + tid, 1);
        fence_mbar_init();
    }
    if (warp >= WARPS && elect_one()) { tma_prefetch_desc(&k_map); tma_prefetch_desc(&v_map); }
    grid_dep_launch();
    grid_dep_wait();

    // ---- the lengths, as numbers of chunks, summed up
    const int ps = a.c.page_size, shift = a.c.page_shift, items = a.c.heads * a.chunks_of_heads;
    int total, cost, all_chunks, sequences;
    {
        static_assert(KV_SEQS <= K::THREADS, "a sequence to a thread");
        int len = tid < a.batch ? a.lens[tid] : 0;
        // a short page table into L1 meanwhile, a line to a thread (0.1 to 0.2 us of a call)
        const int lines = (a.width + 31) >> 5;
        if (tid < a.batch * lines) {
            int entry;
            const int b = tid / lines;
            asm volatile("ld.global.ca.b32 %0, [%1];" : "=r"(entry) : "l"(a.pages + b * a.ldp + (tid - b * lines) * 32));
        }
        if (len < 0 || len > (int64_t)a.width * ps) { atomicExch(a.bad, ERR_KV_LENGTH); len = 0; }
        const int n = (len + KEYS - 1) / KEYS;
        int2 all;
        const int2 before = block_scan<WARPS + K::TEAMS>(make_int2(n, n > 0 ? n + KV_ITEM_COST : 0), all, sh.scan);
        if (tid < a.batch) { sh.prefix[tid] = before.x; sh.cost[tid] = before.y; sh.len[tid] = len; }
        if (tid == 0) sh.prefix[a.batch] = all.x;
        all_chunks = all.x;
        sequences = (all.y - all.x) / KV_ITEM_COST;      // that are not empty
        total = all.x * items;
        cost = all.y * items;
        __syncthreads();
    }
    // ---- a team's part of the stream: equal costs, where each item costs some chunks more than it has; ends inside an item that is not worth a join are moved
    // (A team has at least four chunks, one to a warp; eight where sequences are long, which halves the parts to join: one sequence of 2000 rows of bf16 10.3 us, with four
    // 11.7; of 600 rows 9.1 and 8.5.)
    const int least = all_chunks > 48 * sequences ? 2 * KV_TEAM : KV_TEAM, most = gridDim.x * K::TEAMS, wanted = sequences * items;
    const int teams = solo ? min(KV_TEAM * most, wanted) : min(most, max((total + least - 1) / least, wanted));       // (solo: warps)
    const int share = teams > 0 ? total / teams : 0, each = teams > 0 ? cost / teams : 0, over = cost - each * teams;
    const int keep = max(KV_KEEP, wanted <= most ? each + (each >> 1) - KV_ITEM_COST : share >> 2);
    auto cost_of = [&](int id) { return each * id + over * id / teams; };         // cost * id / teams, in 32 bits (over and id are below 1921)
    auto begin_of = [&](int id) {
        if (id >= teams) return total;
        const int at = cost_of(id);
        int lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sh.cost[mid] * items <= at) lo = mid; else hi = mid - 1;
        }
        const int n = sh.prefix[lo + 1] - sh.prefix[lo], rel = at - sh.cost[lo] * items, item = rel / (n + KV_ITEM_COST);
        int c = rel - item * (n + KV_ITEM_COST);
        if (n <= keep) c = 2 * c < n + KV_ITEM_COST ? 0 : n;      // the nearer end
        else c = min(c, n);
        return sh.prefix[lo] * items + item * n + c;
    };
    auto part_of = [&](int id, int lane, int& c0, int& c1) {        // both ends at once
        const int at = begin_of(id + (lane & 1));
        c0 = __shfl_sync(0xffffffffu, at, 0);
        c1 = __shfl_sync(0xffffffffu, at, 1);
    };

    if (warp >= WARPS) {
        // ---- the team's loading warp
        const int team = warp - WARPS, id = team * gridDim.x + blockIdx.x;
        // (solo: lane w has the part of warp w)
        const int by = solo ? 1 : KV_TEAM, at_end = begin_of((solo ? (team * KV_TEAM + (lane >> 1 & 3)) * gridDim.x + blockIdx.x : id) + (lane & 1));
        int f = __shfl_sync(0xffffffffu, at_end, solo ? lane * 2 & 7 : 0), c1 = __shfl_sync(0xffffffffu, at_end, solo ? (lane * 2 & 7) + 1 : 1), place[2] = {-1, -1};
        if (!solo) f += lane;
        if (lane >= KV_TEAM) c1 = 0;
        KvWalk at = {};
        auto look = [&]() {        // the chunk's rows of the cache, 16 at a time; -1: none, -2: a page outside the cache
            const int tok = at.c * KEYS, len = sh.len[at.b], head = a.chunks_of_heads == 1 ? at.item : at.item / a.chunks_of_heads;
#pragma unroll
            for (int h = 0; h < KEYS / 16; ++h) {
                const int token = tok + 16 * h, p = shift >= 0 ? token >> shift : token / ps;
                place[h] = -1;
                if (token >= len) continue;
                const int page = a.pages[at.b * a.ldp + p];
                place[h] = -2;
                if ((unsigned)page >= (unsigned)a.c.pages) atomicExch(a.bad, ERR_KV_PLACE);
                else place[h] = (page * a.c.heads + head) * ps + token - p * ps;
            }
        };
        const int failed = a.kn ? error_word(a.err) : 0;       // a kernel before this one: no row goes into the cache
        if (f < c1) { at.seek(f, sh.prefix, a.batch, items); look(); }
        bool ok = true;
        int issued = 0;          // of the lane's warp
        for (int round = 0; ok; ++round) {
            unsigned left = __ballot_sync(0xffffffffu, f < c1);
            if (!left) break;
            const int now[2] = {place[0], place[1]}, slot = round % STAGES;
            f += by;
            if (f < c1) { at.step(by, sh.prefix, items); look(); }
            for (; left && ok; left &= left - 1) {
                const int mate = __ffs(left) - 1, w = team * KV_TEAM + mate, p0 = __shfl_sync(0xffffffffu, now[0], mate), p1 = KEYS == 32 ? __shfl_sync(0xffffffffu, now[1], mate) : -1;
                uint64_t* const full = &sh.full[w][slot];
                if (elect_one()) {
                    ok = mbar_wait(&sh.empty[w][slot], ((round / STAGES) & 1) ^ 1);
                    if (!ok) atomicExch(a.err, ERR_KV_WAIT);
                    else {
                        if (a.kn) { sh.rows[w][slot][0] = failed ? -1 : p0; sh.rows[w][slot][1] = failed ? -1 : p1; }
                        const int r0 = max(p0, 0), r1 = p1 == -2 ? 0 : p1;       // (of a page outside, the cache's first rows are loaded)
                        uint8_t* const dst = smem + (w * STAGES + slot) * KV_STAGE_BYTES;
                        const uint32_t scales = smem_u32(smem) + K::SCALES + (w * STAGES + slot) * 256;
                        if (TYPE == KV_BF16) {
                            mbar_expect_tx(full, 8192);
                            tma_load_2d(dst, &k_map, full, 0, r0);
                            tma_load_2d(dst + 2048, &k_map, full, 64, r0);
                            tma_load_2d(dst + 4096, &v_map, full, 0, r0);
                            tma_load_2d(dst + 6144, &v_map, full, 64, r0);
                        } else if (a.flags & 8) {
                            mbar_expect_tx(full, 8192 + 256);
                            tma_load_2d(dst, &k_map, full, 0, r0);
                            tma_load_2d(dst + 4096, &v_map, full, 0, r0);
                            bulk_load(scales, a.c.ks + r0, 128, full);
                            bulk_load(scales + 128, a.c.vs + r0, 128, full);
                        } else {
                            mbar_expect_tx(full, r1 >= 0 ? 8192 + 256 : 4096 + 128);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int r = h ? r1 : r0;
                                if (r < 0) break;
                                tma_load_2d(dst + h * 2048, &k_map, full, 0, r);
                                tma_load_2d(dst + 4096 + h * 2048, &v_map, full, 0, r);
                                bulk_load(scales + h * 64, a.c.ks + r, 64, full);
                                bulk_load(scales + 128 + h * 64, a.c.vs + r, 64, full);
                            }
                        }
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (lane == mate && ok) ++issued;
            }
        }
        // Copies land before the block ends, also where a consumer has given up waiting for them: its shared memory is another block's then.
        if (lane < KV_TEAM)
            for (int r = max(0, issued - STAGES); r < issued; ++r) mbar_wait(&sh.full[team * KV_TEAM + lane][r % STAGES], (r / STAGES) & 1);
        return;
    }

    const int team = warp / KV_TEAM, mate = warp % KV_TEAM, g = lane >> 2, t = lane & 3, gp = kv_perm(g), id = team * gridDim.x + blockIdx.x;
    // ---- sequences without rows
    for (int b = id; b < a.batch; b += gridDim.x * K::TEAMS) {
        if (sh.len[b] > 0) continue;
        for (int i = mate * 32 + lane; i < a.heads * KV_D; i += KV_TEAM * 32) a.out[b * a.ldo + i] = 0;
        if (a.lse) for (int i = mate * 32 + lane; i < a.heads; i += KV_TEAM * 32) a.lse[(int64_t)b * a.heads + i] = -INFINITY;
    }
    int c0, c1;
    part_of(solo ? (team * KV_TEAM + mate) * gridDim.x + blockIdx.x : id, lane, c0, c1);
    if (c0 >= c1) return;

    auto head_of = [&](int item) {         // the first query head of an item
        const int kvh = a.chunks_of_heads == 1 ? item : item / a.chunks_of_heads;
        return kvh * a.group + (item - kvh * a.chunks_of_heads) * (8 * HG);
    };
    auto heads_of = [&](int item) { return a.chunks_of_heads == 1 ? a.group : min(8 * HG, a.group - item % a.chunks_of_heads * (8 * HG)); };
    // queries: rows g (and g + 8) of the A operand; the 16-byte pieces 4i + t of a key row are this thread's.  Up to four heads are there twice: rows 4 to 7 of the
    // probabilities are then the second parts of rows 0 to 3, and one product has both (582 MB of fp8 without a pause, at the 1620 MHz that 1000 W allow: 107 us, with two
    // products 109.5; a chunk of bf16 has half as many products, and gains nothing)
    const bool twice = HG == 1 && TYPE != KV_BF16 && a.group <= 4;
    const bool second = twice && g >= 4;
    uint32_t qa[HG][16];
    auto ask_queries = [&](int b, int item) {
        const int head0 = head_of(item), heads = heads_of(item);
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            const int row = twice ? g & 3 : g + 8 * h;
            const bool on = row < heads;
            const uint16_t* src = a.q + b * a.ldq + (head0 + row) * KV_D;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = TYPE == KV_BF16 ? (4 * i + t) * 8 : (4 * (i >> 1) + t) * 16 + (i & 1) * 8;
                const uint4 v = !on ? make_uint4(0, 0, 0, 0) : (a.flags & 1) ? load8<true>(src + at) : load8<false>(src + at);
                qa[h][4 * i] = v.x; qa[h][4 * i + 1] = v.y; qa[h][4 * i + 2] = v.z; qa[h][4 * i + 3] = v.w;
            }
        }
    };
    // segments: what the team has of one item; the first warp writes the next one down while all work on this one (solo: each warp its own)
    auto describe = [&](int f, typename K::Segment& to) {
        KvWalk at;
        at.seek(f, sh.prefix, a.batch, items);
        if (lane == 0) to = {at.b, at.item, f - at.c, f, min(c1, f - at.c + at.n), at.n};
    };
    typename K::Segment* const segs = solo ? reinterpret_cast<typename K::Segment*>(smem + K::JOIN) + 2 * warp : sh.seg[team];      // (solo: where no warps are joined)
    auto together = [&]() { if (solo) __syncwarp(); else team_sync(team); };
    if (solo || mate == 0) describe(c0, segs[0]);
    together();
    ask_queries(segs[0].b, segs[0].item);
    if (!solo && mate == KV_TEAM - 1 && lane < 2) {
        // the items that the team's part begins and ends in, while the first rows are under way: teams from ... to share one, in groups of `fan`; the first
        // one's part is in slot `late`
        KvWalk w;
        w.seek(lane ? c1 - 1 : c0, sh.prefix, a.batch, items);
        const int f0 = (lane ? c1 - 1 : c0) - w.c;
        typename K::Share& to = sh.share[team][lane];
        if ((c0 <= f0 && f0 + w.n <= c1) || (lane && f0 <= c0)) to.here = 0;         // whole, or slot 0's
        else {
            const int at = sh.cost[w.b] * items + w.item * (w.n + KV_ITEM_COST);
            auto owner = [&](int v) {
                int o = min(teams - 1, (int)((float)v * ((float)teams / (float)cost)));
                while (cost_of(o) > v) --o;
                while (o + 1 < teams && cost_of(o + 1) <= v) ++o;
                return o;
            };
            const int from = owner(at), last = owner(at + w.n - 1), late = f0 != begin_of(from), count = last - from + 1;
            const int fan = count <= KV_FLAT ? count : KV_FAN, mine = (id - from) / fan, first = 2 * (from + mine * fan) + (mine == 0 ? late : 0);
            to = {first, min(fan, count - mine * fan), fan, 2 * from + late, (count + fan - 1) / fan, w.b, head_of(w.item), heads_of(w.item)};
        }
    }
    float* const buf = reinterpret_cast<float*>(smem + K::JOIN + team * KV_JOIN_BYTES);
    const int by = solo ? 1 : KV_TEAM;
    int f = solo ? c0 : c0 + mate, slot = 0, parity = 0;
    bool ok = true;
#pragma unroll 1
    for (int k = 0;; ++k) {
        const typename K::Segment seg = segs[k & 1];
        if ((solo || mate == 0) && seg.end < c1) describe(seg.end, segs[(k + 1) & 1]);
        float z_scale[HG], acc[HG][8][4], m[HG], l[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            z_scale[h] = a.scale * 1.4426950408889634f;
            if (TYPE != KV_BF16) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) top = max(top, max(qa[h][i] & 0x7FFFu, (qa[h][i] >> 16) & 0x7FFFu));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the largest one to between 2^15 and 2^16, the top of f16's range: values down to 2^-29 of it keep their eight bits, so that a large one
                // whose keys are small costs the others nothing
                const uint32_t e = min(max(top >> 7, 16u), 254u);         // the largest one's exponent
                const float down = __uint_as_float((269u - e) << 23);
                z_scale[h] *= __uint_as_float(e << 23);              // (the 2^15 goes with the keys' scales, which keeps scores as far from fp32's end as they were)
#pragma unroll
                for (int i = 0; i < 16; ++i) qa[h][i] = pack_f16x2(bf16lo(qa[h][i]) * down, bf16hi(qa[h][i]) * down);
            }
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[h][j][0] = acc[h][j][1] = acc[h][j][2] = acc[h][j][3] = 0.f;
        }

        int valid = sh.len[seg.b] - (f - seg.first) * KEYS;       // rows that the sequence has from the warp's chunk on
#pragma unroll 1
        for (; f < seg.end; f += by, valid -= by * KEYS) {
            const uint32_t st = smem_u32(smem) + (warp * STAGES + slot) * KV_STAGE_BYTES, scales = smem_u32(smem) + K::SCALES + (warp * STAGES + slot) * 256;
            const bool append = a.kn && valid <= KEYS;
            uint4 fresh = make_uint4(0, 0, 0, 0);
            if (append) {
                const int kvh = a.chunks_of_heads == 1 ? seg.item : seg.item / a.chunks_of_heads;
                const uint16_t* src = (lane < 16 ? a.kn + seg.b * a.ldk : a.vn + seg.b * a.ldv) + kvh * KV_D + (lane & 15) * 8;
                fresh = (a.flags & 4) ? load8<true>(src) : load8<false>(src);
            }
            if (ok && !mbar_wait(&sh.full[warp][slot], parity)) { ok = false; atomicExch(a.err, ERR_KV_WAIT); }
            __syncwarp();
            if (append) {     // the sequence's last row is the new one: into the ring, and into the cache
                const int r = valid - 1, part = lane & 15, row = ok ? sh.rows[warp][slot][r >> 4] : -1;
                const bool store = (a.chunks_of_heads == 1 || seg.item % a.chunks_of_heads == 0) && row >= 0;
                const int64_t at = (int64_t)row + (r & 15);
                const uint32_t dst = st + (lane < 16 ? 0 : 4096) + r * 128;
                uint8_t* const base = lane < 16 ? a.c.k : a.c.v;
                if (TYPE == KV_BF16) {
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (part >> 3) * 2048 + (((part & 7) ^ (r & 7)) << 4)), "r"(fresh.x), "r"(fresh.y), "r"(fresh.z), "r"(fresh.w) : "memory");
                    if (store) reinterpret_cast<uint4*>(base)[at * 16 + part] = fresh;
                } else {
                    float sc;
                    const uint2 codes = quantise8(fresh, TYPE, sc);
                    asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(dst + (((part >> 1) ^ (r & 7)) << 4) + (part & 1) * 8), "r"(codes.x), "r"(codes.y) : "memory");
                    if (part == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + (lane >> 4) * 128 + r * 4), "f"(sc) : "memory");
                    if (store) {
                        reinterpret_cast<uint2*>(base)[at * 16 + part] = codes;
                        if (part == 0) (lane < 16 ? a.c.ks : a.c.vs)[at] = sc;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
            }

            // scores of 8 keys a tile; a tile's column n is its key kv_perm(n), so keys t and t + 4 are this thread's
            float s[TILES][4];
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                const uint32_t row = st + n * 1024 + gp * 128;
#pragma unroll
                for (int i = 0; i < (TYPE == KV_BF16 ? 4 : 2); ++i) {
                    const uint4 k = lds128(row + (i >> 1) * 2048 + (((4 * (i & 1) + t) ^ gp) << 4));
                    const uint32_t w[4] = {k.x, k.y, k.z, k.w};
                    if (TYPE == KV_BF16) {
#pragma unroll
                        for (int j = 0; j < 4; j += 2)
                            mma16<TYPE>(s[n], qa[0][4 * i + j], HG == 2 ? qa[HG - 1][4 * i + j] : 0, qa[0][4 * i + j + 1], HG == 2 ? qa[HG - 1][4 * i + j + 1] : 0, w[j], w[j + 1]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t b0, b1;
                            codes_to_f16<TYPE>(w[j], b0, b1);
                            mma16<TYPE>(s[n], qa[0][8 * i + 2 * j], HG == 2 ? qa[HG - 1][8 * i + 2 * j] : 0, qa[0][8 * i + 2 * j + 1], HG == 2 ? qa[HG - 1][8 * i + 2 * j + 1] : 0, b0, b1);
                        }
                    }
                }
            }
            float vs[TILES][2];
            if (TYPE != KV_BF16) {
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float ks = lds_f32(scales + (8 * n + 4 * j + t) * 4) * 3.0517578125e-05f;      // 2^-15
                        vs[n][j] = lds_f32(scales + 128 + (8 * n + 4 * j + t) * 4);
#pragma unroll
                        for (int h = 0; h < HG; ++h) s[n][2 * h + j] *= ks;
                    }
                }
            }
            if (valid < KEYS) {        // what the memory behind a sequence holds, NaN too, takes no part
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (8 * n + 4 * j + t < valid) continue;
                        vs[n][j] = 0.f;
#pragma unroll
                        for (int h = 0; h < HG; ++h) s[n][2 * h + j] = -INFINITY;
                    }
                }
            }
            // running maximum and sum; a tile's accumulators become the probabilities
            float alpha[HG];
            bool moved = false;
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) top = fmaxf(top, s[n][2 * h + j]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m[h], top * z_scale[h]), ref = (m_new == -INFINITY ? 0.f : m_new) - KV_LIFT;
                alpha[h] = exp2_fast(m[h] - KV_LIFT - ref);
                moved = moved || alpha[h] != 1.f;
                m[h] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) { s[n][2 * h + j] = exp2_fast(__fmaf_rn(s[n][2 * h + j], z_scale[h], -ref)); sum += s[n][2 * h + j]; }
                }
                l[h] = l[h] * alpha[h] + sum;
                if (TYPE != KV_BF16) {
#pragma unroll
                    for (int n = 0; n < TILES; ++n) { s[n][2 * h] *= vs[n][0]; s[n][2 * h + 1] *= vs[n][1]; }
                }
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    const float a0 = __shfl_sync(0xffffffffu, alpha[h], 8 * t), a1 = __shfl_sync(0xffffffffu, alpha[h], 8 * t + 4);
#pragma unroll
                    for (int j = 0; j < 8; ++j) { acc[h][j][0] *= a0; acc[h][j][1] *= a1; acc[h][j][2] *= a0; acc[h][j][3] *= a1; }
                }
            }
            // out^T += V^T P^T, 16 keys a step: this thread's rows are keys t, t + 4, t + 8, t + 12
#pragma unroll
            for (int u = 0; u < KEYS / 16; ++u) {
                uint32_t p_hi[HG][2], p_lo[HG][2];
#pragma unroll
                for (int h = 0; h < HG; ++h) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        two_parts(s[2 * u + j][2 * h], s[2 * u + j][2 * h + 1], p_hi[h][j], p_lo[h][j]);
                        if (second) p_hi[h][j] = p_lo[h][j];
                    }
                }
                constexpr int PIECES = TYPE == KV_BF16 ? 2 : 1;
                uint4 v[4][PIECES];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
#pragma unroll
                    for (int i = 0; i < PIECES; ++i)
                        v[r][i] = lds128(st + 4096 + (u + i) * 2048 + (t + 4 * r) * 128 + ((gp ^ (t + 4 * (r & 1))) << 4));
                }
                if (valid < KEYS) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (u * 16 + t + 4 * r < valid) continue;
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) v[r][i] = make_uint4(0, 0, 0, 0);
                    }
                }
                // pairs of keys (t, t + 4), (t + 8, t + 12), of the columns that a word of each row holds: bf16 8 gp + 2 w, + 1 and 64 + those, codes 16 gp + 4 w ... + 3 and 8 + those
                constexpr int EACH = TYPE == KV_BF16 ? 2 : 4;
#pragma unroll
                for (int w = 0; w < 8 / EACH; ++w) {
                    uint32_t pair[2][2][EACH];       // [keys][columns' half]
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint4 x4 = v[2 * r][TYPE == KV_BF16 ? half : 0], y4 = v[2 * r + 1][TYPE == KV_BF16 ? half : 0];
                            const int at = TYPE == KV_BF16 ? w : w + 2 * half;
                            const uint32_t x = at == 0 ? x4.x : at == 1 ? x4.y : at == 2 ? x4.z : x4.w, y = at == 0 ? y4.x : at == 1 ? y4.y : at == 2 ? y4.z : y4.w;
                            if (TYPE == KV_BF16) {
                                pair[r][half][0] = __byte_perm(x, y, 0x5410);
                                pair[r][half][1] = __byte_perm(x, y, 0x7632);
                            } else {
                                pair[r][half][0] = pair_to_bf16<TYPE, 0>(x, y);
                                pair[r][half][1] = pair_to_bf16<TYPE, 1>(x, y);
                                pair[r][half][EACH - 2] = pair_to_bf16<TYPE, 2>(x, y);
                                pair[r][half][EACH - 1] = pair_to_bf16<TYPE, 3>(x, y);
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < HG; ++h) {
#pragma unroll
                        for (int j = 0; j < EACH; ++j) {
                            mma_bf16(acc[h][EACH * w + j], pair[0][0][j], pair[0][1][j], pair[1][0][j], pair[1][1][j], p_hi[h][0], p_hi[h][1]);
                            if (!twice) mma_bf16(acc[h][EACH * w + j], pair[0][0][j], pair[0][1][j], pair[1][0][j], pair[1][1][j], p_lo[h][0], p_lo[h][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[warp][slot]);
            if (++slot == STAGES) { slot = 0; parity ^= 1; }
        }

        const int head0 = head_of(seg.item), heads = heads_of(seg.item);
        together();
        if (seg.end < c1) ask_queries(segs[(k + 1) & 1].b, segs[(k + 1) & 1].item);
        if (twice) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[0][j][c] += __shfl_xor_sync(0xffffffffu, acc[0][j][c], 2);
            }
        }
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
        // a thread's accumulators, of heads 2t, 2t + 1 (and 8 + those): columns 64 half + 8 gp + tile of bf16, 16 gp + 8 half + tile of codes
        auto column = [&](int quarter, int p) { return (TYPE == KV_BF16 ? 64 * (quarter >> 1) + 8 * p : 8 * (quarter >> 1) + 16 * p) + (quarter & 1) * 4; };
        if (solo) {
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                if (a.lse && t == 0 && 8 * h + g < heads) a.lse[(int64_t)seg.b * a.heads + head0 + 8 * h + g] = (m[h] - KV_LIFT + log2f(l[h])) * 0.6931471805599453f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int head = 8 * h + 2 * t + j;
                    const float inv = 1.0f / __shfl_sync(0xffffffffu, l[h], 8 * t + 4 * j);
                    if (head >= heads) continue;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int c = 2 * (q >> 1) + j, four = (q & 1) * 4;
                        store_row4(a.out + seg.b * a.ldo + (head0 + head) * KV_D + column(q, gp), make_float4(acc[h][four][c], acc[h][four + 1][c], acc[h][four + 2][c], acc[h][four + 3][c]), inv, a.flags & 2);
                    }
                }
            }
            if (seg.end == c1) return;
            continue;
        }
        // ---- the warps' parts together, 32 columns at a time or as many as fit the team's buffer
        const int log_q = heads <= 4 ? 2 : heads <= 8 ? 1 : 0, quarters = 1 << log_q;
#pragma unroll
        for (int h = 0; h < HG; ++h)
            if (t == 0) { sh.m[team][mate][8 * h + g] = m[h]; sh.l[team][mate][8 * h + g] = l[h]; }
        const bool whole = seg.begin == seg.first && seg.end == seg.first + seg.n;
        const int64_t mine = (int64_t)(2 * id + (seg.begin == c0 ? 0 : 1)) * a.per_item;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at_q = q & (quarters - 1);
            if (q > 0 && at_q == 0) team_sync(team);
#pragma unroll
            for (int h = 0; h < HG; ++h) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int head = 8 * h + 2 * t + j, c = 2 * (q >> 1) + j, four = (q & 1) * 4;
                    if (head < heads)
                        *reinterpret_cast<float4*>(buf + ((mate * heads + head) * quarters + at_q) * 32 + 4 * g) =
                            make_float4(acc[h][four][c], acc[h][four + 1][c], acc[h][four + 2][c], acc[h][four + 3][c]);
                }
            }
            if (at_q + 1 < quarters) continue;
            team_sync(team);
            const int i = mate * 32 + lane, at = i & 7, qq = (i >> 3) & (quarters - 1), head = i >> (3 + log_q);
            if (head >= heads) continue;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < KV_TEAM; ++w) top = fmaxf(top, sh.m[team][w][head]);
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < KV_TEAM; ++w) {
                const float e = exp2_fast(sh.m[team][w][head] - (top == -INFINITY ? 0.f : top));
                const float4 x = *reinterpret_cast<const float4*>(buf + ((w * heads + head) * quarters + qq) * 32 + 4 * at);
                o.x += x.x * e; o.y += x.y * e; o.z += x.z * e; o.w += x.w * e;
                sum += sh.l[team][w][head] * e;
            }
            const int quarter = q - quarters + 1 + qq, col = column(quarter, kv_perm(at));
            const bool one = at == 0 && quarter == 0;
            if (whole) {
                store_row4(a.out + seg.b * a.ldo + (head0 + head) * KV_D + col, o, 1.0f / sum, a.flags & 2);
                if (a.lse && one) a.lse[(int64_t)seg.b * a.heads + head0 + head] = (top - KV_LIFT + log2f(sum)) * 0.6931471805599453f;
            } else {
                *reinterpret_cast<float4*>(a.parts + (mine + head) * KV_D + col) = o;
                if (one) a.stats[mine + head] = make_float2(top, sum);
            }
        }
        if (seg.end == c1) break;
    }
    // ---- items that the team shares with others: it is known for both at once whether all have come
    team_sync(team);
    const typename K::Share (&shares)[2] = sh.share[team];
    if (shares[0].here + shares[1].here == 0) return;
    if (mate == 0 && lane < 2) sh.last[team][lane] = shares[lane].here > 0 && all_came(a.arrived + shares[lane].first, shares[lane].here);
    team_sync(team);
#pragma unroll 1
    for (int level = 0; level < 2; ++level) {
        int done = 0, again = 0;         // heads to join before this part's
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            if (!sh.last[team][i]) continue;
            const typename K::Share s = shares[i];
            again |= level == 0 && s.groups > 1;
            for (int head = (mate - done) & (KV_TEAM - 1); head < s.heads; head += 2 * HG * KV_TEAM)
                kv_join<2 * HG>(a, level ? s.item : s.first, level ? s.fan : 1, level ? s.groups : s.here, s.b, head, s.heads, s.head0, level || s.groups == 1);
            done += s.heads;
        }
        if (!again) break;
        team_sync(team);
        if (mate == 0 && lane < 2 && sh.last[team][lane])       // the groups of an item
            sh.last[team][lane] = shares[lane].groups > 1 && all_came(a.arrived + 2 * KV_TEAMS_MAX + shares[lane].item, shares[lane].groups);
        team_sync(team);
    }
}

template <int TYPE, int HG, bool SOLO>
static cudaError_t launch_attention(const CUtensorMap& k_map, const CUtensorMap& v_map, const KvAttn& a, int blocks, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    using K = KvKernel<TYPE, HG>;
    static_assert(K::SMEM <= 232448, "more than an SM's block can have");
    if (!func_attr_once(done, (const void*)kv_attention_kernel<TYPE, HG, SOLO>, K::SMEM, "kv_attention")) return cudaErrorInvalidValue;
    return launch_chained(kv_attention_kernel<TYPE, HG, SOLO>, dim3((unsigned)blocks), dim3(K::THREADS), K::SMEM, st, 1, 1, k_map, v_map, a);
}
template <int TYPE, int HG>
static cudaError_t launch_attention(const CUtensorMap& k_map, const CUtensorMap& v_map, const KvAttn& a, int64_t item_chunks, int64_t items, cudaStream_t st) {
    const int most = min(sm_count(), KV_TEAMS_MAX / KvKernel<TYPE, HG>::TEAMS), teams = most * KvKernel<TYPE, HG>::TEAMS;
    // A table of few tokens for more items than teams: an item to a warp, where its chunks one after the other take less than a team's items with their joins.
    // us, to warps and to teams: 200 sequences of 30 rows of fp8, 8 kv heads 7.7 and 20; 62 of 54 of bf16, 16 kv heads 9.7 and 12.7; 128 of up to 100 of bf16 11.6 and 13.3.
    // (Chosen on the device instead, by the lengths, it cost all other calls 0.4 us: one kernel with both.)
    if (items > teams && item_chunks <= KV_SOLO && item_chunks * teams <= KV_TEAM * items) return launch_attention<TYPE, HG, true>(k_map, v_map, a, most, st);
    return launch_attention<TYPE, HG, false>(k_map, v_map, a, (int)max((int64_t)1, min((int64_t)most, max((item_chunks * items + KV_TEAM - 1) / KV_TEAM, items))), st);
}

static bool aligned16(const void* p, int64_t ld) { return (((uintptr_t)p) & 15) == 0 && (ld & 7) == 0; }

static hd_status kv_view(const o1_kv_cache* c, KvView* out, const char* what) {
    if (!c || !c->k || !c->v) { set_error("%s: null cache", what); return HD_ERR_MISSING; }
    if (c->type != O1_KV_BF16 && c->type != O1_KV_FP8 && c->type != O1_KV_INT8) { set_error("%s: unknown cache type %d", what, c->type); return HD_ERR_UNSUPPORTED; }
    if (c->head_dim != KV_D) { set_error("%s: head_dim %d (must be 128)", what, c->head_dim); return HD_ERR_UNSUPPORTED; }
    if (c->pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->page_size % 16) {
        set_error("%s: pages %d, kv_heads %d, page_size %d (a multiple of 16)", what, c->pages, c->kv_heads, c->page_size);
        return HD_ERR_UNSUPPORTED;
    }
    if ((int64_t)c->kv_heads > 4096) { set_error("%s: kv_heads %d (at most 4096)", what, c->kv_heads); return HD_ERR_UNSUPPORTED; }
    if (c->type != O1_KV_BF16 && (!c->k_scale || !c->v_scale)) { set_error("%s: a quantised cache needs k_scale and v_scale", what); return HD_ERR_MISSING; }
    if ((((uintptr_t)c->k) | ((uintptr_t)c->v) | ((uintptr_t)(c->type == O1_KV_BF16 ? nullptr : c->k_scale)) |
         ((uintptr_t)(c->type == O1_KV_BF16 ? nullptr : c->v_scale))) & 15) {
        set_error("%s: cache tensors must be 16-byte aligned", what);
        return HD_ERR_UNSUPPORTED;
    }
    int shift = -1;
    if ((c->page_size & (c->page_size - 1)) == 0)
        for (shift = 0; (1 << shift) < c->page_size; ++shift) {}
    *out = {(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, c->pages, shift, c->page_size, c->kv_heads};
    return HD_OK;
}

}  // namespace o1

using namespace o1;

extern "C" {
void o1_launch_count_add(int n);

hd_status o1_kv_write(const o1_kv_cache* cache, const void* k, int64_t ldk, const void* v, int64_t ldv, const int64_t* slots, int rows) {
    KvView c;
    hd_status st = kv_view(cache, &c, "kv_write");
    if (st != HD_OK) return st;
    if (rows < 0) { set_error("kv_write: rows %d", rows); return HD_ERR_UNSUPPORTED; }
    if (rows == 0) return HD_OK;
    if (!k || !v || !slots) { set_error("kv_write: null argument"); return HD_ERR_MISSING; }
    const int64_t row = (int64_t)c.heads * KV_D;
    if (ldk < row || ldv < row) { set_error("kv_write: row pitch below %lld", (long long)row); return HD_ERR_UNSUPPORTED; }
    const bool vec = aligned16(k, ldk) && aligned16(v, ldv);
    const int most = INT32_MAX / c.heads;      // of a launch, which counts units in 32 bits
    for (int first = 0; first < rows; first += most) {
        const unsigned units = (unsigned)min(most, rows - first) * c.heads;
        const bool few = units < KV_FEW_UNITS;
        const unsigned block = 4 * (few ? KV_EACH_OF_FEW : KV_EACH);
        auto kern = few ? (vec ? kv_write_kernel<true, KV_EACH_OF_FEW> : kv_write_kernel<false, KV_EACH_OF_FEW>) : vec ? kv_write_kernel<true, KV_EACH> : kv_write_kernel<false, KV_EACH>;
        if (!launch_ok(launch_chained(kern, dim3((units + block - 1) / block), dim3(128), 0, current_stream(), 1, 1, c, cache->type, (const uint16_t*)k + first * ldk, ldk,
                                      (const uint16_t*)v + first * ldv, ldv, slots + first, units, (const int*)device_error_word(), device_table_word()), "kv_write"))
            return HD_ERR_RUNTIME;
        o1_launch_count_add(1);
        if (rows - first <= most) break;
    }
    return HD_OK;
}

hd_status o1_kv_read(const o1_kv_cache* cache, void* k, int64_t ldk, void* v, int64_t ldv, const int64_t* slots, int rows) {
    KvView c;
    hd_status st = kv_view(cache, &c, "kv_read");
    if (st != HD_OK) return st;
    if (rows < 0) { set_error("kv_read: rows %d", rows); return HD_ERR_UNSUPPORTED; }
    if (rows == 0) return HD_OK;
    if (!k || !v || !slots) { set_error("kv_read: null argument"); return HD_ERR_MISSING; }
    const int64_t row = (int64_t)c.heads * KV_D;
    if (ldk < row || ldv < row) { set_error("kv_read: row pitch below %lld", (long long)row); return HD_ERR_UNSUPPORTED; }
    const bool vec = aligned16(k, ldk) && aligned16(v, ldv);
    const int most = INT32_MAX / c.heads;      // of a launch, which counts units in 32 bits
    for (int first = 0; first < rows; first += most) {
        const unsigned units = (unsigned)min(most, rows - first) * c.heads;
        const bool few = units < KV_FEW_UNITS;
        const unsigned block = 4 * (few ? KV_EACH_OF_FEW : KV_EACH);
        auto kern = few ? (vec ? kv_read_kernel<true, KV_EACH_OF_FEW> : kv_read_kernel<false, KV_EACH_OF_FEW>) : vec ? kv_read_kernel<true, KV_EACH> : kv_read_kernel<false, KV_EACH>;
        if (!launch_ok(launch_chained(kern, dim3((units + block - 1) / block), dim3(128), 0, current_stream(), 1, 1, c, cache->type, (uint16_t*)k + first * ldk, ldk,
                                      (uint16_t*)v + first * ldv, ldv, slots + first, units, device_table_word()), "kv_read"))
            return HD_ERR_RUNTIME;
        o1_launch_count_add(1);
        if (rows - first <= most) break;
    }
    return HD_OK;
}

// Two counters and, for every head of an item, 128 values, a maximum and a sum, for each team's two parts.
int64_t o1_kv_attention_workspace_bytes(int heads, int kv_heads) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads) return -1;
    return (int64_t)KV_TEAMS_MAX * 2 * (2 * 4 + min(heads / kv_heads, 16) * (KV_D + 2) * 4);
}

hd_status o1_kv_attention(const o1_kv_cache* cache, const void* q, int64_t ldq, const void* k_new, int64_t ldk, const void* v_new, int64_t ldv,
                          const int32_t* pages, int64_t ldp, int width, const int32_t* lens, void* out, int64_t ldo, float* lse, int batch, int heads,
                          float scale, void* workspace, int64_t workspace_bytes) {
    KvView c;
    hd_status st = kv_view(cache, &c, "kv_attention");
    if (st != HD_OK) return st;
    if (batch < 0 || heads <= 0 || heads % c.heads || width < 0) {
        set_error("kv_attention: batch %d, heads %d (a multiple of kv_heads %d), width %d", batch, heads, c.heads, width);
        return HD_ERR_UNSUPPORTED;
    }
    if (batch == 0) return HD_OK;
    if (!q || (!pages && width > 0) || !lens || !out || !workspace || (!k_new != !v_new)) { set_error("kv_attention: null argument"); return HD_ERR_MISSING; }
    const int64_t qrow = (int64_t)heads * KV_D, krow = (int64_t)c.heads * KV_D;
    if (ldq < qrow || ldo < qrow || ldp < width || (k_new && (ldk < krow || ldv < krow))) { set_error("kv_attention: a row pitch is below the row"); return HD_ERR_UNSUPPORTED; }
    if (!(scale > 0.f) || scale > 3.0e38f) { set_error("kv_attention: scale %g", scale); return HD_ERR_UNSUPPORTED; }
    if (workspace_bytes < o1_kv_attention_workspace_bytes(heads, c.heads) || (((uintptr_t)workspace) & 15)) { set_error("kv_attention: workspace too small or unaligned"); return HD_ERR_OOM; }
    const int group = heads / c.heads, hg = group <= 8 ? 1 : 2, of_heads = (group + 8 * hg - 1) / (8 * hg), keys = cache->type == O1_KV_BF16 ? 16 : 32;
    // the stream's index and costs are ints: fewer sequences a launch where the table allows for more, and a limit of items of a sequence
    const int64_t item_chunks = ((int64_t)width * c.page_size + keys - 1) / keys, each = item_chunks * c.heads * of_heads;
    if ((int64_t)width * c.page_size > INT32_MAX - 64 || each > (1 << 30) || (int64_t)c.heads * of_heads > (1 << 18) || (int64_t)c.pages * c.heads * c.page_size > INT32_MAX) { set_error("kv_attention: a table of %d pages of %d tokens for %d heads, or a cache of %d pages, is too large", width, c.page_size, heads, c.pages); return HD_ERR_UNSUPPORTED; }
    const int step = (int)min((int64_t)KV_SEQS, each > 0 ? max((int64_t)1, (int64_t)(1 << 30) / each) : (int64_t)KV_SEQS);
    const int per_item = min(group, 8 * hg);
    KvAttn a = {};
    a.c = c;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldp = ldp; a.ldo = ldo;
    a.arrived = (unsigned*)workspace;
    a.parts = (float*)(a.arrived + 4 * KV_TEAMS_MAX);
    a.stats = (float2*)(a.parts + (int64_t)2 * KV_TEAMS_MAX * per_item * KV_D);
    a.heads = heads; a.group = group; a.chunks_of_heads = of_heads; a.per_item = per_item; a.width = width;
    a.scale = scale;
    a.err = device_error_word();
    a.bad = device_table_word();
    a.flags = (aligned16(q, ldq) ? 1 : 0) | (aligned16(out, ldo) ? 2 : 0) | (aligned16(k_new, ldk) && aligned16(v_new, ldv) ? 4 : 0);
    // maps of the rows, 128 bytes (64 columns of bf16, all codes) x 16, or 32 where a chunk of codes never crosses a page
    const bool wide = keys == 32 && c.page_size % 32 == 0;
    if (wide) a.flags |= 8;
    const uint64_t rows_all = (uint64_t)c.pages * c.heads * c.page_size, cols = cache->type == O1_KV_BF16 ? 128 : 64;
    CUtensorMap k_map, v_map;
    if (!make_tmap_bf16(&k_map, c.k, rows_all, cols, cols, wide ? 32 : 16) || !make_tmap_bf16(&v_map, c.v, rows_all, cols, cols, wide ? 32 : 16)) return HD_ERR_RUNTIME;
    for (int b = 0; b < batch; b += step) {
        a.batch = min(step, batch - b);
        a.q = (const uint16_t*)q + b * ldq;
        a.kn = k_new ? (const uint16_t*)k_new + b * ldk : nullptr;
        a.vn = v_new ? (const uint16_t*)v_new + b * ldv : nullptr;
        a.pages = pages + b * ldp;
        a.lens = lens + b;
        a.out = (uint16_t*)out + b * ldo;
        a.lse = lse ? lse + (int64_t)b * heads : nullptr;
        const int64_t items = (int64_t)c.heads * of_heads * a.batch;
        cudaError_t e;
        if (cache->type == O1_KV_BF16) e = hg == 1 ? launch_attention<KV_BF16, 1>(k_map, v_map, a, item_chunks, items, current_stream()) : launch_attention<KV_BF16, 2>(k_map, v_map, a, item_chunks, items, current_stream());
        else if (cache->type == O1_KV_FP8) e = hg == 1 ? launch_attention<KV_FP8, 1>(k_map, v_map, a, item_chunks, items, current_stream()) : launch_attention<KV_FP8, 2>(k_map, v_map, a, item_chunks, items, current_stream());
        else e = hg == 1 ? launch_attention<KV_INT8, 1>(k_map, v_map, a, item_chunks, items, current_stream()) : launch_attention<KV_INT8, 2>(k_map, v_map, a, item_chunks, items, current_stream());
        if (!launch_ok(e, "kv_attention")) return HD_ERR_RUNTIME;
        o1_launch_count_add(1);
    }
    return HD_OK;
}

}  // extern "C"
