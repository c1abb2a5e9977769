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

#include <algorithm>

namespace o1 {

using std::max;
using std::min;

enum { KV_BF16 = O1_KV_BF16, KV_FP8 = O1_KV_FP8, KV_INT8 = O1_KV_INT8 };
static constexpr int KV_D = 128;
// Codes of the device's error word: what a kernel found in a table on the device.  Nothing is read or written for such an entry.
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
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
    const int i = __float2int_rn(a), j = __float2int_rn(b), k = __float2int_rn(c), l = __float2int_rn(d);
    return __byte_perm(__byte_perm(i, j, 0x0040), __byte_perm(k, l, 0x0040), 0x5410);
}

// Quantising a row of 128, eight values to each of 16 lanes.  The scale is the row's largest magnitude over the
// largest code (127, or e4m3's 448), so no code saturates and one row's outlier costs no other row anything; codes are x times the
// reciprocal, rounded to nearest even (as are scale and reciprocal, in fp32).  A maximum below 2^-100 counts as 2^-100: its reciprocal stays finite and a
// row of zeros gets codes of zero.  A row with an Inf or NaN gets a NaN scale: it reads as NaN, as its bf16 form would
// carry it into the attention, where int8 has no code for either.
__device__ __forceinline__ uint2 quantise8(const uint4& x, int type, float& scale) {
    uint32_t top = 0;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top = max(top, w[i] & 0x7FFFu);
        top = max(top, (w[i] >> 16) & 0x7FFFu);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool finite = top < 0x7F80u;
    const float a = fmaxf(__uint_as_float(top << 16), 7.888609052210118e-31f);
    const float q = type == KV_INT8 ? 127.0f : 448.0f;
    scale = finite ? __fdiv_rn(a, q) : __uint_as_float(0x7FC00000u);
    const float inv = finite ? __fdiv_rn(q, a) : 0.0f;
    if (!finite) return make_uint2(0, 0);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf16lo(w[i]) * inv; f[2 * i + 1] = bf16hi(w[i]) * inv; }
    if (type == KV_INT8) return make_uint2(int8x4(f[0], f[1], f[2], f[3]), int8x4(f[4], f[5], f[6], f[7]));
    return make_uint2(f32_to_e4m3x2(f[0], f[1]) | (f32_to_e4m3x2(f[2], f[3]) << 16), f32_to_e4m3x2(f[4], f[5]) | (f32_to_e4m3x2(f[6], f[7]) << 16));
}
__device__ __forceinline__ uint4 dequantise8(const uint2& c, int type, float scale) {
    float f[8];
    const uint32_t w[2] = {c.x, c.y};
    if (type == KV_INT8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * scale;
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

// Slot of a new row of sequence b: its last one, by the page table.  -1: nothing to write.
__device__ __forceinline__ int64_t last_slot(const int32_t* pages, int64_t ldp, int width, const int32_t* lens, int b, const KvView& c, int* err) {
    const int n = lens[b];
    if (n == 0) return -1;
    if (n < 0 || n > (int64_t)width * c.page_size) { atomicExch(err, ERR_KV_LENGTH); return -1; }
    const int page = pages[b * ldp + (n - 1) / c.page_size];
    if ((unsigned)page >= (unsigned)c.pages) { atomicExch(err, ERR_KV_PLACE); return -1; }
    return (int64_t)page * c.page_size + (n - 1) % c.page_size;
}

// Row r's place in a [pages][heads][page_size] array, -1: none.
__device__ __forceinline__ int64_t place(int64_t slot, int head, const KvView& c, int* err) {
    if (slot < 0) return -1;
    if (slot >= (int64_t)c.pages * c.page_size) { atomicExch(err, ERR_KV_PLACE); return -1; }
    const int64_t page = slot / c.page_size;
    return (page * c.heads + head) * c.page_size + slot - page * c.page_size;
}

// One row of 128 of one of the tensors to 16 lanes.  HBM bound for many rows: 2 bytes in, 1 (or 2) and the scale out a value.
template <bool VEC>
__global__ void __launch_bounds__(256)
kv_write_kernel(KvView c, int type, const uint16_t* __restrict__ k, int64_t ldk, const uint16_t* __restrict__ v, int64_t ldv,
                const int64_t* __restrict__ slots, const int32_t* __restrict__ pages, int64_t ldp, int width,
                const int32_t* __restrict__ lens, int rows, int* err) {
    grid_dep_launch();
    grid_dep_wait();
    const int64_t unit = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int lane = threadIdx.x & 15;
    const int64_t row = unit / (2 * c.heads);
    const int part = (int)(unit - row * 2 * c.heads), head = part >> 1;
    const bool is_v = part & 1, on = row < rows;
    uint4 x = make_uint4(0, 0, 0, 0);
    int64_t at = -1;
    if (on) {
        x = load8<VEC>((is_v ? v + row * ldv : k + row * ldk) + head * KV_D + lane * 8);
        at = place(slots ? slots[row] : last_slot(pages, ldp, width, lens, (int)row, c, err), head, c, err);
    }
    uint8_t* base = is_v ? c.v : c.k;
    if (type == KV_BF16) {
        if (at >= 0) reinterpret_cast<uint4*>(base)[at * 16 + lane] = x;
        return;
    }
    float scale;
    const uint2 codes = quantise8(x, type, scale);
    if (at >= 0) {
        reinterpret_cast<uint2*>(base)[at * 16 + lane] = codes;
        if (lane == 0) (is_v ? c.vs : c.ks)[at] = scale;
    }
}

template <bool VEC>
__global__ void __launch_bounds__(256)
kv_read_kernel(KvView c, int type, uint16_t* __restrict__ k, int64_t ldk, uint16_t* __restrict__ v, int64_t ldv,
               const int64_t* __restrict__ slots, int rows, int* err) {
    grid_dep_launch();
    grid_dep_wait();
    const int64_t unit = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int lane = threadIdx.x & 15;
    const int64_t row = unit / (2 * c.heads);
    if (row >= rows) return;
    const int part = (int)(unit - row * 2 * c.heads), head = part >> 1;
    const bool is_v = part & 1;
    const int64_t at = place(slots[row], head, c, err);
    const uint8_t* base = is_v ? c.v : c.k;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (at >= 0) {
        if (type == KV_BF16) x = reinterpret_cast<const uint4*>(base)[at * 16 + lane];
        else x = dequantise8(reinterpret_cast<const uint2*>(base)[at * 16 + lane], type, (is_v ? c.vs : c.ks)[at]);
    }
    store8<VEC>((is_v ? v + row * ldv : k + row * ldk) + head * KV_D + lane * 8, x);
}

// ------------------------------------------------------------------ attention of a new row
// HBM bound: every cached value is read once and used by the G = heads / kv_heads queries that share it, 2 G multiply-adds for its one or two bytes,
// so all that counts is that enough bytes are on their way at all times, on all SMs, whatever the lengths are.
//
//  * The work is one stream of chunks (16 tokens, 32 of a quantised cache: 8 KB of keys and values) over sequences, kv heads and length, and every
//    block takes an equal, contiguous part of it.  Lengths are only on the device: each block sums them up itself.
//  * A warp takes every KV_WARPS-th chunk of its block's part through a ring of its own (cp.async, KV_STAGES chunks), so its loads run ahead over the ends of
//    sequences; no barrier but those at such an end.
//  * Products on the tensor cores (mma.sync: at most 16 rows of queries, tcgen05's tiles have 64 at least).  Scores: A = queries (rows = heads), B = keys.
//    Their accumulators are, packed in pairs, the B operand of the second product, A = values transposed (rows = columns of a head).  The operands' k and row
//    indices are permuted so that a thread's part of a key or value row is 16 contiguous bytes; the ring's 16-byte pieces are swizzled to be read without
//    bank conflicts.
//  * One pass with a running maximum and sum (in base 2) for each warp; warps join in shared memory, blocks that share a (sequence, kv head) over the
//    workspace: the last one to finish adds all parts in their order, so the result does not depend on who that is.
//  * Rounding: scores and sums in fp32.  Probabilities (times v's scale) enter the second product as two parts of bf16, value and rest, 16 bits of significand; codes
//    of a byte are exact in f16 and bf16.  Keys' codes go through f16, which takes fewer instructions, with queries scaled to f16 by a power of two for each head;
//    values' codes through bf16, whose range a probability needs.  The result is rounded once.
static constexpr int KV_WARPS = 4, KV_STAGES = 3;
static constexpr int KV_STAGE_BYTES = 8192;            // keys and values of a chunk
static constexpr int KV_BLOCKS_MAX = 320;
static constexpr int KV_SEQS = 512;                    // sequences of a launch
static constexpr int KV_PART = 16 * (KV_D + 2);        // floats of a block's part: up to 16 heads, each with its maximum and sum

struct KvAttn {
    KvView c;
    const uint16_t *q, *kn, *vn;
    int64_t ldq, ldk, ldv, ldp, ldo;
    const int32_t *pages, *lens;
    uint16_t* out;
    float* lse;
    float* parts;          // [KV_BLOCKS_MAX][2][KV_PART]
    unsigned* arrived;     // [KV_BLOCKS_MAX]
    int batch, heads, group, chunks_of_heads, width, flags;    // flags: 1 = queries in 16-byte pieces, 2 = results, 4 = new rows
    float scale;
    int* err;
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
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));      // (results below 2^-126 too: a probability may multiply a large value)
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
// Swizzle of a row's 16-byte pieces: the eight threads that one step of a shared-memory load serves read two rows 2m, 2m+1 (keys) or four rows 2t (values)
// of the ring, and this puts their pieces into eight different sets of banks.
__device__ __forceinline__ int kv_swizzle(int row) { return (row & 2) | ((((row >> 2) ^ row) & 1) << 2); }

template <int TYPE, int HG>
struct KvKernel {
    static constexpr int KEYS = TYPE == KV_BF16 ? 16 : 32, ROWB = TYPE == KV_BF16 ? 256 : 128, TILES = KEYS / 8;
    static constexpr int STAGE = KV_STAGE_BYTES + (TYPE == KV_BF16 ? 0 : 2 * KEYS * 4);
    static constexpr int RING = KV_WARPS * KV_STAGES * STAGE;
    static constexpr int JOIN = KV_WARPS * 8 * 64 * 4;
    static constexpr int SMEM = RING + JOIN;
};

// Position in the stream: flat index f = (sum of the chunks before sequence b) * items + item * (chunks of b) + chunk.
struct KvWalk {
    int b, base, n;
    __device__ __forceinline__ void load(const int* prefix, int items) { base = prefix[b] * items; n = prefix[b + 1] - prefix[b]; }
    __device__ __forceinline__ void seek(int f, const int* prefix, int items) {
        while (f - base >= n * items) { ++b; load(prefix, items); }
    }
};

template <int TYPE, int HG>
__global__ void __launch_bounds__(KV_WARPS * 32, 2)
kv_attention_kernel(const KvAttn a) {
    using K = KvKernel<TYPE, HG>;
    constexpr int KEYS = K::KEYS, ROWB = K::ROWB, TILES = K::TILES;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int prefix[KV_SEQS + 1];
    __shared__ float s_m[KV_WARPS][16], s_l[KV_WARPS][16];
    __shared__ int s_sum[KV_WARPS];
    __shared__ bool s_last;
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, tid = threadIdx.x;
    grid_dep_launch();
    grid_dep_wait();

    // ---- the lengths, as numbers of chunks, summed up
    const int ps = a.c.page_size, shift = a.c.page_shift;
    {
        const int per = (a.batch + KV_WARPS * 32 - 1) / (KV_WARPS * 32);
        int mine = 0;
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            int n = b < a.batch ? a.lens[b] : 0;
            if (n < 0 || n > (int64_t)a.width * ps) { atomicExch(a.err, ERR_KV_LENGTH); n = 0; }
            n = (n + KEYS - 1) / KEYS;
            if (b < a.batch) prefix[b + 1] = mine + n;
            mine += n;
        }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) s_sum[warp] = sum;
        if (tid == 0) prefix[0] = 0;
        __syncthreads();
        int before = sum - mine;
#pragma unroll
        for (int w = 0; w < KV_WARPS; ++w) before += w < warp ? s_sum[w] : 0;
        for (int i = 0; i < per; ++i)
            if (tid * per + i < a.batch) prefix[tid * per + i + 1] += before;
        __syncthreads();
    }
    // ---- sequences without rows
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (prefix[b + 1] != prefix[b]) continue;
        for (int i = tid; i < a.heads * KV_D; i += KV_WARPS * 32) a.out[b * a.ldo + i] = 0;
        if (a.lse) for (int i = tid; i < a.heads; i += KV_WARPS * 32) a.lse[(int64_t)b * a.heads + i] = -INFINITY;
    }

    const int items = a.c.heads * a.chunks_of_heads;
    const int total = prefix[a.batch] * items;
    const int blocks = min((int)gridDim.x, (total + KV_WARPS - 1) / KV_WARPS);
    if ((int)blockIdx.x >= blocks) return;
    const int c0 = (int)((int64_t)total * blockIdx.x / blocks), c1 = (int)((int64_t)total * (blockIdx.x + 1) / blocks);

    KvWalk ld, cur;
    {
        int lo = 0, hi = a.batch - 1;       // the last sequence that begins at or before c0 and has chunks
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] * items <= c0) lo = mid; else hi = mid - 1;
        }
        cur.b = lo;
        cur.load(prefix, items);
        cur.seek(c0, prefix, items);
        ld = cur;
    }
    const uint32_t ring = smem_u32(smem) + warp * KV_STAGES * K::STAGE;
    float* join = reinterpret_cast<float*>(smem + K::RING);

    // ---- the load side: what the next chunk is, its pages asked for one chunk ahead
    int lf = c0 + warp, l_off[2], l_page[2], l_head = 0, l_slot = 0;
    bool l_two = false;
    auto look = [&]() {
        if (lf >= c1) return;
        ld.seek(lf, prefix, items);
        const int rel = lf - ld.base, item = rel / ld.n, tok = (rel - item * ld.n) * KEYS;
        l_head = item / a.chunks_of_heads;
        const int32_t* row = a.pages + ld.b * a.ldp;
        const int p0 = shift >= 0 ? tok >> shift : tok / ps;
        l_off[0] = tok - p0 * ps;
        l_page[0] = row[p0];
        if (KEYS == 32) {
            l_two = tok + 16 < a.lens[ld.b];
            const int p1 = shift >= 0 ? (tok + 16) >> shift : (tok + 16) / ps;
            l_off[1] = tok + 16 - p1 * ps;
            l_page[1] = l_two ? row[p1] : 0;
        }
    };
    auto issue = [&]() {
        if (lf < c1) {
            const uint32_t dst = ring + l_slot * K::STAGE;
#pragma unroll
            for (int h = 0; h < KEYS / 16; ++h) {
                if (h == 1 && !l_two) break;
                int page = l_page[h];
                if ((unsigned)page >= (unsigned)a.c.pages) { if (lane == 0) atomicExch(a.err, ERR_KV_PLACE); page = 0; }
                const int64_t at = ((int64_t)page * a.c.heads + l_head) * ps + l_off[h];
                constexpr int LANES = ROWB / 16, ROWS = 32 / LANES;      // lanes of a row, rows of a step
#pragma unroll
                for (int i = 0; i < 16 / ROWS; ++i) {
                    const int r = h * 16 + i * ROWS + lane / LANES, piece = lane % LANES;
                    const uint32_t to = r * ROWB + ((piece ^ kv_swizzle(r)) << 4);
                    const int64_t from = at * ROWB + i * 512 + lane * 16;
                    cp_async16(dst + to, a.c.k + from);
                    cp_async16(dst + 4096 + to, a.c.v + from);
                }
                if (TYPE != KV_BF16 && lane < 8)
                    cp_async16(dst + 8192 + (lane & 4) * 32 + h * 64 + (lane & 3) * 16, (lane < 4 ? a.c.ks : a.c.vs) + at + (lane & 3) * 4);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        l_slot = l_slot + 1 == KV_STAGES ? 0 : l_slot + 1;
        lf += KV_WARPS;
        look();
    };
    look();
    for (int i = 0; i < KV_STAGES; ++i) issue();

    // ---- segments: what the block has of one (sequence, kv head, up to 16 query heads)
    int f = c0 + warp, slot = 0;
    for (int seg = c0; seg < c1;) {
        cur.seek(seg, prefix, items);
        const int item = (seg - cur.base) / cur.n, first = cur.base + item * cur.n, end = min(c1, first + cur.n);
        const int kvh = item / a.chunks_of_heads, head0 = kvh * a.group + (item - kvh * a.chunks_of_heads) * (8 * HG);
        const int heads = min(8 * HG, (kvh + 1) * a.group - head0), b = cur.b, len = a.lens[b];

        // queries: rows g (and g + 8) of the A operand; the 16-byte pieces 4i + t of a key row are this thread's
        uint32_t qa[HG][16];
        float z_scale[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            const bool on = g + 8 * h < heads;
            const uint16_t* src = a.q + b * a.ldq + (head0 + g + 8 * h) * KV_D;
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = TYPE == KV_BF16 ? (4 * i + t) * 8 : (4 * (i >> 1) + t) * 16 + (i & 1) * 8;
                v[i] = !on ? make_uint4(0, 0, 0, 0) : (a.flags & 1) ? load8<true>(src + at) : load8<false>(src + at);
            }
            z_scale[h] = a.scale * 1.4426950408889634f;
            if (TYPE == KV_BF16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { qa[h][4 * i] = v[i].x; qa[h][4 * i + 1] = v[i].y; qa[h][4 * i + 2] = v[i].z; qa[h][4 * i + 3] = v[i].w; }
            } else {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7FFFu, (w[j] >> 16) & 0x7FFFu));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t e = min(max(top >> 7, 1u), 253u);         // the largest one's exponent
                const float down = __uint_as_float((254u - e) << 23);
                z_scale[h] *= __uint_as_float(e << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) qa[h][4 * i + j] = pack_f16x2(bf16lo(w[j]) * down, bf16hi(w[j]) * down);
                }
            }
        }
        float acc[HG][8][4], m[HG], l[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[h][j][0] = acc[h][j][1] = acc[h][j][2] = acc[h][j][3] = 0.f;
        }

        for (; f < end; f += KV_WARPS) {
            const int valid = len - (f - first) * KEYS;        // rows of the chunk that the sequence has, >= 1
            const uint32_t st = ring + slot * K::STAGE;
            uint4 fresh = make_uint4(0, 0, 0, 0);
            const bool append = a.kn && valid <= KEYS;
            if (append) {
                const uint16_t* src = (lane < 16 ? a.kn + b * a.ldk : a.vn + b * a.ldv) + kvh * KV_D + (lane & 15) * 8;
                fresh = (a.flags & 4) ? load8<true>(src) : load8<false>(src);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(KV_STAGES - 1) : "memory");
            __syncwarp();
            if (append) {     // the sequence's last row is the new one: into the ring, and into the cache
                const int r = valid - 1, tok = len - 1, pi = tok / ps;
                const int page = a.pages[b * a.ldp + pi];
                const bool store = item == kvh * a.chunks_of_heads && (unsigned)page < (unsigned)a.c.pages;
                const int64_t at = ((int64_t)page * a.c.heads + kvh) * ps + tok - pi * ps;
                const uint32_t dst = st + (lane < 16 ? 0 : 4096) + r * ROWB;
                uint8_t* const base = lane < 16 ? a.c.k : a.c.v;
                if (TYPE == KV_BF16) {
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (((lane & 15) ^ kv_swizzle(r)) << 4)), "r"(fresh.x), "r"(fresh.y), "r"(fresh.z), "r"(fresh.w) : "memory");
                    if (store) reinterpret_cast<uint4*>(base)[at * 16 + (lane & 15)] = fresh;
                } else {
                    float sc;
                    const uint2 codes = quantise8(fresh, TYPE, sc);
                    asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(dst + ((((lane & 15) >> 1) ^ kv_swizzle(r)) << 4) + (lane & 1) * 8), "r"(codes.x), "r"(codes.y) : "memory");
                    if ((lane & 15) == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(st + 8192 + (lane >> 4) * 128 + r * 4), "f"(sc) : "memory");
                    if (store) {
                        reinterpret_cast<uint2*>(base)[at * 16 + (lane & 15)] = codes;
                        if ((lane & 15) == 0) (lane < 16 ? a.c.ks : a.c.vs)[at] = sc;
                    }
                }
                __syncwarp();
            }

            // scores of 8 keys a tile
            float s[TILES][4];
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                const uint32_t row = st + (n * 8 + g) * ROWB;
#pragma unroll
                for (int i = 0; i < ROWB / 64; ++i) {
                    const uint4 k = lds128(row + (((4 * i + t) ^ kv_swizzle(g)) << 4));
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
            // this thread's keys: 8n + 2t and the next
            float vs[TILES][2];
            if (TYPE != KV_BF16) {
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    float2 ks, v2;
                    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(ks.x), "=f"(ks.y) : "r"(st + 8192 + (8 * n + 2 * t) * 4));
                    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v2.x), "=f"(v2.y) : "r"(st + 8192 + 128 + (8 * n + 2 * t) * 4));
                    s[n][0] *= ks.x; s[n][1] *= ks.y;
                    if (HG == 2) { s[n][2] *= ks.x; s[n][3] *= ks.y; }
                    vs[n][0] = 8 * n + 2 * t < valid ? v2.x : 0.f;
                    vs[n][1] = 8 * n + 2 * t + 1 < valid ? v2.y : 0.f;
                }
            }
            // running maximum and sum; a tile's accumulators become the probabilities
            float alpha[HG];
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float z = s[n][2 * h + j] * z_scale[h];
                        if (8 * n + 2 * t + j >= valid) z = -INFINITY;
                        s[n][2 * h + j] = z;
                        top = fmaxf(top, z);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m[h], top), ref = m_new == -INFINITY ? 0.f : m_new;
                alpha[h] = exp2_fast(m[h] - ref);
                m[h] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) { s[n][2 * h + j] = exp2_fast(s[n][2 * h + j] - ref); sum += s[n][2 * h + j]; }
                }
                l[h] = l[h] * alpha[h] + sum;
                if (TYPE != KV_BF16) {
#pragma unroll
                    for (int n = 0; n < TILES; ++n) { s[n][2 * h] *= vs[n][0]; s[n][2 * h + 1] *= vs[n][1]; }
                }
            }
            bool moved = false;
#pragma unroll
            for (int h = 0; h < HG; ++h) moved = moved || alpha[h] != 1.f;
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    const float a0 = __shfl_sync(0xffffffffu, alpha[h], 8 * t), a1 = __shfl_sync(0xffffffffu, alpha[h], 8 * t + 4);
#pragma unroll
                    for (int j = 0; j < 8; ++j) { acc[h][j][0] *= a0; acc[h][j][1] *= a1; acc[h][j][2] *= a0; acc[h][j][3] *= a1; }
                }
            }
            // out^T += V^T P^T, 16 keys a step
#pragma unroll
            for (int u = 0; u < KEYS / 16; ++u) {
                uint32_t p_hi[HG][2], p_lo[HG][2];
#pragma unroll
                for (int h = 0; h < HG; ++h) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) two_parts(s[2 * u + j][2 * h], s[2 * u + j][2 * h + 1], p_hi[h][j], p_lo[h][j]);
                }
                const uint32_t base = st + 4096 + u * 16 * ROWB;
                // rows of this thread: 2t, 2t+1, 2t+8, 2t+9 of the 16; masked rows as zeros, whatever the memory behind a sequence holds
                uint4 v[4][ROWB / 128];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = 2 * t + (r & 1) + (r >> 1) * 8;
#pragma unroll
                    for (int i = 0; i < ROWB / 128; ++i) {
                        v[r][i] = lds128(base + key * ROWB + ((g ^ kv_swizzle(key)) << 4) + 128 * i);
                        if (valid < KEYS && u * 16 + key >= valid) v[r][i] = make_uint4(0, 0, 0, 0);
                    }
                }
                uint32_t pair[2][16];      // [rows 2t, 2t+1 | 2t+8, 2t+9][16 columns: bf16 8g + j and 64 + 8g + j, codes 16g + j]
#pragma unroll
                for (int r = 0; r < 2; ++r) {
#pragma unroll
                    for (int i = 0; i < ROWB / 128; ++i) {
                        const uint32_t x[4] = {v[2 * r][i].x, v[2 * r][i].y, v[2 * r][i].z, v[2 * r][i].w};
                        const uint32_t y[4] = {v[2 * r + 1][i].x, v[2 * r + 1][i].y, v[2 * r + 1][i].z, v[2 * r + 1][i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (TYPE == KV_BF16) {
                                pair[r][8 * i + 2 * j] = __byte_perm(x[j], y[j], 0x5410);
                                pair[r][8 * i + 2 * j + 1] = __byte_perm(x[j], y[j], 0x7632);
                            } else {
                                pair[r][4 * j] = pair_to_bf16<TYPE, 0>(x[j], y[j]);
                                pair[r][4 * j + 1] = pair_to_bf16<TYPE, 1>(x[j], y[j]);
                                pair[r][4 * j + 2] = pair_to_bf16<TYPE, 2>(x[j], y[j]);
                                pair[r][4 * j + 3] = pair_to_bf16<TYPE, 3>(x[j], y[j]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < HG; ++h) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        mma_bf16(acc[h][j], pair[0][j], pair[0][8 + j], pair[1][j], pair[1][8 + j], p_hi[h][0], p_hi[h][1]);
                        mma_bf16(acc[h][j], pair[0][j], pair[0][8 + j], pair[1][j], pair[1][8 + j], p_lo[h][0], p_lo[h][1]);
                    }
                }
            }
            __syncwarp();
            issue();
            slot = slot + 1 == KV_STAGES ? 0 : slot + 1;
        }

        // ---- the warps' parts together
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (t == 0) { s_m[warp][8 * h + g] = m[h]; s_l[warp][8 * h + g] = l[h]; }
        }
        __syncthreads();
        const bool whole = seg == first && end == first + cur.n;
        float* part = a.parts + ((size_t)blockIdx.x * 2 + (seg == c0 ? 0 : 1)) * KV_PART;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            float fac[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < KV_WARPS; ++w) top = fmaxf(top, s_m[w][8 * h + 2 * t + j]);
                fac[j] = exp2_fast(s_m[warp][8 * h + 2 * t + j] - (top == -INFINITY ? 0.f : top));
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (h + half > 0) __syncthreads();
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float* to = join + (warp * 8 + 2 * t + j) * 64 + 8 * g;
#pragma unroll
                    for (int i = 0; i < 8; i += 4)
                        *reinterpret_cast<float4*>(to + i) = make_float4(acc[h][i][2 * half + j] * fac[j], acc[h][i + 1][2 * half + j] * fac[j],
                                                                         acc[h][i + 2][2 * half + j] * fac[j], acc[h][i + 3][2 * half + j] * fac[j]);
                }
                __syncthreads();
                for (int i = tid; i < 8 * 16; i += KV_WARPS * 32) {       // four columns of a head each
                    const int head = 8 * h + (i >> 4), at = (i & 15) * 4;
                    if (head >= heads) continue;
                    float top = -INFINITY, sum = 0.f;
                    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
                    for (int w = 0; w < KV_WARPS; ++w) top = fmaxf(top, s_m[w][head]);
#pragma unroll
                    for (int w = 0; w < KV_WARPS; ++w) {
                        const float4 x = *reinterpret_cast<const float4*>(join + (w * 8 + (i >> 4)) * 64 + at);
                        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
                        sum += s_l[w][head] * exp2_fast(s_m[w][head] - (top == -INFINITY ? 0.f : top));
                    }
                    // columns of the join buffer: bf16 64 half + at; codes 16 (at / 8) + 8 half + at % 8
                    const int col = TYPE == KV_BF16 ? 64 * half + at : 16 * (at >> 3) + 8 * half + (at & 7);
                    if (whole) {
                        const float inv = 1.0f / sum;
                        uint16_t* dst = a.out + b * a.ldo + (head0 + head) * KV_D + col;
                        const uint2 r = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                        if (a.flags & 2) *reinterpret_cast<uint2*>(dst) = r;
                        else { dst[0] = (uint16_t)r.x; dst[1] = (uint16_t)(r.x >> 16); dst[2] = (uint16_t)r.y; dst[3] = (uint16_t)(r.y >> 16); }
                        if (a.lse && at == 0 && half == 0) a.lse[(int64_t)b * a.heads + head0 + head] = (top + log2f(sum)) * 0.6931471805599453f;
                    } else {
                        *reinterpret_cast<float4*>(part + head * KV_D + col) = o;
                        if (at == 0 && half == 0) { part[16 * KV_D + head] = top; part[16 * KV_D + 16 + head] = sum; }
                    }
                }
            }
        }

        // ---- blocks that share the item: the last one joins all parts, in their order
        if (!whole) {
            const int from = (int)((((int64_t)first + 1) * blocks - 1) / total), to = (int)(((int64_t)(first + cur.n) * blocks - 1) / total);
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(a.arrived + from, 1u) == (unsigned)(to - from);
            __syncthreads();
            if (s_last) {
                __threadfence();
                if (tid == 0) a.arrived[from] = 0;
                const bool late = first != (int)((int64_t)total * from / blocks);       // the item begins inside the first block's part
                for (int head = warp; head < heads; head += KV_WARPS) {
                    float top = -INFINITY, sum = 0.f;
                    float4 o = make_float4(0, 0, 0, 0);
                    for (int p = from; p <= to; ++p) top = fmaxf(top, __ldcg(a.parts + ((size_t)p * 2 + (p == from && late)) * KV_PART + 16 * KV_D + head));
                    const float ref = top == -INFINITY ? 0.f : top;
                    for (int p = from; p <= to; ++p) {
                        const float* src = a.parts + ((size_t)p * 2 + (p == from && late)) * KV_PART;
                        const float w = exp2_fast(__ldcg(src + 16 * KV_D + head) - ref);
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(src + head * KV_D) + lane);
                        o.x += x.x * w; o.y += x.y * w; o.z += x.z * w; o.w += x.w * w;
                        sum += __ldcg(src + 16 * KV_D + 16 + head) * w;
                    }
                    const float inv = 1.0f / sum;
                    uint16_t* dst = a.out + b * a.ldo + (head0 + head) * KV_D + lane * 4;
                    const uint2 r = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                    if (a.flags & 2) *reinterpret_cast<uint2*>(dst) = r;
                    else { dst[0] = (uint16_t)r.x; dst[1] = (uint16_t)(r.x >> 16); dst[2] = (uint16_t)r.y; dst[3] = (uint16_t)(r.y >> 16); }
                    if (a.lse && lane == 0) a.lse[(int64_t)b * a.heads + head0 + head] = (top + log2f(sum)) * 0.6931471805599453f;
                }
            }
        }
        __syncthreads();        // s_m, s_l and the join buffer are free again
        seg = end;
    }
}

template <int TYPE, int HG>
static cudaError_t launch_attention(const KvAttn& a, int64_t chunks, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    using K = KvKernel<TYPE, HG>;
    if (!func_attr_once(done, (const void*)kv_attention_kernel<TYPE, HG>, K::SMEM, "kv_attention")) return cudaErrorInvalidValue;
    const int64_t most = min((int64_t)2 * sm_count(), (int64_t)KV_BLOCKS_MAX), want = (chunks + KV_WARPS - 1) / KV_WARPS;
    return launch_chained(kv_attention_kernel<TYPE, HG>, dim3((unsigned)max((int64_t)1, min(most, want))), dim3(KV_WARPS * 32), K::SMEM, st, 1, 1, a);
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
    const int64_t units = (int64_t)rows * c.heads * 2;
    auto kern = aligned16(k, ldk) && aligned16(v, ldv) ? kv_write_kernel<true> : kv_write_kernel<false>;
    if (!launch_ok(launch_chained(kern, dim3((unsigned)((units + 15) / 16)), dim3(256), 0, current_stream(), 1, rows, c, cache->type, (const uint16_t*)k, ldk,
                                  (const uint16_t*)v, ldv, slots, (const int32_t*)nullptr, (int64_t)0, 0, (const int32_t*)nullptr, rows, device_error_word()), "kv_write"))
        return HD_ERR_RUNTIME;
    o1_launch_count_add(1);
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
    const int64_t units = (int64_t)rows * c.heads * 2;
    auto kern = aligned16(k, ldk) && aligned16(v, ldv) ? kv_read_kernel<true> : kv_read_kernel<false>;
    if (!launch_ok(launch_chained(kern, dim3((unsigned)((units + 15) / 16)), dim3(256), 0, current_stream(), 1, rows, c, cache->type, (uint16_t*)k, ldk,
                                  (uint16_t*)v, ldv, slots, rows, device_error_word()), "kv_read"))
        return HD_ERR_RUNTIME;
    o1_launch_count_add(1);
    return HD_OK;
}

int64_t o1_kv_attention_workspace_bytes(int heads) {
    (void)heads;      // a block's part has room for the 16 heads that it takes at a time
    return (int64_t)KV_BLOCKS_MAX * (2 * KV_PART * sizeof(float) + sizeof(unsigned));
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
    if (workspace_bytes < o1_kv_attention_workspace_bytes(heads) || (((uintptr_t)workspace) & 15)) { set_error("kv_attention: workspace too small or unaligned"); return HD_ERR_OOM; }
    const int group = heads / c.heads, hg = group <= 8 ? 1 : 2, of_heads = (group + 8 * hg - 1) / (8 * hg), keys = cache->type == O1_KV_BF16 ? 16 : 32;
    // the stream's index is an int: fewer sequences a launch where the table allows for more
    const int64_t each = ((int64_t)width * c.page_size + keys - 1) / keys * c.heads * of_heads;
    if ((int64_t)width * c.page_size > INT32_MAX - 64 || each > (1 << 30)) { set_error("kv_attention: a table of %d pages of %d is too long for %d heads", width, c.page_size, heads); return HD_ERR_UNSUPPORTED; }
    const int step = (int)min((int64_t)KV_SEQS, each > 0 ? max((int64_t)1, (int64_t)(1 << 30) / each) : (int64_t)KV_SEQS);
    KvAttn a = {c, nullptr, nullptr, nullptr, ldq, ldk, ldv, ldp, ldo, nullptr, nullptr, nullptr, nullptr, (float*)workspace,
                (unsigned*)((float*)workspace + (size_t)KV_BLOCKS_MAX * 2 * KV_PART), 0, heads, group, of_heads, width, 0, scale, device_error_word()};
    a.flags = (aligned16(q, ldq) ? 1 : 0) | (aligned16(out, ldo) ? 2 : 0) | (aligned16(k_new, ldk) && aligned16(v_new, ldv) ? 4 : 0);
    for (int b = 0; b < batch; b += step) {
        a.batch = min(step, batch - b);
        a.q = (const uint16_t*)q + b * ldq;
        a.kn = k_new ? (const uint16_t*)k_new + b * ldk : nullptr;
        a.vn = v_new ? (const uint16_t*)v_new + b * ldv : nullptr;
        a.pages = pages + b * ldp;
        a.lens = lens + b;
        a.out = (uint16_t*)out + b * ldo;
        a.lse = lse ? lse + (int64_t)b * heads : nullptr;
        const int64_t chunks = each * a.batch;
        cudaError_t e;
        if (cache->type == O1_KV_BF16) e = hg == 1 ? launch_attention<KV_BF16, 1>(a, chunks, current_stream()) : launch_attention<KV_BF16, 2>(a, chunks, current_stream());
        else if (cache->type == O1_KV_FP8) e = hg == 1 ? launch_attention<KV_FP8, 1>(a, chunks, current_stream()) : launch_attention<KV_FP8, 2>(a, chunks, current_stream());
        else e = hg == 1 ? launch_attention<KV_INT8, 1>(a, chunks, current_stream()) : launch_attention<KV_INT8, 2>(a, chunks, current_stream());
        if (!launch_ok(e, "kv_attention")) return HD_ERR_RUNTIME;
        o1_launch_count_add(1);
    }
    return HD_OK;
}

}  // extern "C"
