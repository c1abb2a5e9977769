// A paged cache of keys and values and the attention of one new row per sequence over it.
//
// Layout: k and v each [pages][kv_heads][page_size][128], a head's rows of a page behind one another, so that what one
// (sequence, kv head) pair reads of a page is contiguous.  Stored as bf16, or as fp8 (e4m3) or int8 codes with one fp32 scale for each token
// and head in arrays [pages][kv_heads][page_size]: x ~ code * scale.  No counterpart in o1.c, which keeps no keys or values
// from one forward to the next.
#include "common.cuh"
#include "kernels.h"
#include "../../include/o1_b200.h"

#include <math.h>

namespace o1 {

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
// One block for each (sequence, query head), a cached row to a warp at a time, four columns to a lane: the running
// maximum, sum and weighted sum of a softmax in one pass over the rows, joined over the four warps at the end.
__global__ void __launch_bounds__(128)
kv_attention_kernel(KvView c, int type, const uint16_t* __restrict__ q, int64_t ldq, const int32_t* __restrict__ pages, int64_t ldp, int width,
                    const int32_t* __restrict__ lens, uint16_t* __restrict__ out, int64_t ldo, float* __restrict__ lse, int heads, float scale, int* err) {
    const int b = blockIdx.x / heads, head = blockIdx.x % heads, kvh = head / (heads / c.heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ float sm[4], sl[4], so[4][KV_D];
    int n = lens[b];
    if (n < 0 || n > (int64_t)width * c.page_size) { if (threadIdx.x == 0) atomicExch(err, ERR_KV_LENGTH); n = 0; }
    float qv[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4; ++i) qv[i] = bf16_to_f32(q[b * ldq + head * KV_D + lane * 4 + i]) * scale;
    for (int t = warp; t < n; t += 4) {
        const int page = pages[b * ldp + t / c.page_size];
        if ((unsigned)page >= (unsigned)c.pages) { if (lane == 0) atomicExch(err, ERR_KV_PLACE); continue; }
        const int64_t at = ((int64_t)page * c.heads + kvh) * c.page_size + t % c.page_size;
        float kf[4], vf[4];
        for (int i = 0; i < 4; ++i) {
            const int64_t e = at * KV_D + lane * 4 + i;
            if (type == KV_BF16) { kf[i] = bf16_to_f32(((const uint16_t*)c.k)[e]); vf[i] = bf16_to_f32(((const uint16_t*)c.v)[e]); }
            else if (type == KV_INT8) { kf[i] = (float)((const int8_t*)c.k)[e] * c.ks[at]; vf[i] = (float)((const int8_t*)c.v)[e] * c.vs[at]; }
            else { kf[i] = f16x2_to_f32(e4m3x2_to_f16x2(c.k[e])).x * c.ks[at]; vf[i] = f16x2_to_f32(e4m3x2_to_f16x2(c.v[e])).x * c.vs[at]; }
        }
        float z = qv[0] * kf[0] + qv[1] * kf[1] + qv[2] * kf[2] + qv[3] * kf[3];
        for (int s = 16; s > 0; s >>= 1) z += __shfl_xor_sync(0xffffffffu, z, s);
        const float mn = fmaxf(m, z), a = m == mn ? 1.f : expf(m - mn), p = expf(z - mn);
        m = mn;
        l = l * a + p;
        for (int i = 0; i < 4; ++i) o[i] = o[i] * a + p * vf[i];
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    for (int i = 0; i < 4; ++i) so[warp][lane * 4 + i] = o[i];
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float total = 0.f, r = 0.f;
    for (int w = 0; w < 4; ++w) {
        const float f = sm[w] == m ? 1.f : expf(sm[w] - m);
        total += sl[w] * f;
        r += so[w][threadIdx.x] * f;
    }
    const bool empty = n == 0;
    out[b * ldo + head * KV_D + threadIdx.x] = f32_to_bf16(empty ? 0.f : r / total);
    if (lse && threadIdx.x == 0) lse[(int64_t)b * heads + head] = empty ? -INFINITY : m + logf(total);
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

int64_t o1_kv_attention_workspace_bytes(int heads) { (void)heads; return 256; }

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
    if (k_new) {
        const int64_t units = (int64_t)batch * c.heads * 2;
        auto kern = aligned16(k_new, ldk) && aligned16(v_new, ldv) ? kv_write_kernel<true> : kv_write_kernel<false>;
        if (!launch_ok(launch_chained(kern, dim3((unsigned)((units + 15) / 16)), dim3(256), 0, current_stream(), 1, batch, c, cache->type, (const uint16_t*)k_new, ldk,
                                      (const uint16_t*)v_new, ldv, (const int64_t*)nullptr, pages, ldp, width, lens, batch, device_error_word()), "kv_attention"))
            return HD_ERR_RUNTIME;
        o1_launch_count_add(1);
    }
    kv_attention_kernel<<<(unsigned)(batch * heads), 128, 0, current_stream()>>>(c, cache->type, (const uint16_t*)q, ldq, pages, ldp, width, lens, (uint16_t*)out, ldo,
                                                                               lse, heads, scale, device_error_word());
    if (!launch_ok(cudaGetLastError(), "kv_attention")) return HD_ERR_RUNTIME;
    o1_launch_count_add(1);
    return HD_OK;
}

}  // extern "C"
