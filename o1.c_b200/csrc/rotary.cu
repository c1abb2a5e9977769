// Rotary positions: each pair of a head's first rot_dim values is turned by position * frequency,
//   (a, b) -> f (a cos - b sin, b cos + a sin),
// the pairs being (i, i + rot_dim / 2) ("half") or (2i, 2i + 1) ("interleaved").  Frequencies are theta^(-2i / rot_dim), scaled for contexts longer than the model was made
// for (o1_rope_turns).  Beside hd_mrope_cos_sin and hd_apply_rotary (o1.c src/cuda/rope.cu), which need tables in memory, know one layout and turn whole heads; their angles are
// fp32 products, which at position 10^6 are 0.03 radians off.
//
// Angles: a frequency is kept in turns a position, as the 64-bit fraction of a turn.  position * frequency mod 1 is then one 64-bit product whose overflow is the whole turns: exact to
// position * 2^-65 turns however far out.  It is reduced to an eighth of a turn around the nearest quarter with all its bits (integers; cut to 32 of them first, the sine of a slow pair's
// first positions was 3 % off), rounded to fp32 once, and the Taylor polynomials of sine and cosine to the 9th and 8th power, whose rest is below 2.5e-8 there, do what remains.
//
// HBM bound: values in, values out; 341 MB (16640 rows of 32 + 8 heads of bf16) in 52.8 us, 6.45 TB/s, 99 % of a copy's rate (neighbours as pairs 54.4); 84 MB (4111 rows of 16 + 4 heads of
// fp32, half of each head turned) in 14.7.  A thread has one 16-byte piece of a head and its partner, of several heads: all its loads are under way while it finds the piece's angles, once for all heads.
#include "common.cuh"
#include "kernels.h"
#include "../../include/o1_b200.h"

#include <limits.h>
#include <math.h>

namespace o1 {

// From so many (row, unit, head) triples for an SM on a thread has several heads' units, whose loads are under way while it finds their angles: four of bf16, two of fp32.
// 16640 rows of 40 heads of bf16: one 66 us, two 63, four 53.8, five 52.9, eight 55.7; 4111 rows of 20 heads of fp32: one 16.8, two 14.2, four 14.7.  With few rows more threads
// count: 1500 rows of 40 heads 9.5 us with one head to a thread, 5.3 with four; 700 rows 5.6 and 5.0, both the call's own time.  (With angles of 32 bits and without the bound on registers.)
static constexpr int ROPE_FEW = 1000;
struct RopeSide { const void* x; void* y; int64_t ldx, ldy; int heads; };
struct RopeArgs {
    RopeSide side[2];
    const uint64_t* turns;
    const void* positions;
    float factor;
    int rows, head_dim, rot, heads, slots, units, rows_a_block, wide_positions, inverse;      // units: pieces of a head; slots: threads of a row
};

// Cosine and sine times their factors, of which the sine's has the sign of the direction.
__device__ __forceinline__ void rope_angle(uint64_t turns, int64_t position, float factor, float factor_s, float& c, float& s) {
    const uint64_t t = turns * (uint64_t)position;
    const unsigned hi = (unsigned)(t >> 32), quarter = (hi + 0x20000000u) >> 30;
    // 2 pi / 2^64 and / 2^32 (two conversions of 32 bits; one of 64 takes as long, and more registers)
    const float a = __fmaf_rn((float)(uint32_t)t, 3.4061215800865545e-19f, (float)(int)(hi - (quarter << 30)) * 1.4629180792671596e-9f);
    const float a2 = a * a;
    const float sn = a * __fmaf_rn(a2, __fmaf_rn(a2, __fmaf_rn(a2, __fmaf_rn(a2, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -0.16666667f), 1.0f);
    const float cs = __fmaf_rn(a2, __fmaf_rn(a2, __fmaf_rn(a2, __fmaf_rn(a2, 2.4801587e-5f, -1.3888889e-3f), 4.1666668e-2f), -0.5f), 1.0f);
    const unsigned half = (quarter << 30) & 0x80000000u;         // half a turn on: both signs
    const bool odd = quarter & 1;
    c = (odd ? -sn : cs) * __uint_as_float(__float_as_uint(factor) ^ half);
    s = (odd ? cs : sn) * __uint_as_float(__float_as_uint(factor_s) ^ half);
}

// The piece p of V values of T at an address.
template <class T, int V>
struct Piece;
template <>
struct Piece<uint16_t, 8> {
    uint4 v;
    __device__ __forceinline__ void load(const uint16_t* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(uint16_t* p) const { *reinterpret_cast<uint4*>(p) = v; }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = bf16lo(w[i]); f[2 * i + 1] = bf16hi(w[i]); }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) { v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])); }
};
template <>
struct Piece<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float4*>(p) = v; }
    __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    __device__ __forceinline__ void set(const float (&f)[4]) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Piece<uint16_t, 1> {
    uint16_t v;
    __device__ __forceinline__ void load(const uint16_t* p) { v = *p; }
    __device__ __forceinline__ void store(uint16_t* p) const { *p = v; }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = bf16_to_f32(v); }
    __device__ __forceinline__ void set(const float (&f)[1]) { v = f32_to_bf16(f[0]); }
};
template <>
struct Piece<float, 1> {
    float v;
    __device__ __forceinline__ void load(const float* p) { v = *p; }
    __device__ __forceinline__ void store(float* p) const { *p = v; }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = v; }
    __device__ __forceinline__ void set(const float (&f)[1]) { v = f[0]; }
};

// V values to a piece.  A unit is two pieces whose values pair up: V values and those half a rotation on (HALF), or 2 V neighbours; behind the turned ones, two pieces as they are.
// A thread has one unit of N heads.  Registers are bounded so that four blocks (fp32: six) share an SM, where values are under way for long: 16640 rows of 40 heads of bf16 54.5 us without,
// 52.8 with, 4111 of 20 of fp32 15.3 and 14.7.
template <class T, int V, bool HALF, int N>
__global__ void __launch_bounds__(256, V * sizeof(T) == 16 && N > 1 ? (sizeof(T) == 2 ? 4 : 6) : 0)
rotary_kernel(const RopeArgs a) {
    grid_dep_launch();
    const int local = threadIdx.x / a.slots;                                   // (slots <= 256: rows side by side in a block; else a row's slots over blockIdx.y)
    const int64_t row = (int64_t)blockIdx.x * a.rows_a_block + (a.rows_a_block > 1 ? local : 0);
    const int slot = a.rows_a_block > 1 ? threadIdx.x - local * a.slots : blockIdx.y * blockDim.x + threadIdx.x;
    if (row >= a.rows || slot >= a.slots || (a.rows_a_block > 1 && local >= a.rows_a_block)) return;
    const int group = slot / a.units, unit = slot - group * a.units, turned = a.rot / 2 / V;
    const bool turns = unit < turned;
    const int at0 = turns ? (HALF ? unit * V : unit * 2 * V) : a.rot + (unit - turned) * 2 * V;
    const int at1 = turns && HALF ? at0 + a.rot / 2 : at0 + V;
    const bool two = at1 < a.head_dim;              // (behind the turned ones the last unit may have one piece)
    const int step = a.slots / a.units;             // heads side by side
    const T* x[N];
    T* y[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        int head = group + k * step;
        const RopeSide& side = a.side[head >= a.side[0].heads];
        if (head >= a.heads) { x[k] = nullptr; continue; }
        if (head >= a.side[0].heads) head -= a.side[0].heads;
        x[k] = (const T*)side.x + row * side.ldx + (int64_t)head * a.head_dim;
        y[k] = (T*)side.y + row * side.ldy + (int64_t)head * a.head_dim;
    }
    grid_dep_wait();
    Piece<T, V> p[N], q[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (!x[k]) continue;
        p[k].load(x[k] + at0);
        if (two) q[k].load(x[k] + at1);
    }
    if (turns) {             // while the values are on their way
        const int64_t position = a.wide_positions ? ((const int64_t*)a.positions)[row] : (int64_t)((const int32_t*)a.positions)[row];
        float c[V], s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            rope_angle(a.turns[unit * V + i], position, a.factor, a.inverse ? -a.factor : a.factor, c[i], s[i]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (!x[k]) continue;
            float u[V], w[V], e[V], f[V];
            p[k].get(u);
            q[k].get(w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int j = 2 * i;
                const float first = HALF ? u[i] : j < V ? u[j % V] : w[j % V], other = HALF ? w[i] : j + 1 < V ? u[(j + 1) % V] : w[(j + 1) % V];
                const float x0 = __fmaf_rn(first, c[i], -__fmul_rn(other, s[i])), x1 = __fmaf_rn(other, c[i], __fmul_rn(first, s[i]));
                if (HALF) { e[i] = x0; f[i] = x1; }
                else {
                    if (j < V) e[j % V] = x0; else f[j % V] = x0;
                    if (j + 1 < V) e[(j + 1) % V] = x1; else f[(j + 1) % V] = x1;
                }
            }
            p[k].set(e);
            q[k].set(f);
            p[k].store(y[k] + at0);
            q[k].store(y[k] + at1);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (!x[k]) continue;
            p[k].store(y[k] + at0);
            if (two) q[k].store(y[k] + at1);
        }
    }
}

template <class T, int V, int N>
static void (*rotary_of(bool half))(const RopeArgs) { return half ? rotary_kernel<T, V, true, N> : rotary_kernel<T, V, false, N>; }
template <class T, int V>
static void (*rotary_of(bool half, int heads))(const RopeArgs) { return heads == 1 ? rotary_of<T, V, 1>(half) : rotary_of<T, V, sizeof(T) == 2 ? 4 : 2>(half); }

// Whether any row of one set of rows and any of another share an address: `rows` of each, wa and wb bytes wide, lda and ldb bytes apart (at least as far as they are wide).
static bool rows_meet(const void* a, int64_t lda, int64_t wa, const void* b, int64_t ldb, int64_t wb, int64_t rows) {
    const int64_t d = (int64_t)((uintptr_t)b - (uintptr_t)a);
    if (wa == 0 || wb == 0 || d >= (rows - 1) * lda + wa || -d >= (rows - 1) * ldb + wb) return false;
    auto below = [](int64_t n, int64_t by) { return n / by - (n % by < 0); };             // the quotient, rounded down
    if (lda == ldb) {        // slices of wider rows, as a rule: b's row i + m is d + m * ld behind a's row i, and only the two nearest can be in its reach
        const int64_t m = -below(d, lda), r = d + m * lda;
        return (r < wa && m < rows && -m < rows) || (r - lda > -wb && m - 1 < rows && 1 - m < rows);
    }
    for (int64_t i = 0; i < rows; ++i) {      // of b's rows those from the first one that ends behind a's row's beginning to the last one that begins before its end
        const int64_t at = i * lda - d, first = below(at - wb, ldb) + 1, last = below(at + wa - 1, ldb);
        if (max(first, (int64_t)0) <= min(last, rows - 1)) return true;
    }
    return false;
}

}  // namespace o1

using namespace o1;

extern "C" {
void o1_launch_count_add(int n);

// Frequencies as turns a position, in 64-bit fractions.
hd_status o1_rope_turns(double theta, int rot_dim, const o1_rope_scaling* scaling, uint64_t* turns_host, float* factor) {
    const int kind = scaling ? scaling->kind : O1_ROPE_PLAIN;
    if (!turns_host || !factor || (kind == O1_ROPE_FACTORS && !scaling->factors)) { set_error("rope_turns: null argument"); return HD_ERR_MISSING; }
    if (!(theta > 1.0) || theta > 1e300 || rot_dim <= 0 || rot_dim % 2 || rot_dim > 65536 || kind < O1_ROPE_PLAIN || kind > O1_ROPE_FACTORS) {
        set_error("rope_turns: theta %g, rot_dim %d (even), scaling %d", theta, rot_dim, kind);
        return HD_ERR_UNSUPPORTED;
    }
    const double by = kind == O1_ROPE_PLAIN ? 1.0 : scaling->factor;
    if (kind != O1_ROPE_PLAIN && kind != O1_ROPE_FACTORS && (!(by >= 1.0) || by > 1e30)) { set_error("rope_turns: factor %g (at least 1)", by); return HD_ERR_UNSUPPORTED; }
    if (kind == O1_ROPE_YARN && (!(scaling->original >= 1.0) || !(scaling->fast > 0.0) || !(scaling->slow > 0.0) || scaling->fast < scaling->slow)) {
        set_error("rope_turns: original %g, fast %g, slow %g", scaling->original, scaling->fast, scaling->slow);
        return HD_ERR_UNSUPPORTED;
    }
    const long double two_pi = 6.283185307179586476925286766559L, n = rot_dim;
    const long double base = kind == O1_ROPE_NTK ? theta * powl((long double)by, n / (rot_dim > 3 ? n - 2 : 1)) : (long double)theta;
    double low = 0, high = 0;
    if (kind == O1_ROPE_YARN) {      // the pairs that turn `fast` and `slow` times within the original length
        auto pair_at = [&](double t) { return rot_dim * log(scaling->original / (t * 2.0 * M_PI)) / (2.0 * log(theta)); };
        low = fmax(floor(pair_at(scaling->fast)), 0.0);
        high = fmin(ceil(pair_at(scaling->slow)), rot_dim - 1.0);
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        long double f = powl(base, -2.0L * i / n);
        if (kind == O1_ROPE_LINEAR) f /= by;
        if (kind == O1_ROPE_YARN) {
            const double ramp = fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
            f = f / by * ramp + f * (1.0L - ramp);
        }
        if (kind == O1_ROPE_FACTORS) {
            if (!(fabs(scaling->factors[i]) > 1e-30) || !(fabs(scaling->factors[i]) < 1e30)) { set_error("rope_turns: factor %g of pair %d", scaling->factors[i], i); return HD_ERR_UNSUPPORTED; }
            f /= scaling->factors[i];
        }
        f /= two_pi;
        f -= floorl(f);                                       // whole turns change nothing
        const long double scaled = roundl(ldexpl(f, 64));
        turns_host[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
    }
    *factor = kind == O1_ROPE_YARN ? (float)(0.1 * log(by) + 1.0) : 1.0f;
    if (scaling && scaling->attention > 0.0) *factor = (float)scaling->attention;
    return HD_OK;
}

hd_status o1_rotary(const o1_rope* rope, const void* positions, int wide_positions, const void* x, int64_t ldx, void* y, int64_t ldy, int heads, const void* x2,
                    int64_t ldx2, void* y2, int64_t ldy2, int heads2, int rows, int type, int inverse) {
    if (!rope || !rope->turns || (rows > 0 && (!positions || (heads > 0 && (!x || !y)) || (heads2 > 0 && (!x2 || !y2))))) { set_error("rotary: null argument"); return HD_ERR_MISSING; }
    if (rope->head_dim <= 0 || rope->head_dim > 4096 || rope->rot_dim <= 0 || rope->rot_dim % 2 || rope->rot_dim > rope->head_dim ||
        (rope->layout != O1_ROPE_HALF && rope->layout != O1_ROPE_INTERLEAVED)) {
        set_error("rotary: head_dim %d (at most 4096), rot_dim %d (even), layout %d", rope->head_dim, rope->rot_dim, rope->layout);
        return HD_ERR_UNSUPPORTED;
    }
    if (type != O1_ROPE_BF16 && type != O1_ROPE_FP32) { set_error("rotary: type %d", type); return HD_ERR_UNSUPPORTED; }
    if (rows < 0 || heads < 0 || heads2 < 0 || (int64_t)heads + heads2 > 65536) { set_error("rotary: rows %d, heads %d and %d (at most 65536)", rows, heads, heads2); return HD_ERR_UNSUPPORTED; }
    const int64_t w = (int64_t)heads * rope->head_dim, w2 = (int64_t)heads2 * rope->head_dim;
    if (ldx < w || ldy < w || (heads2 && (ldx2 < w2 || ldy2 < w2))) { set_error("rotary: a row pitch is below the row"); return HD_ERR_UNSUPPORTED; }
    if (rows == 0 || heads + heads2 == 0) return HD_OK;
    const int size = type == O1_ROPE_BF16 ? 2 : 4, wide = 16 / size;
    if ((((uintptr_t)x | (uintptr_t)y | (uintptr_t)(heads2 ? x2 : nullptr) | (uintptr_t)(heads2 ? y2 : nullptr)) & (size - 1)) || ((uintptr_t)positions & (wide_positions ? 7 : 3))) {
        set_error("rotary: an address is not a multiple of its type's size");
        return HD_ERR_UNSUPPORTED;
    }
    // Threads read and write in no order: a result may take the place of its own rows, and no other's.
    auto meet = [&](const void* p, int64_t ldp, int64_t wp, const void* q, int64_t ldq, int64_t wq) { return rows_meet(p, ldp * size, wp * size, q, ldq * size, wq * size, rows); };
    auto same = [&](const void* p, int64_t ldp, const void* q, int64_t ldq) { return p == q && (ldp == ldq || rows == 1); };
    if ((!same(x, ldx, y, ldy) && meet(x, ldx, w, y, ldy, w)) ||
        (heads2 && ((!same(x2, ldx2, y2, ldy2) && meet(x2, ldx2, w2, y2, ldy2, w2)) || meet(x, ldx, w, y2, ldy2, w2) || meet(x2, ldx2, w2, y, ldy, w) || meet(y, ldy, w, y2, ldy2, w2)))) {
        set_error("rotary: results share memory with rows other than their own (which they may take the place of, row for row), or with one another");
        return HD_ERR_UNSUPPORTED;
    }
    RopeArgs a = {};
    a.side[0] = {x, y, ldx, ldy, heads};
    a.side[1] = {x2, y2, ldx2, ldy2, heads2};
    a.turns = rope->turns; a.positions = positions; a.factor = rope->factor;
    a.rows = rows; a.head_dim = rope->head_dim; a.rot = rope->rot_dim; a.heads = heads + heads2;
    a.wide_positions = wide_positions; a.inverse = inverse;
    // 16 bytes to a piece where pieces begin on such an address and no pair's halves share one
    const bool half = rope->layout == O1_ROPE_HALF;
    bool vec = a.rot % (2 * wide) == 0 && a.head_dim % wide == 0;
    for (const RopeSide& s : a.side)
        if (s.heads) vec = vec && (((uintptr_t)s.x | (uintptr_t)s.y) & 15) == 0 && s.ldx % wide == 0 && s.ldy % wide == 0;
    const int v = vec ? wide : 1;
    a.units = a.rot / 2 / v + (a.head_dim - a.rot + 2 * v - 1) / (2 * v);
    const int per_thread = (int64_t)rows * a.units * a.heads >= (int64_t)sm_count() * ROPE_FEW ? (size == 2 ? 4 : 2) : 1;
    a.slots = a.units * ((a.heads + per_thread - 1) / per_thread);
    a.rows_a_block = a.slots <= 256 ? 256 / a.slots : 1;
    if (a.slots > 256 || a.rows_a_block < 1) a.rows_a_block = 1;
    const dim3 grid((unsigned)(((int64_t)rows + a.rows_a_block - 1) / a.rows_a_block), (unsigned)(a.rows_a_block > 1 ? 1 : (a.slots + 255) / 256));
    if (grid.y > 65535) { set_error("rotary: %d heads of %d are too many", a.heads, a.head_dim); return HD_ERR_UNSUPPORTED; }
    auto kern = type == O1_ROPE_BF16 ? (vec ? rotary_of<uint16_t, 8>(half, per_thread) : rotary_of<uint16_t, 1>(half, per_thread))
                                     : (vec ? rotary_of<float, 4>(half, per_thread) : rotary_of<float, 1>(half, per_thread));
    if (!launch_ok(launch_chained(kern, grid, dim3(256), 0, current_stream(), 1, 1, a), "rotary")) return HD_ERR_RUNTIME;
    o1_launch_count_add(1);
    return HD_OK;
}

}  // extern "C"
