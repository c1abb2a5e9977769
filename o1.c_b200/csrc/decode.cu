// Prompts and the rows after them on cached keys and values: the decoder of o1.c (src/model/block.c:137-385) for text rows that are
// computed once.  o1_prompt_rows runs the rows of one sequence through all blocks and leaves their keys and values in the caches;
// o1_decode_step runs one new row of each of many sequences.  No counterpart in o1.c, which computes all rows in every forward.
//
// A step's launches for a block: q | k | v with norm and rotary, attention (which appends the row), o_proj, residual + norm, gate | up + SwiGLU, down, residual +
// the next block's norm.  The residual stream is rounded to bf16 once an addition, as in the block; its norm is of the unrounded sum.
#include "common.cuh"
#include "kernels.h"
#include "../../include/o1_b200.h"

#include <math.h>

using namespace o1;

extern "C" void o1_launch_count_add(int n);

namespace {

constexpr float EPS = 1e-6f;
constexpr int MIN_ROWS = 8;         // the tensor-core GEMMs' least; rows beyond the batch hold anything and reach no other row

struct Scratch {
    uint16_t *x, *ln, *qkv, *attn, *tmp, *swi;
    float* cs;
    void* attention;
    int64_t attention_bytes, bytes;
};
Scratch carve(void* base, int64_t rows, int heads, int kv_heads, int hidden, int ff, int hd) {
    Scratch s = {};
    uint8_t* p = (uint8_t*)base;
    auto take = [&](int64_t n) { uint8_t* at = p; p += (n + 255) & ~(int64_t)255; return at; };
    rows = rows < MIN_ROWS ? MIN_ROWS : rows;
    s.attention_bytes = o1_kv_attention_workspace_bytes(heads, kv_heads);
    s.attention = take(s.attention_bytes);       // first: the part that stays between calls
    s.x = (uint16_t*)take(rows * hidden * 2);
    s.ln = (uint16_t*)take(rows * hidden * 2);
    s.qkv = (uint16_t*)take(rows * (heads + 2 * kv_heads) * hd * 2);
    s.attn = (uint16_t*)take(rows * heads * hd * 2);
    s.tmp = (uint16_t*)take(rows * hidden * 2);
    s.swi = (uint16_t*)take(rows * ff * 2);
    s.cs = (float*)take(rows * 128 * 4);
    s.bytes = p - (uint8_t*)base;
    return s;
}

#define DEC_TRY(expr, what)                                                                                                   \
    do {                                                                                                                      \
        if (!(expr)) { hd_set_error("decode: %s: %s", what, hd_cuda_last_error()); return HD_ERR_RUNTIME; }                   \
        o1_launch_count_add(1);                                                                                               \
    } while (0)
#define DEC_CALL(expr, what)                                                                                                  \
    do {                                                                                                                      \
        const hd_status st__ = (expr);                                                                                        \
        if (st__ != HD_OK) { hd_set_error("decode: %s: %s", what, hd_cuda_last_error()); return st__; }                       \
    } while (0)

hd_status check(const hd_forward_binding* bw, const o1_kv_cache* caches, int rows, int heads, int kv_heads, int hidden, int ff, int hd) {
    if (!bw || !caches || !bw->blocks || !bw->embed_tokens || !bw->fnorm_w) { hd_set_error("decode: null argument"); return HD_ERR_MISSING; }
    if (bw->n_layers <= 0 || hd != 128 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || hidden <= 0 || hidden % 256 || ff <= 0 || ff % 128) {
        hd_set_error("decode: unsupported dims (head_dim 128, hidden a multiple of 256, ff of 128)");
        return HD_ERR_UNSUPPORTED;
    }
    if (rows < 0) { hd_set_error("decode: %d rows", rows); return HD_ERR_UNSUPPORTED; }
    for (int l = 0; l < bw->n_layers; ++l)
        if (caches[l].kv_heads != kv_heads) { hd_set_error("decode: the cache of layer %d has %d heads, not %d", l, caches[l].kv_heads, kv_heads); return HD_ERR_MISMATCH; }
    return HD_OK;
}

// All blocks and the final norm; `attention` fills s.attn from s.qkv for a layer.
template <class F>
hd_status run(const hd_forward_binding* bw, const Scratch& s, const int64_t* ids, int rows, int heads, int kv_heads, int hidden, int ff, int hd, int vocab,
              void* out, F attention) {
    cudaStream_t st = current_stream();
    const int M = rows < MIN_ROWS ? MIN_ROWS : rows, qc = heads * hd, kc = kv_heads * hd, ld = qc + 2 * kc;
    DEC_TRY(gather_rows(bw->embed_tokens, ids, s.x, rows, hidden, vocab, st), "embedding");
    DEC_TRY(rmsnorm(s.x, bw->blocks[0].input_ln, s.ln, rows, hidden, EPS, st), "input norm");
    for (int l = 0; l < bw->n_layers; ++l) {
        const hd_block_binding& b = bw->blocks[l];
        DEC_TRY(gemm_qkv(s.ln, hidden, b.q_proj, b.k_proj, b.v_proj, s.qkv, ld, M, qc, kc, hidden, b.q_norm, b.k_norm, s.cs, EPS, 0, nullptr, nullptr, nullptr, st), "q | k | v");
        DEC_CALL(attention(l), "attention");
        DEC_TRY(gemm_bf16(s.attn, b.o_proj, nullptr, s.tmp, M, hidden, qc, EPI_STORE, nullptr, nullptr, 0.f, 0, st), "o_proj");
        DEC_CALL(o1_residual_norm(s.x, hidden, s.tmp, hidden, nullptr, nullptr, 1.f, b.post_ln, nullptr, nullptr, 1, s.x, hidden, s.ln, hidden, rows, hidden, EPS), "residual + norm");
        DEC_TRY(gemm_bf16(s.ln, b.gate_proj, b.up_proj, s.swi, M, ff, hidden, EPI_SWIGLU, nullptr, nullptr, 0.f, 0, st), "gate | up");
        DEC_TRY(gemm_bf16(s.swi, b.down_proj, nullptr, s.tmp, M, hidden, ff, EPI_STORE, nullptr, nullptr, 0.f, 0, st), "down_proj");
        const bool last = l + 1 == bw->n_layers;
        DEC_CALL(o1_residual_norm(s.x, hidden, s.tmp, hidden, nullptr, nullptr, 1.f, last ? bw->fnorm_w : bw->blocks[l + 1].input_ln, nullptr, nullptr, 1, s.x, hidden,
                                  last ? out : s.ln, hidden, rows, hidden, EPS), "residual + norm");
    }
    return HD_OK;
}

}  // namespace

extern "C" {

int64_t o1_decode_scratch_bytes(int64_t rows, int heads, int kv_heads, int hidden, int ff_hidden, int head_dim) {
    if (rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || hidden <= 0 || ff_hidden <= 0 || head_dim <= 0) return -1;
    return carve(nullptr, rows, heads, kv_heads, hidden, ff_hidden, head_dim).bytes + 256;
}

hd_status o1_prompt_rows(const hd_forward_binding* bw, const o1_kv_cache* caches, const int64_t* ids, const float* pos_f32, const int64_t* slots, void* scratch,
                         int64_t scratch_bytes, void* out, int rows, int heads, int kv_heads, int hidden, int ff_hidden, int head_dim, int vocab) {
    hd_status st = check(bw, caches, rows, heads, kv_heads, hidden, ff_hidden, head_dim);
    if (st != HD_OK || rows == 0) return st;
    if (!ids || !pos_f32 || !slots || !scratch || !out) { hd_set_error("decode: null argument"); return HD_ERR_MISSING; }
    if (scratch_bytes < o1_decode_scratch_bytes(rows, heads, kv_heads, hidden, ff_hidden, head_dim)) { hd_set_error("decode: scratch too small"); return HD_ERR_OOM; }
    const Scratch s = carve((void*)(((uintptr_t)scratch + 255) & ~(uintptr_t)255), rows, heads, kv_heads, hidden, ff_hidden, head_dim);
    DEC_TRY(mrope_table64_rows(pos_f32, rows, 0, rows, 5000000.0f, s.cs, current_stream()), "rotary table");
    const int qc = heads * head_dim, kc = kv_heads * head_dim, ld = qc + 2 * kc;
    const float scale = (float)(1.0 / sqrt((double)head_dim));
    return run(bw, s, ids, rows, heads, kv_heads, hidden, ff_hidden, head_dim, vocab, out, [&](int l) {
        const hd_status w = o1_kv_write(caches + l, s.qkv + qc, ld, s.qkv + qc + kc, ld, slots, rows);
        if (w != HD_OK) return w;
        // causal over the prompt's own rows (the SwiGLU buffer is idle: partial results of a key-split tail)
        if (!flash_attention(s.qkv, ld, s.qkv + qc, ld, s.qkv + qc + kc, ld, s.attn, qc, rows, heads, kv_heads, rows, scale, current_stream(), s.swi,
                             (size_t)rows * ff_hidden * 2)) return HD_ERR_RUNTIME;
        o1_launch_count_add(1);
        return HD_OK;
    });
}

hd_status o1_decode_step(const hd_forward_binding* bw, const o1_kv_cache* caches, const int64_t* ids, const float* pos_f32, const int32_t* pages, int64_t ldp, int width,
                         const int32_t* lens, void* scratch, int64_t scratch_bytes, void* out, int batch, int heads, int kv_heads, int hidden, int ff_hidden,
                         int head_dim, int vocab) {
    hd_status st = check(bw, caches, batch, heads, kv_heads, hidden, ff_hidden, head_dim);
    if (st != HD_OK || batch == 0) return st;
    if (!ids || !pos_f32 || !pages || !lens || !scratch || !out) { hd_set_error("decode: null argument"); return HD_ERR_MISSING; }
    if (scratch_bytes < o1_decode_scratch_bytes(batch, heads, kv_heads, hidden, ff_hidden, head_dim)) { hd_set_error("decode: scratch too small"); return HD_ERR_OOM; }
    const Scratch s = carve((void*)(((uintptr_t)scratch + 255) & ~(uintptr_t)255), batch, heads, kv_heads, hidden, ff_hidden, head_dim);
    DEC_TRY(mrope_table64_rows(pos_f32, batch, 0, batch, 5000000.0f, s.cs, current_stream()), "rotary table");
    const int qc = heads * head_dim, kc = kv_heads * head_dim, ld = qc + 2 * kc;
    const float scale = (float)(1.0 / sqrt((double)head_dim));
    return run(bw, s, ids, batch, heads, kv_heads, hidden, ff_hidden, head_dim, vocab, out, [&](int l) {
        return o1_kv_attention(caches + l, s.qkv, ld, s.qkv + qc, ld, s.qkv + qc + kc, ld, pages, ldp, width, lens, s.attn, qc, nullptr, batch, heads, scale, s.attention,
                               s.attention_bytes);
    });
}

}  // extern "C"
