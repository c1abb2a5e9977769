// Pages of a cache handed out on the GPU: which pages a sequence has, how many rows, and the list of free pages stay on the device, and requests (new rows, or rows that
// remain, of some of the sequences) are answered there with page tables, slots and positions.  Lengths never go to the host, so a captured step serves new requests at each replay.
// No counterpart in o1.c, which keeps no keys or values from one forward to the next.
//
// With l_b rows of a request's sequence, n_b new ones and pages of s: it needs d_b = ceil((l_b + n_b) / s) - ceil(l_b / s) pages.  Two prefix sums over the requests,
// P_b = d_0 + ... + d_(b-1) and S_b = n_0 + ... + n_(b-1), place everything: its j-th new page is free[count - 1 - P_b - j] (the list is a stack), and row r of the
// requests' rows behind one another is row t = l_b + r - S_b of the sequence b with S_b <= r < S_(b+1), in slot table[b][t / s] * s + t % s.  Giving back is the same
// backwards: a sequence's page i, from the last one that remains on, goes to free[count' - 1 - P_b - i], so what a request took comes back in its order.
//
// Bound by latency: 12 bytes a row leave, a step of 24 sequences moves 20 KB, 1000 requests of 150000 rows 2.4 MB.  So it is one launch whose blocks each do both prefix sums
// (the requests are a few KB from L2) instead of one that sums and one that writes; state changes (lengths, the count of free pages) are left to the last block to
// come, when all have read them.
#include "common.cuh"
#include "kernels.h"
#include "../../include/o1_b200.h"

#include <limits.h>

namespace o1 {

static constexpr int PG_THREADS = 512, PG_SEQS = 8192;
static constexpr int PG_COLS = 128;                // entries of a sequence's table to a warp's step
static constexpr int ERR_PG_SEQUENCE = 70, ERR_PG_LENGTH = 71, ERR_PG_NONE_LEFT = 73;

struct PgArgs {
    int32_t *table, *lens, *free_pages, *state;    // state: free pages; blocks that have come
    int pages, page_size, page_shift, max_seqs, width;
    const int32_t *seqs, *asked;                   // asked: new rows, or rows that remain
    int batch, rows;
    int64_t* slots;
    int32_t *positions, *starts, *lens_out, *tables_out;
    int64_t ldp;
    int* bad;
};

struct PgRequest { int seq, len, pages_before, pages_after; };      // seq < 0: refused (its rows have no slots)

// Sums of v over the block's threads before this one, and over all, of both components.
__device__ __forceinline__ longlong2 pg_scan(longlong2 v, longlong2& all, longlong2* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    longlong2 sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
        if (lane >= o) { sum.x += x; sum.y += y; }
    }
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    longlong2 before = make_longlong2(sum.x - v.x, sum.y - v.y);
    all = make_longlong2(0, 0);
#pragma unroll
    for (int w = 0; w < PG_THREADS / 32; ++w) {
        const longlong2 p = part[w];
        if (w < warp) { before.x += p.x; before.y += p.y; }
        all.x += p.x;
        all.y += p.y;
    }
    __syncthreads();
    return before;
}

template <bool GROW>
__global__ void __launch_bounds__(PG_THREADS)
pages_kernel(const PgArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ longlong2 part[PG_THREADS / 32];
    __shared__ int granted, last;
    PgRequest* const req = reinterpret_cast<PgRequest*>(smem);
    int* const start = reinterpret_cast<int*>(req + a.batch);          // [batch + 1] rows before a request
    int* const taken = start + a.batch + 1;                            // [batch] pages before it
    unsigned *const seen = reinterpret_cast<unsigned*>(taken + a.batch), *const twice = seen + ((a.max_seqs + 31) >> 5);
    const int tid = threadIdx.x, ps = a.page_size, shift = a.page_shift;
    const bool first_block = blockIdx.x == 0;
    grid_dep_launch();
    if (a.seqs) for (int i = tid; i < ((a.max_seqs + 31) >> 5) * 2; i += PG_THREADS) seen[i] = 0;
    if (tid == 0) granted = 0;
    __syncthreads();
    grid_dep_wait();
    auto whole = [&](int64_t rows) { return (int)(shift >= 0 ? (rows + ps - 1) >> shift : (rows + ps - 1) / ps); };

    // ---- the requests
    const int have = min(max(a.state[0], 0), a.pages);
    for (int b = tid; a.seqs && b < a.batch; b += PG_THREADS) {        // a sequence twice: neither request is served
        const int s = a.seqs[b];
        if ((unsigned)s < (unsigned)a.max_seqs && (atomicOr(seen + (s >> 5), 1u << (s & 31)) >> (s & 31) & 1)) atomicOr(twice + (s >> 5), 1u << (s & 31));
    }
    __syncthreads();
    longlong2 base = make_longlong2(0, 0);
    for (int b0 = 0; b0 < a.batch; b0 += PG_THREADS) {
        const int b = b0 + tid;
        PgRequest r = {-1, 0, 0, 0};
        longlong2 mine = make_longlong2(0, 0);
        int code = 0;
        if (b < a.batch) {
            r.seq = a.seqs ? a.seqs[b] : b;
            const int n = a.asked[b];
            if ((unsigned)r.seq >= (unsigned)a.max_seqs || (a.seqs && (twice[r.seq >> 5] >> (r.seq & 31) & 1))) { r.seq = -1; code = ERR_PG_SEQUENCE; }
            else r.len = a.lens[r.seq];
            const int64_t after = GROW ? (int64_t)r.len + n : n;
            if (GROW && n > 0) mine.x = n;
            if (r.seq >= 0 && (n < 0 || r.len < 0 || (GROW ? after : r.len) > (int64_t)a.width * ps || (!GROW && n > r.len))) { r.seq = -1; code = ERR_PG_LENGTH; }
            if (r.seq >= 0) {
                r.pages_before = whole(r.len);
                r.pages_after = whole(after);
                mine.y = GROW ? r.pages_after - r.pages_before : r.pages_before - r.pages_after;
            }
        }
        longlong2 all;
        longlong2 before = pg_scan(mine, all, part);
        before.x += base.x; before.y += base.y;
        base.x += all.x; base.y += all.y;
        if (b < a.batch) {
            // Both sums only grow, so what is refused for want of rows or pages has behind it only requests that are too, or that need no page: pages leave the stack from its top.
            if (GROW && r.seq >= 0 && before.x + mine.x > a.rows && mine.x > 0) { r.seq = -1; code = ERR_PG_LENGTH; }
            if (r.seq >= 0 && mine.y > 0 && before.y + mine.y > (GROW ? have : a.pages - have)) { r.seq = -1; code = ERR_PG_NONE_LEFT; }
            req[b] = r;
            start[b] = (int)min(before.x, (long long)INT_MAX);
            taken[b] = (int)min(before.y, (long long)INT_MAX);
            if (r.seq >= 0 && mine.y > 0) atomicMax(&granted, (int)(before.y + mine.y));
            if (first_block) {
                if (code) atomicExch(a.bad, code);
                if (GROW) {
                    a.starts[b] = start[b];
                    a.lens_out[b] = r.seq >= 0 ? r.len + a.asked[b] : 0;
                }
            }
        }
    }
    if (tid == 0) {
        start[a.batch] = (int)min(base.x, (long long)INT_MAX);
        if (GROW && first_block) a.starts[a.batch] = start[a.batch];
    }
    __syncthreads();
    const int total = granted, top = (GROW ? have : have + total) - 1;

    // ---- the rows, four to a thread
    if (GROW) {
        const int known = min(start[a.batch], a.rows);
        for (int64_t r0 = ((int64_t)blockIdx.x * PG_THREADS + tid) * 4; r0 < a.rows; r0 += (int64_t)gridDim.x * PG_THREADS * 4) {
            long long slot[4];
            int pos[4], b = 0;
            if (r0 < known) {
                int hi = a.batch - 1;
                while (b < hi) {
                    const int mid = (b + hi + 1) >> 1;
                    if (start[mid] <= r0) b = mid; else hi = mid - 1;
                }
            }
            int page_of = -1, page = 0, owner = -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = (int)r0 + i;
                slot[i] = -1;
                pos[i] = 0;
                if (r0 + i >= known) continue;
                while (start[b + 1] <= r) ++b;
                const PgRequest q = req[b];
                if (q.seq < 0) continue;
                const int t = q.len + r - start[b], j = shift >= 0 ? t >> shift : t / ps;
                if (owner != b || page_of != j) {
                    page = j < q.pages_before ? a.table[(int64_t)q.seq * a.width + j] : a.free_pages[top - taken[b] - (j - q.pages_before)];
                    owner = b;
                    page_of = j;
                }
                slot[i] = (long long)page * ps + (t - j * ps);
                pos[i] = t;
            }
            if (r0 + 4 <= a.rows && ((uintptr_t)a.slots & 15) == 0 && ((uintptr_t)a.positions & 15) == 0) {
                *reinterpret_cast<longlong2*>(a.slots + r0) = make_longlong2(slot[0], slot[1]);
                *reinterpret_cast<longlong2*>(a.slots + r0 + 2) = make_longlong2(slot[2], slot[3]);
                *reinterpret_cast<int4*>(a.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) if (r0 + i < a.rows) { a.slots[r0 + i] = slot[i]; a.positions[r0 + i] = pos[i]; }
            }
        }
    }
    // ---- the tables, PG_COLS entries to a warp
    const int lane = tid & 31, pieces = (a.width + PG_COLS - 1) / PG_COLS;
    for (int64_t task = (int64_t)blockIdx.x * (PG_THREADS / 32) + (tid >> 5); task < (int64_t)a.batch * pieces; task += (int64_t)gridDim.x * (PG_THREADS / 32)) {
        const int b = (int)(task / pieces), j0 = (int)(task - (int64_t)b * pieces) * PG_COLS;
        const PgRequest q = req[b];
        int32_t* const row = a.table + (int64_t)max(q.seq, 0) * a.width;
        int32_t* const out = GROW && a.tables_out ? a.tables_out + b * a.ldp : nullptr;
        const int lo = GROW ? q.pages_before : q.pages_after, hi = GROW ? q.pages_after : q.pages_before;         // pages that come or go
        if (!out && (q.seq < 0 || j0 >= hi || j0 + PG_COLS <= lo)) continue;
#pragma unroll
        for (int i = 0; i < PG_COLS / 32; ++i) {
            const int j = j0 + i * 32 + lane;
            if (j >= a.width) break;
            const bool moves = q.seq >= 0 && j >= lo && j < hi;
            if (GROW) {
                int page = -1;
                if (moves) row[j] = page = a.free_pages[top - taken[b] - (j - lo)];
                else if (out && q.seq >= 0 && j < lo) page = row[j];
                if (out) out[j] = page;
            } else if (moves) {
                a.free_pages[top - taken[b] - (j - lo)] = row[j];
                row[j] = -1;
            }
        }
    }
    // ---- lengths and the count of free pages, when all blocks have read them
    __syncthreads();
    if (tid == 0) {
        bool mine = true;
        if (gridDim.x > 1) {
            __threadfence();
            mine = atomicAdd(a.state + 1, 1) == (int)gridDim.x - 1;
            __threadfence();
        }
        last = mine;
    }
    __syncthreads();
    if (!last) return;
    for (int b = tid; b < a.batch; b += PG_THREADS)
        if (req[b].seq >= 0) a.lens[req[b].seq] = GROW ? req[b].len + a.asked[b] : a.asked[b];
    if (tid == 0) {
        a.state[0] = top + 1 - (GROW ? total : 0);
        if (gridDim.x > 1) a.state[1] = 0;
    }
}

__global__ void pages_reset_kernel(const PgArgs a) {
    grid_dep_launch();
    grid_dep_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x, at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t i = at; i < (int64_t)a.max_seqs * a.width; i += step) a.table[i] = -1;
    for (int64_t i = at; i < a.pages; i += step) a.free_pages[i] = a.pages - 1 - (int)i;
    for (int64_t i = at; i < a.max_seqs; i += step) a.lens[i] = 0;
    if (at == 0) { a.state[0] = a.pages; a.state[1] = 0; }
}

static hd_status pages_view(const o1_kv_pages* p, PgArgs* a, const char* what) {
    if (!p || !p->table || !p->lens || !p->free_pages || !p->state) { set_error("%s: null pages", what); return HD_ERR_MISSING; }
    if (p->pages <= 0 || p->page_size <= 0 || p->page_size % 16 || p->max_seqs <= 0 || p->max_seqs > PG_SEQS || p->width <= 0) {
        set_error("%s: pages %d, page_size %d (a multiple of 16), max_seqs %d (at most %d), width %d", what, p->pages, p->page_size, p->max_seqs, PG_SEQS, p->width);
        return HD_ERR_UNSUPPORTED;
    }
    if ((int64_t)p->width * p->page_size > INT_MAX) { set_error("%s: a table of %d pages of %d tokens is too large", what, p->width, p->page_size); return HD_ERR_UNSUPPORTED; }
    *a = {};
    a->table = p->table; a->lens = p->lens; a->free_pages = p->free_pages; a->state = p->state;
    a->pages = p->pages; a->page_size = p->page_size; a->max_seqs = p->max_seqs; a->width = p->width;
    a->page_shift = -1;
    if ((p->page_size & (p->page_size - 1)) == 0)
        for (a->page_shift = 0; (1 << a->page_shift) < p->page_size; ++a->page_shift) {}
    a->bad = device_table_word();
    return HD_OK;
}

template <bool GROW>
static hd_status launch_pages(const PgArgs& a, const char* what) {
    static std::atomic<uint64_t> done{0};
    constexpr int most = PG_SEQS * (int)(sizeof(PgRequest) + 8) + 4 + (PG_SEQS / 32) * 8;
    static_assert(most <= 232448 - 1024, "more than an SM's block can have");
    if (!func_attr_once(done, (const void*)pages_kernel<GROW>, most, what)) return HD_ERR_RUNTIME;
    const size_t smem = a.batch * (sizeof(PgRequest) + 8) + 4 + (a.seqs ? ((a.max_seqs + 31) / 32) * 8 : 0);
    const int64_t work = max((GROW ? (int64_t)a.rows : 0) / 4, (int64_t)a.batch * ((a.width + PG_COLS - 1) / PG_COLS) * 32);
    const int blocks = (int)max((int64_t)1, min((int64_t)sm_count(), (work + PG_THREADS - 1) / PG_THREADS));
    if (!launch_ok(launch_chained(pages_kernel<GROW>, dim3(blocks), dim3(PG_THREADS), smem, current_stream(), 1, 1, a), what)) return HD_ERR_RUNTIME;
    return HD_OK;
}

}  // namespace o1

using namespace o1;

extern "C" {
void o1_launch_count_add(int n);

hd_status o1_kv_pages_reset(const o1_kv_pages* pages) {
    PgArgs a;
    const hd_status st = pages_view(pages, &a, "kv_pages_reset");
    if (st != HD_OK) return st;
    const int64_t most = max((int64_t)a.pages, (int64_t)a.max_seqs * a.width);
    if (!launch_ok(launch_chained(pages_reset_kernel, dim3((unsigned)min((int64_t)sm_count(), (most + 255) / 256)), dim3(256), 0, current_stream(), 1, 1, a), "kv_pages_reset"))
        return HD_ERR_RUNTIME;
    o1_launch_count_add(1);
    return HD_OK;
}

hd_status o1_kv_pages_grow(const o1_kv_pages* pages, const int32_t* seqs, const int32_t* counts, int batch, int64_t* slots, int32_t* positions, int rows,
                           int32_t* starts, int32_t* lens, int32_t* tables, int64_t ldp) {
    PgArgs a;
    hd_status st = pages_view(pages, &a, "kv_pages_grow");
    if (st != HD_OK) return st;
    if (batch < 0 || batch > a.max_seqs || rows < 0) { set_error("kv_pages_grow: batch %d (at most max_seqs %d), rows %d", batch, a.max_seqs, rows); return HD_ERR_UNSUPPORTED; }
    if ((batch > 0 && (!counts || !lens)) || !starts || (rows > 0 && (!slots || !positions))) { set_error("kv_pages_grow: null argument"); return HD_ERR_MISSING; }
    if (tables && ldp < a.width) { set_error("kv_pages_grow: a row pitch is below the row"); return HD_ERR_UNSUPPORTED; }
    a.seqs = seqs; a.asked = counts; a.batch = batch; a.rows = rows;
    a.slots = slots; a.positions = positions; a.starts = starts; a.lens_out = lens; a.tables_out = tables; a.ldp = ldp;
    st = launch_pages<true>(a, "kv_pages_grow");
    if (st == HD_OK) o1_launch_count_add(1);
    return st;
}

hd_status o1_kv_pages_shrink(const o1_kv_pages* pages, const int32_t* seqs, const int32_t* keep, int batch) {
    PgArgs a;
    hd_status st = pages_view(pages, &a, "kv_pages_shrink");
    if (st != HD_OK) return st;
    if (batch < 0 || batch > a.max_seqs) { set_error("kv_pages_shrink: batch %d (at most max_seqs %d)", batch, a.max_seqs); return HD_ERR_UNSUPPORTED; }
    if (batch == 0) return HD_OK;
    if (!keep) { set_error("kv_pages_shrink: null argument"); return HD_ERR_MISSING; }
    a.seqs = seqs; a.asked = keep; a.batch = batch;
    st = launch_pages<false>(a, "kv_pages_shrink");
    if (st == HD_OK) o1_launch_count_add(1);
    return st;
}

}  // extern "C"
