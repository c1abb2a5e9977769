// Pages of a cache handed out on the GPU: which pages a sequence has, how many rows, and the list of free pages stay on the device, and requests (new rows, or rows that
// remain, of some of the sequences) are answered there with page tables, slots and positions.  Lengths never go to the host, so a captured step serves new requests at each replay.
// No counterpart in o1.c, which keeps no keys or values from one forward to the next.
//
// With l_b rows of a request's sequence, n_b new ones and pages of s: it needs d_b = ceil((l_b + n_b) / s) - ceil(l_b / s) pages.  Two prefix sums over the requests,
// P_b = d_0 + ... + d_(b-1) and S_b = n_0 + ... + n_(b-1), place everything: its j-th new page is free[count - 1 - P_b - j] (the list is a stack), and row r of the
// requests' rows behind one another is row t = l_b + r - S_b of the sequence b with S_b <= r < S_(b+1), in slot table[b][t / s] * s + t % s.  Giving back is the same
// backwards: a sequence's page i, from the last one that remains on, goes to free[count' - 1 - P_b - i], so what a request took comes back in its order.
//
// Bound by latency: 12 bytes a row leave, a step of 24 sequences moves 20 KB, 1000 requests of 150000 rows 2.4 MB.  In a stream's chain a launch of one request takes 2.3 us, one of 24
// requests with tables of 132 pages 5.4 (given back: 3.3), 1000 requests 9 (5.4): requests, then lengths, then pages, then results, each a trip to L2, and the barriers of the sums
// between.  So it is one launch whose blocks each do both prefix sums
// (the requests are a few KB from L2) instead of one that sums and one that writes; state changes (lengths, the count of free pages) are left to the last block to
// come, when all have read them.
#include "common.cuh"
#include "kernels.h"
#include "../../include/o1_b200.h"

namespace o1 {

static constexpr int PG_THREADS = 1024, PG_SEQS = 8192;
static constexpr int PG_FULL = 1 << 30;             // sums end here, and no table or result is larger
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

// seq < 0: refused (its rows have no slots); after: its rows when it is done
struct PgRequest { int seq, len, after; };

// (twice PG_FULL is beyond int)
__device__ __forceinline__ int pg_add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)PG_FULL); }

// Sums of v over the block's threads before this one, and over all, of both components, which are between 0 and PG_FULL and stay there.
__device__ __forceinline__ int2 pg_scan(int2 v, int2& all, int2* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int2 sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
        if (lane >= o) { sum.x = pg_add(sum.x, x); sum.y = pg_add(sum.y, y); }
    }
    if (lane == 31) part[warp] = sum;
    int2 before = make_int2(__shfl_up_sync(0xffffffffu, sum.x, 1), __shfl_up_sync(0xffffffffu, sum.y, 1));
    if (lane == 0) before = make_int2(0, 0);
    __syncthreads();
    int2 p = lane < warps ? part[lane] : make_int2(0, 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, p.x, o), y = __shfl_up_sync(0xffffffffu, p.y, o);
        if (lane >= o) { p.x = pg_add(p.x, x); p.y = pg_add(p.y, y); }
    }
    all = make_int2(__shfl_sync(0xffffffffu, p.x, 31), __shfl_sync(0xffffffffu, p.y, 31));
    const int x = __shfl_sync(0xffffffffu, p.x, max(warp - 1, 0)), y = __shfl_sync(0xffffffffu, p.y, max(warp - 1, 0));
    if (warp > 0) before = make_int2(pg_add(before.x, x), pg_add(before.y, y));
    return before;
}

template <bool GROW>
__global__ void __launch_bounds__(PG_THREADS, 1)
pages_kernel(const PgArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int2 part[32];
    __shared__ int granted, last;
    PgRequest* const req = reinterpret_cast<PgRequest*>(smem);
    int* const start = reinterpret_cast<int*>(req + a.batch);          // [batch + 1] rows before a request
    int* const taken = start + a.batch + 1;                            // [batch] pages before it
    unsigned *const seen = reinterpret_cast<unsigned*>(taken + a.batch), *const twice = seen + ((a.max_seqs + 31) >> 5);
    const int tid = threadIdx.x, threads = blockDim.x, ps = a.page_size, shift = a.page_shift;
    const bool first_block = blockIdx.x == 0;
    grid_dep_launch();
    if (a.seqs) for (int i = tid; i < ((a.max_seqs + 31) >> 5) * 2; i += threads) seen[i] = 0;
    if (tid == 0) granted = 0;
    __syncthreads();
    grid_dep_wait();
    auto whole = [&](int64_t rows) { return (int)(shift >= 0 ? (rows + ps - 1) >> shift : (rows + ps - 1) / ps); };

    // ---- the requests; a thread's first one is on its way while sequences that the call names twice are found (neither of their requests is served)
    const int have = min(max(a.state[0], 0), a.pages);
    int seq = -1, asked = 0, len = 0;
    auto ask = [&](int b) {
        if (b >= a.batch) return;
        seq = a.seqs ? a.seqs[b] : b;
        asked = a.asked[b];
        len = (unsigned)seq < (unsigned)a.max_seqs ? a.lens[seq] : -1;
    };
    ask(tid);
    if (a.seqs) {
        for (int b = tid; b < a.batch; b += threads) {
            const int s = b == tid ? seq : a.seqs[b];
            if ((unsigned)s < (unsigned)a.max_seqs && (atomicOr(seen + (s >> 5), 1u << (s & 31)) >> (s & 31) & 1)) atomicOr(twice + (s >> 5), 1u << (s & 31));
        }
        __syncthreads();
    }
    int2 base = make_int2(0, 0);
    for (int b0 = 0; b0 < a.batch; b0 += threads) {
        const int b = b0 + tid;
        if (b0 > 0) ask(b);
        int2 mine = make_int2(0, 0);
        int code = 0;
        const int64_t after = GROW ? (int64_t)len + asked : asked;
        if (b < a.batch) {
            if (GROW) mine.x = min(max(asked, 0), PG_FULL);
            if ((unsigned)seq >= (unsigned)a.max_seqs || (a.seqs && (twice[seq >> 5] >> (seq & 31) & 1))) { seq = -1; code = ERR_PG_SEQUENCE; }
            else if (asked < 0 || len < 0 || (GROW ? after : len) > (int64_t)a.width * ps || (!GROW && asked > len)) { seq = -1; code = ERR_PG_LENGTH; }
            else mine.y = GROW ? whole(after) - whole(len) : whole(len) - whole(after);
        }
        int2 all, before = pg_scan(mine, all, part);
        before = make_int2(pg_add(before.x, base.x), pg_add(before.y, base.y));
        base = make_int2(pg_add(base.x, all.x), pg_add(base.y, all.y));
        if (b < a.batch) {
            // Both sums only grow, so what is refused for want of rows or pages has behind it only requests that are too, or that need no page: pages leave the stack from its top.
            if (GROW && seq >= 0 && mine.x > a.rows - before.x && mine.x > 0) { seq = -1; code = ERR_PG_LENGTH; }
            if (seq >= 0 && mine.y > 0 && mine.y > (GROW ? have : a.pages - have) - before.y) { seq = -1; code = ERR_PG_NONE_LEFT; }
            req[b] = {seq, len, (int)after};
            start[b] = before.x;
            taken[b] = before.y;
            if (seq >= 0 && mine.y > 0) atomicMax(&granted, before.y + mine.y);
            if (first_block) {
                if (code) atomicExch(a.bad, code);
                if (GROW) {
                    a.starts[b] = start[b];
                    a.lens_out[b] = seq >= 0 ? (int)after : 0;
                }
            }
        }
        if (b0 + threads < a.batch) __syncthreads();          // (the scan's sums are read)
    }
    if (tid == 0) {
        start[a.batch] = base.x;
        if (GROW && first_block) a.starts[a.batch] = base.x;
    }
    __syncthreads();
    const int total = granted, top = (GROW ? have : have + total) - 1;

    // ---- the rows, four to a thread
    if (GROW) {
        const int known = min(start[a.batch], a.rows);
        for (int64_t r0 = ((int64_t)blockIdx.x * threads + tid) * 4; r0 < a.rows; r0 += (int64_t)gridDim.x * threads * 4) {
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
                    const int known_pages = whole(q.len);
                    page = j < known_pages ? a.table[(int64_t)q.seq * a.width + j] : a.free_pages[top - taken[b] - (j - known_pages)];
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
    // ---- the tables, PG_COLS entries to a warp, from the last warp on (the first ones have rows); a lane's entries all on their way before the first is stored
    const int lane = tid & 31, pieces = (a.width + PG_COLS - 1) / PG_COLS, warps = threads / 32;
    for (int64_t task = (int64_t)gridDim.x * warps - 1 - ((int64_t)blockIdx.x * warps + (tid >> 5)); task < (int64_t)a.batch * pieces; task += (int64_t)gridDim.x * warps) {
        const int b = (int)(task / pieces), j0 = (int)(task - (int64_t)b * pieces) * PG_COLS;
        const PgRequest q = req[b];
        int32_t* const row = a.table + (int64_t)max(q.seq, 0) * a.width;
        int32_t* const out = GROW && a.tables_out ? a.tables_out + b * a.ldp : nullptr;
        const int lo = whole(GROW ? q.len : q.after), hi = whole(GROW ? q.after : q.len);         // pages that come or go
        if (!out && (q.seq < 0 || j0 >= hi || j0 + PG_COLS <= lo)) continue;
        int page[PG_COLS / 32];
#pragma unroll
        for (int i = 0; i < PG_COLS / 32; ++i) {
            const int j = j0 + i * 32 + lane;
            const bool moves = q.seq >= 0 && j >= lo && j < hi;
            page[i] = -1;
            if (GROW && moves) page[i] = a.free_pages[top - taken[b] - (j - lo)];
            else if (GROW ? out && q.seq >= 0 && j < lo : moves) page[i] = row[j];
        }
#pragma unroll
        for (int i = 0; i < PG_COLS / 32; ++i) {
            const int j = j0 + i * 32 + lane;
            if (j >= a.width) break;
            const bool moves = q.seq >= 0 && j >= lo && j < hi;
            if (GROW && moves) row[j] = page[i];
            if (out) out[j] = page[i];
            if (!GROW && moves) {
                a.free_pages[top - taken[b] - (j - lo)] = page[i];
                row[j] = -1;
            }
        }
    }
    // ---- lengths and the count of free pages, when all blocks have read them
    __syncthreads();
    if (tid == 0) {
        int before = gridDim.x - 1;
        if (gridDim.x > 1) asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(a.state + 1) : "memory");
        last = before == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    for (int b = tid; b < a.batch; b += threads)
        if (req[b].seq >= 0) a.lens[req[b].seq] = req[b].after;
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
    if ((int64_t)p->width * p->page_size > PG_FULL || p->pages > PG_FULL) { set_error("%s: a table of %d pages of %d tokens, or a list of %d pages, is too large", what, p->width, p->page_size, p->pages); return HD_ERR_UNSUPPORTED; }
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
    // as many threads as there are requests or steps of the rows and tables, one block up to PG_THREADS
    const int64_t work = max((GROW ? (int64_t)a.rows : 0) / 4, (int64_t)a.batch * ((a.width + PG_COLS - 1) / PG_COLS) * 32);
    const int threads = (int)min((int64_t)PG_THREADS, max((int64_t)a.batch, work) + 31 & ~(int64_t)31);
    const int blocks = work <= 2 * PG_THREADS ? 1 : (int)min((int64_t)sm_count(), (work + PG_THREADS - 1) / PG_THREADS);
    if (!launch_ok(launch_chained(pages_kernel<GROW>, dim3(blocks), dim3(max(threads, 32)), smem, current_stream(), 1, 1, a), what)) return HD_ERR_RUNTIME;
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
    if (batch < 0 || batch > a.max_seqs || rows < 0 || rows > PG_FULL) { set_error("kv_pages_grow: batch %d (at most max_seqs %d), rows %d (at most 2^30)", batch, a.max_seqs, rows); return HD_ERR_UNSUPPORTED; }
    if ((batch > 0 && (!counts || !lens)) || !starts || (rows > 0 && (!slots || !positions))) { set_error("kv_pages_grow: null argument"); return HD_ERR_MISSING; }
    if (tables && ldp < a.width) { set_error("kv_pages_grow: a row pitch is below the row"); return HD_ERR_UNSUPPORTED; }
    // Blocks read requests and state while others write results.
    struct Range { const void* at; int64_t bytes; };
    const int64_t n = batch, max_seqs = a.max_seqs;
    const Range ranges[] = {{slots, rows * 8ll}, {positions, rows * 4ll}, {starts, (n + 1) * 4}, {lens, n * 4}, {tables, n > 0 && tables ? ((n - 1) * ldp + a.width) * 4 : 0},
                            {counts, n * 4}, {seqs, seqs ? n * 4 : 0}, {a.table, max_seqs * a.width * 4}, {a.lens, max_seqs * 4}, {a.free_pages, a.pages * 4ll}, {a.state, 8}};
    for (int i = 0; i < 5; ++i) {
        for (int j = i + 1; j < 11; ++j) {
            const Range &r = ranges[i], &q = ranges[j];
            if (r.bytes == 0 || q.bytes == 0 || (uintptr_t)r.at + r.bytes <= (uintptr_t)q.at || (uintptr_t)q.at + q.bytes <= (uintptr_t)r.at) continue;
            set_error("kv_pages_grow: a result shares memory with another one, the requests or the pages themselves");
            return HD_ERR_UNSUPPORTED;
        }
    }
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
