// The pages of a paged key-value cache: forking and freeing rows by reference, making room for new tokens (with a copy of a
// shared last page before it is written), copying pages over all layers, moving the live pages together, and gathering rows
// of contiguous state by parent. A page is free when its reference count is 0; there is no other free list, so every choice
// of a page (the lowest free ones, ascending) follows from the counts alone and repeats from run to run.
//
// Bookkeeping is integer work on small arrays, bound by latency (freeing, forking and reserving 128 rows of some 130 pages, a token
// each, with copies of 62 MB: 22 us on a B200, about half of it the copies; a row's new pages are handed out by one thread, one after
// the other, which a prompt of thousands of pages waits for); the copies are bound by HBM, each byte read and written once
// (504 pages of 32 KB in 64 pools 337 us, rows of 1.4 MB 191 us: 6.3 and 6.6 TB/s).
#include "serving.cuh"

namespace tlb {

namespace {

// ---- forking -------------------------------------------------------------------------------------------------------
// Row r becomes a copy of row parents[r]; the permutation acts within a column of the table, so a CTA that holds a slab of
// columns of ALL rows in shared memory needs no other CTA and no second launch. Entries that stay the same are skipped.
// The last CTA does the same with the lengths. Counts change by atomic additions of whole numbers: any order, same result.
constexpr int FORK_THREADS = 256;
constexpr int FORK_SMEM = 196608;

template <int SLAB>
__global__ void __launch_bounds__(FORK_THREADS) k_fork(int* table, int* lengths, int* refs, const int* parents, int n_rows,
                                                       int max_pages, int n_pages, int* status) {
    extern __shared__ int sm[];
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == gridDim.x - 1) {            // the lengths
        for (int r = threadIdx.x; r < n_rows; r += FORK_THREADS) sm[r] = lengths[r];
        __syncthreads();
        for (int r = threadIdx.x; r < n_rows; r += FORK_THREADS) {
            const int parent = parents[r];
            if (parent >= n_rows || parent < -1) atomicExch(status, TL_ERR_INVALID_ARGUMENT);
            else if (parent != r) lengths[r] = parent < 0 ? 0 : sm[parent];
        }
        return;
    }
    const int c0 = blockIdx.x * SLAB;
    int* base = table + c0;
    for (int i = threadIdx.x; i < n_rows * SLAB; i += FORK_THREADS) {
        const int r = i / SLAB, j = i % SLAB;
        sm[i] = c0 + j < max_pages ? base[(long long)r * max_pages + j] : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * SLAB; i += FORK_THREADS) {
        const int r = i / SLAB, j = i % SLAB;
        const int parent = parents[r];
        if (parent >= n_rows || parent < -1) continue;         // not a row: this one stays as it is
        const int o = sm[i], n = parent < 0 ? -1 : sm[parent * SLAB + j];
        if (o == n) continue;
        base[(long long)r * max_pages + j] = n;
        if (n >= 0 && n < n_pages) atomicAdd(refs + n, 1);
        if (o >= 0 && o < n_pages) atomicSub(refs + o, 1);
        if (n >= n_pages || o >= n_pages || n < -1 || o < -1) atomicExch(status, TL_ERR_INVALID_ARGUMENT);
    }
}

// ---- page contents -------------------------------------------------------------------------------------------------
// The first `n` tokens of a page as `runs` runs of contiguous vectors: one run where the page is packed by token, one a head
// where it is packed by head, one a token where only the heads are packed, else one a (token, head).
struct PageShape {
    long long token_stride, head_stride;
    int page_size, heads, dim;
    int vec;                       // halfs a vector: 8 where everything is 16-byte aligned, else 1
    int kind;                      // 0 packed by token, 1 packed by head, 2 heads packed, 3 neither
    FastDiv by_row, by_heads;
};

PageShape page_shape(const PagedView& c) {
    PageShape s{};
    s.token_stride = c.token_stride; s.head_stride = c.head_stride;
    s.page_size = c.page_size; s.heads = c.n_kv_heads; s.dim = c.head_dim;
    s.vec = c.aligned16() ? 8 : 1;
    const bool heads_packed = c.head_stride == c.head_dim;
    if (heads_packed && c.token_stride == (long long)c.n_kv_heads * c.head_dim) s.kind = 0;
    else if (c.token_stride == c.head_dim) s.kind = 1;
    else s.kind = heads_packed ? 2 : 3;
    const int row = s.kind == 2 ? c.n_kv_heads * c.head_dim : c.head_dim;   // kinds 0 and 1 take their run lengths from n
    s.by_row = FastDiv((unsigned)(row / s.vec));
    s.by_heads = FastDiv((unsigned)c.n_kv_heads);
    return s;
}

// n vectors by THREADS threads, eight loads under way each
template <typename V, int THREADS>
__device__ __forceinline__ void copy_run(__half* dst, const __half* src, int n, int tid) {
    const V* s = reinterpret_cast<const V*>(src) + tid;
    V* d = reinterpret_cast<V*>(dst) + tid;
    constexpr int U = 8;
    for (int left = n - tid; left > 0; left -= U * THREADS, s += U * THREADS, d += U * THREADS) {
        V x[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u * THREADS < left) x[u] = s[u * THREADS];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u * THREADS < left) d[u * THREADS] = x[u];
    }
}

template <typename V, int THREADS>
__device__ __forceinline__ void copy_page(const PageShape& s, __half* dst, const __half* src, int n, int tid) {
    constexpr int VEC = sizeof(V) / sizeof(__half);
    if (s.kind <= 1) {
        const bool by_head = s.kind == 1 && !(n == s.page_size && s.head_stride == (long long)n * s.dim);
        const int len = n * s.dim / VEC * (by_head ? 1 : s.heads);
        for (int run = 0; run < (by_head ? s.heads : 1); run++)
            copy_run<V, THREADS>(dst + run * s.head_stride, src + run * s.head_stride, len, tid);
        return;
    }
    const unsigned total = (unsigned)n * (s.kind == 2 ? 1 : s.heads) * s.by_row.d;
    for (unsigned i = tid; i < total; i += THREADS) {
        unsigned run, v, tok, h = 0;
        s.by_row.divmod(i, run, v);
        tok = run;
        if (s.kind == 3) s.by_heads.divmod(run, tok, h);
        const long long at = tok * s.token_stride + h * s.head_stride;
        reinterpret_cast<V*>(dst + at)[v] = reinterpret_cast<const V*>(src + at)[v];
    }
}

constexpr int COPY_THREADS = 256;

// An item is one page of one layer of K or of V; TEAM threads copy it (a CTA, or where pages are small a warp).
struct CopyArgs {
    __half* k; __half* v;
    long long layer_stride, page_stride;
    int n_layers, n_pages, team;
    PageShape shape;
    FastDiv by_each;                              // 2 n_layers items a page
    int* status;
};

template <typename V, int TEAM>
__device__ __forceinline__ void copy_item(const CopyArgs& a, unsigned what, int src, int dst, int tokens) {
    __half* pool = (what & 1) ? a.v : a.k;
    __half* layer = pool + (long long)(what >> 1) * a.layer_stride;
    copy_page<V, TEAM>(a.shape, layer + dst * a.page_stride, layer + src * a.page_stride, tokens, threadIdx.x % TEAM);
}
// f(page pair, what) for the items of n page pairs, below 2^31 in all
template <int TEAM, typename Fn>
__device__ __forceinline__ void each_item(const CopyArgs& a, int n, Fn&& f) {
    constexpr unsigned TEAMS = COPY_THREADS / TEAM;
    const unsigned total = (unsigned)n * a.by_each.d;
    for (unsigned it = blockIdx.x * TEAMS + threadIdx.x / TEAM; it < total; it += gridDim.x * TEAMS) {
        unsigned m, what;
        a.by_each.divmod(it, m, what);
        f((int)m, what);
    }
}

template <typename V, int TEAM>
__global__ void __launch_bounds__(COPY_THREADS, 4) k_copy_pages(CopyArgs a, const int* src, const int* dst, int n) {
    pdl_launch_dependents();
    pdl_wait();
    each_item<TEAM>(a, n, [&](int m, unsigned what) {
        const int s = src[m], d = dst[m];
        if (s == d || s == -1) return;
        if (s < 0 || d < 0 || s >= a.n_pages || d >= a.n_pages) {
            atomicExch(a.status, TL_ERR_INVALID_ARGUMENT);
            return;
        }
        copy_item<V, TEAM>(a, what, s, d, a.shape.page_size);
    });
}

// ---- making room ---------------------------------------------------------------------------------------------------
// Sequential meaning, rows in ascending order: a row whose next token goes into a page that other rows still hold gets a
// copy of its own; the last holder keeps the page. One CTA: the whole is a few dependent passes over n_rows and n_pages
// small integers. Nothing is written to the table before it is known that every row can be served.
constexpr int RES_THREADS = 1024;

struct CowItem { int src, dst, tokens, pad; };
struct ReserveWork {
    int* n_copies; CowItem* copies; int* need; int* freed;
};

__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* warp_sums, unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    unsigned long long before = 0, all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    total = all;
    return before + x - v;
}

__global__ void __launch_bounds__(RES_THREADS, 1) k_reserve(PagedView c, const int* new_tokens, int* result, ReserveWork wk, int* status) {
    __shared__ unsigned long long sums[RES_THREADS / 32];
    __shared__ int bad_sh;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x;
    // Rows r0 .. r1 are this thread's; of the first one, where nearly always there is no other, everything stays in registers.
    const int per = (c.n_rows + RES_THREADS - 1) / RES_THREADS;
    const int r0 = min(c.n_rows, tid * per), r1 = min(c.n_rows, r0 + per);
    constexpr int WRITES = 1 << 30, COPY = 1 << 29;
    // copies and pages are summed in one number: a table of 2^36 entries is more than any memory, and there are fewer than 2^28 rows
    constexpr int COPIES = 36;
    constexpr unsigned long long PAGES = (1ull << COPIES) - 1;
    struct Row { int len, add, pages, slot, last, flag; };     // pages that it holds, slots used of the last one, its id
    auto read = [&](int r) {
        Row x;
        x.len = c.lengths[r];
        x.add = new_tokens[r];
        if (x.len < 0) x.len = -1;
        const unsigned whole = x.len < 0 ? 0u : c.by_page.div((unsigned)x.len);
        x.slot = x.len < 0 ? 0 : (int)((unsigned)x.len - whole * c.by_page.d);
        x.pages = (int)whole + (x.slot != 0);
        x.last = -1;
        x.flag = 0;
        return x;
    };
    auto again = [&](int r) {                     // a row beyond the first, with what was found out about it
        Row x = read(r);
        x.flag = wk.need[r];
        if (x.flag & WRITES) x.last = __ldcg(c.table + (long long)r * c.max_pages + x.pages - 1);
        return x;
    };
    Row mine{};
    if (r0 < r1) mine = read(r0);
    // the free pages among the first 4 RES_THREADS ones, as they are before any count changes
    unsigned free4 = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int pg = tid * 4 + i;
        if (pg < c.n_pages && __ldcg(c.refs + pg) == 0) free4 |= 1u << i;
    }
    if (tid == 0) bad_sh = 0;
    __syncthreads();
    // 1: every row that writes into a page that is there lets go of it
    auto let_go = [&](int r, Row& x) {
        if (x.len < 0 || x.add < 0) { atomicMax(&bad_sh, 2); return; }
        if ((long long)x.len + x.add > (long long)c.max_pages * c.page_size) { atomicMax(&bad_sh, 1); return; }
        if (x.add == 0 || x.slot == 0) return;
        x.last = __ldcg(c.table + (long long)r * c.max_pages + x.pages - 1);
        if (x.last < 0 || x.last >= c.n_pages) { atomicMax(&bad_sh, 2); return; }
        if (atomicSub(c.refs + x.last, 1) <= 0) atomicMax(&bad_sh, 2);
        x.flag = WRITES;
    };
    if (r0 < r1) let_go(r0, mine);
    for (int r = r0 + 1; r < r1; r++) {
        Row x = read(r);
        let_go(r, x);
        wk.need[r] = x.flag;
    }
    __syncthreads();
    if (bad_sh) {                                 // refused: before a count is used as a claim, so that taking back restores each
        auto take_back = [&](const Row& x) {
            if (x.flag & WRITES) atomicAdd(c.refs + x.last, 1);
        };
        if (r0 < r1) take_back(mine);
        for (int r = r0 + 1; r < r1; r++) take_back(again(r));
        if (tid == 0) {
            *result = bad_sh == 2 ? TL_ERR_INVALID_ARGUMENT : TL_ERR_OUT_OF_MEMORY;
            *wk.n_copies = 0;
            if (bad_sh == 2) atomicExch(status, TL_ERR_INVALID_ARGUMENT);
        }
        return;
    }
    // 2: a page that nobody holds any more goes to the highest of the rows that let go of it: its count becomes -(row + 1)
    auto claim = [&](int r, const Row& x) {
        if ((x.flag & WRITES) && __ldcg(c.refs + x.last) <= 0) atomicMin(c.refs + x.last, -(r + 1));
    };
    if (r0 < r1) claim(r0, mine);
    for (int r = r0 + 1; r < r1; r++) claim(r, again(r));
    __syncthreads();
    unsigned long long wants = 0;                 // copies from bit COPIES up, pages below
    auto count = [&](int r, Row& x) {
        if ((x.flag & WRITES) && __ldcg(c.refs + x.last) != -(r + 1)) {
            x.flag |= COPY;
            wants += (1ull << COPIES) + 1;
        }
        if (x.add > 0) wants += (unsigned)((int)c.by_page.div((unsigned)(x.len + x.add - 1)) + 1 - x.pages);
    };
    if (r0 < r1) count(r0, mine);
    for (int r = r0 + 1; r < r1; r++) {
        Row x = again(r);
        count(r, x);
        wk.need[r] = x.flag;
    }
    // 3: the keepers' counts are 1 again (after the barrier in the sum: everyone has looked)
    unsigned long long total;
    const unsigned long long before = block_scan(wants, sums, total);
    const long long pages_wanted = (long long)(total & PAGES);
    auto keep = [&](const Row& x) {
        if ((x.flag & (WRITES | COPY)) == WRITES) atomicExch(c.refs + x.last, 1);
    };
    if (r0 < r1) keep(mine);
    for (int r = r0 + 1; r < r1; r++) keep(again(r));
    __syncthreads();
    // 4: the lowest free pages, ascending
    int found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < pages_wanted; p0 += 4 * RES_THREADS) {
        unsigned mask = free4;
        if (p0 > 0) {
            mask = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int pg = p0 + tid * 4 + i;
                if (pg < c.n_pages && __ldcg(c.refs + pg) == 0) mask |= 1u << i;
            }
        }
        unsigned long long here;
        int at = found + (int)block_scan((unsigned long long)__popc(mask), sums, here);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (mask >> i & 1u) {
                if (at < pages_wanted) wk.freed[at] = p0 + tid * 4 + i;
                at++;
            }
        found += (int)here;
    }
    if (found < pages_wanted) {                   // refused: the counts are as they were, nothing else has changed
        if (r0 < r1 && (mine.flag & COPY)) atomicAdd(c.refs + mine.last, 1);
        for (int r = r0 + 1; r < r1; r++) {
            const Row x = again(r);
            if (x.flag & COPY) atomicAdd(c.refs + x.last, 1);
        }
        if (tid == 0) {
            *result = TL_ERR_OUT_OF_MEMORY;
            *wk.n_copies = 0;
        }
        return;
    }
    __syncthreads();
    // 5: hand them out, rows in order: a row's copy first, then its new pages
    int at = (int)(before & PAGES), copy_at = (int)(before >> COPIES);         // there are that many pages: it fits
    auto hand_out = [&](int r, const Row& x) {
        if (x.add <= 0) return;
        int* row = c.table + (long long)r * c.max_pages;
        if (x.flag & COPY) {
            const int dst = __ldcg(wk.freed + at++);
            wk.copies[copy_at++] = CowItem{x.last, dst, x.slot, 0};
            row[x.pages - 1] = dst;
            c.refs[dst] = 1;
        }
        const int end = (int)c.by_page.div((unsigned)(x.len + x.add - 1)) + 1;
        for (int pg = x.pages; pg < end; pg++) {
            const int dst = __ldcg(wk.freed + at++);
            row[pg] = dst;
            c.refs[dst] = 1;
        }
        c.lengths[r] = x.len + x.add;
    };
    if (r0 < r1) hand_out(r0, mine);
    for (int r = r0 + 1; r < r1; r++) hand_out(r, again(r));
    if (tid == 0) {
        *result = TL_OK;
        *wk.n_copies = (int)(total >> COPIES);
    }
}

// the filled tokens of the shared pages that k_reserve gave a copy
template <typename V, int TEAM>
__global__ void __launch_bounds__(COPY_THREADS, 4) k_copy_shared(CopyArgs a, ReserveWork wk) {
    pdl_launch_dependents();
    pdl_wait();
    each_item<TEAM>(a, *wk.n_copies, [&](int m, unsigned what) {
        const CowItem c = wk.copies[m];
        copy_item<V, TEAM>(a, what, c.src, c.dst, c.tokens);
    });
}

// ---- moving the live pages together --------------------------------------------------------------------------------
// L live pages end up in pages 0 .. L-1: the highest live page moves to the lowest free one, and so on while the one lies
// above the other. Sources lie at or above L and destinations below, so the moves do not touch one another.
constexpr int CMP_THREADS = 256;
constexpr int CMP_PAGES = 1024;                   // pages a CTA counts

struct CompactWork {
    int* moves; int* counts; int* rank; int* src; int* dst;
};

__device__ __forceinline__ int block_sum(int v, int* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    int s = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) s += sh[w];
    return s;
}

__global__ void __launch_bounds__(CMP_THREADS) k_compact_count(const int* refs, int n_pages, CompactWork wk) {
    __shared__ int sh[CMP_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int p0 = blockIdx.x * CMP_PAGES;
    int n = 0;
    for (int p = p0 + threadIdx.x; p < min(n_pages, p0 + CMP_PAGES); p += CMP_THREADS) n += refs[p] > 0;
    n = block_sum(n, sh);
    if (threadIdx.x == 0) wk.counts[blockIdx.x] = n;
}

__global__ void __launch_bounds__(CMP_THREADS) k_compact_plan(const int* refs, int n_pages, int* moved_to, int* live_out, CompactWork wk) {
    __shared__ int sh[CMP_THREADS / 32];
    __shared__ unsigned long long sums[CMP_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    int before = 0, total = 0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += CMP_THREADS) {
        const int n = wk.counts[b];
        total += n;
        if (b < (int)blockIdx.x) before += n;
    }
    before = block_sum(before, sh);
    const int L = block_sum(total, sh);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *live_out = L;
        if (L == n_pages) *wk.moves = 0;          // no page L: nothing lies above
    }
    constexpr int EACH = CMP_PAGES / CMP_THREADS;
    const int q0 = blockIdx.x * CMP_PAGES + threadIdx.x * EACH;
    int live[EACH], n = 0;
#pragma unroll
    for (int j = 0; j < EACH; j++) {
        live[j] = q0 + j < n_pages && refs[q0 + j] > 0;
        n += live[j];
    }
    unsigned long long all;
    int seen = before + (int)block_scan((unsigned long long)n, sums, all);   // live pages below q0
#pragma unroll
    for (int j = 0; j < EACH; j++) {
        const int p = q0 + j;
        if (p >= n_pages) break;
        if (p == L) *wk.moves = L - seen;         // free pages below L = live pages from L on
        if (p < L) {
            moved_to[p] = live[j] ? p : -1;
            if (!live[j]) wk.dst[p - seen] = p;   // k-th free page
        } else if (live[j]) {
            wk.rank[p] = L - 1 - seen;            // counted from the highest live page down
            wk.src[L - 1 - seen] = p;
        } else {
            moved_to[p] = -1;
        }
        seen += live[j];
    }
}

template <typename V, int TEAM>
__global__ void __launch_bounds__(COPY_THREADS, 4) k_compact_move(CopyArgs a, PagedView c, int* moved_to, const int* live_out, CompactWork wk) {
    pdl_launch_dependents();
    pdl_wait();
    const int M = *wk.moves, L = *live_out;
    if (M == 0) return;
    const long long gtid = (long long)blockIdx.x * COPY_THREADS + threadIdx.x, gsize = (long long)gridDim.x * COPY_THREADS;
    for (long long i = gtid; i < (long long)c.n_rows * c.max_pages; i += gsize) {
        const int e = c.table[i];
        if (e >= L && e < c.n_pages) {
            const int k = wk.rank[e];
            if (k >= 0 && k < M && wk.src[k] == e) c.table[i] = wk.dst[k];
        }
    }
    for (long long i = gtid; i < M; i += gsize) moved_to[wk.src[i]] = wk.dst[i];
    each_item<TEAM>(a, M, [&](int m, unsigned what) { copy_item<V, TEAM>(a, what, wk.src[m], wk.dst[m], a.shape.page_size); });
}

// the counts follow their pages
__global__ void __launch_bounds__(CMP_THREADS) k_compact_refs(int* refs, CompactWork wk) {
    pdl_launch_dependents();
    pdl_wait();
    for (int i = blockIdx.x * CMP_THREADS + threadIdx.x; i < *wk.moves; i += gridDim.x * CMP_THREADS) {
        refs[wk.dst[i]] = refs[wk.src[i]];
        refs[wk.src[i]] = 0;
    }
}

// ---- rows of contiguous state --------------------------------------------------------------------------------------
constexpr int GATHER_VECS = 2048;                 // vectors an item

template <typename V>
__global__ void __launch_bounds__(COPY_THREADS, 4) k_gather_rows(const __half* src, __half* dst, const int* parents, int outer, int rows,
                                                              long long used, long long so, long long sr, long long dso, long long dsr,
                                                              int pieces, int* status) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int VEC = sizeof(V) / sizeof(__half);
    const long long vecs = used / VEC;
    for (long long it = blockIdx.x; it < (long long)outer * rows * pieces; it += gridDim.x) {
        const int piece = (int)(it % pieces);
        const long long orow = it / pieces;
        const int o = (int)(orow / rows), r = (int)(orow % rows);
        const int parent = parents[r];
        if (parent == -1) continue;
        if (parent < 0 || parent >= rows) {
            if (threadIdx.x == 0) atomicExch(status, TL_ERR_INVALID_ARGUMENT);
            continue;
        }
        const __half* s = src + o * so + parent * sr;
        __half* d = dst + o * dso + r * dsr;
        const long long v0 = (long long)piece * GATHER_VECS;
        copy_run<V, COPY_THREADS>(d + v0 * VEC, s + v0 * VEC, (int)min((long long)GATHER_VECS, vecs - v0), threadIdx.x);
        if (piece == pieces - 1)
            for (long long i = vecs * VEC + threadIdx.x; i < used; i += COPY_THREADS) d[i] = s[i];
    }
}

CopyArgs copy_args(const PagedView& c) {
    CopyArgs a{c.k, c.v, c.layer_stride, c.page_stride, c.n_layers, c.n_pages, COPY_THREADS, page_shape(c), FastDiv(2u * c.n_layers), device_id_status_word()};
    if ((long long)c.page_size * c.n_kv_heads * c.head_dim / a.shape.vec <= 2 * COPY_THREADS) a.team = 32;
    return a;
}
// the kernel of a copy for vectors of 16 or 2 bytes and a CTA or a warp an item
#define TL_LAUNCH_COPY(KERNEL, ...)                                                                                      \
    (a.shape.vec == 8 ? (a.team == 32 ? launch_pdl(KERNEL<uint4, 32>, __VA_ARGS__) : launch_pdl(KERNEL<uint4, COPY_THREADS>, __VA_ARGS__))   \
                      : (a.team == 32 ? launch_pdl(KERNEL<__half, 32>, __VA_ARGS__) : launch_pdl(KERNEL<__half, COPY_THREADS>, __VA_ARGS__)))
// CTAs of a copy: one an item where that is at all possible. Fewer that loop over items keep too little under way: rows of 1.4 MB
// took 224 us with eight CTAs an SM, 200 with 64, 191 with one an item; pages of 32 KB 360, 343 and 338.
unsigned copy_grid(long long items) {
    const long long most = (long long)sm_count() * 256;
    return (unsigned)(items < 1 ? 1 : (items < most ? items : most));
}
unsigned page_grid(const CopyArgs& a, long long pages) { return copy_grid((pages * 2 * a.n_layers * a.team + COPY_THREADS - 1) / COPY_THREADS); }
}  // namespace

template <int SLAB>
static int launch_fork(const PagedView& c, const int* parents, cudaStream_t st) {
    static PerDeviceOnce once;
    TL_CUDA(once.run([&] { return cudaFuncSetAttribute(k_fork<SLAB>, cudaFuncAttributeMaxDynamicSharedMemorySize, FORK_SMEM); }));
    return launch_pdl(k_fork<SLAB>, (unsigned)((c.max_pages + SLAB - 1) / SLAB + 1), FORK_THREADS, (size_t)c.n_rows * SLAB * 4, st, true, c.table,
                      c.lengths, c.refs, parents, c.n_rows, c.max_pages, c.n_pages, device_id_status_word());
}
int launch_paged_fork(const PagedView& c, const int* parents, cudaStream_t st) {
    // 32 bytes of a row at a time; less where many rows fill shared memory
    if ((long long)c.n_rows * 32 <= FORK_SMEM) return launch_fork<8>(c, parents, st);
    if ((long long)c.n_rows * 4 <= FORK_SMEM) return launch_fork<1>(c, parents, st);
    return set_error(TL_ERR_UNSUPPORTED, "paged_fork: more than 49152 rows");
}

// reserve: 64 bytes of counters, CowItem[n_rows], int need[n_rows], int freed[n_pages];
// compact: 64 bytes, counts[n_pages / 1024], rank, src, dst [n_pages]. Both fit the same formula.
size_t paged_workspace_bytes(int n_rows, int n_pages) { return 4096 + 20 * (size_t)n_rows + 13 * (size_t)n_pages; }

int launch_paged_reserve(const PagedView& c, const int* new_tokens, int* result, void* work, cudaStream_t st) {
    char* w = static_cast<char*>(work);
    ReserveWork wk;
    wk.n_copies = reinterpret_cast<int*>(w);
    wk.copies = reinterpret_cast<CowItem*>(w + 64);
    wk.need = reinterpret_cast<int*>(w + 64 + sizeof(CowItem) * (size_t)c.n_rows);
    wk.freed = wk.need + c.n_rows;
    TL_PROPAGATE(launch_pdl(k_reserve, 1, RES_THREADS, 0, st, true, c, new_tokens, result, wk, device_id_status_word()));
    const CopyArgs a = copy_args(c);
    return TL_LAUNCH_COPY(k_copy_shared, page_grid(a, c.n_rows), COPY_THREADS, 0, st, true, a, wk);
}

int launch_paged_copy(const PagedView& c, const int* src, const int* dst, int n, cudaStream_t st) {
    if (n == 0) return TL_OK;
    const CopyArgs a = copy_args(c);
    return TL_LAUNCH_COPY(k_copy_pages, page_grid(a, n), COPY_THREADS, 0, st, true, a, src, dst, n);
}

int launch_paged_compact(const PagedView& c, int* moved_to, int* live, void* work, cudaStream_t st) {
    CompactWork wk;
    const int blocks = (c.n_pages + CMP_PAGES - 1) / CMP_PAGES;
    wk.moves = static_cast<int*>(work);
    wk.counts = wk.moves + 16;
    wk.rank = wk.counts + blocks;
    wk.src = wk.rank + c.n_pages;
    wk.dst = wk.src + c.n_pages;
    TL_PROPAGATE(launch_pdl(k_compact_count, blocks, CMP_THREADS, 0, st, true, c.refs, c.n_pages, wk));
    TL_PROPAGATE(launch_pdl(k_compact_plan, blocks, CMP_THREADS, 0, st, true, c.refs, c.n_pages, moved_to, live, wk));
    const CopyArgs a = copy_args(c);              // (no more pages can move than half of them)
    TL_PROPAGATE(TL_LAUNCH_COPY(k_compact_move, page_grid(a, c.n_pages / 2 + 1), COPY_THREADS, 0, st, true, a, c, moved_to, live, wk));
    return launch_pdl(k_compact_refs, (unsigned)ceil_div((size_t)c.n_pages / 2 + 1, CMP_THREADS) < 64u ? (unsigned)ceil_div((size_t)c.n_pages / 2 + 1, CMP_THREADS) : 64u,
                      CMP_THREADS, 0, st, true, c.refs, wk);
}

int launch_gather_rows(const __half* src, __half* dst, const int* parents, int outer, int rows, long long used, long long so,
                       long long sr, long long dso, long long dsr, cudaStream_t st) {
    if (outer == 0 || rows == 0 || used == 0) return TL_OK;
    const bool vec = (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0) && so % 8 == 0 && sr % 8 == 0 &&
                     dso % 8 == 0 && dsr % 8 == 0;
    const long long vecs = vec ? used / 8 : used;
    const int pieces = (int)(vecs <= GATHER_VECS ? 1 : (vecs + GATHER_VECS - 1) / GATHER_VECS);
    const unsigned grid = copy_grid((long long)outer * rows * pieces);
    return vec ? launch_pdl(k_gather_rows<uint4>, grid, COPY_THREADS, 0, st, true, src, dst, parents, outer, rows, used, so, sr, dso, dsr,
                            pieces, device_id_status_word())
               : launch_pdl(k_gather_rows<__half>, grid, COPY_THREADS, 0, st, true, src, dst, parents, outer, rows, used, so, sr, dso, dsr,
                            pieces, device_id_status_word());
}

}  // namespace tlb
