// The pages of a paged key-value cache: forking and freeing rows by reference, making room for new tokens (with a copy of a
// shared last page before it is written), copying pages over all layers, moving the live pages together, and gathering rows
// of contiguous state by parent. A page is free when its reference count is 0; there is no other free list, so every choice
// of a page (the lowest free ones, ascending) follows from the counts alone and repeats from run to run.
//
// Bookkeeping is integer work on small arrays, bound by latency; the copies are bound by HBM (each byte read and written
// once).
#include "serving.cuh"

namespace tlb {

namespace {

// ---- forking -------------------------------------------------------------------------------------------------------
// Row r becomes a copy of row parents[r]; the permutation acts within a column of the table, so a CTA that holds a slab of
// columns of ALL rows in shared memory needs no other CTA and no second launch. Entries that stay the same are skipped.
// The last CTA does the same with the lengths. Counts change by atomic additions of whole numbers: any order, same result.
constexpr int FORK_THREADS = 256;

__global__ void __launch_bounds__(FORK_THREADS) k_fork(int* table, int* lengths, int* refs, const int* parents, int n_rows,
                                                       int max_pages, int n_pages, int slab, int* status) {
    extern __shared__ int sm[];
    pdl_launch_dependents();
    pdl_wait();
    const bool is_len = blockIdx.x == gridDim.x - 1;
    const int c0 = is_len ? 0 : blockIdx.x * slab;
    const int w = is_len ? 1 : min(slab, max_pages - c0);
    int* base = is_len ? lengths : table + c0;
    const long long pitch = is_len ? 1 : max_pages;
    for (int i = threadIdx.x; i < n_rows * w; i += FORK_THREADS) sm[i] = base[(i / w) * pitch + i % w];
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * w; i += FORK_THREADS) {
        const int r = i / w, j = i % w;
        const int parent = parents[r];
        if (parent >= n_rows || parent < -1) {    // not a row: this one stays as it is
            atomicExch(status, TL_ERR_INVALID_ARGUMENT);
            continue;
        }
        const int o = sm[i], n = parent < 0 ? (is_len ? 0 : -1) : sm[parent * w + j];
        if (o == n) continue;
        base[r * pitch + j] = n;
        if (is_len) continue;
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

template <typename V>
__device__ __forceinline__ void copy_run(__half* dst, const __half* src, long long n, int tid, int threads) {
    const V* s = reinterpret_cast<const V*>(src);
    V* d = reinterpret_cast<V*>(dst);
    constexpr int U = 8;           // loads in flight a thread
    long long i = tid;
    for (; i + (U - 1) * threads < n; i += U * threads) {
        V x[U];
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = s[i + u * threads];
#pragma unroll
        for (int u = 0; u < U; u++) d[i + u * threads] = x[u];
    }
    for (; i < n; i += threads) d[i] = s[i];
}

template <typename V>
__device__ __forceinline__ void copy_page(const PageShape& s, __half* dst, const __half* src, int n, int tid, int threads) {
    constexpr int VEC = sizeof(V) / sizeof(__half);
    if (s.kind == 0) {
        copy_run<V>(dst, src, (long long)n * s.heads * s.dim / VEC, tid, threads);
        return;
    }
    if (s.kind == 1 && n == s.page_size && s.head_stride == (long long)n * s.dim) {
        copy_run<V>(dst, src, (long long)n * s.heads * s.dim / VEC, tid, threads);
        return;
    }
    if (s.kind == 1) {
        for (int h = 0; h < s.heads; h++)
            copy_run<V>(dst + h * s.head_stride, src + h * s.head_stride, (long long)n * s.dim / VEC, tid, threads);
        return;
    }
    const unsigned total = (unsigned)n * (s.kind == 2 ? 1 : s.heads) * s.by_row.d;
    for (unsigned i = tid; i < total; i += threads) {
        unsigned run, v, tok, h = 0;
        s.by_row.divmod(i, run, v);
        tok = run;
        if (s.kind == 3) s.by_heads.divmod(run, tok, h);
        const long long at = tok * s.token_stride + h * s.head_stride;
        reinterpret_cast<V*>(dst + at)[v] = reinterpret_cast<const V*>(src + at)[v];
    }
}

constexpr int COPY_THREADS = 256;

struct CopyArgs {
    __half* k; __half* v;
    long long layer_stride, page_stride;
    int n_layers, n_pages;
    PageShape shape;
    int* status;
};

__device__ __forceinline__ void copy_item(const CopyArgs& a, int what, int src, int dst, int tokens) {
    __half* pool = (what & 1) ? a.v : a.k;
    __half* layer = pool + (long long)(what >> 1) * a.layer_stride;
    if (a.shape.vec == 8) copy_page<uint4>(a.shape, layer + dst * a.page_stride, layer + src * a.page_stride, tokens, threadIdx.x, COPY_THREADS);
    else copy_page<__half>(a.shape, layer + dst * a.page_stride, layer + src * a.page_stride, tokens, threadIdx.x, COPY_THREADS);
}

// one item = one page of one layer of K or of V
__global__ void __launch_bounds__(COPY_THREADS) k_copy_pages(CopyArgs a, const int* src, const int* dst, int n) {
    pdl_launch_dependents();
    pdl_wait();
    const int each = 2 * a.n_layers;
    for (long long it = blockIdx.x; it < (long long)n * each; it += gridDim.x) {
        const int m = (int)(it / each), what = (int)(it - (long long)m * each);
        const int s = src[m], d = dst[m];
        if (s == d || s == -1) continue;
        if (s < 0 || d < 0 || s >= a.n_pages || d >= a.n_pages) {
            if (threadIdx.x == 0) atomicExch(a.status, TL_ERR_INVALID_ARGUMENT);
            continue;
        }
        copy_item(a, what, s, d, a.shape.page_size);
    }
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

__global__ void __launch_bounds__(RES_THREADS) k_reserve(PagedView c, const int* new_tokens, int* result, ReserveWork wk, int* status) {
    __shared__ unsigned long long sums[RES_THREADS / 32];
    __shared__ int bad_sh;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x;
    const int per = (c.n_rows + RES_THREADS - 1) / RES_THREADS;
    const int r0 = min(c.n_rows, tid * per), r1 = min(c.n_rows, r0 + per);
    if (tid == 0) bad_sh = 0;
    __syncthreads();
    auto last_page = [&](int r, int len) { return __ldcg(c.table + (long long)r * c.max_pages + len / c.page_size); };
    // 1: every row that writes into a page that is there lets go of it
    constexpr int NONE = 0, WRITES = 1 << 30, COPY = 1 << 29;
    for (int r = r0; r < r1; r++) {
        const int len = c.lengths[r], add = new_tokens[r];
        int flag = NONE;
        if (len < 0 || add < 0 || (long long)len + add > (long long)c.max_pages * c.page_size) {
            atomicMax(&bad_sh, add < 0 || len < 0 ? 2 : 1);
        } else if (add > 0 && len % c.page_size != 0) {
            const int page = last_page(r, len);
            if (page < 0 || page >= c.n_pages) atomicMax(&bad_sh, 2);
            else {
                if (atomicSub(c.refs + page, 1) <= 0) atomicMax(&bad_sh, 2);
                flag = WRITES;
            }
        }
        wk.need[r] = flag;
    }
    __syncthreads();
    // 2: a page that nobody holds any more goes to the highest of the rows that let go of it: its count becomes -(row + 1)
    for (int r = r0; r < r1; r++)
        if (wk.need[r] & WRITES) {
            int* ref = c.refs + last_page(r, c.lengths[r]);
            if (__ldcg(ref) <= 0) atomicMin(ref, -(r + 1));
        }
    __syncthreads();
    unsigned long long mine = 0;                  // copies in the upper half, pages in the lower
    for (int r = r0; r < r1; r++) {
        const int len = c.lengths[r], add = new_tokens[r];
        int flag = wk.need[r];
        if (flag & WRITES) {
            if (__ldcg(c.refs + last_page(r, len)) != -(r + 1)) {
                flag |= COPY;
                mine += (1ull << 32) + 1;
            }
            wk.need[r] = flag;
        }
        if (add > 0 && len >= 0)
            mine += (unsigned)(((long long)len + add + c.page_size - 1) / c.page_size - ((long long)len + c.page_size - 1) / c.page_size);
    }
    __syncthreads();
    // 3: the keepers' counts are 1 again
    for (int r = r0; r < r1; r++)
        if ((wk.need[r] & (WRITES | COPY)) == WRITES) atomicExch(c.refs + last_page(r, c.lengths[r]), 1);
    unsigned long long total;
    const unsigned long long before = block_scan(mine, sums, total);
    const int pages_wanted = (int)(total & 0xffffffffu);
    __syncthreads();
    // 4: the lowest free pages, ascending
    int found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < pages_wanted && bad_sh == 0; p0 += RES_THREADS) {
        const int p = p0 + tid;
        const bool is_free = p < c.n_pages && __ldcg(c.refs + p) == 0;
        unsigned long long here;
        const int at = found + (int)block_scan(is_free, sums, here);
        if (is_free && at < pages_wanted) wk.freed[at] = p;
        found += (int)here;
    }
    const int bad = bad_sh;
    if (bad || found < pages_wanted) {            // refused: the counts as they were, nothing else has changed
        for (int r = r0; r < r1; r++)
            if (wk.need[r] & COPY) atomicAdd(c.refs + last_page(r, c.lengths[r]), 1);
        if (tid == 0) {
            *result = bad == 2 ? TL_ERR_INVALID_ARGUMENT : TL_ERR_OUT_OF_MEMORY;
            *wk.n_copies = 0;
            if (bad == 2) atomicExch(status, TL_ERR_INVALID_ARGUMENT);
        }
        return;
    }
    __syncthreads();
    // 5: hand them out, rows in order: a row's copy first, then its new pages
    int at = (int)(before & 0xffffffffu), copy_at = (int)(before >> 32);
    for (int r = r0; r < r1; r++) {
        const int len = c.lengths[r], add = new_tokens[r];
        if (add <= 0) continue;
        int* row = c.table + (long long)r * c.max_pages;
        if (wk.need[r] & COPY) {
            const int dst = __ldcg(wk.freed + at++);
            wk.copies[copy_at++] = CowItem{row[len / c.page_size], dst, len % c.page_size, 0};
            row[len / c.page_size] = dst;
            c.refs[dst] = 1;
        }
        const int p1 = (int)(((long long)len + add + c.page_size - 1) / c.page_size);
        for (int p = (int)(((long long)len + c.page_size - 1) / c.page_size); p < p1; p++) {
            const int dst = __ldcg(wk.freed + at++);
            row[p] = dst;
            c.refs[dst] = 1;
        }
        c.lengths[r] = len + add;
    }
    if (tid == 0) {
        *result = TL_OK;
        *wk.n_copies = (int)(total >> 32);
    }
}

// the filled tokens of the shared pages that k_reserve gave a copy
__global__ void __launch_bounds__(COPY_THREADS) k_copy_shared(CopyArgs a, ReserveWork wk) {
    pdl_launch_dependents();
    pdl_wait();
    const int each = 2 * a.n_layers;
    const long long n = (long long)*wk.n_copies * each;
    for (long long it = blockIdx.x; it < n; it += gridDim.x) {
        const int m = (int)(it / each), what = (int)(it - (long long)m * each);
        const CowItem c = wk.copies[m];
        copy_item(a, what, c.src, c.dst, c.tokens);
    }
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

__global__ void __launch_bounds__(COPY_THREADS) k_compact_move(CopyArgs a, PagedView c, int* moved_to, const int* live_out, CompactWork wk) {
    pdl_launch_dependents();
    pdl_wait();
    const int M = *wk.moves, L = *live_out;
    if (M == 0) return;
    const long long gtid = (long long)blockIdx.x * COPY_THREADS + threadIdx.x, gsize = (long long)gridDim.x * COPY_THREADS;
    for (long long i = gtid; i < (long long)c.n_rows * c.max_pages; i += gsize) {
        const int e = c.table[i];
        if (e >= L && e < c.n_pages && c.refs[e] >= 0) {
            const int k = wk.rank[e];
            if (k >= 0 && k < M && wk.src[k] == e) c.table[i] = wk.dst[k];
        }
    }
    for (long long i = gtid; i < M; i += gsize) moved_to[wk.src[i]] = wk.dst[i];
    const int each = 2 * a.n_layers;
    for (long long it = blockIdx.x; it < (long long)M * each; it += gridDim.x) {
        const int m = (int)(it / each), what = (int)(it - (long long)m * each);
        copy_item(a, what, wk.src[m], wk.dst[m], a.shape.page_size);
    }
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
constexpr int GATHER_VECS = 4096;                 // vectors an item

template <typename V>
__global__ void __launch_bounds__(COPY_THREADS) k_gather_rows(const __half* src, __half* dst, const int* parents, int outer, int rows,
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
        copy_run<V>(d + v0 * VEC, s + v0 * VEC, min((long long)GATHER_VECS, vecs - v0), threadIdx.x, COPY_THREADS);
        if (piece == pieces - 1)
            for (long long i = vecs * VEC + threadIdx.x; i < used; i += COPY_THREADS) d[i] = s[i];
    }
}

CopyArgs copy_args(const PagedView& c) {
    return CopyArgs{c.k, c.v, c.layer_stride, c.page_stride, c.n_layers, c.n_pages, page_shape(c), device_status_word()};
}
unsigned copy_grid(long long items) {
    const long long most = (long long)sm_count() * 8;
    return (unsigned)(items < 1 ? 1 : (items < most ? items : most));
}
}  // namespace

int launch_paged_fork(const PagedView& c, const int* parents, cudaStream_t st) {
    int slab = 8;                                 // 32 bytes of a row; fewer columns where many rows fill shared memory
    while (slab > 1 && (long long)c.n_rows * slab * 4 > 196608) slab /= 2;
    const size_t smem = (size_t)c.n_rows * slab * 4;
    if (smem > 196608) return set_error(TL_ERR_UNSUPPORTED, "paged_fork: more than 49152 rows");
    static PerDeviceOnce once;
    if (once.needed()) TL_CUDA(cudaFuncSetAttribute(k_fork, cudaFuncAttributeMaxDynamicSharedMemorySize, 196608));
    const int grid = (c.max_pages + slab - 1) / slab + 1;
    return launch_pdl(k_fork, grid, FORK_THREADS, smem, st, true, c.table, c.lengths, c.refs, parents, c.n_rows, c.max_pages, c.n_pages,
                      slab, device_status_word());
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
    TL_PROPAGATE(launch_pdl(k_reserve, 1, RES_THREADS, 0, st, true, c, new_tokens, result, wk, device_status_word()));
    return launch_pdl(k_copy_shared, copy_grid((long long)c.n_rows * 2 * c.n_layers), COPY_THREADS, 0, st, true, copy_args(c), wk);
}

int launch_paged_copy(const PagedView& c, const int* src, const int* dst, int n, cudaStream_t st) {
    if (n == 0) return TL_OK;
    return launch_pdl(k_copy_pages, copy_grid((long long)n * 2 * c.n_layers), COPY_THREADS, 0, st, true, copy_args(c), src, dst, n);
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
    const long long most = (long long)(c.n_pages / 2) * 2 * c.n_layers;
    TL_PROPAGATE(launch_pdl(k_compact_move, copy_grid(most), COPY_THREADS, 0, st, true, copy_args(c), c, moved_to, live, wk));
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
                            pieces, device_status_word())
               : launch_pdl(k_gather_rows<__half>, grid, COPY_THREADS, 0, st, true, src, dst, parents, outer, rows, used, so, sr, dso, dsr,
                            pieces, device_status_word());
}

}  // namespace tlb
