// Attention of one new token over a paged cache: out_h = sum_t softmax_t(scale q_h . k_t) v_t over the tokens of the row,
// lse_h = log sum_t exp(scale q_h . k_t). An empty row gives zeros and -inf.
#include "serving.cuh"

namespace tlb {

namespace {

struct AttnLaunch {
    const __half* k; const __half* v;
    const int* table; const int* lengths; const int* rows;
    long long page_stride, token_stride, head_stride;
    int page_size, max_pages, n_pages, n_rows, n_kv, head_dim;
    FastDiv by_page;
    const __half* q; __half* out; float* lse;
    long long q_row, o_row;
    int batch, n_heads, group;
    float scale;
    int* status;
};

// tokens of batch entry b, checked against what the table can hold
__device__ __forceinline__ int row_tokens(const AttnLaunch& p, int b, int& row) {
    row = p.rows ? p.rows[b] : b;
    if (row == -1) return 0;
    if (row < 0 || row >= p.n_rows) {
        atomicExch(p.status, TL_ERR_INVALID_ARGUMENT);
        return 0;
    }
    const int n = p.lengths[row];
    if (n < 0 || (long long)n > (long long)p.max_pages * p.page_size) {
        atomicExch(p.status, TL_ERR_INVALID_ARGUMENT);
        return n < 0 ? 0 : p.max_pages * p.page_size;
    }
    return n;
}

constexpr int ANY_WARPS = 8;
constexpr int ANY_HD = 256;

// Any alignment and stride (48 ragged sequences that the kernel below takes 81 us for: 1340 us): one CTA a (head, batch entry), a warp a token at a time, a lane every 32nd element.
__global__ void __launch_bounds__(ANY_WARPS * 32) k_paged_attn_any(AttnLaunch p) {
    __shared__ float sm_m[ANY_WARPS], sm_l[ANY_WARPS], sm_acc[ANY_WARPS][ANY_HD];
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = h / p.group, hd = p.head_dim;
    int row;
    const int n = row_tokens(p, b, row);
    constexpr int I = ANY_HD / 32;
    float q[I], acc[I], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < I; i++) {
        const int d = lane + 32 * i;
        q[i] = d < hd ? __half2float(p.q[b * p.q_row + (long long)h * hd + d]) * p.scale : 0.f;
        acc[i] = 0.f;
    }
    for (int t = warp; t < n; t += ANY_WARPS) {
        unsigned pg, slot;
        p.by_page.divmod((unsigned)t, pg, slot);
        const int page = p.table[(long long)row * p.max_pages + pg];
        if (page < 0 || page >= p.n_pages) {
            if (lane == 0) atomicExch(p.status, TL_ERR_INVALID_ARGUMENT);
            continue;
        }
        const long long at = page * p.page_stride + slot * p.token_stride + kvh * p.head_stride;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < I; i++) {
            const int d = lane + 32 * i;
            if (d < hd) s = fmaf(q[i], __half2float(p.k[at + d]), s);
        }
        s = warp_sum(s);
        const float mn = fmaxf(m, s);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float keep = expf(m - ref), e = expf(s - ref);
        l = l * keep + e;
        m = mn;
#pragma unroll
        for (int i = 0; i < I; i++) {
            const int d = lane + 32 * i;
            if (d < hd) acc[i] = fmaf(e, __half2float(p.v[at + d]), acc[i] * keep);
        }
    }
    if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < I; i++)
        if (lane + 32 * i < hd) sm_acc[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < ANY_WARPS; w++) M = fmaxf(M, sm_m[w]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < ANY_WARPS; w++) L += sm_l[w] * expf(sm_m[w] - ref);
    for (int d = threadIdx.x; d < hd; d += ANY_WARPS * 32) {
        float a = 0.f;
        for (int w = 0; w < ANY_WARPS; w++) a += sm_acc[w][d] * expf(sm_m[w] - ref);
        p.out[b * p.o_row + (long long)h * hd + d] = __float2half_rn(L == 0.f ? 0.f : a / L);
    }
    if (threadIdx.x == 0 && p.lse) p.lse[(long long)b * p.n_heads + h] = L == 0.f ? -INFINITY : M + logf(L);
}


// ---- the tensor-core kernel ----------------------------------------------------------------------------------------
// For rows of head_dim values that start on 16 bytes. Per KV head the `group` query heads are the columns of the products
//   S^T [16 tokens x 8 heads] = K_tile Q^T,   O^T [dims x 8 heads] += V_tile^T P^T        (mma.m16n8k16, fp32 sums)
// so that eight heads cost what one does. P^T leaves the accumulators of the first product through a transposing register
// move and enters the second as its B operand, split into two fp16 parts. A weight is exp(s - running maximum) times 2^FL_LIFT, the
// largest power of two that fp16 holds, in the sums of weights and of values alike: the factor cancels, and the log-sum takes it
// off. The parts then keep a weight to 2^-22 of itself or 2^-40 of the largest, whichever is more. (Without the factor that is 2^-25 of
// the largest, and what thousands of tokens some 17 nats below one other add to the values was lost or off by a quarter.)
//
// HBM bound: K and V are read once, and a tile of 16 tokens costs some 250 warp instructions against the 360 cycles that an
// SM's share of the memory needs for its 8 KB. Each warp streams its own tiles through a private ring of shared memory
// (cp.async, zero-filled behind the last token and for ids outside the pool, so nothing unwritten is ever multiplied);
// page ids are looked up one tile further ahead. Warps meet only at the end of a (sequence, head group).
//
// The work of all sequences, counted in units of 64 tokens and FL_START more for every (sequence, head group), which is about
// what starting and finishing one costs, is cut into equal contiguous ranges, one a CTA: ragged batches fill the machine
// whatever their lengths, one long sequence as well as many. A (sequence, head group) that falls into one
// range is finished there; one that is cut leaves partial results (max, sum, sums of values) in the workspace, and the CTA
// that comes last joins them, in order of the ranges.
//
// Measured on a B200 (32 query, 8 KV heads of 128): 48 sequences of 200..6000 tokens 81 us = 6.2 TB/s, four of about 115000
// 277 us = 6.9 TB/s; the tensor pipe is 14% busy and DRAM reads are the algorithmic bytes. One sequence of 333 tokens and 32 KV
// heads 6.8 us, of which about 3 pass before the first product (length -> page id -> K and V) and 1.5 in the join.
constexpr int FL_WARPS = 4;
constexpr int FL_THREADS = FL_WARPS * 32;
constexpr int FL_TILE = 16;                       // tokens of a warp's tile
constexpr int FL_UNIT = FL_TILE * FL_WARPS;
constexpr int FL_START = 2;
constexpr float FL_LIFT = 15.f;
constexpr int FL_JOIN = 16;                       // pieces joined at a time
constexpr int FL_MAX_SMS = 160;
constexpr int FL_COUNTER_BYTES = 8192;

struct TiledLaunch {
    AttnLaunch a;
    int chunk, chunks, groups;                    // query heads of a head group, head groups a KV head, head groups in all
    FastDiv by_grid;
    float scale_log2;
    bool out8;                                    // out can be stored 8 bytes at a time
    unsigned int* counters; float* partial;       // workspace: [3 CTAs]; [4 CTAs] partial results
};

template <int HDP, int NT>
struct TiledShape {
    // Stages of a warp's ring and CTAs an SM. More warps beat deeper rings where both keep some 100 KB under way: at 128
    // elements, 3 x 2 against 2 x 3, 32 sequences of 500..2000 tokens took 31.0 against 32.9 us, 256 of 1..100 21.0 against 25.6.
    static constexpr int STAGES = HDP <= 96 ? 3 : (HDP == 256 ? 3 : 2);
    static constexpr int CTAS = HDP == 64 ? 4 : (HDP <= 128 ? 3 : (HDP == 192 ? 2 : 1));
    // The same 16-byte chunk of eight rows lies in different banks: the chunks are turned by the row, where rows are 192 bytes,
    // which alternate between halves of the banks, by every second one. (A pitch 16 bytes longer did the same for the reads,
    // but took 320 us for 283 at four long contexts.)
    static constexpr int PITCH = HDP * 2;
    __device__ static __forceinline__ uint32_t at(int row, int chunk) {
        return row * PITCH + ((chunk ^ (HDP == 96 ? (row >> 1) & 3 : row & 7)) << 4);
    }
    static constexpr int TILE_BYTES = FL_TILE * PITCH;
    static constexpr int RING = FL_WARPS * STAGES * 2 * TILE_BYTES;
    static constexpr int HEADS = 8 * NT;
    static constexpr int SMEM = RING + FL_WARPS * HEADS * 8 + FL_WARPS * STAGES * 4;
    static_assert(HEADS * HDP * 4 <= 2 * TILE_BYTES, "a warp's sums go into one free stage of its ring");
};

// a partial result: [chunk][head_dim] sums, [chunk] (max, sum of weights), 16-byte aligned
__host__ __device__ __forceinline__ long long tiled_slot_floats(int chunk, int head_dim) { return ((long long)chunk * (head_dim + 2) + 3) / 4 * 4; }

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// a place in the flattened (sequence, head group, FL_START + unit) space; a head group is a part of a KV head's query heads
struct Cursor {
    int b, row, len, units, kvh, part, i;
    int left;                                     // of this CTA's range from here on
};

__device__ __forceinline__ int units_of(int len) { return (len + FL_UNIT - 1) / FL_UNIT; }
__device__ __forceinline__ int cost_of(int len) { return len > 0 ? units_of(len) + FL_START : 0; }

__device__ __forceinline__ void advance(const TiledLaunch& p, Cursor& c) {
    if (--c.left <= 0) return;
    if (++c.i < c.units) return;
    c.left -= FL_START;
    if (c.left <= 0) return;
    c.i = 0;
    if (++c.part < p.chunks) return;
    c.part = 0;
    if (++c.kvh < p.a.n_kv) return;
    c.kvh = 0;
    do {
        c.b++;
        c.len = row_tokens(p.a, c.b, c.row);
        c.units = units_of(c.len);
    } while (c.units == 0);
}

// one more arrival of `expected`; true for the last one, which then sees what the others wrote (the caller's CTA has met at a
// barrier before, so its writes are covered) and leaves the counter at 0
__device__ __forceinline__ bool last_to_arrive(unsigned int* counter, int expected) {
    unsigned int before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    if (before != (unsigned)(expected - 1)) return false;
    *counter = 0;
    return true;
}

template <int HDP, int NT>
__global__ void __launch_bounds__(FL_THREADS, TiledShape<HDP, NT>::CTAS) k_paged_attn(TiledLaunch p) {
    using F = TiledShape<HDP, NT>;
    extern __shared__ __align__(128) unsigned char sm[];
    float2* stats = reinterpret_cast<float2*>(sm + F::RING);                                 // [warp][head]: max, sum
    uint32_t* masks = reinterpret_cast<uint32_t*>(sm + F::RING + FL_WARPS * F::HEADS * 8);   // [warp][stage]
    __shared__ int scan_sh[FL_WARPS];
    __shared__ int start_sh, start_b, start_row, start_len;
    __shared__ int last_sh;
    const AttnLaunch& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = a.head_dim;
    pdl_launch_dependents();
    pdl_wait();

    // 1: this CTA's range. Every CTA adds up the costs of all sequences; a thread takes a run of them. (The host has made sure
    // that the sum fits 31 bits.)
    const int per_thread = (a.batch + FL_THREADS - 1) / FL_THREADS;
    const int b0 = min(a.batch, tid * per_thread), b1 = min(a.batch, b0 + per_thread);
    int row0 = 0, len0 = 0, mine = 0;             // the run's first sequence, the run's cost
    if (b0 < b1) {
        len0 = row_tokens(a, b0, row0);
        mine = cost_of(len0);
    }
    for (int b = b0 + 1; b < b1; b++) {
        int row;
        mine += cost_of(row_tokens(a, b, row));
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) scan_sh[warp] = upto;
    __syncthreads();
    int before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < FL_WARPS; w++) {
        if (w < warp) before += scan_sh[w];
        total += scan_sh[w];
    }
    const int U = total * p.groups;
    const int per = (int)p.by_grid.div((unsigned)U + gridDim.x - 1);
    const int u0 = per * (int)blockIdx.x, u1 = min(u0 + per, U);
    // sequences with nothing to attend to
    auto empty_rows = [&] {
        for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
            int row;
            if (row_tokens(a, b, row) == 0) {
                for (int i = tid; i < a.n_heads * hd; i += FL_THREADS) a.out[b * a.o_row + i] = __float2half_rn(0.f);
                if (a.lse)
                    for (int h = tid; h < a.n_heads; h += FL_THREADS) a.lse[(long long)b * a.n_heads + h] = -INFINITY;
            }
        }
    };
    if (u0 >= u1) {
        empty_rows();
        return;
    }
    if (u0 >= before * p.groups && u0 < (before + mine) * p.groups) {      // one thread's run holds the start
        int b = b0, at = before;
        while (u0 >= (at + cost_of(len0)) * p.groups) {
            at += cost_of(len0);
            len0 = row_tokens(a, ++b, row0);
        }
        start_sh = at * p.groups;
        start_b = b;
        start_row = row0;
        start_len = len0;
    }
    __syncthreads();
    Cursor cur;                                   // what is computed next
    cur.b = start_b;
    cur.row = start_row;
    cur.len = start_len;
    cur.units = units_of(cur.len);
    {
        const unsigned in = (unsigned)(u0 - start_sh), cost = (unsigned)cur.units + FL_START;
        const int hg = (int)(in / cost);
        cur.i = (int)(in - (unsigned)hg * cost) - FL_START;
        cur.kvh = p.chunks == 1 ? hg : hg / p.chunks;
        cur.part = hg - cur.kvh * p.chunks;
    }
    cur.left = u1 - u0;
    if (cur.i < 0) {
        cur.left += cur.i;
        cur.i = 0;
    }
    Cursor ahead = cur;                           // what is looked up next

    // 2: loads. lookup(): the page id of this lane's token (lanes 16.. repeat 0..15); issue(): the tile's rows.
    struct Look { int page, slot, kvh; };
    auto lookup = [&]() {
        Look k{0, -1, 0};
        if (ahead.left > 0) {
            const int tok = ahead.i * FL_UNIT + warp * FL_TILE + (lane & 15);
            k.kvh = ahead.kvh;
            if (tok < ahead.len) {
                unsigned pg, s;
                a.by_page.divmod((unsigned)tok, pg, s);
                k.slot = (int)s;
                k.page = a.table[(long long)ahead.row * a.max_pages + pg];
            }
            advance(p, ahead);
        }
        return k;
    };
    constexpr int CPR = HDP / 8;                  // 16-byte chunks a row
    unsigned char* ring = sm + warp * F::STAGES * 2 * F::TILE_BYTES;
    auto issue = [&](int stage, const Look& k) {
        long long off = -1;
        if (k.slot >= 0) {
            if ((unsigned)k.page < (unsigned)a.n_pages) off = k.page * a.page_stride + k.slot * a.token_stride + k.kvh * a.head_stride;
            else atomicExch(a.status, TL_ERR_INVALID_ARGUMENT);
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, off >= 0) & 0xffffu;
        if (lane == 0) masks[warp * F::STAGES + stage] = mask;
        if (mask) {
            const uint32_t kd = smem_addr(ring + stage * 2 * F::TILE_BYTES), vd = kd + F::TILE_BYTES;
#pragma unroll
            for (int i0 = 0; i0 < FL_TILE * CPR; i0 += 32) {
                const int r = (i0 + lane) / CPR, chunk = (i0 + lane) % CPR;
                const long long o = __shfl_sync(0xffffffffu, off, r);
                const bool ok = o >= 0 && chunk * 8 < hd;
                const long long at = ok ? o + chunk * 8 : 0;
                const uint32_t d = F::at(r, chunk);
                cp_async16(kd + d, a.k + at, ok ? 16 : 0);
                cp_async16(vd + d, a.v + at, ok ? 16 : 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    Look look;                                    // of the next tile to load
    {
        Look first[F::STAGES - 1];                // their lookups are under way together
#pragma unroll
        for (int s = 0; s < F::STAGES - 1; s++) first[s] = lookup();
        look = lookup();
#pragma unroll
        for (int s = 0; s < F::STAGES - 1; s++) issue(s, first[s]);
    }
    empty_rows();

    // 3: the range, segment by segment (one (sequence, head group) each)
    const int g = lane >> 2, t = lane & 3;        // fragment row and column pair
    int stage = 0;
    while (cur.left > 0) {
        const int h0 = cur.kvh * a.group + cur.part * p.chunk, heads = min(p.chunk, (cur.kvh + 1) * a.group - h0);
        const int seg_units = min(cur.units - cur.i, cur.left);
        const int seg_b = cur.b, seg_i = cur.i, seg_n = cur.units;
        const int base = u1 - cur.left - seg_i;                              // where its first unit lies
        uint32_t q[NT][HDP / 16][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int ks = 0; ks < HDP / 16; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int h = n * 8 + g, d = ks * 16 + j * 8 + t * 2;
                    q[n][ks][j] = h < heads && d < hd ? *reinterpret_cast<const uint32_t*>(a.q + seg_b * a.q_row + (long long)(h0 + h) * hd + d) : 0u;
                }
        float o[NT][HDP / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int j = 0; j < HDP / 16; j++) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
        }
        for (int u = 0; u < seg_units; u++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(F::STAGES - 2) : "memory");
            __syncwarp();
            const uint32_t mask = masks[warp * F::STAGES + stage];
            {
                const int next = stage == 0 ? F::STAGES - 1 : stage - 1;       // the stage computed last
                issue(next, look);
                look = lookup();
            }
            if (mask) {
                const uint32_t ks_base = smem_addr(ring + stage * 2 * F::TILE_BYTES), vs_base = ks_base + F::TILE_BYTES;
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                const int kr = lane & 15;
#pragma unroll
                for (int ks = 0; ks < HDP / 16; ks++) {
                    uint32_t f[4];
                    ldsm4(f, ks_base + F::at(kr, 2 * ks + (lane >> 4)));
#pragma unroll
                    for (int n = 0; n < NT; n++) mma16816(s[n], f, q[n][ks][0], q[n][ks][1]);
                }
                const bool in0 = mask >> g & 1, in1 = mask >> (g + 8) & 1;
                uint32_t ph[NT][2], pl[NT][2];
                float keep[NT][2];
                bool moved = false;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float x0 = in0 ? s[n][j] * p.scale_log2 : -INFINITY, x1 = in1 ? s[n][j + 2] * p.scale_log2 : -INFINITY;
                        float mx = fmaxf(x0, x1);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mn = fmaxf(m[n][j], mx);
                        const float ref = mn == -INFINITY ? 0.f : mn;
                        keep[n][j] = exp2f(m[n][j] - ref);
                        moved |= mn != m[n][j];
                        m[n][j] = mn;
                        s[n][j] = exp2f(x0 - ref + FL_LIFT);
                        s[n][j + 2] = exp2f(x1 - ref + FL_LIFT);
                        l[n][j] = l[n][j] * keep[n][j] + (s[n][j] + s[n][j + 2]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const __half2 hi = __floats2half2_rn(s[n][2 * j], s[n][2 * j + 1]);
                        const float2 hf = __half22float2(hi);
                        const __half2 lo = __floats2half2_rn(s[n][2 * j] - hf.x, s[n][2 * j + 1] - hf.y);
                        ph[n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
                        pl[n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&lo));
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < HDP / 16; j++) {
                            o[n][j][0] *= keep[n][0];
                            o[n][j][1] *= keep[n][1];
                            o[n][j][2] *= keep[n][0];
                            o[n][j][3] *= keep[n][1];
                        }
                }
                const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;
#pragma unroll
                for (int j = 0; j < HDP / 16; j++) {
                    uint32_t f[4];
                    ldsm4t(f, vs_base + F::at(vr, 2 * j + vc));
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma16816(o[n][j], f, ph[n][0], ph[n][1]);
                        mma16816(o[n][j], f, pl[n][0], pl[n][1]);
                    }
                }
            }
            __syncwarp();
            stage = stage + 1 == F::STAGES ? 0 : stage + 1;
            advance(p, cur);
        }
        // 4: the warps' results become one. Each leaves its sums in the stage of its ring that was computed last (the others are
        // being filled), the head's words turned by 8 for each pair of heads, which spreads an accumulator register's stores
        // over all banks.
        const int freed = stage == 0 ? F::STAGES - 1 : stage - 1;
        auto sums = [&](int w) { return reinterpret_cast<float*>(sm + (w * F::STAGES + freed) * 2 * F::TILE_BYTES); };
        {
            float* mine_at = sums(warp);
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
                    l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
                    if (g == 0) stats[warp * F::HEADS + n * 8 + 2 * t + j] = make_float2(m[n][j], l[n][j]);
                }
#pragma unroll
                for (int j = 0; j < HDP / 16; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mine_at[(n * 8 + 2 * t + (e & 1)) * HDP + ((j * 16 + g + (e >> 1) * 8) ^ (t * 8))] = o[n][j][e];
            }
        }
        __syncthreads();
        const bool whole = seg_i == 0 && seg_units == seg_n;
        const long long slot_floats = tiled_slot_floats(p.chunk, hd);
        float* part = p.partial + (2ll * blockIdx.x + (seg_i == 0)) * slot_floats;
        auto finish = [&](int h, int d, float4 x, float M, float L) {     // four elements of a head's result
            const float inv = L == 0.f ? 0.f : 1.f / L;                      // (a NaN stays one)
            const __half2 lo = __floats2half2_rn(x.x * inv, x.y * inv), hi = __floats2half2_rn(x.z * inv, x.w * inv);
            __half* at = a.out + seg_b * a.o_row + (long long)(h0 + h) * hd + d;
            if (p.out8) {
                *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
            } else {
                at[0] = __low2half(lo); at[1] = __high2half(lo); at[2] = __low2half(hi); at[3] = __high2half(hi);
            }
            if (d == 0 && a.lse) a.lse[(long long)seg_b * a.n_heads + h0 + h] = L == 0.f ? -INFINITY : (M + (log2f(L) - FL_LIFT)) * 0.69314718055994531f;
        };
        for (int i = tid; i < heads * (HDP / 4); i += FL_THREADS) {
            const int h = i / (HDP / 4), d = i % (HDP / 4) * 4;
            if (d >= hd) continue;
            float2 st[FL_WARPS];
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < FL_WARPS; w++) {
                st[w] = stats[w * F::HEADS + h];
                M = fmaxf(M, st[w].x);
            }
            const float ref = M == -INFINITY ? 0.f : M;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < FL_WARPS; w++) {
                const float f = exp2f(st[w].x - ref);
                const float4 y = *reinterpret_cast<const float4*>(sums(w) + h * HDP + (d ^ ((h >> 1 & 3) * 8)));
                L += st[w].y * f;
                x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
            }
            if (whole) {
                finish(h, d, x, M, L);
            } else {
                *reinterpret_cast<float4*>(part + h * hd + d) = x;
                if (d == 0) *reinterpret_cast<float2*>(part + p.chunk * hd + 2 * h) = make_float2(M, L);
            }
        }
        if (!whole) {
            // The ranges that hold a piece of it: CTAs first .. first + pieces - 1. Up to FL_JOIN consecutive pieces are joined by
            // the last of them to arrive; where there are more groups than one, the last group to arrive joins the groups'
            // results the same way, in order.
            const int first = (int)((unsigned)base / (unsigned)per), pieces = (int)((unsigned)(base + seg_n - 1) / (unsigned)per) - first + 1;
            auto join = [&](int n, auto&& piece, bool final, float* to) {       // piece(c): partial result c < n
                for (int i = tid; i < heads * (HDP / 4); i += FL_THREADS) {
                    const int h = i / (HDP / 4), d = i % (HDP / 4) * 4;
                    if (d >= hd) continue;
                    float M = -INFINITY, L = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int AT_ONCE = 4;
                    for (int c0 = 0; c0 < n; c0 += AT_ONCE) {
                        float2 st[AT_ONCE];
                        float4 y[AT_ONCE];
#pragma unroll
                        for (int c = 0; c < AT_ONCE; c++) {
                            const bool in = c0 + c < n;
                            const float* from = piece(in ? c0 + c : 0);
                            st[c] = in ? __ldcg(reinterpret_cast<const float2*>(from + p.chunk * hd + 2 * h)) : make_float2(-INFINITY, 0.f);
                            y[c] = in ? __ldcg(reinterpret_cast<const float4*>(from + h * hd + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                        float top = M;
#pragma unroll
                        for (int c = 0; c < AT_ONCE; c++) top = fmaxf(top, st[c].x);
                        const float ref = top == -INFINITY ? 0.f : top;
                        const float old = exp2f(M - ref);
                        L *= old; x.x *= old; x.y *= old; x.z *= old; x.w *= old;
                        M = top;
#pragma unroll
                        for (int c = 0; c < AT_ONCE; c++) {
                            const float f = exp2f(st[c].x - ref);
                            L += st[c].y * f;
                            x.x += y[c].x * f; x.y += y[c].y * f; x.z += y[c].z * f; x.w += y[c].w * f;
                        }
                    }
                    if (final) {
                        finish(h, d, x, M, L);
                    } else {
                        *reinterpret_cast<float4*>(to + h * hd + d) = x;
                        if (d == 0) *reinterpret_cast<float2*>(to + p.chunk * hd + 2 * h) = make_float2(M, L);
                    }
                }
            };
            // the first piece is its range's last segment (odd slot), the others are their ranges' first ones (even slots)
            auto slot_of = [&](int c) { return 2ll * (first + c) + (c == 0); };
            const int c = (int)blockIdx.x - first, group = c / FL_JOIN, groups = (pieces + FL_JOIN - 1) / FL_JOIN;
            const int members = min(FL_JOIN, pieces - group * FL_JOIN);
            const long long joined0 = 2ll * gridDim.x;                          // groups' results lie behind the pieces
            __syncthreads();
            if (tid == 0) last_sh = last_to_arrive(p.counters + slot_of(group * FL_JOIN), members);
            __syncthreads();
            if (last_sh) {
                join(members, [&](int k) { return p.partial + slot_of(group * FL_JOIN + k) * slot_floats; }, groups == 1,
                     p.partial + (joined0 + slot_of(group * FL_JOIN)) * slot_floats);
                if (groups > 1) {
                    __syncthreads();
                    if (tid == 0) last_sh = last_to_arrive(p.counters + 2 * gridDim.x + first, groups);
                    __syncthreads();
                    if (last_sh) join(groups, [&](int k) { return p.partial + (joined0 + slot_of(k * FL_JOIN)) * slot_floats; }, true, nullptr);
                }
            }
        }
        __syncthreads();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int HDP, int NT>
int launch_tiled(const TiledLaunch& p, cudaStream_t st) {
    using F = TiledShape<HDP, NT>;
    static PerDeviceOnce once;
    TL_CUDA(once.run([&] { return cudaFuncSetAttribute(k_paged_attn<HDP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM); }));
    TiledLaunch q = p;
    const int grid = (sm_count() < FL_MAX_SMS ? sm_count() : FL_MAX_SMS) * F::CTAS;
    q.by_grid = FastDiv((unsigned)grid);
    return launch_pdl(k_paged_attn<HDP, NT>, grid, FL_THREADS, F::SMEM, st, true, q);
}

// query heads of a head group: as few groups as 16 columns allow (8 at 256 elements a head, where 16 would not fit the
// registers), of even size
int tiled_chunk(int group, int head_dim) {
    const int most = head_dim > 128 ? 8 : 16;
    const int chunks = (group + most - 1) / most;
    return (group + chunks - 1) / chunks;
}

}  // namespace

size_t paged_attn_workspace_bytes(int n_heads, int n_kv_heads, int head_dim) {
    const int ctas = FL_MAX_SMS * (head_dim <= 64 ? TiledShape<64, 1>::CTAS : (head_dim <= 128 ? TiledShape<128, 1>::CTAS :
                                   (head_dim <= 192 ? TiledShape<192, 1>::CTAS : TiledShape<256, 1>::CTAS)));
    static_assert(TiledShape<96, 1>::CTAS == TiledShape<128, 1>::CTAS, "one formula for both");
    static_assert(3 * FL_MAX_SMS * TiledShape<64, 1>::CTAS * 4 <= FL_COUNTER_BYTES, "counters");
    return FL_COUNTER_BYTES + 4 * (size_t)ctas * tiled_slot_floats(tiled_chunk(n_heads / n_kv_heads, head_dim), head_dim) * 4;
}

int launch_paged_attn(const PagedView& c, const PagedAttnArgs& a, cudaStream_t st) {
    if (a.batch == 0) return TL_OK;
    AttnLaunch p{};
    p.k = c.k; p.v = c.v; p.table = c.table; p.lengths = c.lengths; p.rows = a.rows;
    p.page_stride = c.page_stride; p.token_stride = c.token_stride; p.head_stride = c.head_stride;
    p.page_size = c.page_size; p.max_pages = c.max_pages; p.n_pages = c.n_pages; p.n_rows = c.n_rows; p.n_kv = c.n_kv_heads;
    p.head_dim = c.head_dim; p.by_page = c.by_page;
    p.q = a.q; p.out = a.out; p.lse = a.lse; p.q_row = a.q_row; p.o_row = a.o_row;
    p.batch = a.batch; p.n_heads = a.n_heads; p.group = a.n_heads / c.n_kv_heads; p.scale = a.scale;
    p.status = device_id_status_word();
    const bool fast = c.aligned16() && (reinterpret_cast<uintptr_t>(a.q) & 3) == 0 && a.q_row % 2 == 0;
    if (!fast) return launch_pdl(k_paged_attn_any, dim3(a.n_heads, a.batch), ANY_WARPS * 32, 0, st, true, p);
    // the cost of the whole batch has to fit 31 bits
    const long long cost = ((long long)c.max_pages * c.page_size + FL_UNIT - 1) / FL_UNIT + FL_START;
    if (cost * a.batch * a.n_heads >= (1ll << 31) - 1024)
        return set_error(TL_ERR_UNSUPPORTED, "paged_attn_decode: batch * n_heads * (max_pages * page_size / 64 + 3) has to stay below 2^31");
    TiledLaunch f{};
    f.a = p;
    f.chunk = tiled_chunk(p.group, p.head_dim);
    f.chunks = (p.group + f.chunk - 1) / f.chunk;
    f.groups = p.n_kv * f.chunks;
    f.scale_log2 = a.scale * 1.4426950408889634f;
    f.out8 = (reinterpret_cast<uintptr_t>(a.out) & 7) == 0 && a.o_row % 4 == 0;
    f.counters = static_cast<unsigned int*>(a.work);
    f.partial = reinterpret_cast<float*>(static_cast<char*>(a.work) + FL_COUNTER_BYTES);
    if (p.head_dim <= 64) return f.chunk <= 8 ? launch_tiled<64, 1>(f, st) : launch_tiled<64, 2>(f, st);
    if (p.head_dim <= 96) return f.chunk <= 8 ? launch_tiled<96, 1>(f, st) : launch_tiled<96, 2>(f, st);
    if (p.head_dim <= 128) return f.chunk <= 8 ? launch_tiled<128, 1>(f, st) : launch_tiled<128, 2>(f, st);
    return p.head_dim <= 192 ? launch_tiled<192, 1>(f, st) : launch_tiled<256, 1>(f, st);
}

}  // namespace tlb
