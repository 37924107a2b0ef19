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

// Any alignment and stride: one CTA a (head, batch entry), a warp a token at a time, a lane every 32nd element.
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
        const float keep = mn == -INFINITY ? 1.f : expf(m - mn), e = mn == -INFINITY ? 0.f : expf(s - mn);
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
        p.out[b * p.o_row + (long long)h * hd + d] = __float2half_rn(L > 0.f ? a / L : 0.f);
    }
    if (threadIdx.x == 0 && p.lse) p.lse[(long long)b * p.n_heads + h] = L > 0.f ? M + logf(L) : -INFINITY;
}

}  // namespace

size_t paged_attn_workspace_bytes(int, int, int) { return 0; }

int launch_paged_attn(const PagedView& c, const PagedAttnArgs& a, cudaStream_t st) {
    if (a.batch == 0) return TL_OK;
    AttnLaunch p{};
    p.k = c.k; p.v = c.v; p.table = c.table; p.lengths = c.lengths; p.rows = a.rows;
    p.page_stride = c.page_stride; p.token_stride = c.token_stride; p.head_stride = c.head_stride;
    p.page_size = c.page_size; p.max_pages = c.max_pages; p.n_pages = c.n_pages; p.n_rows = c.n_rows; p.n_kv = c.n_kv_heads;
    p.head_dim = c.head_dim; p.by_page = c.by_page;
    p.q = a.q; p.out = a.out; p.lse = a.lse; p.q_row = a.q_row; p.o_row = a.o_row;
    p.batch = a.batch; p.n_heads = a.n_heads; p.group = a.n_heads / c.n_kv_heads; p.scale = a.scale;
    p.status = device_status_word();
    return launch_pdl(k_paged_attn_any, dim3(a.n_heads, a.batch), ANY_WARPS * 32, 0, st, true, p);
}

}  // namespace tlb
