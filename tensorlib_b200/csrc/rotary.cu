// Rotary positions: pair i of a head (elements 2i, 2i+1, or i, i + rot/2) is turned by the angle position * freqs[i] and
// scaled by `magnitude`; elements from rot on pass through. With a paged cache the keys go, rotated, and the values, as
// they are, straight into their pages: one pass over q, k and v.
//
// The angle: position * freqs[i] / (2 pi) in 64 bits, reduced to the nearest turn there, so that position 10^6 loses
// nothing; the fraction (at most half a turn) is exact to 2^-24 of a turn in 32 bits, and sincospif takes it from there.
// The rotation itself is in 32 bits with one rounding to fp16.
//
// Bound: HBM at many tokens (every element is read and written once), launch and one dependent load chain
// (position -> cos/sin -> store) at one token. One CTA a token: its cos/sin (rot/2 pairs) are computed once and shared by
// all heads through shared memory.
#include "serving.cuh"

namespace tlb {

namespace {

constexpr int ROT_THREADS = 256;
constexpr int MAX_ROT_PAIRS = 512;

struct RotLaunch {
    RotaryArgs a;
    __half* kc; __half* vc; int* table;           // cache (kc == nullptr: none)
    long long page_stride, token_stride, head_stride;
    int n_kv, n_rows, max_pages, n_pages;
    FastDiv by_page, by_items;
    int items;                                    // work items of a head
    int* status;
};

// VEC = 8: 16-byte items. Interleaved: one vector = four pairs. Half layout: one item = the vectors at i and i + rot/2.
// VEC = 1: any alignment, one pair or one passed-through element an item.
template <int VEC>
__global__ void __launch_bounds__(ROT_THREADS) k_rotary(RotLaunch p) {
    __shared__ float2 cs[MAX_ROT_PAIRS];
    __shared__ long long slot_sh;
    pdl_launch_dependents();
    pdl_wait();
    const RotaryArgs& a = p.a;
    const int pairs = a.rot / 2;
    for (int t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int pos = a.positions[t];
        __syncthreads();
        if (pos < 0) continue;                    // padding: nothing is written
        for (int i = threadIdx.x; i < pairs; i += ROT_THREADS) {
            const double turns = (double)pos * (a.freqs[i] * 0.15915494309189533577);
            const float frac = (float)(turns - rint(turns));
            float s, c;
            sincospif(2.f * frac, &s, &c);
            cs[i] = make_float2(c * a.magnitude, (a.inverse ? -s : s) * a.magnitude);
        }
        if (threadIdx.x == 0 && p.kc) {
            const int row = a.rows ? a.rows[t] : t;
            const unsigned pg = p.by_page.div((unsigned)pos);
            long long slot = -1;
            if (row >= 0 && row < p.n_rows && (int)pg < p.max_pages) {
                const int page = p.table[(long long)row * p.max_pages + pg];
                if (page >= 0 && page < p.n_pages)
                    slot = page * p.page_stride + (long long)((unsigned)pos - pg * p.by_page.d) * p.token_stride;
            }
            if (slot < 0) atomicExch(p.status, TL_ERR_INVALID_ARGUMENT);
            slot_sh = slot;
        }
        __syncthreads();
        const long long slot = p.kc ? slot_sh : -1;
        const int heads = a.n_heads + (slot >= 0 ? 2 * p.n_kv : 0);
        for (int w = threadIdx.x; w < heads * p.items; w += ROT_THREADS) {
            unsigned h, i;
            p.by_items.divmod((unsigned)w, h, i);
            const __half* in;
            __half* out;
            bool rotate = true;
            if ((int)h < a.n_heads) {
                in = a.q + t * a.q_token + h * a.q_head;
                out = a.q_out + t * a.qo_token + h * a.qo_head;
            } else if ((int)h < a.n_heads + p.n_kv) {
                in = a.k + t * a.kv_token + (long long)(h - a.n_heads) * a.head_dim;
                out = p.kc + slot + (long long)(h - a.n_heads) * p.head_stride;
            } else {
                in = a.v + t * a.kv_token + (long long)(h - a.n_heads - p.n_kv) * a.head_dim;
                out = p.vc + slot + (long long)(h - a.n_heads - p.n_kv) * p.head_stride;
                rotate = false;
            }
            if constexpr (VEC == 8) {
                if (a.half_layout && (int)i < a.rot / 16) {
                    const int d = (int)i * 8;
                    const uint4 x = *reinterpret_cast<const uint4*>(in + d), y = *reinterpret_cast<const uint4*>(in + d + pairs);
                    uint4 xo = x, yo = y;
                    if (rotate) {
                        const __half2* xh = reinterpret_cast<const __half2*>(&x);
                        const __half2* yh = reinterpret_cast<const __half2*>(&y);
                        __half2* xq = reinterpret_cast<__half2*>(&xo);
                        __half2* yq = reinterpret_cast<__half2*>(&yo);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float2 u = __half22float2(xh[j]), v = __half22float2(yh[j]);
                            const float2 c0 = cs[d + 2 * j], c1 = cs[d + 2 * j + 1];
                            xq[j] = __floats2half2_rn(u.x * c0.x - v.x * c0.y, u.y * c1.x - v.y * c1.y);
                            yq[j] = __floats2half2_rn(u.x * c0.y + v.x * c0.x, u.y * c1.y + v.y * c1.x);
                        }
                    }
                    *reinterpret_cast<uint4*>(out + d) = xo;
                    *reinterpret_cast<uint4*>(out + d + pairs) = yo;
                } else {
                    const int d = a.half_layout ? a.rot + ((int)i - a.rot / 16) * 8 : (int)i * 8;
                    const uint4 x = *reinterpret_cast<const uint4*>(in + d);
                    uint4 xo = x;
                    if (rotate && d < a.rot) {
                        const __half2* xh = reinterpret_cast<const __half2*>(&x);
                        __half2* xq = reinterpret_cast<__half2*>(&xo);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float2 u = __half22float2(xh[j]);
                            const float2 c = cs[d / 2 + j];
                            xq[j] = __floats2half2_rn(u.x * c.x - u.y * c.y, u.x * c.y + u.y * c.x);
                        }
                    }
                    *reinterpret_cast<uint4*>(out + d) = xo;
                }
            } else {
                if ((int)i < pairs) {
                    const int d0 = a.half_layout ? (int)i : 2 * (int)i, d1 = a.half_layout ? (int)i + pairs : 2 * (int)i + 1;
                    const __half xh = in[d0], yh = in[d1];
                    if (rotate) {
                        const float x = __half2float(xh), y = __half2float(yh);
                        const float2 c = cs[i];
                        out[d0] = __float2half_rn(x * c.x - y * c.y);
                        out[d1] = __float2half_rn(x * c.y + y * c.x);
                    } else {
                        out[d0] = xh;
                        out[d1] = yh;
                    }
                } else {
                    const int d = a.rot + (int)i - pairs;
                    out[d] = in[d];
                }
            }
        }
    }
}

}  // namespace

int launch_rotary(const RotaryArgs& a, const PagedView* cache, cudaStream_t st) {
    if (a.tokens == 0) return TL_OK;
    RotLaunch p{};
    p.a = a;
    p.status = device_status_word();
    auto on16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    bool vec = a.head_dim % 8 == 0 && a.rot % 8 == 0 && (!a.half_layout || a.rot % 16 == 0);
    if (a.n_heads > 0)
        vec = vec && on16(a.q) && on16(a.q_out) && a.q_token % 8 == 0 && a.q_head % 8 == 0 && a.qo_token % 8 == 0 && a.qo_head % 8 == 0;
    if (cache) {
        p.kc = cache->k; p.vc = cache->v; p.table = cache->table;
        p.page_stride = cache->page_stride; p.token_stride = cache->token_stride; p.head_stride = cache->head_stride;
        p.n_kv = cache->n_kv_heads; p.n_rows = cache->n_rows; p.max_pages = cache->max_pages; p.n_pages = cache->n_pages;
        p.by_page = cache->by_page;
        vec = vec && cache->aligned16() && on16(a.k) && on16(a.v) && a.kv_token % 8 == 0;
    }
    if (vec) p.items = a.half_layout ? a.rot / 16 + (a.head_dim - a.rot) / 8 : a.head_dim / 8;
    else p.items = a.rot / 2 + (a.head_dim - a.rot);
    p.by_items = FastDiv((unsigned)p.items);
    const int grid = a.tokens < 148 * 64 ? a.tokens : 148 * 64;
    return vec ? launch_pdl(k_rotary<8>, grid, ROT_THREADS, 0, st, true, p)
               : launch_pdl(k_rotary<1>, grid, ROT_THREADS, 0, st, true, p);
}

}  // namespace tlb
