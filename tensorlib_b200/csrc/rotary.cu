// Rotary positions: pair i of a head (elements 2i, 2i+1, or i, i + rot/2) is turned by the angle position * freqs[i] and
// scaled by `magnitude`; elements from rot on pass through. With a paged cache the keys go, rotated, and the values, as
// they are, straight into their pages: one pass over q, k and v.
//
// The angle: position * freqs[i] / (2 pi) in 64 bits, reduced to the nearest turn there, so that position 10^6 loses
// nothing; the fraction (at most half a turn) is exact to 2^-24 of a turn in 32 bits. Within half a turn the hardware's sine and
// cosine are good to 2^-20.5, a seven-hundredth of the rounding of the result to fp16. The rotation itself is in 32 bits with
// that one rounding.
//
// Bound: HBM at many tokens (every element is read and written once), launch and one dependent load chain
// (position -> cos/sin -> store) at one token. What has to be small for that is the number of instructions a vector: a form
// that found token, head and element of every vector anew issued 190 of them and took 83 us for 16384 tokens of 40 heads of
// 128, at 83% of the issue slots. So a thread keeps to one vector of the head and steps through (token, head) rows with
// pointers that only grow; the cos/sin of a CTA's tokens are worked out once, for all heads, in shared memory, while the first
// vectors arrive.
#include <type_traits>

#include "serving.cuh"

namespace tlb {

namespace {

constexpr int ROT_THREADS = 256;
// CTAs of an SM: what the registers of the rows under way allow. 16384 tokens of 40 heads of 128: interleaved 58 us with five (64
// with four), in halves 59 us with four (65 with five).
constexpr int rot_ctas(bool half_layout) { return half_layout ? 4 : 5; }
constexpr int ROT_ROWS = 16;                      // rows of a thread; twice that where three tensors are set up
constexpr int ROT_MAX_GROUP = 64;                 // tokens of a CTA
constexpr int ROT_MAX_PAIRS = 1024;               // their pairs in shared memory (one token has at most 512)

// One of the tensors that a call moves: rows (token, head) of head_dim values.
struct RotPlane {
    const __half* in; __half* out;
    long long in_token, in_head, out_token, out_head;      // out_token: only where rows do not go to pages
    int heads;
    bool turned, paged;                           // rotated; stored at the token's slot of the page
    int heads_at_once, tokens_at_once;            // of a CTA
    FastDiv by_heads_at_once;
};

struct RotLaunch {
    RotaryArgs a;
    RotPlane plane[3];
    int planes;
    const int* table;                             // of the cache, if there is one
    long long page_stride, token_stride;
    int n_rows, max_pages, n_pages;
    bool paged;
    FastDiv by_page, by_items, by_pairs;
    int items, group, turn_stride;                // items of a head; tokens of a CTA; floats between a token's cos and sin
    int* status;
};

// cos and sin of pair i at `pos`, times the magnitude
__device__ __forceinline__ float2 turn_of(const RotaryArgs& a, int pos, int i) {
    const double turns = (double)pos * (a.freqs[i] * 0.15915494309189533577);
    const float angle = (float)(turns - rint(turns)) * 6.2831853071795865f;
    const float s = __sinf(angle), c = __cosf(angle);
    return make_float2(c * a.magnitude, (a.inverse ? -s : s) * a.magnitude);
}
// where token t goes in its page, -1 if its row, position or page is not there
__device__ __forceinline__ long long slot_of(const RotLaunch& p, int t, int pos) {
    const int row = p.a.rows ? p.a.rows[t] : t;
    const unsigned pg = p.by_page.div((unsigned)pos);
    if (row >= 0 && row < p.n_rows && (int)pg < p.max_pages) {
        const int page = p.table[(long long)row * p.max_pages + pg];
        if (page >= 0 && page < p.n_pages) return page * p.page_stride + (long long)((unsigned)pos - pg * p.by_page.d) * p.token_stride;
    }
    atomicExch(p.status, TL_ERR_INVALID_ARGUMENT);
    return -1;
}

template <int N> struct FloatVec;
template <> struct FloatVec<4> { using T = float4; };
template <> struct FloatVec<2> { using T = float2; };
template <> struct FloatVec<1> { using T = float; };
template <int VEC> struct HalfVec;
template <> struct HalfVec<8> { using T = uint4; };
template <> struct HalfVec<4> { using T = uint2; };
template <> struct HalfVec<2> { using T = unsigned; };

// x (and y, the vector half a rotated part further) turned by the cos and sin of its pairs, which lie at c and c + stride
template <int VEC, bool HALF, typename V>
__device__ __forceinline__ void turn_item(V& x, V& y, const float* c, int stride) {
    constexpr int PAIRS = HALF ? VEC : VEC / 2, W = PAIRS < 4 ? PAIRS : 4;
    using F = typename FloatVec<W>::T;            // W pairs by one load each
    __half2* xh = reinterpret_cast<__half2*>(&x);
    __half2* yh = reinterpret_cast<__half2*>(&y);
#pragma unroll
    for (int j0 = 0; j0 < PAIRS; j0 += W) {
        const F cv = *reinterpret_cast<const F*>(c + j0), sv = *reinterpret_cast<const F*>(c + stride + j0);
        const float* co = reinterpret_cast<const float*>(&cv);
        const float* si = reinterpret_cast<const float*>(&sv);
        if constexpr (HALF) {
#pragma unroll
            for (int j = 0; j < W; j += 2) {
                __half2 &xv = xh[(j0 + j) / 2], &yv = yh[(j0 + j) / 2];
                const float2 f = __half22float2(xv), g = __half22float2(yv);
                xv = __floats2half2_rn(f.x * co[j] - g.x * si[j], f.y * co[j + 1] - g.y * si[j + 1]);
                yv = __floats2half2_rn(f.x * si[j] + g.x * co[j], f.y * si[j + 1] + g.y * co[j + 1]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float2 f = __half22float2(xh[j0 + j]);
                xh[j0 + j] = __floats2half2_rn(f.x * co[j] - f.y * si[j], f.x * si[j] + f.y * co[j]);
            }
        }
    }
}

// Items of VEC values. Interleaved pairs: an item is a vector, VEC / 2 pairs. Half layout: an item is the vectors at i and
// i + rot / 2, VEC pairs; behind rot, one vector.
// BY: how the rows that a thread has under way follow one another: ROT_BY_HEAD within a token, ROT_BY_TOKEN (all heads of a token
// are moved at once) from token to token, ROT_EITHER as each tensor wants it, which takes more registers.
enum { ROT_BY_HEAD, ROT_BY_TOKEN, ROT_EITHER };
template <int VEC, bool HALF, int BY>
__global__ void __launch_bounds__(ROT_THREADS, rot_ctas(HALF)) k_rotary(RotLaunch p) {
    using V = typename HalfVec<VEC>::T;
    extern __shared__ __align__(16) float turns[];             // [group]: cos [stride], sin [stride]
    __shared__ long long places[2][ROT_MAX_GROUP];             // where the token goes: its row of q, its slot in the page; -1: nowhere
    pdl_launch_dependents();
    pdl_wait();
    const RotaryArgs& a = p.a;
    const int pairs = a.rot / 2, stride = p.turn_stride, t0 = blockIdx.x * p.group, n_tokens = min(p.group, a.tokens - t0);
    unsigned r, item;
    p.by_items.divmod(threadIdx.x, r, item);
    const bool pair = HALF && (int)item < pairs / VEC, mine = HALF ? pair : (int)item * VEC < a.rot;
    const int d = !HALF || pair ? (int)item * VEC : a.rot + ((int)item - pairs / VEC) * VEC;
    // all planes one after the other, or (few tokens) one a CTA
    const int first = gridDim.y > 1 ? blockIdx.y : 0, end = gridDim.y > 1 ? first + 1 : p.planes;
    constexpr int U = HALF ? 2 : (BY == ROT_EITHER ? 3 : 4);    // rows under way a thread
    V x[U], y[U];
    bool ready = false;
    for (int w = first; w < end; w++) {
        const int heads = p.plane[w].heads, at_once = p.plane[w].heads_at_once, tokens_at_once = p.plane[w].tokens_at_once;
        const bool paged = p.plane[w].paged, turn = p.plane[w].turned && mine;
        const long long in_step = (long long)at_once * p.plane[w].in_head, out_step = (long long)at_once * p.plane[w].out_head;
        unsigned tt, h0;
        p.plane[w].by_heads_at_once.divmod(r, tt, h0);
        const int left = (int)tt < tokens_at_once ? heads - (int)h0 : 0;       // rows of a token: 0, at_once, .. below this
        const __half* in_token = p.plane[w].in + (long long)(t0 + tt) * p.plane[w].in_token + h0 * p.plane[w].in_head + d;
        __half* const out0 = p.plane[w].out + h0 * p.plane[w].out_head + d;
        // a thread's rows under way: heads of one token, or, where all its heads are moved at once, tokens
        auto move = [&](auto by_token_c) {
            constexpr bool by_token = decltype(by_token_c)::value;
            const int more_tokens = by_token ? tokens_at_once : 0, t_step = by_token ? U * tokens_at_once : tokens_at_once;
            const long long in_more = by_token ? tokens_at_once * p.plane[w].in_token : in_step, out_more = by_token ? 0 : out_step;
            const long long in_next = t_step * p.plane[w].in_token;
            for (int t = (int)tt;; t += t_step, in_token += in_next) {
                const __half* in = in_token;
                int h = 0;
                do {
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (t + u * more_tokens < n_tokens && (by_token ? left > 0 : h + u * at_once < left)) {
                            x[u] = *reinterpret_cast<const V*>(in + u * in_more);
                            if (pair) y[u] = *reinterpret_cast<const V*>(in + u * in_more + pairs);
                        }
                    if (!ready) {                 // the turns and places of the CTA's tokens, while the first rows arrive
                        for (int j = threadIdx.x; j < n_tokens; j += ROT_THREADS) {
                            const int pos = a.positions[t0 + j];          // below 0: padding
                            places[0][j] = pos >= 0 ? (t0 + j) * p.plane[0].out_token : -1;
                            places[1][j] = p.paged && pos >= 0 ? slot_of(p, t0 + j, pos) : -1;
                        }
                        const int todo = p.plane[first].turned ? n_tokens * pairs : 0;      // (values alone need no turns)
                        for (int j = threadIdx.x; j < todo; j += ROT_THREADS) {
                            unsigned k, i;
                            p.by_pairs.divmod((unsigned)j, k, i);
                            const float2 c = turn_of(a, a.positions[t0 + (int)k], (int)i);
                            turns[k * 2 * stride + i] = c.x;
                            turns[(k * 2 + 1) * stride + i] = c.y;
                        }
                        __syncthreads();
                        ready = true;
                    }
                    if (t >= n_tokens || left <= 0) return;
                    __half* out = out0 + (h == 0 ? 0 : (long long)(h / at_once) * out_step);
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int tu = t + u * more_tokens;
                        if (tu >= n_tokens || (!by_token && h + u * at_once >= left)) continue;
                        const long long at = places[paged][tu];
                        if (at < 0) continue;
                        if (turn) turn_item<VEC, HALF>(x[u], y[u], turns + tu * 2 * stride + (HALF ? d : d / 2), stride);
                        *reinterpret_cast<V*>(out + at + u * out_more) = x[u];
                        if (pair) *reinterpret_cast<V*>(out + at + u * out_more + pairs) = y[u];
                    }
                    in += U * in_step;
                    h += U * at_once;
                } while (!by_token && h < left);
            }
        };
        if constexpr (BY == ROT_BY_HEAD) move(std::false_type{});
        else if constexpr (BY == ROT_BY_TOKEN) move(std::true_type{});
        else if (at_once == heads) move(std::true_type{});
        else move(std::false_type{});
    }
}

// Any alignment: one pair or one passed-through element an item, one token a CTA.
__global__ void __launch_bounds__(ROT_THREADS) k_rotary_any(RotLaunch p) {
    extern __shared__ float2 cs[];
    __shared__ long long slot_sh;
    pdl_launch_dependents();
    pdl_wait();
    const RotaryArgs& a = p.a;
    const int pairs = a.rot / 2;
    // (unsigned counters: a step beyond the last token or item may pass 2^31)
    for (unsigned t = blockIdx.x; t < (unsigned)a.tokens; t += gridDim.x) {
        const int pos = a.positions[t];
        __syncthreads();
        if (pos < 0) continue;                    // padding: nothing is written
        for (int i = threadIdx.x; i < pairs; i += ROT_THREADS) cs[i] = turn_of(a, pos, i);
        if (threadIdx.x == 0 && p.paged) slot_sh = slot_of(p, (int)t, pos);
        __syncthreads();
        const long long slot = p.paged ? slot_sh : -1;
        for (int w = 0; w < p.planes; w++) {
            const RotPlane& q = p.plane[w];
            if (q.paged && slot < 0) continue;
            for (unsigned k = threadIdx.x; k < (unsigned)(q.heads * p.items); k += ROT_THREADS) {
                unsigned h, i;
                p.by_items.divmod(k, h, i);
                const __half* in = q.in + t * q.in_token + h * q.in_head;
                __half* out = q.out + (q.paged ? slot : t * q.out_token) + h * q.out_head;
                if ((int)i < pairs) {
                    const int d0 = a.half_layout ? (int)i : 2 * (int)i, d1 = a.half_layout ? (int)i + pairs : 2 * (int)i + 1;
                    const __half xh = in[d0], yh = in[d1];
                    if (q.turned) {
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

template <int VEC, bool HALF>
int launch_by(const RotLaunch& p, dim3 grid, size_t smem, cudaStream_t st) {
    int by_token = 0;
    for (int w = 0; w < p.planes; w++) by_token += p.plane[w].heads_at_once == p.plane[w].heads;
    return by_token == 0 ? launch_pdl(k_rotary<VEC, HALF, ROT_BY_HEAD>, grid, ROT_THREADS, smem, st, true, p)
         : by_token == p.planes ? launch_pdl(k_rotary<VEC, HALF, ROT_BY_TOKEN>, grid, ROT_THREADS, smem, st, true, p)
                                : launch_pdl(k_rotary<VEC, HALF, ROT_EITHER>, grid, ROT_THREADS, smem, st, true, p);
}
template <int VEC>
int launch_vec(const RotLaunch& p, dim3 grid, size_t smem, cudaStream_t st) {
    return p.a.half_layout ? launch_by<VEC, true>(p, grid, smem, st) : launch_by<VEC, false>(p, grid, smem, st);
}

}  // namespace

int launch_rotary(const RotaryArgs& a, const PagedView* cache, cudaStream_t st) {
    if (a.tokens == 0) return TL_OK;
    RotLaunch p{};
    p.a = a;
    p.status = device_id_status_word();
    if (a.n_heads > 0)
        p.plane[p.planes++] = RotPlane{a.q, a.q_out, a.q_token, a.q_head, a.qo_token, a.qo_head, a.n_heads, true, false};
    if (cache) {
        p.paged = true;
        p.table = cache->table; p.page_stride = cache->page_stride; p.token_stride = cache->token_stride;
        p.n_rows = cache->n_rows; p.max_pages = cache->max_pages; p.n_pages = cache->n_pages; p.by_page = cache->by_page;
        p.plane[p.planes++] = RotPlane{a.k, cache->k, a.kv_token, a.head_dim, 0, cache->head_stride, cache->n_kv_heads, true, true};
        p.plane[p.planes++] = RotPlane{a.v, cache->v, a.kv_token, a.head_dim, 0, cache->head_stride, cache->n_kv_heads, false, true};
    }
    // the widest vectors that every row, the rotated part and its halves allow
    const int pairs = a.rot / 2;
    auto fits = [&](int vec) {
        auto on = [&](const void* x) { return reinterpret_cast<uintptr_t>(x) % (2 * vec) == 0; };
        bool ok = a.head_dim % vec == 0 && (a.half_layout ? pairs : a.rot) % vec == 0;
        if (cache) ok = ok && cache->page_stride % vec == 0 && cache->token_stride % vec == 0;
        for (int w = 0; w < p.planes; w++) {
            const RotPlane& q = p.plane[w];
            ok = ok && on(q.in) && on(q.out) && q.in_token % vec == 0 && q.in_head % vec == 0 && q.out_token % vec == 0 && q.out_head % vec == 0;
        }
        return ok;
    };
    int vec = fits(8) ? 8 : (fits(4) ? 4 : (fits(2) ? 2 : 1));
    if (vec > 1) {
        p.items = (a.half_layout ? pairs : a.rot) / vec + (a.head_dim - a.rot) / vec;
        if (p.items > ROT_THREADS) vec = 1;       // a thread keeps to an item of the head
    }
    if (vec == 1) {
        p.items = pairs + (a.head_dim - a.rot);
        p.by_items = FastDiv((unsigned)p.items);
        return launch_pdl(k_rotary_any, a.tokens < sm_count() * 64 ? a.tokens : sm_count() * 64, ROT_THREADS, (size_t)pairs * 8, st, true, p);
    }
    p.by_items = FastDiv((unsigned)p.items);
    p.by_pairs = FastDiv((unsigned)(pairs > 0 ? pairs : 1));
    const int rows = ROT_THREADS / p.items;
    int heads = 0;
    for (int w = 0; w < p.planes; w++) {
        RotPlane& q = p.plane[w];
        q.heads_at_once = rows < q.heads ? rows : q.heads;
        q.tokens_at_once = rows / q.heads_at_once;
        q.by_heads_at_once = FastDiv((unsigned)q.heads_at_once);
        heads += q.heads;
    }
    // Tokens a CTA: enough that setting up a tensor is small against moving its rows (about ROT_ROWS a thread), and so that the
    // CTAs make whole rounds of those that are resident. Where a token is a CTA, so is each tensor of it.
    const long long resident = (long long)rot_ctas(a.half_layout != 0) * sm_count();
    long long most = (long long)ROT_ROWS * (p.planes > 1 ? 2 : 1) * rows / heads;
    if (pairs > 0 && most > ROT_MAX_PAIRS / pairs) most = ROT_MAX_PAIRS / pairs;
    if (most > ROT_MAX_GROUP) most = ROT_MAX_GROUP;
    if (most < 1) most = 1;
    const long long rounds = (a.tokens + most * resident - 1) / (most * resident);
    p.group = (int)((a.tokens + rounds * resident - 1) / (rounds * resident));
    p.turn_stride = (pairs + 3) / 4 * 4;
    const dim3 grid((unsigned)(((long long)a.tokens + p.group - 1) / p.group), p.group == 1 ? p.planes : 1);
    const size_t smem = (size_t)p.group * p.turn_stride * 8;
    return vec == 8 ? launch_vec<8>(p, grid, smem, st) : (vec == 4 ? launch_vec<4>(p, grid, smem, st) : launch_vec<2>(p, grid, smem, st));
}

}  // namespace tlb
