// Beam selection: of all candidates (beam w, token j) of a batch entry, valued score_w + logit_wj - lse_w, the k best, ties
// to the lowest flat index w * vocab + j.
#include "serving.cuh"

namespace tlb {

namespace {

constexpr int BEAM_THREADS = 512;

// a logit as it counts: NaN is never chosen, +inf is the largest finite value
__device__ __forceinline__ float beam_logit(__half h) {
    const float x = __half2float(h);
    return x != x ? -INFINITY : fminf(x, 65504.f);
}
__device__ __forceinline__ double beam_score(float s) { return s != s ? -INFINITY : (double)fminf(s, 3.402823466e38f); }

// Plain form for what one CTA cannot join or 32 chunks cannot hold (many beams times many results, vocabularies beyond 2 million):
// right, and two orders of magnitude slower (four beams of 32000, which the kernel below takes 8 us for: 865 us): one CTA a batch entry; lse of its rows, then k rounds of an arg-maximum over what comes after
// the last one chosen.
__global__ void __launch_bounds__(BEAM_THREADS) k_beam_any(BeamArgs a) {
    extern __shared__ double lse[];               // [beams], and the scores [beams]: out_scores may be their place
    __shared__ double red[BEAM_THREADS / 32];
    __shared__ long long red_i[BEAM_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double* score = lse + a.beams;
    for (int w = tid; w < a.beams; w += BEAM_THREADS) score[w] = beam_score(a.scores[b * a.beams + w]);
    for (int w = 0; w < a.beams; w++) {
        const __half* x = a.logits + (long long)(b * a.beams + w) * a.pitch;
        float m = -INFINITY;
        for (unsigned j = tid; j < (unsigned)a.vocab; j += BEAM_THREADS) m = fmaxf(m, beam_logit(x[j]));    // (a step may pass 2^31)
        m = warp_max(m);
        __syncthreads();
        if (lane == 0) red[warp] = m;
        __syncthreads();
        double M = red[0];
        for (int i = 1; i < BEAM_THREADS / 32; i++) M = fmax(M, red[i]);
        __syncthreads();
        double s = 0.0;
        if (M > -INFINITY)
            for (unsigned j = tid; j < (unsigned)a.vocab; j += BEAM_THREADS) s += (double)expf(beam_logit(x[j]) - (float)M);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        if (tid == 0) {
            double S = 0.0;
            for (int i = 0; i < BEAM_THREADS / 32; i++) S += red[i];
            lse[w] = M > -INFINITY ? M + log(S) : 0.0;
        }
    }
    __syncthreads();
    double last = INFINITY;
    long long last_i = -1;
    const long long n = (long long)a.beams * a.vocab;
    for (int r = 0; r < a.k; r++) {
        double best = -INFINITY;
        long long best_i = n;
        for (long long i = tid; i < n; i += BEAM_THREADS) {
            const int w = (int)(i / a.vocab), j = (int)(i - (long long)w * a.vocab), row = b * a.beams + w;
            const double sc = score[w];
            double v;
            if (a.finished && a.finished[row]) v = j == a.pad ? sc : -INFINITY;
            else v = sc + ((double)beam_logit(a.logits[(long long)row * a.pitch + j]) - lse[w]);
            if ((v < last || (v == last && i > last_i)) && (v > best || (v == best && i < best_i))) { best = v; best_i = i; }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, best, o);
            const long long i = __shfl_xor_sync(0xffffffffu, best_i, o);
            if (v > best || (v == best && i < best_i)) { best = v; best_i = i; }
        }
        __syncthreads();
        if (lane == 0) { red[warp] = best; red_i[warp] = best_i; }
        __syncthreads();
        for (int w = 0; w < BEAM_THREADS / 32; w++)
            if (red[w] > best || (red[w] == best && red_i[w] < best_i)) { best = red[w]; best_i = red_i[w]; }
        last = best;
        last_i = best_i;
        if (tid == 0) {
            const long long at = (long long)b * a.k + r;
            a.out_scores[at] = (float)best;
            a.out_parents[at] = b * a.beams + (int)(best_i / a.vocab);
            a.out_tokens[at] = (int)(best_i % a.vocab);
        }
        __syncthreads();
    }
}


// ---- one pass over the logits ----------------------------------------------------------------------------------------
// A CTA streams a chunk of one row through registers, a window of W vectors a thread at a time, the next window's loads under
// way: the maximum and sum of exponentials (32-bit exponentials, 64-bit sums), and the k best of the chunk under the order
// (logit descending, index ascending). The first window gives a border that at least k values reach, later ones raise it;
// vectors that reach it are set aside whole in shared memory (taking them apart at once, in diverged warps, cost as much as all
// the rest), and what reaches the last border is ranked at the end. Many of them (equal or masked logits) are taken apart in
// between and cut back to the k best. The last CTA of a batch entry joins: the rows' log-sums, the candidates' values in 64
// bits, and a border and ranks over the sorted lists.
//
// Bound: with few rows the chain load -> border -> list -> arrival -> log-sum -> ranks; with many no unit (half the issue slots, a third
// of the exponentials' pipe) but what a row costs beyond its stream. Measured on a B200: 512 rows of 32000 logits, 16 of eight beams
// each, 21 us (floor 4.7), of which the last window is done at 10, its list is ranked and the CTA arrives at 13.4, and the join takes
// 4; 19 warp instructions for 32 logits, of which the stream is 6 by the source. Four rows 8.5 us. Rows in several chunks took 30 us, for the part of a chunk that does
// not shrink with it.
constexpr int SEL_THREADS = 256;
constexpr int SEL_ASIDE = 256;                    // vectors set aside that wait for the end; more are taken apart
constexpr int SEL_BATCH = SEL_THREADS / 2;        // vectors taken apart at a time, two threads each
constexpr int SEL_LONG = 1024;                    // a list of values longer than this is cut back
constexpr int SEL_MAX_SPLITS = 32;                // a lane each in the join
constexpr int SEL_MAX_CHUNK = 65536;              // indices in a chunk have 16 bits
constexpr int SEL_MAX_MERGE = 8192;               // candidates that one CTA joins
constexpr int SEL_ENTRIES = 4096;                 // batch entries of a launch: their counters have a place of their own in the workspace,
                                                  // so that calls of other sizes never find results where they expect a counter at 0

struct SelStat { double sum; float max; float pad; };

struct SelLaunch {
    BeamArgs a;
    int splits, chunk;                            // chunks of a row, logits of a chunk (a multiple of 8)
    int groups;                                   // the power of two from 8 to 128 at or above k
    int row0;                                     // row of the whole call that this launch begins with
    unsigned int* counters; SelStat* stats; unsigned int* keys;     // [SEL_ENTRIES], [row][split], [row][split][k]
};

// order of fp16 values as 16-bit integers; 0 stands below every value
__device__ __forceinline__ unsigned ord16(unsigned h) { return (h & 0x8000u) ? 0xffffu - h : h + 0x8000u; }
__device__ __forceinline__ float ord16_value(unsigned o) {
    const unsigned short h = (unsigned short)(o & 0x8000u ? o - 0x8000u : 0xffffu - o);
    __half_raw r;
    r.x = h;
    return __half2float(__half(r));
}
// order of doubles as 64-bit integers
__device__ __forceinline__ unsigned long long ord64(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double ord64_value(unsigned long long o) {
    return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}
// two 32-bit operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 c;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 c;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
// 2^x to 2^-22, results below the normal range as 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool dead_row(const BeamArgs& a, int row) {
    const float s = a.scores[row];
    return !(s > -INFINITY);
}

// A row's lists hold its largest logits, and so its largest values, but where distinct logits have the same value in 64 bits not the
// first tokens of the least value that is taken. For rows whose score makes that possible: logits differ by 2^-24 at least, and values
// below 2^28 are rounded by 2^-26 at most, so up to SEL_ROOM distinct logits have distinct values. The n-th largest value
// in the lists is the row's n-th largest; what lies above it stays, and the entries that equal it become the lowest tokens that do,
// found by the whole CTA in one pass that ends when there are enough.
constexpr double SEL_ROOM = 134217728.0;          // 2^27
__device__ __noinline__ void settle_ties(const __half* x, unsigned vocab, unsigned at0, int n, double score, double lse, unsigned long long* val,
                                         unsigned* idx, int places) {
    constexpr int EACH = 8;                       // tokens of a thread at a time
    __shared__ unsigned first[128];               // the lowest tokens of that value
    __shared__ int found_sh[SEL_THREADS / 32], above_sh;
    __shared__ unsigned long long least_sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __syncthreads();
    for (int i = tid; i < places; i += SEL_THREADS) {
        if (idx[i] == ~0u) continue;
        int above = 0, equal = 0;
        for (int j = 0; j < places; j++) {        // (places that no candidate fills are 0, below every value)
            above += val[j] > val[i];
            equal += val[j] == val[i];
        }
        if (above < n && above + equal >= n) { least_sh = val[i]; above_sh = above; }        // the same from all that write
    }
    __syncthreads();
    const unsigned long long least = least_sh;
    const int need = n - above_sh;
    int got = 0;
    for (unsigned j0 = 0; j0 < vocab && got < need; j0 += SEL_THREADS * EACH) {
        unsigned hits = 0;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const unsigned j = j0 + tid * EACH + e;
            if (j < vocab && ord64(score + ((double)beam_logit(x[j]) - lse)) == least) hits |= 1u << e;
        }
        int upto = __popc(hits);
        const int mine = upto;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        __syncthreads();
        if (lane == 31) found_sh[warp] = upto;
        __syncthreads();
        int at = got + upto - mine;
        for (int w = 0; w < SEL_THREADS / 32; w++) {
            if (w < warp) at += found_sh[w];
            got += found_sh[w];
        }
        for (int e = 0; e < EACH; e++)
            if (hits >> e & 1u) {
                if (at < need) first[at] = j0 + tid * EACH + e;
                at++;
            }
    }
    __syncthreads();
    for (int i = tid; i < places; i += SEL_THREADS) {
        if (val[i] != least || idx[i] == ~0u) continue;
        int before = 0;
        for (int j = 0; j < i; j++) before += val[j] == least;
        idx[i] = before < min(need, got) ? at0 + first[before] : ~0u;  // (~0: a place that no candidate fills)
    }
    __syncthreads();
}

// keys: (ord16 of the logit) << 16 | 0xffff - index in the chunk: unique, larger = earlier in the order
template <int W>
__global__ void __launch_bounds__(SEL_THREADS, 4) k_beam_select(SelLaunch p) {
    extern __shared__ __align__(16) unsigned char dyn[];         // the list; later the join's candidates
    __shared__ __align__(16) unsigned short tops[SEL_THREADS];
    __shared__ unsigned kept[128];
    __shared__ int red_i[SEL_THREADS / 32];
    __shared__ float red_f[SEL_THREADS / 32];
    __shared__ double red_d[SEL_THREADS / 32];
    __shared__ int count_sh, listed_sh, last_sh, large_sh;
    const BeamArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, entry = row / a.beams;
    pdl_launch_dependents();
    pdl_wait();
    if (!dead_row(a, row) && !(a.finished && a.finished[row])) {
        constexpr int SPAN = SEL_THREADS * 8 * W;
        constexpr float L2E = 1.4426950408889634f;
        uint4* aside = reinterpret_cast<uint4*>(dyn);            // [W * SEL_THREADS + SEL_ASIDE]: a window's vectors always fit
        unsigned* aside_at = reinterpret_cast<unsigned*>(aside + W * SEL_THREADS + SEL_ASIDE);
        unsigned* list = aside_at + W * SEL_THREADS + SEL_ASIDE; // [SEL_LONG + 8 * SEL_ASIDE]
        const int first = split * p.chunk, n = min(p.chunk, a.vocab - first);
        const __half* x = a.logits + row * a.pitch + first;
        const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) >> 1);
        const uint4* xv = reinterpret_cast<const uint4*>(x - skew);
        // cut the list back to its k best (it holds more): the k-th largest of the unique keys, bit by bit
        unsigned border = 0;
        auto shrink = [&](int have) {
            unsigned least = 0;
            for (int bit = 31; bit >= 0; bit--) {
                const unsigned c = least | 1u << bit;
                int reach = 0;
                for (int i = tid; i < have; i += SEL_THREADS) reach += list[i] >= c;
                reach = __reduce_add_sync(0xffffffffu, reach);
                __syncthreads();
                if (lane == 0) red_i[warp] = reach;
                __syncthreads();
                int all = 0;
#pragma unroll
                for (int w = 0; w < SEL_THREADS / 32; w++) all += red_i[w];
                if (all >= a.k) least = c;
            }
            if (tid == 0) listed_sh = 0;
            __syncthreads();
            for (int i = tid; i < have; i += SEL_THREADS)
                if (list[i] >= least) kept[atomicAdd(&listed_sh, 1)] = list[i];
            __syncthreads();
            if (tid < a.k) list[tid] = kept[tid];
            border = max(border, least >> 16);
            __syncthreads();
        };
        // take `have` vectors apart: what reaches the border goes on the list
        auto take_apart = [&](int have) {
            for (int i0 = 0; i0 < have; i0 += SEL_BATCH) {
                const int i = i0 + (tid >> 1);
                if (i < have) {
                    const uint2 half = reinterpret_cast<const uint2*>(aside + i)[tid & 1];
                    const unsigned e0 = aside_at[i] * 8 + (tid & 1) * 4;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const unsigned h = ((r < 2 ? half.x : half.y) >> (16 * (r & 1))) & 0xffffu;
                        const unsigned o = (h & 0x7fffu) > 0x7c00u ? 0x3ffu : ord16(h == 0x8000u ? 0u : h);     // NaN is -inf, -0 is 0
                        if (e0 + r < (unsigned)n && o >= border) list[atomicAdd(&listed_sh, 1)] = o << 16 | (0xffffu - (e0 + r));
                    }
                }
                if ((i0 + SEL_BATCH) % SEL_ASIDE != 0 && i0 + SEL_BATCH < have) continue;      // the list holds that many more
                __syncthreads();
                const int listed = listed_sh;
                __syncthreads();
                if (listed > SEL_LONG) shrink(listed);
            }
        };
        // A thread's values go by their index in the chunk, not by where the row happens to start, so equal rows give equal
        // sums to the last bit: rows off the 16-byte grid take each vector from the two aligned ones that it lies in (each
        // holds at least one value of the row, so nothing beyond its 16-byte neighbours is touched).
        auto index_of = [&](int w, int j) { return (w * W + j) * SEL_THREADS + tid; };     // in vectors
        uint4 next[W];
        auto fetch = [&](int w) {
#pragma unroll
            for (int j = 0; j < W; j++) {
                const int i = index_of(w, j);
                if (i * 8 < n) next[j] = __ldcs(xv + i);
            }
        };
        if (skew == 0) fetch(0);
        const int windows = (n + SPAN - 1) / SPAN;
        const __half2 ninf = __half2half2(__ushort_as_half(0xfc00)), top = __half2half2(__ushort_as_half(0x7bff));
        // The border: a value that at least k values seen so far reach. The threads form `groups` >= k groups (by their index
        // modulo that number, so none is empty where as many threads hold values); the least of the groups' maxima is one, and
        // about k ln k values reach it. Fewer threads than groups: it stays below every value. Also the largest value.
        unsigned best = 0;                        // largest value of this thread so far, as ord16; 0: it holds none
        auto publish = [&] {
            unsigned mine = best;
            for (int o = 16; o >= p.groups; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
            tops[tid] = (unsigned short)mine;
        };
        auto raise_border = [&] {
            unsigned g[8];
#pragma unroll
            for (int i = 0; i < 8; i++) g[i] = tops[i * 32 + lane];
#pragma unroll
            for (int i = 0; i < 4; i++) g[i] = max(g[i], g[i + 4]);                 // threads equal modulo 128
            const unsigned all = max(max(g[0], g[2]), max(g[1], g[3]));
            const unsigned b = p.groups == 128 ? min(min(g[0], g[1]), min(g[2], g[3])) : (p.groups == 64 ? min(max(g[0], g[2]), max(g[1], g[3])) : all);
            border = max(border, __reduce_min_sync(0xffffffffu, b));
            return __reduce_max_sync(0xffffffffu, all);
        };
        float ref = -INFINITY;                    // what this thread's sum is relative to
        double sum = 0.0;
        for (int w = 0; w < windows; w++) {
            // 1: the window; -inf outside the row
            __half2 v[W][4];
#pragma unroll
            for (int j = 0; j < W; j++) {
                const int i = index_of(w, j), e = i * 8;
                uint4 raw = next[j];
                if (skew) {
                    unsigned q[8] = {};
                    if (e < n) {
                        const uint4 lo = __ldcs(xv + i);
                        q[0] = lo.x; q[1] = lo.y; q[2] = lo.z; q[3] = lo.w;
                    }
                    if (e + 8 - skew < n) {
                        const uint4 hi = __ldcs(xv + i + 1);
                        q[4] = hi.x; q[5] = hi.y; q[6] = hi.z; q[7] = hi.w;
                    }
                    if (skew & 4) {
#pragma unroll
                        for (int r = 0; r < 6; r++) q[r] = q[r + 2];
                    }
                    if (skew & 2) {
#pragma unroll
                        for (int r = 0; r < 5; r++) q[r] = q[r + 1];
                    }
                    const unsigned odd = (skew & 1) * 16;
                    raw = make_uint4(__funnelshift_r(q[0], q[1], odd), __funnelshift_r(q[1], q[2], odd), __funnelshift_r(q[2], q[3], odd),
                                     __funnelshift_r(q[3], q[4], odd));
                }
                unsigned word[4] = {raw.x, raw.y, raw.z, raw.w};
                if (e + 8 > n) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if (e + 2 * r >= n) word[r] = 0xfc00fc00u;
                        else if (e + 2 * r + 1 >= n) word[r] = (word[r] & 0xffffu) | 0xfc000000u;
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) v[j][r] = *reinterpret_cast<__half2*>(&word[r]);
            }
            if (skew == 0 && w + 1 < windows) fetch(w + 1);
            // 2: its maximum (NaN loses against any value). +inf counts as 65504, NaN as -inf: cleaned where one turns up, +inf by
            // the maximum, NaN by the sum.
            auto clean = [&] {
#pragma unroll
                for (int j = 0; j < W; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) v[j][r] = __hmin2(__hmax2(v[j][r], ninf), top);
            };
            __half2 vm[W], mx = ninf;
#pragma unroll
            for (int j = 0; j < W; j++) {
                vm[j] = __hmax2(__hmax2(v[j][0], v[j][1]), __hmax2(v[j][2], v[j][3]));
                mx = __hmax2(mx, vm[j]);
            }
            float my_max = fmaxf(__low2float(mx), __high2float(mx));
            if (my_max == INFINITY) {
                clean();
                my_max = 65504.f;
            }
            if ((w * W * SEL_THREADS + tid) * 8 < n) best = max(best, ord16(__half_as_ushort(__float2half_rn(my_max + 0.f))));
            if (w == 0) {
                publish();
                if (tid == 0) count_sh = listed_sh = 0;
                __syncthreads();
                ref = ord16_value(raise_border());
                if (windows > 1) __syncthreads();  // before tops is written again
            } else if (my_max > ref) {
                if (ref > -INFINITY) sum *= (double)exp2f((ref - my_max) * L2E);
                ref = my_max;
            }
            // 3: the sum: exp2((x - ref) * log2 e), two at a time (x - ref is exact or nearly so, and small where it counts)
            if (ref > -INFINITY) {
                auto add_up = [&] {
                    double total = 0.0;
                    const float2 minus = make_float2(-ref, -ref), scale = make_float2(L2E, L2E);
#pragma unroll
                    for (int j = 0; j < W; j++) {
                        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float2 f = mul2(add2(__half22float2(v[j][r]), minus), scale);
                            s2 = add2(s2, make_float2(ex2(f.x), ex2(f.y)));
                        }
                        total += (double)(s2.x + s2.y);
                    }
                    return total;
                };
                double part = add_up();
                if (part != part) {
                    clean();
                    part = add_up();
                }
                sum += part;
            }
            // 4: vectors that reach the border are set aside; a border below every value lets all pass
            const bool all_pass = border <= 0x3ffu;
            const __half2 edge = __half2half2(__float2half_rn(all_pass ? -INFINITY : ord16_value(border)));
#pragma unroll
            for (int j = 0; j < W; j++) {
                const int i = index_of(w, j);
                if ((all_pass || __hge2_mask(vm[j], edge)) && i * 8 < n) {
                    const int at = atomicAdd(&count_sh, 1);
                    aside[at] = *reinterpret_cast<const uint4*>(&v[j][0]);
                    aside_at[at] = (unsigned)i;
                }
            }
            if (w + 1 < windows) {
                publish();
                __syncthreads();
                const int have = count_sh;
                raise_border();
                __syncthreads();
                if (have > SEL_ASIDE) {
                    take_apart(have);
                    if (tid == 0) count_sh = 0;
                    __syncthreads();
                }
            }
        }
        // 5: the chunk's statistics and its k best, in order
        const float M = [&] {
            const float m = warp_max(ref);
            if (lane == 0) red_f[warp] = m;
            __syncthreads();
            float all = red_f[0];
#pragma unroll
            for (int w = 1; w < SEL_THREADS / 32; w++) all = fmaxf(all, red_f[w]);
            return all;
        }();
        if (ref > -INFINITY) sum *= (double)exp2f((ref - M) * L2E);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) red_d[warp] = sum;
        publish();
        const int have = count_sh;
        __syncthreads();
        raise_border();                           // over the whole chunk now
        take_apart(have);
        const int found = listed_sh;
        if (tid == 0) {
            double S = 0.0;
#pragma unroll
            for (int w = 0; w < SEL_THREADS / 32; w++) S += red_d[w];
            p.stats[(long long)row * p.splits + split] = SelStat{S, M, 0.f};
        }
        unsigned* out = p.keys + ((long long)row * p.splits + split) * a.k;
        const unsigned edge = border << 16;       // values listed before the border rose
        for (int i = tid; i < found; i += SEL_THREADS) {
            const unsigned key = list[i];
            if (key < edge) continue;
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < found; j++) rank += list[j] > key;
            if (rank < a.k) out[rank] = key;
        }
    }
    // 6: the last CTA of the entry joins (the barrier makes the release cover all threads' results)
    __syncthreads();
    if (tid == 0) {
        unsigned seen;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(seen) : "l"(p.counters + entry) : "memory");
        last_sh = seen == (unsigned)(a.beams * p.splits - 1);
        if (last_sh) p.counters[entry] = 0;
        count_sh = large_sh = 0;
    }
    __syncthreads();
    if (!last_sh) return;
    const int lists = a.beams * p.splits, total = lists * a.k;
    unsigned long long* val = reinterpret_cast<unsigned long long*>(dyn);           // [total]
    unsigned long long* some_val = val + total;                                     // [total]
    double* lse = reinterpret_cast<double*>(some_val + total);                      // [beams]
    unsigned* idx = reinterpret_cast<unsigned*>(lse + a.beams);                     // [total] flat index, ~0 where a list is short
    unsigned* some_idx = idx + total;                                               // [total]
    for (int w = warp; w < a.beams; w += SEL_THREADS / 32) {                        // a warp a row, a lane a chunk
        const int r = entry * a.beams + w;
        if (dead_row(a, r) || (a.finished && a.finished[r])) continue;
        const SelStat* s = p.stats + (long long)r * p.splits;
        const float m = lane < p.splits ? __ldcg(&s[lane].max) : -INFINITY;
        double S = lane < p.splits ? __ldcg(&s[lane].sum) : 0.0;
        const float M = warp_max(m);
        S = m > -INFINITY ? S * (double)expf(m - M) : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
        if (lane == 0) lse[w] = M > -INFINITY ? (double)M + log(S) : 0.0;
    }
    __syncthreads();
    // the heads of the lists (as many of each as make 4 k candidates): their k-th bounds the result from below, closely
    const int heads = min(a.k, (4 * a.k + lists - 1) / lists), some = heads * lists;
    for (int i = tid; i < total; i += SEL_THREADS) {
        const int l = i / a.k, j = i - l * a.k, w = l / p.splits, s = l - w * p.splits, r = entry * a.beams + w;
        const double score = beam_score(a.scores[r]);
        unsigned long long o = 0;
        unsigned at = ~0u;
        const bool dead = dead_row(a, r), fin = a.finished && a.finished[r];
        if (dead || fin) {                        // no logits: the lowest tokens at -inf, and a finished beam's pad token before them
            if (s == 0 && j < a.vocab) {
                int tok = j;
                double v = -INFINITY;
                if (!dead) {
                    tok = j == 0 ? a.pad : (j <= a.pad ? j - 1 : j);
                    if (j == 0) v = score;
                }
                o = ord64(v);
                at = (unsigned)w * (unsigned)a.vocab + (unsigned)tok;
            }
        } else {
            const int first = s * p.chunk;
            if (j < min(p.chunk, a.vocab - first)) {
                const unsigned key = __ldcg(p.keys + ((long long)r * p.splits + s) * a.k + j);
                o = ord64(score + ((double)ord16_value(key >> 16) - lse[w]));
                at = (unsigned)w * (unsigned)a.vocab + (unsigned)first + (0xffffu - (key & 0xffffu));
                if (fabs(score) >= SEL_ROOM) large_sh = 1;
            }
        }
        val[i] = o;
        idx[i] = at;
        if (j < heads) {
            some_val[l * heads + j] = o;
            some_idx[l * heads + j] = at;
        }
    }
    __shared__ unsigned long long border_val;
    __shared__ unsigned border_idx;
    if (tid == 0) { border_val = 0; border_idx = ~0u; }
    __syncthreads();
    auto rank_among = [&](unsigned long long o, unsigned at, int n) {
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) {
            const unsigned long long y = some_val[j];
            rank += (int)(y > o) | ((int)(y == o) & (int)(some_idx[j] < at));
        }
        return rank;
    };
    unsigned long long bv = 0;
    unsigned bi = ~0u;
    for (int i = tid; i < some; i += SEL_THREADS)
        if (some_idx[i] != ~0u && rank_among(some_val[i], some_idx[i], some) == a.k - 1) { border_val = some_val[i]; border_idx = some_idx[i]; }
    __syncthreads();
    bv = border_val;
    bi = border_idx;
    if (large_sh)
        for (int w = 0; w < a.beams; w++) {
            const int r = entry * a.beams + w, l0 = w * p.splits;
            const double score = beam_score(a.scores[r]);
            if (fabs(score) < SEL_ROOM || dead_row(a, r) || (a.finished && a.finished[r])) continue;
            unsigned long long most = 0;          // a list begins with its largest value
            for (int s = 0; s < p.splits; s++) most = max(most, val[(l0 + s) * a.k]);
            int above = 0;
            for (int i0 = 0; i0 < total && above < a.k; i0 += SEL_THREADS) above += __syncthreads_count(i0 + tid < total && val[i0 + tid] > most);
            if (above < a.k)                      // else (a beam marked by -1e9, say) none of it is taken
                settle_ties(a.logits + r * a.pitch, (unsigned)a.vocab, (unsigned)w * (unsigned)a.vocab, min(a.k, a.vocab), score, lse[w],
                            val + l0 * a.k, idx + l0 * a.k, p.splits * a.k);
        }
    for (int i = tid; i < total; i += SEL_THREADS) {
        const unsigned long long o = val[i];
        const unsigned at = idx[i];
        if (at != ~0u && (o > bv || (o == bv && at <= bi))) {
            const int q = atomicAdd(&count_sh, 1);
            some_val[q] = o;
            some_idx[q] = at;
        }
    }
    __syncthreads();
    const int n = count_sh;
    for (int i = tid; i < n; i += SEL_THREADS) {
        const unsigned long long o = some_val[i];
        const unsigned x = some_idx[i];
        const int rank = rank_among(o, x, n);
        if (rank < a.k) {
            const long long at = (long long)entry * a.k + rank;
            const unsigned w = x / (unsigned)a.vocab;
            a.out_scores[at] = (float)ord64_value(o);
            a.out_parents[at] = p.row0 + entry * a.beams + (int)w;
            a.out_tokens[at] = (int)(x - w * (unsigned)a.vocab);
        }
    }
}

// Chunks of a row: four CTAs an SM where the rows alone are fewer, but no chunk below one vector a thread, and no more
// candidates than the join holds: between `least` and `most`, whatever the batch; least = 0: the plain kernel. (148: the workspace
// is asked for where there may be no device.)
constexpr int SEL_CTAS = 4 * 148;
struct SelSplits { int least, most; };
SelSplits sel_split_limits(int beams, int vocab, int k) {
    const int least = (int)(((long long)vocab + SEL_MAX_CHUNK - 1) / SEL_MAX_CHUNK);
    if (least > SEL_MAX_SPLITS || (long long)beams * least * k > SEL_MAX_MERGE) return {0, 0};
    int most = 16;
    while (most > least && (beams * most * k > 1024 || vocab / most < SEL_THREADS * 4)) most--;
    return {least, most > least ? most : least};
}
int sel_splits(int batch, int beams, int vocab, int k) {
    const SelSplits limits = sel_split_limits(beams, vocab, k);
    const long long want = SEL_CTAS / ((long long)batch * beams);
    return (int)(want < limits.least ? limits.least : (want < limits.most ? want : limits.most));
}
int sel_chunk(int vocab, int splits) { return ((vocab + splits - 1) / splits + 7) / 8 * 8; }

template <int W>
int launch_sel(const SelLaunch& p, cudaStream_t st) {
    const size_t total = (size_t)p.a.beams * p.splits * p.a.k, join = total * 24 + (size_t)p.a.beams * 8;
    const size_t list = (size_t)(SEL_THREADS * W + SEL_ASIDE) * 20 + (SEL_LONG + 8 * SEL_ASIDE) * 4, smem = list > join ? list : join;
    static PerDeviceOnce once;
    TL_CUDA(once.run([&] { return cudaFuncSetAttribute(k_beam_select<W>, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_MAX_MERGE * 24 + 128 * 8); }));
    return launch_pdl(k_beam_select<W>, p.a.batch * p.a.beams * p.splits, SEL_THREADS, smem, st, true, p);
}

}  // namespace

size_t beam_workspace_bytes(int batch, int beams, int vocab, int k) {
    // Never less than what a smaller batch asks for, whose rows may be cut into more chunks: rows times chunks are at most
    // rows * most and SEL_CTAS, or rows * least where that is more.
    const SelSplits limits = sel_split_limits(beams, vocab, k);
    const size_t rows = (size_t)(batch < SEL_ENTRIES ? batch : SEL_ENTRIES) * beams, least = rows * limits.least, most = rows * limits.most;
    const size_t cut = most < (size_t)SEL_CTAS ? most : (size_t)SEL_CTAS;
    return SEL_ENTRIES * 4 + (cut > least ? cut : least) * (sizeof(SelStat) + 4 * (size_t)k);
}

int launch_beam_select(const BeamArgs& a, cudaStream_t st) {
    if (a.batch == 0) return TL_OK;
    SelLaunch p{};
    p.a = a;
    p.splits = sel_splits(a.batch, a.beams, a.vocab, a.k);
    if (p.splits == 0)
        return launch_pdl(k_beam_any, a.batch, BEAM_THREADS, (size_t)a.beams * 16, st, true, a);
    p.chunk = sel_chunk(a.vocab, p.splits);
    p.groups = 8;
    while (p.groups < a.k) p.groups *= 2;
    char* w = static_cast<char*>(a.work);
    const int most = a.batch < SEL_ENTRIES ? a.batch : SEL_ENTRIES;
    p.counters = reinterpret_cast<unsigned int*>(w);
    p.stats = reinterpret_cast<SelStat*>(w + SEL_ENTRIES * 4);
    p.keys = reinterpret_cast<unsigned int*>(p.stats + (size_t)most * a.beams * p.splits);
    for (int e0 = 0; e0 < a.batch; e0 += most) {  // launches behind one another share the workspace
        p.row0 = e0 * a.beams;
        p.a.batch = a.batch - e0 < most ? a.batch - e0 : most;
        p.a.logits = a.logits + (long long)p.row0 * a.pitch;
        p.a.scores = a.scores + p.row0;
        p.a.finished = a.finished ? a.finished + p.row0 : nullptr;
        p.a.out_scores = a.out_scores + (long long)e0 * a.k;
        p.a.out_parents = a.out_parents + (long long)e0 * a.k;
        p.a.out_tokens = a.out_tokens + (long long)e0 * a.k;
        // one vector a thread where that covers the chunk: the shortest chain; else four, loaded ahead
        TL_PROPAGATE(p.chunk <= SEL_THREADS * 8 ? launch_sel<1>(p, st) : launch_sel<4>(p, st));
        if (a.batch - e0 <= most) break;          // (e0 may not pass 2^31 - 1)
    }
    return TL_OK;
}

}  // namespace tlb
