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

// Plain form for any shape: one CTA a batch entry; lse of its rows, then k rounds of an arg-maximum over what comes after
// the last one chosen.
__global__ void __launch_bounds__(BEAM_THREADS) k_beam_any(BeamArgs a) {
    extern __shared__ double lse[];               // [beams]
    __shared__ double red[BEAM_THREADS / 32];
    __shared__ long long red_i[BEAM_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int w = 0; w < a.beams; w++) {
        const __half* x = a.logits + (long long)(b * a.beams + w) * a.pitch;
        float m = -INFINITY;
        for (int j = tid; j < a.vocab; j += BEAM_THREADS) m = fmaxf(m, beam_logit(x[j]));
        m = warp_max(m);
        __syncthreads();
        if (lane == 0) red[warp] = m;
        __syncthreads();
        double M = red[0];
        for (int i = 1; i < BEAM_THREADS / 32; i++) M = fmax(M, red[i]);
        __syncthreads();
        double s = 0.0;
        if (M > -INFINITY)
            for (int j = tid; j < a.vocab; j += BEAM_THREADS) s += (double)expf(beam_logit(x[j]) - (float)M);
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
            const double sc = beam_score(a.scores[row]);
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
// A CTA holds a chunk of one row in registers: its maximum and its sum of exponentials (32-bit exponentials, 64-bit sums),
// and the k best of the chunk under the order (logit descending, index ascending). The K-th largest of the threads' maxima
// bounds the K-th largest logit from below, so what reaches it is a short list, ranked by counting; only where that list is
// long (many equal or masked logits) is the exact border searched. The last CTA of a batch entry joins: the rows' log-sums,
// the candidates' values in 64 bits, and the same bound-and-rank over the sorted lists.
//
// Bound: HBM with many rows (each logit is read once); with few rows the chain load -> maximum -> sum -> list -> join.
constexpr int SEL_THREADS = 256;
constexpr int SEL_CAP = 1024;                     // candidates of a chunk that are ranked by counting
constexpr int SEL_MAX_SPLITS = 16;
constexpr int SEL_MAX_MERGE = 8192;               // candidates that one CTA joins

struct SelStat { double sum; float max; float pad; };

struct SelLaunch {
    BeamArgs a;
    int splits, chunk;                            // chunks of a row, logits of a chunk (a multiple of 8)
    int groups;                                   // the power of two from 8 to 128 at or above k
    unsigned int* counters; SelStat* stats; unsigned int* keys;     // [batch], [row][split], [row][split][k]
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
__device__ __forceinline__ bool dead_row(const BeamArgs& a, int row) {
    const float s = a.scores[row];
    return !(s > -INFINITY);
}

// keys: (ord16 of the logit) << 16 | 0xffff - index in the chunk: unique, larger = earlier in the order
template <int VPT>
__global__ void __launch_bounds__(SEL_THREADS, VPT <= 2 ? 6 : (VPT == 4 ? 4 : (VPT == 8 ? 2 : 1))) k_beam_select(SelLaunch p) {
    extern __shared__ unsigned char dyn[];        // the join's candidates
    __shared__ unsigned list[SEL_CAP];
    __shared__ __align__(16) unsigned short tops[SEL_THREADS];
    __shared__ int red_i[SEL_THREADS / 32];
    __shared__ double red_d[SEL_THREADS / 32];
    __shared__ int count_sh, last_sh;
    const BeamArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits, entry = row / a.beams;
    pdl_launch_dependents();
    pdl_wait();
    if (!dead_row(a, row) && !(a.finished && a.finished[row])) {
        // 1: the chunk into registers. A thread's values go by their index in the chunk, not by where the row happens to start,
        // so equal rows give equal sums to the last bit: rows off the 16-byte grid take each vector from the two aligned ones
        // that it lies in (which hold at least one value of the row each, so nothing beyond its 16-byte neighbours is touched).
        const int first = split * p.chunk, n = min(p.chunk, a.vocab - first);
        const __half* x = a.logits + row * a.pitch + first;
        const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) >> 1);
        const uint4* xv = reinterpret_cast<const uint4*>(x - skew);
        // values cleaned (NaN -> -inf, +inf -> 65504, -0 -> +0); outside: bit pattern NONE, a NaN that cleaning never leaves
        constexpr unsigned NONE = 0xffffu;
        unsigned v[VPT][4];
        const __half2 ninf = __half2half2(__ushort_as_half(0xfc00)), top = __half2half2(__ushort_as_half(0x7bff)), zero = __half2half2(__ushort_as_half(0));
        __half2 mx = ninf;
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            const int e = (tid + j * SEL_THREADS) * 8;                              // chunk index of the vector's first value
            uint4 raw = make_uint4(~0u, ~0u, ~0u, ~0u);
            if (e < n) raw = __ldcs(xv + tid + j * SEL_THREADS);
            if (skew) {
                uint4 hi = make_uint4(~0u, ~0u, ~0u, ~0u);
                if (e + 8 - skew < n) hi = __ldcs(xv + tid + j * SEL_THREADS + 1);
                unsigned w[8] = {raw.x, raw.y, raw.z, raw.w, hi.x, hi.y, hi.z, hi.w};
                if (skew & 4) {
#pragma unroll
                    for (int i = 0; i < 6; i++) w[i] = w[i + 2];
                }
                if (skew & 2) {
#pragma unroll
                    for (int i = 0; i < 5; i++) w[i] = w[i + 1];
                }
                const unsigned odd = (skew & 1) * 16;
                raw = make_uint4(__funnelshift_r(w[0], w[1], odd), __funnelshift_r(w[1], w[2], odd), __funnelshift_r(w[2], w[3], odd),
                                 __funnelshift_r(w[3], w[4], odd));
            }
            v[j][0] = raw.x; v[j][1] = raw.y; v[j][2] = raw.z; v[j][3] = raw.w;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (e + 2 * i >= n) v[j][i] = 0xfc00fc00u;
                else if (e + 2 * i + 1 >= n) v[j][i] = (v[j][i] & 0xffffu) | 0xfc000000u;
                __half2 y = *reinterpret_cast<__half2*>(&v[j][i]);
                y = __hadd2(__hmin2(__hmax2(y, ninf), top), zero);
                mx = __hmax2(mx, y);
                v[j][i] = *reinterpret_cast<unsigned*>(&y);
                if (e + 2 * i >= n) v[j][i] |= NONE;
                if (e + 2 * i + 1 >= n) v[j][i] |= NONE << 16;
            }
        }
        // 2: the maximum, and a border that at least k values reach: the threads form `groups` >= k groups (by their index modulo
        // that number, so none is empty where as many threads hold values), and the least of the groups' maxima is one. About
        // k ln k values reach it. Fewer threads than groups: the border is below every value, and they hold less than SEL_CAP.
        unsigned mine = tid * 8 < n ? ord16(__half_as_ushort(__hmax(__low2half(mx), __high2half(mx)))) : 0u;
        for (int o = 16; o >= p.groups; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        tops[tid] = (unsigned short)mine;
        if (tid == 0) count_sh = 0;
        __syncthreads();
        unsigned e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = tops[i * 32 + lane];
        unsigned g4[4], border;
#pragma unroll
        for (int i = 0; i < 4; i++) g4[i] = max(e[i], e[i + 4]);                    // threads equal modulo 128
        if (p.groups == 128) border = min(min(g4[0], g4[1]), min(g4[2], g4[3]));
        else border = p.groups == 64 ? min(max(g4[0], g4[2]), max(g4[1], g4[3])) : max(max(g4[0], g4[2]), max(g4[1], g4[3]));
        border = __reduce_min_sync(0xffffffffu, border);
        const float M = ord16_value(__reduce_max_sync(0xffffffffu, max(max(g4[0], g4[2]), max(g4[1], g4[3]))));
        // 3: the sum
        double sum = 0.0;
        if (M > -INFINITY) {
            constexpr float L2E = 1.4426950408889634f;
#pragma unroll
            for (int j = 0; j < VPT; j++) {
                float s8 = 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&v[j][i]));
                    // NONE is a NaN: fmaxf leaves -inf, whose exponential is 0
                    s8 += exp2f((fmaxf(f.x, -INFINITY) - M) * L2E) + exp2f((fmaxf(f.y, -INFINITY) - M) * L2E);
                }
                sum += (double)s8;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) red_d[warp] = sum;
        // 4: what reaches the border
        const int want = min(a.k, n);
        {
            // compared in pairs; a border below every value lets all pass (NONE is a NaN and never does)
            const __half2 edge = __half2half2(__float2half_rn(border <= 0x3ffu ? -INFINITY : ord16_value(border)));
#pragma unroll
            for (int j = 0; j < VPT; j++) {
                unsigned hit[4], any = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    hit[i] = __hge2_mask(*reinterpret_cast<__half2*>(&v[j][i]), edge);
                    any |= hit[i];
                }
                if (any) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (hit[i >> 1] >> (16 * (i & 1)) & 1u) {
                            const int at = atomicAdd(&count_sh, 1);
                            const unsigned h = (v[j][i >> 1] >> (16 * (i & 1))) & 0xffffu;
                            if (at < SEL_CAP) list[at] = ord16(h) << 16 | (0xffffu - (unsigned)((tid + j * SEL_THREADS) * 8 + i));
                        }
                }
            }
        }
        __syncthreads();
        int found = count_sh;
        if (tid == 0) {
            double S = 0.0;
#pragma unroll
            for (int w = 0; w < SEL_THREADS / 32; w++) S += red_d[w];
            p.stats[(long long)row * p.splits + split] = SelStat{S, M, 0.f};
        }
        if (found > SEL_CAP) {                    // many equal ones: the exact border among the unique keys
            auto each = [&](auto&& f) {
#pragma unroll
                for (int j = 0; j < VPT; j++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const unsigned h = (v[j][i >> 1] >> (16 * (i & 1))) & 0xffffu;
                        if (h != NONE) f(ord16(h) << 16 | (0xffffu - (unsigned)((tid + j * SEL_THREADS) * 8 + i)));
                    }
            };
            unsigned least = 0;
            for (int bit = 31; bit >= 0; bit--) {
                const unsigned c = least | 1u << bit;
                int have = 0;
                each([&](unsigned key) { have += key >= c; });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) have += __shfl_xor_sync(0xffffffffu, have, o);
                __syncthreads();
                if (lane == 0) red_i[warp] = have;
                __syncthreads();
                int all = 0;
#pragma unroll
                for (int w = 0; w < SEL_THREADS / 32; w++) all += red_i[w];
                if (all >= want) least = c;
            }
            if (tid == 0) count_sh = 0;
            __syncthreads();
            each([&](unsigned key) { if (key >= least) list[atomicAdd(&count_sh, 1)] = key; });
            __syncthreads();
            found = count_sh;
        }
        // 5: their ranks
        unsigned* out = p.keys + ((long long)row * p.splits + split) * a.k;
        for (int i = tid; i < found; i += SEL_THREADS) {
            const unsigned key = list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < found; j++) rank += list[j] > key;
            if (rank < a.k) out[rank] = key;
        }
    }
    // 6: the last CTA of the entry joins (the barrier before the fence makes it cover all threads' results)
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        last_sh = atomicAdd(p.counters + entry, 1u) == (unsigned)(a.beams * p.splits - 1);
        if (last_sh) p.counters[entry] = 0;
        __threadfence();
        count_sh = 0;
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
    // the heads of the lists (as many of each as make k candidates): their k-th bounds the result from below
    const int heads = (a.k + lists - 1) / lists, some = heads * lists;
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
            a.out_parents[at] = entry * a.beams + (int)w;
            a.out_tokens[at] = (int)(x - w * (unsigned)a.vocab);
        }
    }
}

// Chunks of a row: enough CTAs for the machine, at most SEL_MAX_SPLITS and what the join can hold; 0 = the plain kernel.
int sel_splits(int batch, int beams, int vocab, int k) {
    const int widest = SEL_THREADS * 8 * 16;      // logits that fit the registers of a CTA
    const int least = (vocab + widest - 1) / widest;
    if (least > SEL_MAX_SPLITS || (long long)beams * least * k > SEL_MAX_MERGE) return 0;
    long long want = (4 * 148 + (long long)batch * beams - 1) / ((long long)batch * beams);
    const int light = (vocab + 8191) / 8192;      // four vectors a thread: several CTAs fit an SM
    if (want < light) want = light;
    want = want < SEL_MAX_SPLITS ? want : SEL_MAX_SPLITS;
    while (want > least && (beams * want * k > 1024 || vocab / want < SEL_THREADS * 8)) want--;
    return (int)(want > least ? want : least);
}
int sel_chunk(int vocab, int splits) { return ((vocab + splits - 1) / splits + 7) / 8 * 8; }

template <int VPT>
int launch_sel(const SelLaunch& p, size_t smem, cudaStream_t st) {
    static PerDeviceOnce once;
    if (once.needed()) TL_CUDA(cudaFuncSetAttribute(k_beam_select<VPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_MAX_MERGE * 24 + 128 * 8));
    return launch_pdl(k_beam_select<VPT>, p.a.batch * p.a.beams * p.splits, SEL_THREADS, smem, st, true, p);
}

}  // namespace

size_t beam_workspace_bytes(int batch, int beams, int vocab, int k) {
    const int splits = sel_splits(batch > 0 ? batch : 1, beams, vocab, k);
    const size_t rows = (size_t)batch * beams;
    return ((size_t)batch * 4 + 15) / 16 * 16 + rows * splits * (sizeof(SelStat) + 4 * (size_t)k);
}

int launch_beam_select(const BeamArgs& a, cudaStream_t st) {
    if (a.batch == 0) return TL_OK;
    SelLaunch p{};
    p.a = a;
    p.splits = sel_splits(a.batch, a.beams, a.vocab, a.k);
    if (p.splits == 0 || (long long)a.batch * a.beams * p.splits >= (1ll << 31))
        return launch_pdl(k_beam_any, a.batch, BEAM_THREADS, (size_t)a.beams * 8, st, true, a);
    p.chunk = sel_chunk(a.vocab, p.splits);
    p.groups = 8;
    while (p.groups < a.k) p.groups *= 2;
    char* w = static_cast<char*>(a.work);
    const size_t lists = (size_t)a.batch * a.beams * p.splits;
    p.counters = reinterpret_cast<unsigned int*>(w);
    p.stats = reinterpret_cast<SelStat*>(w + ((size_t)a.batch * 4 + 15) / 16 * 16);
    p.keys = reinterpret_cast<unsigned int*>(p.stats + lists);
    const size_t total = (size_t)a.beams * p.splits * a.k, smem = total * 24 + (size_t)a.beams * 8;
    const int vecs = (p.chunk + SEL_THREADS * 8 - 1) / (SEL_THREADS * 8);
    if (vecs <= 1) return launch_sel<1>(p, smem, st);
    if (vecs <= 2) return launch_sel<2>(p, smem, st);
    if (vecs <= 4) return launch_sel<4>(p, smem, st);
    if (vecs <= 8) return launch_sel<8>(p, smem, st);
    return launch_sel<16>(p, smem, st);
}

}  // namespace tlb
