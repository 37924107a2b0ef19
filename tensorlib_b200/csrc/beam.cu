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

}  // namespace

size_t beam_workspace_bytes(int, int, int, int) { return 0; }

int launch_beam_select(const BeamArgs& a, cudaStream_t st) {
    if (a.batch == 0) return TL_OK;
    return launch_pdl(k_beam_any, a.batch, BEAM_THREADS, (size_t)a.beams * 8, st, true, a);
}

}  // namespace tlb
