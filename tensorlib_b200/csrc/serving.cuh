// Shared by the operators that serve many sequences at once: rotary positions (rotary.cu), the paged key-value cache
// (paged.cu, paged_attn.cu) and beam selection (beam.cu). Launchers only enqueue on `st` and return a tl_status; the
// C entry points with their argument checks are in api_serving.cu.
#pragma once

#include "common.cuh"

namespace tlb {

// What kernels here set to TL_ERR_INVALID_ARGUMENT for an id outside its table. It is not the word of the bounded waits: that one says
// that the results of the call which finds it are not valid, and its value is not to be lost.
int* device_id_status_word();
int init_device();

// Calls may come from a thread whose current device is another one: the pointers belong to the device of tl_init.
struct OnLibraryDevice {
    int before = -1;
    cudaError_t err = cudaSuccess;
    OnLibraryDevice() {
        int now = 0;
        err = cudaGetDevice(&now);
        if (err == cudaSuccess && now != init_device()) {
            before = now;
            err = cudaSetDevice(init_device());
        }
    }
    ~OnLibraryDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// n / d for n < 2^31 by one multiplication (Granlund and Montgomery, Division by Invariant Integers using Multiplication): m = ceil(2^32 * 2^s / d) with 2^s >= d, so the error term n * (m d - 2^(32+s))
// stays below 2^(32+s) (round-up method); d = 1 .. 2^31 - 1. The top bit of m is implied, hence the extra addition.
struct FastDiv {
    unsigned int m, s, d;
    FastDiv() : m(0), s(0), d(1) {}
    explicit FastDiv(unsigned int div) : m(0), s(0), d(div) {
        while ((1ull << s) < d) s++;
        m = (unsigned int)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
    __host__ __device__ __forceinline__ unsigned int div(unsigned int n) const {
#ifdef __CUDA_ARCH__
        return (__umulhi(m, n) + n) >> s;
#else
        return (unsigned int)((((unsigned long long)m * n >> 32) + n) >> s);
#endif
    }
    __host__ __device__ __forceinline__ void divmod(unsigned int n, unsigned int& q, unsigned int& r) const {
        q = div(n);
        r = n - q * d;
    }
};

// tl_paged_cache with the divisors the kernels need
struct PagedView {
    __half* k; __half* v;                                        // of the layer asked for (layer 0 where every layer is meant)
    long long layer_stride, page_stride, token_stride, head_stride;
    int n_layers, n_pages, page_size, n_kv_heads, head_dim, n_rows, max_pages;
    int* table; int* lengths; int* refs;
    FastDiv by_page;
    explicit PagedView(const tl_paged_cache& c, int layer = 0)
        : k(reinterpret_cast<__half*>(c.k_pages) + (long long)layer * c.layer_stride),
          v(reinterpret_cast<__half*>(c.v_pages) + (long long)layer * c.layer_stride), layer_stride(c.layer_stride),
          page_stride(c.page_stride), token_stride(c.token_stride), head_stride(c.head_stride), n_layers(c.n_layers),
          n_pages(c.n_pages), page_size(c.page_size), n_kv_heads(c.n_kv_heads), head_dim(c.head_dim), n_rows(c.n_rows),
          max_pages(c.max_pages), table(c.page_table), lengths(c.lengths), refs(c.ref_counts), by_page((unsigned)c.page_size) {}
    // every head's row of every token starts on 16 bytes
    bool aligned16() const {
        return head_dim % 8 == 0 && page_stride % 8 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0 &&
               (n_layers == 1 || layer_stride % 8 == 0) && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    }
};

// ---- rotary.cu ---------------------------------------------------------------------------------------------------
struct RotaryArgs {
    // rows to rotate: q (or the plain operand) ...
    const __half* q; __half* q_out;
    long long q_token, q_head, qo_token, qo_head;
    int n_heads;
    // ... and, where a cache is given, k (rotated) and v (copied) into their pages
    const __half* k; const __half* v;
    long long kv_token;
    const int* rows;
    const int* positions; const double* freqs;
    float magnitude;
    int tokens, head_dim, rot, half_layout, inverse;
};
int launch_rotary(const RotaryArgs& a, const PagedView* cache, cudaStream_t st);

// ---- paged.cu ----------------------------------------------------------------------------------------------------
int launch_paged_fork(const PagedView& c, const int* parents, cudaStream_t st);
size_t paged_workspace_bytes(int n_rows, int n_pages);
int launch_paged_reserve(const PagedView& c, const int* new_tokens, int* result, void* work, cudaStream_t st);
int launch_paged_copy(const PagedView& c, const int* src, const int* dst, int n, cudaStream_t st);
int launch_paged_compact(const PagedView& c, int* moved_to, int* live, void* work, cudaStream_t st);
int launch_gather_rows(const __half* src, __half* dst, const int* parents, int outer, int rows, long long used, long long so,
                       long long sr, long long dso, long long dsr, cudaStream_t st);

// ---- paged_attn.cu -----------------------------------------------------------------------------------------------
struct PagedAttnArgs {
    const __half* q; __half* out; float* lse;
    const int* rows;
    int batch, n_heads;
    float scale;
    long long q_row, o_row;
    void* work;
};
size_t paged_attn_workspace_bytes(int n_heads, int n_kv_heads, int head_dim);
int launch_paged_attn(const PagedView& c, const PagedAttnArgs& a, cudaStream_t st);

// ---- beam.cu -----------------------------------------------------------------------------------------------------
struct BeamArgs {
    const __half* logits; long long pitch;
    const float* scores; const unsigned char* finished;
    int pad, batch, beams, vocab, k;
    float* out_scores; int* out_parents; int* out_tokens;
    void* work;
};
size_t beam_workspace_bytes(int batch, int beams, int vocab, int k);
int launch_beam_select(const BeamArgs& a, cudaStream_t st);

}  // namespace tlb
