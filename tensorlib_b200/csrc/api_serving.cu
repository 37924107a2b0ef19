// extern "C" entry points of the operators that serve many sequences: argument checks, then the launchers of rotary.cu,
// paged.cu, paged_attn.cu and beam.cu. Arguments are checked before the device is asked for, so the refusals are the same
// with and without one.
#include <cmath>

#include "serving.cuh"

using namespace tlb;

namespace {
inline const __half* H(const tl_half* p) { return reinterpret_cast<const __half*>(p); }
inline __half* H(tl_half* p) { return reinterpret_cast<__half*>(p); }

#define TL_ON_LIBRARY_DEVICE()      \
    TL_CHECK_INIT();                \
    OnLibraryDevice on_device_;     \
    TL_CUDA(on_device_.err)

// what every use of a cache needs; the arrays that only some calls touch are checked there
int check_cache(const tl_paged_cache* c, bool pools, const char* who) {
    TL_REQUIRE(c != nullptr, "%s: null cache", who);
    TL_REQUIRE(c->n_layers > 0 && c->n_pages > 0 && c->page_size > 0 && c->n_kv_heads > 0 && c->head_dim > 0 && c->n_rows > 0 &&
                   c->max_pages > 0, "%s: cache sizes must be positive", who);
    TL_REQUIRE((long long)c->max_pages * c->page_size <= (1ll << 31) - 128, "%s: a row of more than 2^31 - 128 tokens", who);
    TL_REQUIRE(c->n_rows < (1 << 28), "%s: 2^28 rows or more", who);
    TL_REQUIRE(c->page_table, "%s: null page table", who);
    if (pools) {
        TL_REQUIRE(c->k_pages && c->v_pages, "%s: null page pool", who);
        TL_REQUIRE(c->page_stride > 0 && c->token_stride > 0 && c->head_stride > 0 && (c->n_layers == 1 || c->layer_stride > 0),
                   "%s: cache strides must be positive", who);
        TL_REQUIRE((long long)c->page_size * c->n_kv_heads * c->head_dim < (1ll << 31), "%s: a page of more than 2^31 - 1 values", who);
        TL_REQUIRE(2ll * c->n_layers * ((long long)c->n_pages + c->n_rows) < (1ll << 31), "%s: more than 2^31 - 1 pages over all layers", who);
    }
    return TL_OK;
}
}  // namespace

extern "C" {

int tl_rotary_frequencies(int rot_dim, double base, int scaling, double factor, double trained_len, double low, double high,
                          double* freqs_host, float* magnitude_host) {
    TL_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && freqs_host && magnitude_host, "rotary_frequencies: bad arguments");
    TL_REQUIRE(base > 1.0 && std::isfinite(base), "rotary_frequencies: base must be above 1");
    TL_REQUIRE(scaling >= TL_ROPE_UNSCALED && scaling <= TL_ROPE_RAMP, "rotary_frequencies: unknown scaling %d", scaling);
    if (scaling != TL_ROPE_UNSCALED) TL_REQUIRE(factor >= 1.0 && std::isfinite(factor), "rotary_frequencies: factor must be at least 1");
    if (scaling == TL_ROPE_PARTS || scaling == TL_ROPE_RAMP)
        TL_REQUIRE(trained_len > 0 && std::isfinite(trained_len) && low > 0 && high > low && std::isfinite(high),
                   "rotary_frequencies: needs trained_len > 0 and 0 < low < high");
    const double two_pi = 6.283185307179586476925;
    const int n = rot_dim / 2;
    double b = base;
    if (scaling == TL_ROPE_BASE && rot_dim > 2) b = base * std::pow(factor, (double)rot_dim / (rot_dim - 2));
    *magnitude_host = 1.0f;
    double lo = 0, hi = 0;
    bool all = false;                             // not even the first pair turns more than `low` times
    if (scaling == TL_ROPE_RAMP) {
        // pair index at which a pair turns x times over the trained length
        auto index_of = [&](double turns) { return rot_dim * std::log(trained_len / (turns * two_pi)) / (2 * std::log(base)); };
        lo = std::fmax(std::floor(index_of(high)), 0.0);
        hi = std::fmin(std::ceil(index_of(low)), rot_dim - 1.0);
        all = index_of(low) <= 0;
        *magnitude_host = (float)(0.1 * std::log(factor) + 1.0);
    }
    for (int i = 0; i < n; i++) {
        double f = std::pow(b, -2.0 * i / rot_dim);
        if (scaling == TL_ROPE_LINEAR) f /= factor;
        if (scaling == TL_ROPE_PARTS) {
            const double s = std::fmin(1.0, std::fmax(0.0, (trained_len * f / two_pi - low) / (high - low)));
            f = (1 - s) * f / factor + s * f;
        }
        if (scaling == TL_ROPE_RAMP) {
            const double s = all ? 1.0 : std::fmin(1.0, std::fmax(0.0, (i - lo) / std::fmax(hi - lo, 0.001)));
            f = (1 - s) * f + s * f / factor;
        }
        freqs_host[i] = f;
    }
    return TL_OK;
}

int tl_rotary_f16(const tl_half* in, tl_half* out, const int* positions, const double* freqs, float magnitude, int tokens, int n_heads,
                  int head_dim, int rot_dim, int half_layout, int inverse, long long in_token_stride, long long in_head_stride,
                  long long out_token_stride, long long out_head_stride, tl_stream stream) {
    TL_REQUIRE(tokens >= 0 && n_heads > 0 && head_dim > 0, "rotary: bad sizes");
    TL_REQUIRE(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_dim && rot_dim <= 1024, "rotary: rot_dim must be even, at most head_dim and 1024");
    TL_REQUIRE((long long)n_heads * head_dim < (1ll << 31), "rotary: a token of more than 2^31 - 1 values");
    TL_REQUIRE(half_layout == 0 || half_layout == 1, "rotary: half_layout is 0 or 1");
    if (tokens == 0) {
        TL_CHECK_INIT();
        return TL_OK;
    }
    TL_REQUIRE(in && out && positions && (freqs || rot_dim == 0), "rotary: null pointer");
    TL_REQUIRE(in_token_stride >= 0 && in_head_stride >= 0 && out_token_stride >= 0 && out_head_stride >= 0, "rotary: negative stride");
    TL_REQUIRE(in != out || (in_token_stride == out_token_stride && in_head_stride == out_head_stride),
               "rotary: in place needs the same strides on both sides");
    TL_ON_LIBRARY_DEVICE();
    RotaryArgs a{};
    a.q = H(in); a.q_out = H(out);
    a.q_token = in_token_stride; a.q_head = in_head_stride; a.qo_token = out_token_stride; a.qo_head = out_head_stride;
    a.n_heads = n_heads; a.positions = positions; a.freqs = freqs; a.magnitude = magnitude;
    a.tokens = tokens; a.head_dim = head_dim; a.rot = rot_dim; a.half_layout = half_layout; a.inverse = inverse != 0;
    return launch_rotary(a, nullptr, as_stream(stream));
}

int tl_rotary_append_f16(const tl_paged_cache* cache, int layer, const tl_half* q, tl_half* q_out, const tl_half* k, const tl_half* v,
                         const int* rows, const int* positions, const double* freqs, float magnitude, int tokens, int n_heads, int rot_dim,
                         int half_layout, long long q_token_stride, long long q_out_token_stride, long long kv_token_stride,
                         tl_stream stream) {
    TL_PROPAGATE(check_cache(cache, true, "rotary_append"));
    TL_REQUIRE(layer >= 0 && layer < cache->n_layers, "rotary_append: layer %d out of range", layer);
    TL_REQUIRE(tokens >= 0 && n_heads >= 0, "rotary_append: bad sizes");
    TL_REQUIRE(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= cache->head_dim && rot_dim <= 1024,
               "rotary_append: rot_dim must be even, at most head_dim and 1024");
    TL_REQUIRE(((long long)n_heads + 2ll * cache->n_kv_heads) * cache->head_dim < (1ll << 31), "rotary_append: a token of more than 2^31 - 1 values");
    TL_REQUIRE(half_layout == 0 || half_layout == 1, "rotary_append: half_layout is 0 or 1");
    if (tokens == 0) {
        TL_CHECK_INIT();
        return TL_OK;
    }
    TL_REQUIRE(k && v && positions && (freqs || rot_dim == 0) && (n_heads == 0 || (q && q_out)), "rotary_append: null pointer");
    TL_REQUIRE(rows || tokens <= cache->n_rows, "rotary_append: more tokens than rows without a row list");
    TL_REQUIRE(q_token_stride >= 0 && q_out_token_stride >= 0 && kv_token_stride >= 0, "rotary_append: negative stride");
    TL_REQUIRE(n_heads == 0 || q != q_out || q_token_stride == q_out_token_stride, "rotary_append: in place needs the same strides on both sides");
    TL_ON_LIBRARY_DEVICE();
    RotaryArgs a{};
    a.q = H(q); a.q_out = H(q_out);
    a.q_token = q_token_stride; a.q_head = cache->head_dim; a.qo_token = q_out_token_stride; a.qo_head = cache->head_dim;
    a.n_heads = n_heads; a.k = H(k); a.v = H(v); a.kv_token = kv_token_stride;
    a.rows = rows; a.positions = positions; a.freqs = freqs; a.magnitude = magnitude;
    a.tokens = tokens; a.head_dim = cache->head_dim; a.rot = rot_dim; a.half_layout = half_layout; a.inverse = 0;
    const PagedView view(*cache, layer);
    return launch_rotary(a, &view, as_stream(stream));
}

int tl_paged_attn_workspace(int n_heads, int n_kv_heads, int head_dim, size_t* bytes) {
    TL_REQUIRE(bytes && n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && head_dim > 0 && head_dim <= 256,
               "paged_attn_workspace: bad arguments");
    *bytes = paged_attn_workspace_bytes(n_heads, n_kv_heads, head_dim);
    return TL_OK;
}

int tl_paged_attn_decode_f16(const tl_paged_cache* cache, int layer, const tl_half* q, tl_half* out, float* lse, const int* rows, int batch,
                             int n_heads, float scale, long long q_row_stride, long long out_row_stride, void* workspace,
                             size_t workspace_bytes, tl_stream stream) {
    TL_PROPAGATE(check_cache(cache, true, "paged_attn_decode"));
    TL_REQUIRE(layer >= 0 && layer < cache->n_layers, "paged_attn_decode: layer %d out of range", layer);
    TL_REQUIRE(batch >= 0 && n_heads > 0 && n_heads % cache->n_kv_heads == 0, "paged_attn_decode: n_heads must be a multiple of the cache's");
    if (cache->head_dim > 256) return set_error(TL_ERR_UNSUPPORTED, "paged_attn_decode: head_dim above 256");
    // scores are exponentiated to base 2
    TL_REQUIRE(std::isfinite(scale * 1.4426950408889634f), "paged_attn_decode: scale times log2 e must be finite");
    TL_REQUIRE(batch <= 65535 && n_heads <= 65535, "paged_attn_decode: more than 65535 rows or heads");
    if (batch == 0) {
        TL_CHECK_INIT();
        return TL_OK;
    }
    TL_REQUIRE(q && out && cache->lengths, "paged_attn_decode: null pointer");
    TL_REQUIRE(q_row_stride >= 0 && out_row_stride >= 0, "paged_attn_decode: negative stride");
    TL_REQUIRE(rows || batch <= cache->n_rows, "paged_attn_decode: more queries than rows without a row list");
    TL_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "paged_attn_decode: the workspace must be 16-byte aligned");
    const size_t need = paged_attn_workspace_bytes(n_heads, cache->n_kv_heads, cache->head_dim);
    TL_REQUIRE(workspace_bytes >= need, "paged_attn_decode: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    TL_ON_LIBRARY_DEVICE();
    PagedAttnArgs a{};
    a.q = H(q); a.out = H(out); a.lse = lse; a.rows = rows; a.batch = batch; a.n_heads = n_heads; a.scale = scale;
    a.q_row = q_row_stride; a.o_row = out_row_stride; a.work = workspace;
    return launch_paged_attn(PagedView(*cache, layer), a, as_stream(stream));
}

int tl_paged_fork(const tl_paged_cache* cache, const int* parents, tl_stream stream) {
    TL_PROPAGATE(check_cache(cache, false, "paged_fork"));
    TL_REQUIRE(parents && cache->lengths && cache->ref_counts, "paged_fork: null pointer");
    TL_ON_LIBRARY_DEVICE();
    return launch_paged_fork(PagedView(*cache), parents, as_stream(stream));
}

int tl_paged_workspace(int n_rows, int n_pages, size_t* bytes) {
    TL_REQUIRE(bytes && n_rows > 0 && n_pages > 0, "paged_workspace: bad arguments");
    *bytes = paged_workspace_bytes(n_rows, n_pages);
    return TL_OK;
}

static int check_paged_work(const tl_paged_cache* c, const void* workspace, size_t bytes, const char* who) {
    TL_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be 16-byte aligned", who);
    const size_t need = paged_workspace_bytes(c->n_rows, c->n_pages);
    TL_REQUIRE(bytes >= need, "%s: workspace of %zu bytes, %zu needed", who, bytes, need);
    return TL_OK;
}

int tl_paged_reserve_f16(const tl_paged_cache* cache, const int* new_tokens, int* result, void* workspace, size_t workspace_bytes,
                         tl_stream stream) {
    TL_PROPAGATE(check_cache(cache, true, "paged_reserve"));
    TL_REQUIRE(new_tokens && result && cache->lengths && cache->ref_counts, "paged_reserve: null pointer");
    TL_PROPAGATE(check_paged_work(cache, workspace, workspace_bytes, "paged_reserve"));
    TL_ON_LIBRARY_DEVICE();
    return launch_paged_reserve(PagedView(*cache), new_tokens, result, workspace, as_stream(stream));
}

int tl_paged_copy_f16(const tl_paged_cache* cache, const int* src, const int* dst, int n, tl_stream stream) {
    TL_PROPAGATE(check_cache(cache, true, "paged_copy"));
    TL_REQUIRE(n >= 0 && (n == 0 || (src && dst)) && 2ll * n * cache->n_layers < (1ll << 31), "paged_copy: bad arguments");
    TL_ON_LIBRARY_DEVICE();
    return launch_paged_copy(PagedView(*cache), src, dst, n, as_stream(stream));
}

int tl_paged_compact_f16(const tl_paged_cache* cache, int* moved_to, int* live, void* workspace, size_t workspace_bytes, tl_stream stream) {
    TL_PROPAGATE(check_cache(cache, true, "paged_compact"));
    TL_REQUIRE(moved_to && live && cache->ref_counts, "paged_compact: null pointer");
    TL_PROPAGATE(check_paged_work(cache, workspace, workspace_bytes, "paged_compact"));
    TL_ON_LIBRARY_DEVICE();
    return launch_paged_compact(PagedView(*cache), moved_to, live, workspace, as_stream(stream));
}

static int check_beam_sizes(int batch, int beams, int vocab, int k) {
    TL_REQUIRE(batch >= 0 && beams > 0 && vocab > 0 && k > 0, "beam_select: bad sizes");
    TL_REQUIRE(beams <= 128 && k <= 128, "beam_select: more than 128 beams or results");
    TL_REQUIRE((long long)beams * vocab < (1ll << 31) && (long long)batch * beams < (1ll << 31) && (long long)batch * k < (1ll << 31),
               "beam_select: more than 2^31 - 1 candidates or rows");
    TL_REQUIRE((long long)k <= (long long)beams * vocab, "beam_select: k exceeds the number of candidates");
    return TL_OK;
}

int tl_beam_select_workspace(int batch, int beams, int vocab, int k, size_t* bytes) {
    TL_REQUIRE(bytes != nullptr, "beam_select_workspace: null output");
    TL_PROPAGATE(check_beam_sizes(batch, beams, vocab, k));
    *bytes = beam_workspace_bytes(batch, beams, vocab, k);
    return TL_OK;
}

int tl_beam_select_f16(const tl_half* logits, long long row_stride, const float* scores, const unsigned char* finished, int pad_token,
                       int batch, int beams, int vocab, int k, float* out_scores, int* out_parents, int* out_tokens, void* workspace,
                       size_t workspace_bytes, tl_stream stream) {
    TL_PROPAGATE(check_beam_sizes(batch, beams, vocab, k));
    if (batch == 0) {
        TL_CHECK_INIT();
        return TL_OK;
    }
    TL_REQUIRE(logits && scores && out_scores && out_parents && out_tokens, "beam_select: null pointer");
    TL_REQUIRE(!finished || (pad_token >= 0 && pad_token < vocab), "beam_select: pad_token out of range");
    TL_REQUIRE(row_stride >= vocab || (long long)batch * beams == 1, "beam_select: row stride smaller than the row");
    TL_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "beam_select: the workspace must be 16-byte aligned");
    const size_t need = beam_workspace_bytes(batch, beams, vocab, k);
    TL_REQUIRE(workspace_bytes >= need, "beam_select: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    TL_ON_LIBRARY_DEVICE();
    BeamArgs a{H(logits), row_stride, scores, finished, pad_token, batch, beams, vocab, k, out_scores, out_parents, out_tokens, workspace};
    return launch_beam_select(a, as_stream(stream));
}

int tl_beam_reorder_f16(const tl_half* src, tl_half* dst, const int* parents, int outer, int rows, long long used, long long src_outer_stride,
                        long long src_row_stride, long long dst_outer_stride, long long dst_row_stride, tl_stream stream) {
    TL_REQUIRE(outer >= 0 && rows >= 0 && used >= 0, "beam_reorder: bad sizes");
    if (outer == 0 || rows == 0 || used == 0) {
        TL_CHECK_INIT();
        return TL_OK;
    }
    TL_REQUIRE(src && dst && parents && src != dst, "beam_reorder: null pointer, or in place");
    TL_REQUIRE(src_row_stride >= used && dst_row_stride >= used, "beam_reorder: row stride smaller than the row");
    TL_REQUIRE(src_outer_stride >= 0 && dst_outer_stride >= 0, "beam_reorder: negative stride");
    TL_REQUIRE(used < (1ll << 40) && (long long)outer * rows < (1ll << 31), "beam_reorder: too large");
    TL_ON_LIBRARY_DEVICE();
    return launch_gather_rows(H(src), H(dst), parents, outer, rows, used, src_outer_stride, src_row_stride, dst_outer_stride, dst_row_stride,
                              as_stream(stream));
}

}  // extern "C"
