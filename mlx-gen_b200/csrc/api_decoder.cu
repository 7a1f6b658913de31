// api_decoder.cu -- the extern "C" entry points of the decoder operators (residual norm,
// rotary positions, paged attention, page copies, step planning, sampling).  Everything the host can know is checked
// here before a launch; sizes and indices that live on the device are bounds-checked by the
// kernels, which report them in the device error word.
#include <math.h>
#include <stdlib.h>

#include "attn_common.cuh"

namespace ql {

int launch_norm_residual(const normres::Params &, int, int, int64_t, bool, cudaStream_t);
int launch_rope(const ropek::Params &, int, int64_t, bool, bool, cudaStream_t);
int launch_copy_pages(void *, int64_t, int64_t, int64_t, int64_t, const int32_t *, const int32_t *, int64_t,
                      cudaStream_t);
size_t paged_attention_workspace(int64_t, int, int, int, int64_t, int64_t, int64_t, int64_t);
int launch_paged_attention(attn::Params &, int, int, int64_t, void *, cudaStream_t);
int launch_plan_step(const plank::Params &, cudaStream_t);
int launch_sample(const samplek::Params &, int, int64_t, cudaStream_t);

static int elem_bytes(int dt) { return dt == QL_F32 ? 4 : 2; }
static bool elem_aligned(const void *p, int dt) { return (reinterpret_cast<uintptr_t>(p) % elem_bytes(dt)) == 0; }
static bool aligned32(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }
static bool pow2(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }
static int log2i(int64_t v) {
    int s = 0;
    while (((int64_t)1 << s) < v) ++s;
    return s;
}

// Whether the n bytes at `a` touch one of the rows of `width` bytes, `stride` >= width apart, from `base` on.
static bool touches_rows(const void *a, int64_t n, const void *base, int64_t rows, int64_t stride, int64_t width) {
    if (n <= 0 || rows <= 0 || width <= 0) return false;
    const int64_t from = (int64_t)(reinterpret_cast<intptr_t>(a) - reinterpret_cast<intptr_t>(base));
    if (from + n <= 0 || from >= (__int128)(rows - 1) * stride + width) return false;  // (nearly always)
    const int64_t row = from < width ? 0 : (from - width) / stride + 1;  // the first that ends behind a
    return row < rows && row * stride < from + n;
}

static int check_attention(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv) {
    if (T < 0 || T > INT32_MAX || B < 0 || B > 65535)
        return fail(QL_EINVAL_SHAPE, "ql_paged_attention: bad token or sequence count (T=%lld, B=%lld; at most 65535 sequences)",
                    (long long)T, (long long)B);
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv) return fail(QL_EINVAL_SHAPE, "Hq=%d must be a positive multiple of Hkv=%d", Hq, Hkv);
    if (D != 64 && D != 96 && D != 128 && D != 256)
        return fail(QL_EUNSUPPORTED, "head dimension must be 64, 96, 128 or 256 (got %d)", D);
    if (max_q < 0 || max_q > T || max_kv < 0 || max_kv > (1 << 30))
        return fail(QL_EINVAL_SHAPE, "max_q=%lld must be in [0, T], max_kv=%lld in [0, 2^30]", (long long)max_q, (long long)max_kv);
    // rows of a kv head: ints in the kernels; row blocks of 16 times Hkv are a grid's x, tiles of 256
    // (heads of 64 and 128) its y
    const int64_t rows = max_q * (Hq / Hkv);
    if (rows > (1 << 30) || (rows + 15) / 16 * Hkv > INT32_MAX || ((D == 64 || D == 128) && rows > (int64_t)65535 * attn::SM100_ROWS))
        return fail(QL_EUNSUPPORTED, "max_q * Hq / Hkv = %lld is too large for one call; split the chunk", (long long)rows);
    return QL_OK;
}

}  // namespace ql

extern "C" {

int ql_norm_residual(const void *y, int y_dtype, int64_t y_stride, const void *residual, int r_dtype, int64_t r_stride,
                     int64_t M, int64_t D, const void *weight, float weight_offset, const void *post_weight,
                     const void *gate, int64_t gate_period, float alpha, const void *scale, int64_t scale_period,
                     float eps, void *h, void *r_out, void *stream) {
    g_err[0] = 0;
    if (M < 0 || M > INT32_MAX || D <= 0 || D > normres::MAX_D)
        return fail(QL_EINVAL_SHAPE, "ql_norm_residual: D must be in [1, %d] (M=%lld D=%lld)", normres::MAX_D, (long long)M,
                    (long long)D);
    if (!valid_dtype(y_dtype) || !valid_dtype(r_dtype) || (r_dtype != y_dtype && r_dtype != QL_F32))
        return fail(QL_EUNSUPPORTED, "ql_norm_residual: the residual is in y's dtype or f32");
    if (y_stride < D || r_stride < D) return fail(QL_EINVAL_SHAPE, "row strides must be at least D");
    if (gate_period < 0 || scale_period < 0) return fail(QL_EINVAL_ARG, "periods must be >= 0");
    if (M == 0) return QL_OK;
    if (!y || !residual || !weight || !h || !r_out) return fail(QL_EINVAL_ARG, "ql_norm_residual: NULL pointer");
    const void *vecs[] = {y, weight, post_weight, gate, scale, h};
    const int ye = elem_bytes(y_dtype), re = elem_bytes(r_dtype);
    bool vec = D % 8 == 0 && y_stride * ye % 16 == 0 && r_stride * re % 16 == 0 && aligned16(residual) && aligned16(r_out);
    for (const void *v : vecs) {
        if (!elem_aligned(v, y_dtype)) return fail(QL_EINVAL_ARG, "ql_norm_residual: pointer not aligned to its dtype");
        vec = vec && aligned16(v);
    }
    if (!elem_aligned(residual, r_dtype) || !elem_aligned(r_out, r_dtype))
        return fail(QL_EINVAL_ARG, "ql_norm_residual: pointer not aligned to its dtype");
    const normres::Params p{y,     residual,    y_stride, r_stride, (int)D, 1.0f / (float)D, alpha, weight_offset, eps,
                            post_weight, weight, gate,  scale,    gate_period, scale_period, h, r_out};
    return launch_norm_residual(p, y_dtype, r_dtype, M, vec, (cudaStream_t)stream);
}

static int rope_common(ql::ropek::Params &p, int dtype, int64_t T, int64_t page_size, int layout, void *stream) {
    if (T < 0 || T > INT32_MAX || p.Hq < 0 || p.Hk < 0 || p.Hq + p.Hk <= 0 || p.D <= 0 || p.D > 1024)
        return fail(QL_EINVAL_SHAPE, "rotary positions: bad sizes (T=%lld Hq=%d Hk=%d D=%d, D at most 1024)", (long long)T,
                    p.Hq, p.Hk, p.D);
    if (p.rot < 2 || p.rot > p.D || p.rot % 2)
        return fail(QL_EINVAL_SHAPE, "rotary dimension must be even and in [2, D] (got %d)", p.rot);
    if (!valid_dtype(dtype)) return fail(QL_EUNSUPPORTED, "unknown dtype");
    if (layout != QL_ROPE_HALF && layout != QL_ROPE_INTERLEAVED) return fail(QL_EINVAL_ARG, "unknown rotary layout %d", layout);
    if (p.P < 0) return fail(QL_EINVAL_SHAPE, "negative table length");
    if (T == 0) return QL_OK;
    if (!p.table || !p.positions || (p.Hq && (!p.q || !p.q_out)) || (p.Hk && !p.k))
        return fail(QL_EINVAL_ARG, "rotary positions: NULL pointer");
    const int e = elem_bytes(dtype);
    const void *ptrs[] = {p.q, p.k, p.v, p.q_out, p.k_out, p.k_cache, p.v_cache};
    const int64_t strides[] = {p.q_token, p.q_head, p.k_token, p.k_head, p.v_token, p.v_head, p.page_stride};
    bool vec = p.D % 8 == 0 && p.rot % 16 == 0 && aligned16(p.table);
    for (const void *q : ptrs) {
        if (!elem_aligned(q, dtype)) return fail(QL_EINVAL_ARG, "rotary positions: pointer not aligned to its dtype");
        vec = vec && aligned16(q);
    }
    for (int64_t s : strides) vec = vec && s * e % 16 == 0;
    if (!elem_aligned(p.table, QL_F32)) return fail(QL_EINVAL_ARG, "rotary table not aligned");
    return launch_rope(p, dtype, T, layout == QL_ROPE_HALF, vec, (cudaStream_t)stream);
}

int ql_rope(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k, int64_t k_token_stride,
            int64_t k_head_stride, int dtype, int64_t T, int Hq, int Hk, int D, int rotary_dim, int layout,
            const float *table, int64_t table_rows, const int64_t *positions, void *q_out, void *k_out, void *stream) {
    g_err[0] = 0;
    if (T > 0 && Hk > 0 && !k_out) return fail(QL_EINVAL_ARG, "ql_rope: NULL pointer");
    ql::ropek::Params p{};
    p.q = q, p.q_token = q_token_stride, p.q_head = q_head_stride;
    p.k = k, p.k_token = k_token_stride, p.k_head = k_head_stride;
    p.Hq = Hq, p.Hk = Hk, p.D = D, p.rot = rotary_dim;
    p.table = table, p.P = table_rows, p.positions = positions;
    p.q_out = q_out, p.k_out = k_out;
    return rope_common(p, dtype, T, 1, layout, stream);
}

int ql_rope_append(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k, int64_t k_token_stride,
                   int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                   int64_t T, int Hq, int Hkv, int D, int rotary_dim, int layout, const float *table,
                   int64_t table_rows, const int64_t *positions, const int64_t *slots, void *k_cache, void *v_cache,
                   int64_t num_pages, int64_t page_stride, int page_size, void *q_out, void *stream) {
    g_err[0] = 0;
    if (Hkv <= 0) return fail(QL_EINVAL_SHAPE, "ql_rope_append: Hkv must be positive");
    if (!pow2(page_size)) return fail(QL_EUNSUPPORTED, "page size must be a power of two (got %d)", page_size);
    if (num_pages <= 0 || page_stride < (int64_t)Hkv * page_size * D)
        return fail(QL_EINVAL_SHAPE, "ql_rope_append: no pages, or a page stride below Hkv * page_size * D");
    if (T > 0 && (!v || !slots || !k_cache || !v_cache)) return fail(QL_EINVAL_ARG, "ql_rope_append: NULL pointer");
    ql::ropek::Params p{};
    p.q = q, p.q_token = q_token_stride, p.q_head = q_head_stride;
    p.k = k, p.k_token = k_token_stride, p.k_head = k_head_stride;
    p.v = v, p.v_token = v_token_stride, p.v_head = v_head_stride;
    p.Hq = Hq, p.Hk = Hkv, p.D = D, p.rot = rotary_dim;
    p.table = table, p.P = table_rows, p.positions = positions, p.slots = slots;
    p.q_out = q_out;
    p.k_cache = k_cache, p.v_cache = v_cache;
    p.page_stride = page_stride, p.num_slots = num_pages * page_size, p.page_shift = log2i(page_size);
    return rope_common(p, dtype, T, page_size, layout, stream);
}

static int64_t effective_window(int64_t window, int64_t max_kv) { return window <= 0 || window >= max_kv ? 0 : window; }

size_t ql_paged_attention_workspace_size(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv,
                                         int64_t window) {
    if (check_attention(T, Hq, Hkv, D, B, max_q, max_kv) || T == 0 || B == 0) return 0;
    return paged_attention_workspace(T, Hq, Hkv, D, B, max_q, max_kv, effective_window(window, max_kv));
}

static int attention(const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int Hq,
                     int Hkv, int D, const void *k_cache, const void *v_cache, int64_t num_pages,
                     int64_t page_stride, int page_size, const int32_t *page_table, int64_t table_stride,
                     const int32_t *q_starts, const int32_t *kv_lens, int64_t B, int64_t max_q, int64_t max_kv,
                     float scale, int causal, int64_t window, int64_t sinks, void *out, void *workspace,
                     size_t workspace_bytes, void *stream) {
    g_err[0] = 0;
    if (int rc = check_attention(T, Hq, Hkv, D, B, max_q, max_kv)) return rc;
    if (dtype != QL_BF16 && dtype != QL_F16) return fail(QL_EUNSUPPORTED, "ql_paged_attention: bf16 or f16");
    if (page_size < 16 || page_size > 1024 || !pow2(page_size))
        return fail(QL_EUNSUPPORTED, "page size must be a power of two in [16, 1024] (got %d)", page_size);
    if (num_pages <= 0 || num_pages > INT32_MAX || page_stride < (int64_t)Hkv * page_size * D || page_stride % 8)
        return fail(QL_EINVAL_SHAPE, "ql_paged_attention: no pages, or a page stride below Hkv * page_size * D or not a "
                                     "multiple of 8");
    if (table_stride < (max_kv + page_size - 1) / page_size)
        return fail(QL_EINVAL_SHAPE, "the page table's rows (%lld) hold fewer pages than max_kv=%lld needs",
                    (long long)table_stride, (long long)max_kv);
    if (!(scale > 0.f) || !isfinite(scale)) return fail(QL_EINVAL_ARG, "scale must be positive and finite");
    if (window < 0 || (window && !causal)) return fail(QL_EINVAL_ARG, "window must be >= 0, and needs causal");
    if (sinks < 0 || (sinks && !window)) return fail(QL_EINVAL_ARG, "sinks must be >= 0, and need a window");
    if (sinks > attn::MAX_SINKS) return fail(QL_EUNSUPPORTED, "at most %d sinks (got %lld)", attn::MAX_SINKS, (long long)sinks);
    if (T == 0 || B == 0) return QL_OK;
    if (!q || !k_cache || !v_cache || !page_table || !q_starts || !kv_lens || !out)
        return fail(QL_EINVAL_ARG, "ql_paged_attention: NULL pointer");
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned32(out) || q_token_stride % 8 ||
        q_head_stride % 8)
        return fail(QL_EINVAL_ARG, "q and the caches must be 16-byte aligned, out 32-byte, q's strides multiples of 8");
    window = effective_window(window, max_kv);
    const size_t need = paged_attention_workspace(T, Hq, Hkv, D, B, max_q, max_kv, window);
    if (need && (!workspace || workspace_bytes < need || !aligned32(workspace)))
        return fail(QL_EINVAL_ARG, "ql_paged_attention needs a 32-byte aligned workspace of %zu bytes (got %zu)", need,
                    workspace_bytes);
    ql::attn::Params p{};
    p.q = q, p.q_token = q_token_stride, p.q_head = q_head_stride, p.T = T;
    p.Hq = Hq, p.Hkv = Hkv, p.G = Hq / Hkv;
    p.k_cache = k_cache, p.v_cache = v_cache;
    p.page_stride = page_stride, p.num_pages = (int)num_pages, p.page_shift = log2i(page_size);
    p.table = page_table, p.table_stride = table_stride, p.q_starts = q_starts, p.kv_lens = kv_lens;
    p.max_q = (int)max_q, p.max_kv = (int)max_kv;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.causal = causal != 0, p.window = (int)window;
    p.sinks = window ? (int)sinks : 0;  // (a window that holds everything is none)
    p.out = out;
    return launch_paged_attention(p, dtype, D, B, workspace, (cudaStream_t)stream);
}

int ql_paged_attention(const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int Hq,
                       int Hkv, int D, const void *k_cache, const void *v_cache, int64_t num_pages,
                       int64_t page_stride, int page_size, const int32_t *page_table, int64_t table_stride,
                       const int32_t *q_starts, const int32_t *kv_lens, int64_t B, int64_t max_q, int64_t max_kv,
                       float scale, int causal, int64_t window, void *out, void *workspace, size_t workspace_bytes,
                       void *stream) {
    return attention(q, dtype, q_token_stride, q_head_stride, T, Hq, Hkv, D, k_cache, v_cache, num_pages, page_stride, page_size,
                     page_table, table_stride, q_starts, kv_lens, B, max_q, max_kv, scale, causal, window, 0, out, workspace,
                     workspace_bytes, stream);
}

int ql_sink_attention(const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int Hq,
                      int Hkv, int D, const void *k_cache, const void *v_cache, int64_t num_pages, int64_t page_stride,
                      int page_size, const int32_t *page_table, int64_t table_stride, const int32_t *q_starts,
                      const int32_t *kv_lens, int64_t B, int64_t max_q, int64_t max_kv, float scale, int64_t window,
                      int64_t sinks, void *out, void *workspace, size_t workspace_bytes, void *stream) {
    return attention(q, dtype, q_token_stride, q_head_stride, T, Hq, Hkv, D, k_cache, v_cache, num_pages, page_stride, page_size,
                     page_table, table_stride, q_starts, kv_lens, B, max_q, max_kv, scale, 1, window, sinks, out, workspace,
                     workspace_bytes, stream);
}

int ql_plan_step(int32_t *page_table, int64_t table_stride, int64_t table_width, const int32_t *lengths,
                 const int32_t *new_tokens, int64_t B, int page_size, int64_t max_tokens, const int32_t *free_pages,
                 int64_t num_free, const int32_t *taken, int64_t *positions, int64_t *slots, int32_t *q_starts,
                 int32_t *kv_lens, int32_t *taken_out, void *stream) {
    return ql_plan_step_within(page_table, table_stride, table_width, lengths, new_tokens, B, page_size, max_tokens, INT32_MAX,
                               free_pages, num_free, taken, positions, slots, q_starts, kv_lens, taken_out, stream);
}

int ql_plan_step_within(int32_t *page_table, int64_t table_stride, int64_t table_width, const int32_t *lengths,
                        const int32_t *new_tokens, int64_t B, int page_size, int64_t max_tokens, int64_t max_kv,
                        const int32_t *free_pages, int64_t num_free, const int32_t *taken, int64_t *positions,
                        int64_t *slots, int32_t *q_starts, int32_t *kv_lens, int32_t *taken_out, void *stream) {
    g_err[0] = 0;
    if (B < 0 || B > INT32_MAX - 1 || max_tokens < 0 || max_tokens > INT32_MAX || num_free < 0 || num_free > INT32_MAX ||
        max_kv < 0 || max_kv > INT32_MAX)
        return fail(QL_EINVAL_SHAPE, "ql_plan_step: bad sizes (B=%lld, max_tokens=%lld, max_kv=%lld, num_free=%lld)", (long long)B,
                    (long long)max_tokens, (long long)max_kv, (long long)num_free);
    if (!pow2(page_size)) return fail(QL_EUNSUPPORTED, "page size must be a power of two (got %d)", page_size);
    if (table_width < 0 || (B > 1 && table_stride < table_width))
        return fail(QL_EINVAL_SHAPE, "ql_plan_step: the page table's rows overlap (%lld entries, stride %lld)", (long long)table_width,
                    (long long)table_stride);
    if (B && (!lengths || !new_tokens || !kv_lens || (table_width && !page_table))) return fail(QL_EINVAL_ARG, "ql_plan_step: NULL pointer");
    if (!q_starts || (max_tokens && (!positions || !slots))) return fail(QL_EINVAL_ARG, "ql_plan_step: NULL pointer");
    if (free_pages && (!taken || !taken_out)) return fail(QL_EINVAL_ARG, "ql_plan_step: a free list needs taken and taken_out");
    const void *words[] = {page_table, lengths, new_tokens, free_pages, taken, q_starts, kv_lens, taken_out};
    for (const void *w : words)
        if (reinterpret_cast<uintptr_t>(w) % 4) return fail(QL_EINVAL_ARG, "ql_plan_step: pointer not aligned to its dtype");
    if (reinterpret_cast<uintptr_t>(positions) % 8 || reinterpret_cast<uintptr_t>(slots) % 8)
        return fail(QL_EINVAL_ARG, "ql_plan_step: pointer not aligned to its dtype");
    // What is written may not be read or written as something else: CTAs that still read would see it.  (In place is what
    // the kernel waits for: kv_lens over lengths, taken_out over taken.)
    struct Range {
        const void *at;
        int64_t bytes;
        bool written;
    };
    const Range all[] = {{lengths, 4 * B, false}, {new_tokens, 4 * B, false}, {free_pages, 4 * num_free, false}, {taken, free_pages ? 4 : 0, false},
                         {positions, 8 * max_tokens, true}, {slots, 8 * max_tokens, true}, {q_starts, 4 * (B + 1), true}, {kv_lens, 4 * B, true},
                         {taken_out, free_pages ? 4 : 0, true}};
    for (const Range &w : all) {
        if ((w.written || free_pages) && touches_rows(w.at, w.bytes, page_table, B, 4 * table_stride, 4 * table_width))
            return fail(QL_EINVAL_ARG, "ql_plan_step: the page table overlaps another argument");
        if (!w.written) continue;
        for (const Range &r : all) {
            const bool in_place = w.at == r.at && ((&w == &all[7] && &r == &all[0]) || (&w == &all[8] && &r == &all[3]));
            if (&r != &w && !in_place && touches_rows(r.at, r.bytes, w.at, 1, w.bytes, w.bytes))
                return fail(QL_EINVAL_ARG, "ql_plan_step: an output overlaps another argument");
        }
    }
    const ql::plank::Params p{page_table, table_stride, table_width, lengths, new_tokens, B, max_tokens, max_kv, log2i(page_size),
                              free_pages, num_free, taken, positions, slots, q_starts, kv_lens, taken_out};
    return launch_plan_step(p, (cudaStream_t)stream);
}

int ql_sample(const void *logits, int dtype, int64_t row_stride, int64_t B, int64_t V, const float *u,
              const float *temperature, double temperature_all, const int32_t *top_k, int64_t top_k_all,
              const float *top_p, double top_p_all, const float *min_p, double min_p_all, int64_t *tokens,
              float *logprobs, void *stream) {
    g_err[0] = 0;
    if (!valid_dtype(dtype)) return fail(QL_EUNSUPPORTED, "unknown dtype");
    if (B < 0 || V < 1 || row_stride < 0)
        return fail(QL_EINVAL_SHAPE, "ql_sample: bad sizes (B=%lld, V=%lld, row stride %lld)", (long long)B, (long long)V,
                    (long long)row_stride);
    if (V > samplek::MAX_ROW / elem_bytes(dtype))
        return fail(QL_EUNSUPPORTED, "ql_sample: a row of %lld logits is too long (at most %d bytes)", (long long)V, samplek::MAX_ROW);
    if ((!temperature && !(temperature_all >= 0.0)) || (!top_p && !(top_p_all >= 0.0)) || (!min_p && !(min_p_all >= 0.0 && min_p_all <= 1.0)) ||
        (!top_k && top_k_all < 0))
        return fail(QL_EINVAL_ARG, "ql_sample: temperature, top_k and top_p must not be negative, min_p in [0, 1]");
    if (B == 0) return QL_OK;
    if (!logits || !u || !tokens) return fail(QL_EINVAL_ARG, "ql_sample: NULL pointer");
    if (!elem_aligned(logits, dtype) || reinterpret_cast<uintptr_t>(tokens) % 8) return fail(QL_EINVAL_ARG, "ql_sample: pointer not aligned to its dtype");
    const void *words[] = {u, temperature, top_k, top_p, min_p, logprobs};
    for (const void *w : words)
        if (reinterpret_cast<uintptr_t>(w) % 4) return fail(QL_EINVAL_ARG, "ql_sample: pointer not aligned to its dtype");
    // weights are whole numbers up to 2^scale, sums of V of them fit 63 bits
    const int scale = 63 - log2i(V) < 46 ? 63 - log2i(V) : 46;
    const ql::samplek::Params p{logits, row_stride, (int)V, 0, scale, u, temperature, top_p, min_p, top_k,
                                temperature_all, top_p_all, min_p_all, top_k_all, tokens, logprobs};
    return launch_sample(p, dtype, B, (cudaStream_t)stream);
}

int ql_copy_pages(void *pool, int64_t planes, int64_t plane_stride, int64_t num_pages, int64_t page_stride,
                  int64_t page_bytes, const int32_t *src, const int32_t *dst, int64_t n, void *stream) {
    g_err[0] = 0;
    if (planes < 0 || num_pages < 0 || num_pages > INT32_MAX || n < 0 || page_bytes <= 0 || page_stride < page_bytes)
        return fail(QL_EINVAL_SHAPE, "ql_copy_pages: bad sizes");
    if (page_bytes % 16 || page_stride % 16 || plane_stride % 16)
        return fail(QL_EINVAL_SHAPE, "ql_copy_pages: the page's bytes and both strides must be multiples of 16");
    if (planes > 1 && num_pages > 0 && plane_stride < (num_pages - 1) * page_stride + page_bytes)
        return fail(QL_EINVAL_SHAPE, "ql_copy_pages: planes overlap");
    if (n == 0 || planes == 0) return QL_OK;
    if (!pool || !src || !dst) return fail(QL_EINVAL_ARG, "ql_copy_pages: NULL pointer");
    if (!aligned16(pool)) return fail(QL_EINVAL_ARG, "pool must be 16-byte aligned");
    // every index in range, no destination twice, no destination that is a source: the copies
    // are then independent of their order
    uint8_t *seen = static_cast<uint8_t *>(calloc((size_t)num_pages, 1));
    if (!seen) return fail(QL_EINVAL_ARG, "ql_copy_pages: out of host memory");
    int rc = QL_OK;
    for (int64_t i = 0; i < n && !rc; ++i) {
        if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
            rc = fail(QL_EINVAL_ARG, "ql_copy_pages: pair %lld (%d -> %d) is outside the %lld pages", (long long)i, src[i],
                      dst[i], (long long)num_pages);
        else if (seen[dst[i]]) rc = fail(QL_EINVAL_ARG, "ql_copy_pages: page %d is a destination twice", dst[i]);
        else seen[dst[i]] = 1;
    }
    for (int64_t i = 0; i < n && !rc; ++i)
        if (seen[src[i]]) rc = fail(QL_EINVAL_ARG, "ql_copy_pages: page %d is both source and destination", src[i]);
    free(seen);
    if (rc) return rc;
    return launch_copy_pages(pool, planes, plane_stride, page_stride, page_bytes, src, dst, n, (cudaStream_t)stream);
}

}  // extern "C"
