// device_ops.cu — the C entries of the operators on device tensors (include/llama_b200.h, "operators on device tensors"): argument checks and the choice
// among types (those of routed experts: device_ops_experts.cu).  Nothing is allocated here and nothing waits for the device.
#include <cmath>

#include "dev_entry.cuh"
#include "dev_gemm_i8.cuh"
#include "dev_norm_q8.cuh"
#include "dev_q4_attn.cuh"
#include "dev_q4_cache.cuh"
#include "dev_q4_prompt.cuh"

namespace {

using namespace dev;

int check_pages(const char* op, const b200_q4_pages& c) {
    if (!c.data) return bad(op, "null cache");
    if (off16(c.data)) return bad(op, "the cache must start on 16 bytes");
    if (c.head_dim != 64 && c.head_dim != 128) return dev_fail(B200_ERR_UNSUPPORTED, (std::string(op) + ": head_dim must be 64 or 128").c_str());
    if (c.page_size < 16 || c.page_size > 1024 || c.page_size % 16) return bad(op, "page_size must be a multiple of 16 up to 1024");
    if (c.n_kv_heads < 1 || c.n_kv_heads > 1024 || c.n_pages < 1 || c.n_pages >= kMost) return shape(op, "bad number of pages or kv heads");
    return B200_OK;
}

}  // namespace

extern "C" int b200_dev_watchdog(int device, int* out) {
    const char* op = "watchdog";
    return entry(op, [&]() -> int {
        if (!out) return bad(op, "null pointer");
        return on_device(op, device, [&] {
            const int zero = 0;
            cudaError_t e = cudaMemcpyFromSymbol(out, dev_watchdog, sizeof(int));
            if (e == cudaSuccess && *out) e = cudaMemcpyToSymbol(dev_watchdog, &zero, sizeof(int));
            return e;
        });
    });
}

extern "C" int b200_dev_add_rms_norm_q8(int device, void* stream, uint32_t type, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* sum, int64_t lds,
                                        const float* weight, float eps, int8_t* q, int64_t ldq, float* scales, int64_t rows, int64_t hidden) {
    const char* op = "add_rms_norm_q8";
    return entry(op, [&]() -> int {
        if (!type_bytes(type)) return bad_type(op, type);
        if (rows < 0 || rows >= kMost || hidden < 1 || hidden > 65536) return shape(op, "0 <= rows < 2^31 and 1 <= hidden <= 65536 expected");
        if (ldx < 0 || ldq < hidden || (residual && (ldr < 0 || lds < hidden))) return shape(op, "negative distance, or rows of an output overlap");
        if (!(eps >= 0.0f)) return bad(op, "eps must not be negative");
        if (rows == 0) return B200_OK;
        if (!x || !weight || !q || !scales || (residual && !sum)) return bad(op, "null pointer");
        if ((sum == x && lds != ldx) || (sum == residual && lds != ldr)) return bad(op, "sum in place needs the same row distance");
        NormQ8Args a{x, residual, residual ? sum : nullptr, weight, q, scales, ldx, ldr, lds, ldq, rows, (int)hidden, eps};
        return on_device(op, device, [&] { return by_type(type, [&](auto t) { return add_rms_norm_q8<decltype(t)>(a, (cudaStream_t)stream); }); });
    });
}

extern "C" int b200_dev_read_q8(int device, void* stream, uint32_t type, const int8_t* q, int64_t ldq, const float* scales, void* out, int64_t ldo, int64_t rows, int64_t n) {
    const char* op = "read_q8";
    return entry(op, [&]() -> int {
        if (!type_bytes(type)) return bad_type(op, type);
        if (rows < 0 || rows >= kMost || n < 1 || n >= kMost) return shape(op, "0 <= rows < 2^31 and 1 <= n < 2^31 expected");
        if (ldq < 0 || ldo < n) return shape(op, "negative distance, or rows of an output overlap");
        if (rows == 0) return B200_OK;
        if (!q || !scales || !out) return bad(op, "null pointer");
        const ReadQ8Args a{q, scales, out, ldq, ldo, rows, n};
        return on_device(op, device, [&] { return by_type(type, [&](auto t) { return read_q8<decltype(t)>(a, (cudaStream_t)stream); }); });
    });
}

extern "C" int b200_dev_mat_mat_i8(int device, void* stream, uint32_t out_type, const int8_t* a, int64_t lda, const float* a_scales, const int8_t* w, int64_t ldw,
                                   const float* w_scales, const float* bias, void* out, int64_t ldo, int64_t t_rows, int64_t k, int64_t n) {
    const char* op = "mat_mat_i8";
    return entry(op, [&]() -> int {
        if (!type_bytes(out_type)) return bad_type(op, out_type);
        if (t_rows < 0 || t_rows > kMostTiled || n < 1 || n > kMostTiled || k < 1) return shape(op, "empty or oversized shape");
        if (k > 131071) return shape(op, "k must be at most 131071 (32-bit sums)");
        if (lda < k || ldw < k || ldo < n) return shape(op, "rows overlap");
        if (t_rows == 0) return B200_OK;
        if (!a || !a_scales || !w || !w_scales || !out) return bad(op, "null pointer");
        if (off16(a) || off16(w) || lda % 16 || ldw % 16) return bad(op, "a and w must start on 16 bytes, with rows a multiple of 16 bytes apart");
        const GemmI8Args g{a_scales, w_scales, bias, out, ldo, (int)t_rows, (int)k, (int)n, 1};
        return on_device(op, device, [&] { return by_type(out_type, [&](auto t) { return gemm_i8<decltype(t)>(a, lda, w, ldw, g, (cudaStream_t)stream); }); });
    });
}

extern "C" int b200_debug_i8_plan(int64_t t, int64_t k, int64_t n, int* out4) {
    const char* op = "b200_debug_i8_plan";
    return entry(op, [&]() -> int {
        if (!out4 || t < 1 || t > kMostTiled || n < 1 || n > kMostTiled || k < 1 || k > 131071) return bad(op, "bad argument");
        const GemmI8Plan p = gemm_i8_plan(t, k, n);
        out4[0] = p.tn;
        out4[1] = p.splits;
        out4[2] = p.wide;
        out4[3] = p.pair;
        return B200_OK;
    });
}

extern "C" int b200_dev_rope_append_q4(const b200_q4_append* a) {
    const char* op = "rope_append_q4";
    return entry(op, [&]() -> int {
        if (!a) return bad(op, "null pointer");
        if (!type_bytes(a->type)) return bad_type(op, a->type);
        int rc = check_pages(op, a->cache);
        if (rc) return rc;
        if (a->rot_dims < 2 || a->rot_dims > a->cache.head_dim || a->rot_dims % 2) return shape(op, "rot_dims must be even, from 2 to head_dim");
        if (a->tokens < 0 || a->table_rows < 1) return shape(op, "bad number of tokens or table rows");
        if (a->q && (a->n_heads < 1 || a->n_heads > 65536)) return shape(op, "bad number of query heads");
        if (a->tokens * ((a->q ? a->n_heads : 0) + 2LL * a->cache.n_kv_heads) >= kMost || a->tokens >= kMost) return shape(op, "too many rows for one call");
        if (a->q && overlap(a->tokens, a->q_out_token, a->n_heads, a->q_out_head, a->cache.head_dim)) return shape(op, "rows of q_out overlap");
        if (a->tokens == 0) return B200_OK;
        if (!a->k || !a->v || !a->cos_sin || !a->positions || !a->slots || (a->q && !a->q_out)) return bad(op, "null pointer");
        if (a->q && a->q == a->q_out && (a->q_token != a->q_out_token || a->q_head != a->q_out_head)) return bad(op, "q in place needs the same strides");
        const int e = 16 / type_bytes(a->type);
        bool vec = !off16(a->k) && !off16(a->v) && a->k_token % e == 0 && a->k_head % e == 0 && a->v_token % e == 0 && a->v_head % e == 0 && a->rot_dims % 16 == 0 && !off16(a->cos_sin);
        if (a->q) vec = vec && !off16(a->q) && !off16(a->q_out) && a->q_token % e == 0 && a->q_head % e == 0 && a->q_out_token % e == 0 && a->q_out_head % e == 0;
        return on_device(op, a->device, [&] {
            return by_type(a->type, [&](auto t) {
                using T = decltype(t);
                return a->cache.head_dim == 64 ? rope_append_q4<T, 64>(*a, vec, (cudaStream_t)a->stream) : rope_append_q4<T, 128>(*a, vec, (cudaStream_t)a->stream);
            });
        });
    });
}

extern "C" int b200_dev_read_q4(int device, void* stream, uint32_t type, const b200_q4_pages* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out, int32_t* status) {
    const char* op = "read_q4";
    return entry(op, [&]() -> int {
        if (!cache) return bad(op, "null pointer");
        if (!type_bytes(type)) return bad_type(op, type);
        int rc = check_pages(op, *cache);
        if (rc) return rc;
        if (tokens < 0 || tokens >= kMost || tokens * 2 * cache->n_kv_heads >= kMost) return shape(op, "too many rows for one call");
        if (tokens == 0 || (!k_out && !v_out)) return B200_OK;
        if (!slots) return bad(op, "null pointer");
        if (off16(k_out) || off16(v_out)) return bad(op, "the outputs must start on 16 bytes");
        const ReadQ4Args a{*cache, slots, tokens, k_out, v_out, status};
        return on_device(op, device, [&] {
            return by_type(type, [&](auto t) {
                using T = decltype(t);
                return cache->head_dim == 64 ? read_q4<T, 64>(a, (cudaStream_t)stream) : read_q4<T, 128>(a, (cudaStream_t)stream);
            });
        });
    });
}

static int check_attention(const char* op, const b200_q4_attention* a) {
    if (!a) return bad(op, "null pointer");
    if (!type_bytes(a->type)) return bad_type(op, a->type);
    int rc = check_pages(op, a->cache);
    if (rc) return rc;
    if (a->n_heads < 1 || a->n_heads > 65536 || a->n_heads % a->cache.n_kv_heads) return shape(op, "the query heads must be a multiple of the kv heads");
    if (a->seqs < 0 || a->tokens < 0 || a->table_pages < 0 || a->table_stride < 0 || a->max_q < 0) return shape(op, "negative size");
    if (a->tokens * a->n_heads >= kMost || a->tokens >= kMost || (int64_t)a->table_pages * a->cache.page_size > kMostTiled) return shape(op, "too many rows or positions for one call");
    if (!a->q_starts && a->tokens != a->seqs) return shape(op, "without q_starts every sequence has one token");
    if (a->window < 0) return bad(op, "window must not be negative");
    if (!std::isfinite(a->scale)) return bad(op, "scale is not finite");
    return B200_OK;
}

extern "C" int b200_dev_attention_paged_q4_workspace(const b200_q4_attention* a, size_t* bytes) {
    const char* op = "attention_paged_q4";
    return entry(op, [&]() -> int {
        int rc = check_attention(op, a);
        if (rc) return rc;
        if (!bytes) return bad(op, "null pointer");
        *bytes = attention_q4_workspace(*a);
        return B200_OK;
    });
}

extern "C" int b200_debug_q4_prompt_blocks(const b200_q4_attention* a, int64_t* blocks) {
    const char* op = "b200_debug_q4_prompt_blocks";
    return entry(op, [&]() -> int {
        int rc = check_attention(op, a);
        if (rc) return rc;
        if (!blocks) return bad(op, "null pointer");
        *blocks = attention_q4_has_prompts(*a) ? attention_q4_prompt_blocks(*a) * a->cache.n_kv_heads : 0;
        return B200_OK;
    });
}

extern "C" int b200_dev_attention_paged_q4(const b200_q4_attention* a) {
    const char* op = "attention_paged_q4";
    return entry(op, [&]() -> int {
        int rc = check_attention(op, a);
        if (rc) return rc;
        if (overlap(a->tokens, a->out_token, a->n_heads, a->out_head, a->cache.head_dim)) return shape(op, "rows of out overlap");
        if (a->tokens == 0 || a->seqs == 0) return B200_OK;
        if (!a->q || !a->out || !a->kv_lens || (a->table_pages > 0 && !a->page_table)) return bad(op, "null pointer");
        const size_t need = attention_q4_workspace(*a);
        if (need && (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255) || a->workspace_bytes < need)) return bad(op, "workspace missing, too small or not on 256 bytes");
        return on_device(op, a->device, [&] {
            return by_type(a->type, [&](auto t) {
                using T = decltype(t);
                return a->cache.head_dim == 64 ? attention_q4<T, 64>(*a, (cudaStream_t)a->stream) : attention_q4<T, 128>(*a, (cudaStream_t)a->stream);
            });
        });
    });
}
