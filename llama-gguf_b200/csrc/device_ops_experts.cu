// device_ops_experts.cu — the C entries of the operators on device tensors for feed-forwards with 4-bit weights and routed experts (include/llama_b200.h, "operators on device tensors").
#include <cmath>

#include "dev_entry.cuh"
#include "dev_gated_norm.cuh"
#include "dev_glu_q8.cuh"
#include "dev_mat_i4.cuh"
#include "dev_route.cuh"

using namespace dev;

extern "C" int b200_dev_route_experts(const b200_route* a) {
    const char* op = "route_experts";
    return entry(op, [&]() -> int {
        if (!a) return bad(op, "null pointer");
        if (!type_bytes(a->type)) return bad_type(op, a->type);
        if (a->tokens < 0 || a->tokens >= kMost || a->n < 1 || a->n > ROUTE_MOST) return shape(op, "0 <= tokens < 2^31 and 1 to 1024 experts expected");
        if (a->groups < 1 || a->groups > ROUTE_GROUPS || a->n % a->groups) return shape(op, "groups must divide the experts, up to 32 of them");
        if (a->top_groups < 1 || a->top_groups > a->groups) return shape(op, "top_groups must be from 1 to groups");
        if (a->top < 1 || a->top > 32 || a->top > a->n / a->groups * a->top_groups) return shape(op, "top must be from 1 to 32 and to the experts of the chosen groups");
        if (a->ld < 0) return shape(op, "negative distance");
        if (!std::isfinite(a->scale)) return bad(op, "scale is not finite");
        if (a->tokens == 0) return B200_OK;
        if (!a->logits || !a->experts || !a->weights) return bad(op, "null pointer");
        const RouteArgs r{a->logits, a->correction, a->experts, a->weights, a->ld, a->tokens, a->n, a->top, a->groups, a->top_groups, a->sigmoid != 0, a->renormalise != 0, a->scale,
                          ((1u << 20) + a->n / a->groups - 1) / (a->n / a->groups)};
        return on_device(op, a->device, [&] { return by_type(a->type, [&](auto t) { return route_experts<decltype(t)>(r, (cudaStream_t)a->stream); }); });
    });
}

extern "C" int b200_dev_mat_mat_i4(const b200_i4_product* a) {
    const char* op = "mat_mat_i4";
    return entry(op, [&]() -> int {
        if (!a) return bad(op, "null pointer");
        if (!type_bytes(a->out_type)) return bad_type(op, a->out_type);
        if (!type_bytes(a->scale_type)) return bad_type(op, a->scale_type);
        if (a->group != 32 && a->group != 64 && a->group != 128) return dev_fail(B200_ERR_UNSUPPORTED, (std::string(op) + ": group must be 32, 64 or 128").c_str());
        if (a->tokens < 0 || a->n < 1 || a->n > kMostTiled || a->k < 1 || a->k > kMostTiled) return shape(op, "empty or oversized shape");
        if (a->k % a->group) return shape(op, "k must be a multiple of group");
        if (a->experts && (a->top < 1 || a->top > 32 || a->n_experts < 1 || a->n_experts > ROUTE_MOST)) return shape(op, "1 to 32 places of 1 to 1024 experts expected");
        if (!a->experts && a->tokens && (a->top || a->n_experts || a->rows_per_pair)) return bad(op, "top, n_experts or rows_per_pair without experts");
        if (a->tokens > kMostTiled / (a->experts ? a->top : 1)) return shape(op, "too many rows for one call");
        if (a->experts && a->n > (1 << 23)) return shape(op, "too many rows of weights for one call");      // (chunks times tiles are a 32-bit number)
        if (a->lda < a->k || a->ldo < a->n) return shape(op, "rows overlap");
        if (a->tokens == 0) return B200_OK;
        if (!a->a || !a->a_scales || !a->w || !a->w_scales || !a->out) return bad(op, "null pointer");
        if (off16(a->a) || off16(a->w) || a->lda % 16) return bad(op, "a and w must start on 16 bytes, with rows of a a multiple of 16 bytes apart");
        if (off16(a->w_scales)) return bad(op, "the scales must start on 16 bytes");
        MatI4Args m{};
        m.a = a->a;
        m.a_scales = a->a_scales;
        m.w = (const uint8_t*)a->w;
        m.ws = a->w_scales;
        m.bias = a->bias;
        m.experts = a->experts;
        m.out = a->out;
        m.status = a->status;
        m.lda = a->lda;
        m.ldo = a->ldo;
        m.rows = (int)(a->tokens * (a->experts ? a->top : 1));
        m.tokens = (int)a->tokens;
        m.k = (int)a->k;
        m.n = (int)a->n;
        m.div = a->experts && !a->rows_per_pair ? a->top : 1;
        m.n_experts = a->experts ? a->n_experts : 0;
        m.steps = (m.k + 63) / 64;
        m.groups = m.k / a->group;
        m.tiles = (m.n + 15) / 16;
        m.out_type = a->out_type;
        return on_device(op, a->device, [&] {
            return by_type(a->scale_type, [&](auto t) {
                using S = decltype(t);
                const cudaStream_t st = (cudaStream_t)a->stream;
                return a->group == 32 ? mat_mat_i4<S, 32>(m, st) : a->group == 64 ? mat_mat_i4<S, 64>(m, st) : mat_mat_i4<S, 128>(m, st);
            });
        });
    });
}

extern "C" int b200_dev_glu_q8(int device, void* stream, uint32_t type, int act, const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scales, int64_t rows, int64_t ff) {
    const char* op = "glu_q8";
    return entry(op, [&]() -> int {
        if (!type_bytes(type)) return bad_type(op, type);
        if (act < GLU_SILU || act > GLU_RELU) return bad(op, "unknown act");
        if (rows < 0 || rows >= kMost || ff < 1 || ff > 65536) return shape(op, "0 <= rows < 2^31 and 1 <= ff <= 65536 expected");
        if (ldx < 0 || ldq < ff) return shape(op, "negative distance, or rows of an output overlap");
        if (rows == 0) return B200_OK;
        if (!x || !q || !scales) return bad(op, "null pointer");
        const GluQ8Args a{x, q, scales, ldx, ldq, rows, (int)ff, act};
        return on_device(op, device, [&] { return by_type(type, [&](auto t) { return glu_q8<decltype(t)>(a, (cudaStream_t)stream); }); });
    });
}

extern "C" int b200_dev_add_gated_norm_q8(const b200_gated_norm* a) {
    const char* op = "add_gated_norm_q8";
    return entry(op, [&]() -> int {
        if (!a) return bad(op, "null pointer");
        if (!type_bytes(a->type)) return bad_type(op, a->type);
        if (a->rows < 0 || a->rows >= kMost || a->hidden < 1 || a->hidden > 65536) return shape(op, "0 <= rows < 2^31 and 1 <= hidden <= 65536 expected");
        if (a->mix && (a->top < 1 || a->top > 32)) return shape(op, "1 to 32 rows of y per row expected");
        if (a->ldy < 0 || a->ldr < 0 || a->gate_row < 0 || a->gate_col < 0 || a->lds < a->hidden || (a->weight && a->ldq < a->hidden)) return shape(op, "negative distance, or rows of an output overlap");
        if (!(a->eps >= 0.0f)) return bad(op, "eps must not be negative");
        if (!std::isfinite(a->scale)) return bad(op, "scale is not finite");
        if (a->rows == 0) return B200_OK;
        if (!a->y || !a->residual || !a->sum || (a->weight && (!a->q || !a->scales))) return bad(op, "null pointer");
        if (a->sum == a->residual && a->lds != a->ldr) return bad(op, "sum in place needs the same row distance");
        if (a->sum == a->y || (a->gate && a->sum == a->gate)) return bad(op, "sum must not be y or gate");
        const GatedNormArgs g{a->y, a->residual, a->gate, a->sum, a->mix, a->post_weight, a->weight, a->q, a->scales, a->ldy, a->ldr, a->lds, a->ldq, a->gate_row, a->gate_col, a->rows,
                              (int)a->hidden, a->mix ? a->top : 1, a->scale, a->eps, 1.0 / (double)a->hidden};
        return on_device(op, a->device, [&] { return by_type(a->type, [&](auto t) { return add_gated_norm<decltype(t)>(g, (cudaStream_t)a->stream); }); });
    });
}
