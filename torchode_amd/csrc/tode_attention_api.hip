// C entries of cross attention: what the kernels assume of sizes and pointers is checked here.
#include "tode_attention.h"

namespace tode {

static int check(const tode_cross_attention_args *a, bool backward) {
    if (!a) return fail(TODE_E_INVALID, "null argument struct");
    if (a->dtype != TODE_F32 && a->dtype != TODE_BF16 && a->dtype != TODE_F16) return fail(TODE_E_UNSUPPORTED, "cross attention is built for float32, bfloat16 and float16 (dtype %d)", a->dtype);
    if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads || a->head_dim < 1)
        return fail(TODE_E_INVALID, "bad sizes: batch=%lld queries=%lld keys=%lld heads=%d kv_heads=%d head_dim=%d", (long long)a->batch, (long long)a->queries, (long long)a->keys, a->heads,
                    a->kv_heads, a->head_dim);
    const int most = a->dtype == TODE_F32 ? TODE_ATTENTION_MAX_HEAD_DIM_F32 : TODE_ATTENTION_MAX_HEAD_DIM;
    if (a->head_dim > most) return fail(TODE_E_UNSUPPORTED, "head_dim %d, at most %d", a->head_dim, most);
    // rows and keys are counted in 32 bits, workgroups too
    const long long limit = 1ll << 30, share = a->heads / a->kv_heads;
    if (a->heads > 65536 || a->batch > limit || a->queries > limit / share || a->keys > limit) return fail(TODE_E_UNSUPPORTED, "sizes beyond 2^30");
    const long long groups = a->batch * a->kv_heads + 7;
    if (groups > limit || (a->queries * share + 31) / 32 > limit / groups || (a->keys + 31) / 32 > limit / groups || a->batch * a->queries > (limit * 64) / a->heads)
        return fail(TODE_E_UNSUPPORTED, "more than 2^30 tiles");
    // (a row's place in a tile is a 32-bit number where its stride is below 2^24, which one of less than -2^31 would be too)
    for (int i = 0; i < 3; ++i)
        if (a->q_strides[i] < 0 || a->k_strides[i] < 0 || a->v_strides[i] < 0 || (backward && a->grad_strides[i] < 0)) return fail(TODE_E_INVALID, "strides must not be negative");
    if (a->mask_stride < 0) return fail(TODE_E_INVALID, "strides must not be negative");
    if (!(a->scale - a->scale == 0)) return fail(TODE_E_INVALID, "scale must be finite");
    return TODE_OK;
}

}  // namespace tode

extern "C" {

using namespace tode;

int64_t tode_cross_attention_workspace_bytes(const tode_cross_attention_args *a, int32_t backward) {
    if (int rc = check(a, backward != 0)) return rc;
    if (a->batch == 0) return 0;
    switch (a->dtype) {
        case TODE_F32: return backward ? attention_backward_bytes_float(*a) : attention_forward_bytes_float(*a);
        case TODE_BF16: return backward ? attention_backward_bytes_bf16(*a) : attention_forward_bytes_bf16(*a);
        default: return backward ? attention_backward_bytes_f16(*a) : attention_forward_bytes_f16(*a);
    }
}

static int ready(const tode_cross_attention_args *a, int backward) {
    if (int rc = check(a, backward != 0)) return rc;
    if (a->batch == 0) return TODE_OK;
    if (a->queries > 0 && (!a->q || !a->out)) return fail(TODE_E_INVALID, "null pointer");
    if (a->keys > 0 && (!a->k || !a->v)) return fail(TODE_E_INVALID, "null pointer");
    if (backward && a->queries > 0 && (!a->grad_out || !a->lse)) return fail(TODE_E_INVALID, "null pointer");
    if (!a->dk != !a->dv) return fail(TODE_E_INVALID, "dk and dv are computed together");
    const int64_t need = tode_cross_attention_workspace_bytes(a, backward);
    if (a->workspace_bytes < need || (need > 0 && !a->workspace)) return fail(TODE_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)a->workspace_bytes, (long long)need);
    return TODE_OK;
}

int tode_cross_attention(const tode_cross_attention_args *a, void *stream) {
    if (int rc = ready(a, 0)) return rc;
    if (a->batch == 0 || a->queries == 0) return TODE_OK;
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == TODE_F32 ? attention_forward_float(*a, s) : a->dtype == TODE_BF16 ? attention_forward_bf16(*a, s) : attention_forward_f16(*a, s);
}

int tode_cross_attention_backward(const tode_cross_attention_args *a, void *stream) {
    if (int rc = ready(a, 1)) return rc;
    if (a->batch == 0) return TODE_OK;
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == TODE_F32 ? attention_backward_float(*a, s) : a->dtype == TODE_BF16 ? attention_backward_bf16(*a, s) : attention_backward_f16(*a, s);
}

}  // extern "C"
