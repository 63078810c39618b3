// Entry points of the ragged cross attention (attention.h: formulas): the checks of their arguments, and of the offsets on the device.
#include <cmath>

#include "attention.h"
#include "ops.h"

namespace dctr {

__global__ void attn_check_kernel(AttnView a, int32_t* status) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < a.n_seg) flag_segment(a, b, status);
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
static int check_attention(const dctr_attention* a) {
    DCTR_REQUIRE(a != nullptr, "null attention description");
    DCTR_REQUIRE(a->dtype == DCTR_TYPE_F32 || a->dtype == DCTR_TYPE_BF16, "attention: unknown element type %d", a->dtype);
    DCTR_REQUIRE(a->n_seg <= 1 << 26, "attention: %d segments (at most 2^26)", a->n_seg);       // (products of sizes stay within 64 bits)
    DCTR_REQUIRE(a->n_seg >= 0 && a->max_q >= 0 && a->max_k >= 0 && a->total_q >= 0 && a->total_k >= 0, "attention: negative size");
    DCTR_REQUIRE(a->total_q <= INT32_MAX && a->total_k <= INT32_MAX, "attention: more rows than int32 offsets reach");
    DCTR_REQUIRE(a->max_q <= DCTR_MAX_POSITION && a->max_k <= DCTR_MAX_POSITION, "attention: segments of %d x %d rows (at most %d)", a->max_q, a->max_k,
                 DCTR_MAX_POSITION);                                    // (so that differences of positions and boundaries stay within 32 bits)
    DCTR_REQUIRE(a->heads >= 1 && a->heads <= 1024 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0,
                 "attention: %d heads (1..1024) over %d key heads (must divide them)", a->heads, a->kv_heads);
    DCTR_REQUIRE(a->head_dim >= 8 && a->head_dim <= 128 && a->head_dim % 8 == 0, "attention: head_dim %d (a multiple of 8, 8..128)", a->head_dim);
    DCTR_REQUIRE(std::isfinite(a->scale), "attention: scale is not finite");
    DCTR_REQUIRE(a->n_buckets >= 0 && a->n_buckets <= DCTR_MAX_REL_BUCKETS, "attention: %d buckets (0..%d)", a->n_buckets, DCTR_MAX_REL_BUCKETS);
    for (int u = 0; u + 1 < a->n_buckets; ++u) {
        DCTR_REQUIRE(a->boundaries[u] >= -DCTR_MAX_POSITION && a->boundaries[u] <= DCTR_MAX_POSITION, "attention: boundary %d out of range", a->boundaries[u]);
        DCTR_REQUIRE(u == 0 || a->boundaries[u] > a->boundaries[u - 1], "attention: boundaries must ascend (%d after %d)", a->boundaries[u],
                     a->boundaries[u - 1]);
    }
    if (a->n_buckets > 1)
        DCTR_REQUIRE(a->boundaries[a->n_buckets - 2] - a->boundaries[0] <= DCTR_MAX_REL_SPAN, "attention: boundaries span %d (at most %d)",
                     a->boundaries[a->n_buckets - 2] - a->boundaries[0], DCTR_MAX_REL_SPAN);
    return DCTR_OK;
}

// rows of `heads` heads: 16-byte aligned, wide enough
static int check_rows(const dctr_attention* a, const char* what, const void* p, int64_t ld, int heads, int elem, int64_t rows) {
    if (rows == 0) return DCTR_OK;
    DCTR_REQUIRE(p != nullptr, "attention: %s is null", what);
    DCTR_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * elem) % 16 == 0, "attention: rows of %s must be 16-byte aligned", what);
    DCTR_REQUIRE(ld >= (int64_t)heads * a->head_dim, "attention: row stride %lld of %s is below %d", (long long)ld, what, heads * a->head_dim);
    return DCTR_OK;
}

static int make_view(const dctr_attention* a, const void* q, int q_ld, const void* k, int k_ld, const void* v, int v_ld, const int32_t* q_off,
                     const int32_t* k_off, const int32_t* q_start, const uint8_t* keep, const float* bias, AttnView* view) {
    DCTR_TRY(check_attention(a));
    const int elem = a->dtype == DCTR_TYPE_F32 ? 4 : 2;
    DCTR_TRY(check_rows(a, "q", q, q_ld, a->heads, elem, a->total_q));
    DCTR_TRY(check_rows(a, "k", k, k_ld, a->kv_heads, elem, a->total_k));
    DCTR_TRY(check_rows(a, "v", v, v_ld, a->kv_heads, elem, a->total_k));
    if (a->n_seg > 0) DCTR_REQUIRE(q_off != nullptr && k_off != nullptr, "attention: null offsets");
    DCTR_REQUIRE((a->n_buckets > 0) == (bias != nullptr), "attention: d_rel_bias goes with n_buckets > 0");
    *view = AttnView{q, k, v, q_ld, k_ld, v_ld, q_off, k_off, q_start, keep, bias, a->total_q, a->total_k, a->n_seg, a->heads,
                     a->heads / a->kv_heads, a->head_dim, a->max_q, a->max_k, a->causal != 0, a->scale, {}};
    view->rel.n = a->n_buckets;
    for (int u = 0; u < DCTR_MAX_REL_BUCKETS; ++u) view->rel.edge[u] = u + 1 < a->n_buckets ? a->boundaries[u] : INT32_MAX;
    return DCTR_OK;
}

// Every launch of a call, before the first one.
static int check_launches(const dctr_attention* a, int backward) {
    const int64_t blocks = std::max(attn_fwd_blocks(a), backward ? attn_bwd_blocks(a) : 0);
    DCTR_REQUIRE(blocks <= MAX_BLOCKS, "attention: %lld blocks in one launch (at most %lld): too many segments, heads or rows a segment", (long long)blocks,
                 (long long)MAX_BLOCKS);
    return DCTR_OK;
}

static int64_t workspace_bytes(const dctr_attention* a, int backward) {
    return std::max(attn_fwd_workspace(a), backward ? attn_bwd_workspace(a) : 0);
}

static int check_workspace(const dctr_attention* a, int backward, const void* ws, size_t bytes) {
    DCTR_TRY(check_launches(a, backward));
    const int64_t need = workspace_bytes(a, backward);
    DCTR_REQUIRE(need == 0 || (ws != nullptr && (int64_t)bytes >= need), "attention: workspace of %lld bytes needed, %lld given", (long long)need,
                 ws != nullptr ? (long long)bytes : 0ll);
    DCTR_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "attention: workspace must be 16-byte aligned");
    return DCTR_OK;
}

}  // namespace dctr

using namespace dctr;

extern "C" {

int dctr_cross_attention_workspace_bytes(const dctr_attention* a, int backward, int64_t* bytes) {
    DCTR_REQUIRE(bytes != nullptr, "null out pointer");
    DCTR_TRY(check_attention(a));
    DCTR_TRY(check_launches(a, backward));
    *bytes = workspace_bytes(a, backward);
    return DCTR_OK;
}

int dctr_cross_attention_fwd(const dctr_attention* a, const void* d_q, int q_ld, const void* d_k, int k_ld, const void* d_v, int v_ld,
                             const int32_t* d_q_offsets, const int32_t* d_k_offsets, const int32_t* d_q_start, const uint8_t* d_key_keep,
                             const float* d_rel_bias, void* d_out, int out_ld, float* d_lse, int32_t* d_status,
                             void* d_workspace, size_t workspace_bytes, void* stream) {
    AttnView v;
    DCTR_TRY(make_view(a, d_q, q_ld, d_k, k_ld, d_v, v_ld, d_q_offsets, d_k_offsets, d_q_start, d_key_keep, d_rel_bias, &v));
    const bool f32 = a->dtype == DCTR_TYPE_F32;
    DCTR_TRY(check_rows(a, "out", d_out, out_ld, a->heads, f32 ? 4 : 2, a->total_q));
    DCTR_TRY(check_workspace(a, 0, d_workspace, workspace_bytes));
    hipStream_t st = as_stream(stream);
    if (a->n_seg == 0) return DCTR_OK;
    const bool none = a->total_q == 0 || a->max_q == 0;                  // (otherwise the forward's blocks look at their segments)
    if (none && d_status != nullptr) {
        attn_check_kernel<<<ceil_div(a->n_seg, 256), 256, 0, st>>>(v, d_status);
        DCTR_LAUNCH_CHECK();
    }
    return none ? DCTR_OK : attn_fwd(a, v, d_out, out_ld, d_lse, d_status, (float*)d_workspace, st);
}

int dctr_cross_attention_bwd(const dctr_attention* a, const void* d_q, int q_ld, const void* d_k, int k_ld, const void* d_v, int v_ld,
                             const int32_t* d_q_offsets, const int32_t* d_k_offsets, const int32_t* d_q_start, const uint8_t* d_key_keep,
                             const float* d_rel_bias, const void* d_out, int out_ld, const float* d_lse, const void* d_dout, int dout_ld,
                             void* d_dq, int dq_ld, void* d_dk, int dk_ld, void* d_dv, int dv_ld, float* d_drel_bias, void* d_workspace,
                             size_t workspace_bytes, void* stream) {
    AttnView v;
    DCTR_TRY(make_view(a, d_q, q_ld, d_k, k_ld, d_v, v_ld, d_q_offsets, d_k_offsets, d_q_start, d_key_keep, d_rel_bias, &v));
    const int elem = a->dtype == DCTR_TYPE_F32 ? 4 : 2;
    DCTR_TRY(check_rows(a, "out", d_out, out_ld, a->heads, elem, a->total_q));
    DCTR_TRY(check_rows(a, "dout", d_dout, dout_ld, a->heads, elem, a->total_q));
    DCTR_TRY(check_rows(a, "dq", d_dq, dq_ld, a->heads, elem, a->total_q));
    DCTR_TRY(check_rows(a, "dk", d_dk, dk_ld, a->kv_heads, elem, a->total_k));
    DCTR_TRY(check_rows(a, "dv", d_dv, dv_ld, a->kv_heads, elem, a->total_k));
    DCTR_REQUIRE(a->total_q == 0 || d_lse != nullptr, "attention: lse is null");
    DCTR_REQUIRE(d_drel_bias == nullptr || a->n_buckets > 0, "attention: a bias gradient without a bias");
    DCTR_TRY(check_workspace(a, 1, d_workspace, workspace_bytes));
    hipStream_t st = as_stream(stream);
    if (a->n_buckets > 0 && d_drel_bias != nullptr && (a->n_seg == 0 || a->total_q == 0 || a->max_q == 0)) {
        DCTR_TRY(zero_words(d_drel_bias, (size_t)a->n_buckets * a->heads, st));
        d_drel_bias = nullptr;
    }
    if (a->n_seg == 0) return DCTR_OK;
    return attn_bwd(a, v, AttnGrads{d_out, out_ld, d_lse, d_dout, dout_ld, d_dq, dq_ld, d_dk, dk_ld, d_dv, dv_ld, d_drel_bias}, (float*)d_workspace, st);
}

}  // extern "C"
