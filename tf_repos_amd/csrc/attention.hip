// Entry points of the ragged cross attention (attention.h holds the formulas) and its kernels: one wave per (query row, head) forward and
// for dq / the bias gradient, one per (key row, key head) for dk and dv.  64 keys (queries) at a time: each lane first takes one pair's
// scores, then the lanes share the head's columns for the weighted sums.
#include <cmath>

#include "attention.h"

namespace dctr {

constexpr int WAVES = 4;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

template <typename T>
__device__ __forceinline__ float row_dot(const T* a, const T* b, int dim) {
    float s = 0.f;
    for (int d = 0; d < dim; ++d) s = fmaf(to_f32(a[d]), to_f32(b[d]), s);
    return s;
}

__device__ __forceinline__ bool key_seen(const AttnView& a, const Segment& s, int i, int j) {
    return j < s.nk && (a.keep == nullptr || a.keep[s.k0 + j] != 0) && (!a.causal || j <= s.start + i);
}

template <typename T>
__device__ __forceinline__ float score(const AttnView& a, const Segment& s, const T* qi, const T* kj, int i, int j, int h) {
    const float z = a.scale * row_dot(qi, kj, a.dim);
    return a.rel.n > 0 ? z + a.bias[bucket_of(a.rel, j - s.start - i) * a.heads + h] : z;
}

__global__ void attn_check_kernel(AttnView a, int32_t* status) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < a.n_seg && segment_is_bad(a, b)) { status[0] = 1; status[1] = b; }
}

// dq, and this row's share of the bias gradient: part[(q0 + i), h, bucket]
template <typename T>
__global__ __launch_bounds__(64 * WAVES) void attn_bwd_q_kernel(AttnView a, const float* lse, const T* dout, int64_t dout_ld, T* dq, int64_t dq_ld, float* part) {
    const int64_t item = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, h = (int)(item % a.heads);
    const int64_t r = item / a.heads;
    const int i = (int)(r % a.max_q), b = (int)(r / a.max_q);
    if (b >= a.n_seg) return;
    const Segment s = load_segment(a, b);
    if (i >= s.nq) return;
    const int64_t row = s.q0 + i, hd = (int64_t)h * a.dim, gd = (int64_t)(h / a.group) * a.dim;
    const T* qi = (const T*)a.q + row * a.q_ld + hd;
    const T* doi = dout + row * dout_ld + hd;
    const T* K = (const T*)a.k + s.k0 * a.k_ld + gd;
    const T* V = (const T*)a.v + s.k0 * a.v_ld + gd;
    const float L = lse[row * a.heads + h];
    // <do_i, o_i> = sum_j p_ij <do_i, v_j>, taken from the unrounded p: the bias gradient is f32 whatever out was rounded to
    float delta = 0.f;
    if (L != -INFINITY)
        for (int j = lane; j < s.nk; j += 64)
            if (key_seen(a, s, i, j)) delta = fmaf(expf(score(a, s, qi, K + j * a.k_ld, i, j, h) - L), row_dot(doi, V + j * a.v_ld, a.dim), delta);
    delta = wave_sum(delta);
    float acc0 = 0.f, acc1 = 0.f, bin0 = 0.f, bin1 = 0.f;
    for (int j0 = 0; j0 < s.nk; j0 += 64) {
        const int j = j0 + lane;
        const bool on = L != -INFINITY && key_seen(a, s, i, j);
        float ds = 0.f;
        if (on) ds = expf(score(a, s, qi, K + j * a.k_ld, i, j, h) - L) * (row_dot(doi, V + j * a.v_ld, a.dim) - delta);
        const int bin = a.rel.n > 0 ? bucket_of(a.rel, j - s.start - i) : 0;
        const uint64_t seen = __ballot(on);
        for (int t = 0; t < 64; ++t) {
            const float w = __shfl(ds, t);
            const int u = __shfl(bin, t);
            if (!(seen >> t & 1)) continue;
            const T* k = K + (j0 + t) * a.k_ld;
            if (lane < a.dim) acc0 = fmaf(w, to_f32(k[lane]), acc0);
            if (64 + lane < a.dim) acc1 = fmaf(w, to_f32(k[64 + lane]), acc1);
            if (u == lane) bin0 += w;
            if (u == 64 + lane) bin1 += w;
        }
    }
    for (int d = lane; d < a.dim; d += 64) dq[row * dq_ld + hd + d] = (T)((d < 64 ? acc0 : acc1) * a.scale);
    if (part != nullptr)
        for (int u = lane; u < a.rel.n; u += 64) part[(row * a.heads + h) * a.rel.n + u] = u < 64 ? bin0 : bin1;
}

// one block per (bucket, head): the rows' shares in a fixed order
__global__ __launch_bounds__(256) void attn_bias_grad_kernel(AttnView a, const float* part, float* dbias) {
    const int u = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
    float sum = 0.f;
    for (int b = 0; b < a.n_seg; ++b) {
        const Segment s = load_segment(a, b);
        for (int i = threadIdx.x; i < s.nq; i += 256) sum += part[((s.q0 + i) * a.heads + h) * a.rel.n + u];
    }
    __shared__ float red[WAVES];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) dbias[u * a.heads + h] = red[0] + red[1] + red[2] + red[3];
}

// item = (segment, key row j < max_k, key head): the sums run over the queries of every head that reads it
template <typename T>
__global__ __launch_bounds__(64 * WAVES) void attn_bwd_kv_kernel(AttnView a, const T* out, int64_t out_ld, const float* lse, const T* dout,
                                                                 int64_t dout_ld, T* dk, int64_t dk_ld, T* dv, int64_t dv_ld) {
    const int64_t item = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    const int kv_heads = a.heads / a.group;
    const int lane = threadIdx.x & 63, g = (int)(item % kv_heads);
    const int64_t r = item / kv_heads;
    const int j = (int)(r % a.max_k), b = (int)(r / a.max_k);
    if (b >= a.n_seg) return;
    const Segment s = load_segment(a, b);
    if (j >= s.nk) return;
    const int64_t row = s.k0 + j, gd = (int64_t)g * a.dim;
    const T* kj = (const T*)a.k + row * a.k_ld + gd;
    const T* vj = (const T*)a.v + row * a.v_ld + gd;
    float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
    for (int h = g * a.group; h < (g + 1) * a.group; ++h) {
        const int64_t hd = (int64_t)h * a.dim;
        const T* Q = (const T*)a.q + s.q0 * a.q_ld + hd;
        const T* DO = dout + s.q0 * dout_ld + hd;
        for (int i0 = 0; i0 < s.nq; i0 += 64) {
            const int i = i0 + lane;
            float p = 0.f, ds = 0.f;
            bool on = i < s.nq && key_seen(a, s, i, j);
            if (on) {
                const float L = lse[(s.q0 + i) * a.heads + h];
                on = L != -INFINITY;
                if (on) {
                    float delta = 0.f, dp = 0.f;
                    for (int d = 0; d < a.dim; ++d) {
                        const float go = to_f32(DO[i * dout_ld + d]);
                        delta = fmaf(go, to_f32(out[(s.q0 + i) * out_ld + hd + d]), delta);
                        dp = fmaf(go, to_f32(vj[d]), dp);
                    }
                    p = expf(score(a, s, Q + i * a.q_ld, kj, i, j, h) - L);
                    ds = p * (dp - delta);
                }
            }
            const uint64_t seen = __ballot(on);
            for (int t = 0; t < 64; ++t) {
                const float pw = __shfl(p, t), dw = __shfl(ds, t);
                if (!(seen >> t & 1)) continue;
                const T *q = Q + (i0 + t) * a.q_ld, *go = DO + (i0 + t) * dout_ld;
                if (lane < a.dim) { k0 = fmaf(dw, to_f32(q[lane]), k0); v0 = fmaf(pw, to_f32(go[lane]), v0); }
                if (64 + lane < a.dim) { k1 = fmaf(dw, to_f32(q[64 + lane]), k1); v1 = fmaf(pw, to_f32(go[64 + lane]), v1); }
            }
        }
    }
    for (int d = lane; d < a.dim; d += 64) {
        dk[row * dk_ld + gd + d] = (T)((d < 64 ? k0 : k1) * a.scale);
        dv[row * dv_ld + gd + d] = (T)(d < 64 ? v0 : v1);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
static int check_attention(const dctr_attention* a) {
    DCTR_REQUIRE(a != nullptr, "null attention description");
    DCTR_REQUIRE(a->dtype == DCTR_TYPE_F32 || a->dtype == DCTR_TYPE_BF16, "attention: unknown element type %d", a->dtype);
    DCTR_REQUIRE(a->n_seg >= 0 && a->max_q >= 0 && a->max_k >= 0 && a->total_q >= 0 && a->total_k >= 0, "attention: negative size");
    DCTR_REQUIRE(a->total_q <= INT32_MAX && a->total_k <= INT32_MAX, "attention: more rows than int32 offsets reach");
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
    for (int u = 0; u + 1 < a->n_buckets; ++u) view->rel.edge[u] = a->boundaries[u];
    return DCTR_OK;
}

static int64_t workspace_bytes(const dctr_attention* a, int backward) {
    return backward ? 4 * a->total_q * a->heads * (int64_t)a->n_buckets : attn_fwd_workspace(a);
}

static int check_workspace(const dctr_attention* a, int backward, const void* ws, size_t bytes) {
    const int64_t need = workspace_bytes(a, backward);
    DCTR_REQUIRE(need == 0 || (ws != nullptr && (int64_t)bytes >= need), "attention: workspace of %lld bytes needed, %lld given", (long long)need,
                 ws != nullptr ? (long long)bytes : 0ll);
    DCTR_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "attention: workspace must be 16-byte aligned");
    return DCTR_OK;
}

static int grid_of(int64_t blocks, unsigned* grid) {
    DCTR_REQUIRE(blocks <= INT32_MAX, "attention: too many rows for one launch");
    *grid = (unsigned)blocks;
    return DCTR_OK;
}

template <typename T>
static int run_bwd(const AttnView& a, const void* out, int64_t out_ld, const float* lse, const void* dout, int64_t dout_ld, void* dq, int64_t dq_ld,
                   void* dk, int64_t dk_ld, void* dv, int64_t dv_ld, float* dbias, float* part, hipStream_t st) {
    unsigned grid;
    DCTR_TRY(grid_of(((int64_t)a.n_seg * a.max_q * a.heads + WAVES - 1) / WAVES, &grid));
    if (grid > 0) {
        attn_bwd_q_kernel<T><<<grid, 64 * WAVES, 0, st>>>(a, lse, (const T*)dout, dout_ld, (T*)dq, dq_ld, dbias != nullptr ? part : nullptr);
        DCTR_LAUNCH_CHECK();
    }
    if (dbias != nullptr) {
        attn_bias_grad_kernel<<<a.rel.n * a.heads, 256, 0, st>>>(a, part, dbias);
        DCTR_LAUNCH_CHECK();
    }
    DCTR_TRY(grid_of(((int64_t)a.n_seg * a.max_k * (a.heads / a.group) + WAVES - 1) / WAVES, &grid));
    if (grid > 0) {
        attn_bwd_kv_kernel<T><<<grid, 64 * WAVES, 0, st>>>(a, (const T*)out, out_ld, lse, (const T*)dout, dout_ld, (T*)dk, dk_ld, (T*)dv, dv_ld);
        DCTR_LAUNCH_CHECK();
    }
    return DCTR_OK;
}

}  // namespace dctr

using namespace dctr;

extern "C" {

int dctr_cross_attention_workspace_bytes(const dctr_attention* a, int backward, int64_t* bytes) {
    DCTR_REQUIRE(bytes != nullptr, "null out pointer");
    DCTR_TRY(check_attention(a));
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
    if (d_status != nullptr) {
        attn_check_kernel<<<ceil_div(a->n_seg, 256), 256, 0, st>>>(v, d_status);
        DCTR_LAUNCH_CHECK();
    }
    if (a->total_q == 0) return DCTR_OK;
    return attn_fwd(a, v, d_out, out_ld, d_lse, (float*)d_workspace, st);
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
    float* part = (float*)d_workspace;
    return elem == 4 ? run_bwd<float>(v, d_out, out_ld, d_lse, d_dout, dout_ld, d_dq, dq_ld, d_dk, dk_ld, d_dv, dv_ld, d_drel_bias, part, st)
                     : run_bwd<__bf16>(v, d_out, out_ld, d_lse, d_dout, dout_ld, d_dq, dq_ld, d_dk, dk_ld, d_dv, dv_ld, d_drel_bias,
                                               part, st);
}

}  // extern "C"
