// Softmax cross entropy over a large vocabulary from the hidden rows and the vocabulary's table: the [N, V] logits exist 64 at a time.
//     z_nv = <x_n, w_v> + b_v        lse_n = log sum_v exp(z_nv)        loss_n = lse_n - z_n,label(n)
//     g_nv = c_n (exp(z_nv - lse_n) - [v = label(n)]),  c_n = scale row_scale_n (0 for a row without a label)
//     dx_n = sum_v g_nv w_v          dw_v = sum_n g_nv x_n              db_v = sum_n g_nv
// The forward's sums leave the label out and add it at the end: with e the sum of the others, 1 - p_label = e / (e + exp(z_label - m)) has
// no cancellation however sure the model is, nor has loss = log1p(e) where the label is the row's largest.
#include <cmath>

#include "attention.h"

namespace dctr {

struct VocabView {
    const void *x, *w;
    int64_t x_ld, w_ld, V;
    const float* b;                 // [V] or null
    const int32_t* labels;
    const float* row_scale;         // [N] or null
    float scale;
    int32_t N, D;
};

constexpr int VS_WAVES = 4;

template <typename T>
__device__ __forceinline__ float logit(const VocabView& a, const T* x, int64_t v) {
    const T* w = (const T*)a.w + v * a.w_ld;
    float s = 0.f;
    for (int d = 0; d < a.D; ++d) s = fmaf(to_f32(x[d]), to_f32(w[d]), s);
    return a.b != nullptr ? s + a.b[v] : s;
}

__device__ __forceinline__ float vs_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float vs_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// one wave per row
template <typename T>
__global__ __launch_bounds__(64 * VS_WAVES) void vocab_fwd_kernel(VocabView a, float* loss, float* lse, T* dx, int64_t dx_ld, int32_t* status) {
    const int n = blockIdx.x * VS_WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (n >= a.N) return;
    const T* x = (const T*)a.x + n * a.x_ld;
    const int label = a.labels[n];
    const bool on = label >= 0 && label < a.V;
    if (label >= a.V && lane == 0 && status != nullptr) { status[0] = 1; status[1] = label; }
    float m = on ? logit<T>(a, x, label) : -INFINITY, e = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const float mine = m;
    for (int64_t v0 = 0; v0 < a.V; v0 += 64) {
        const int64_t v = v0 + lane;
        const float z = v < a.V && v != label ? logit<T>(a, x, v) : -INFINITY;
        const float top = fmaxf(m, vs_max(z)), base = top == -INFINITY ? 0.f : top;
        const float p = expf(z - base), shrink = expf(m - base);
        e = e * shrink + vs_sum(p);
        m = top;
        if (dx == nullptr) continue;
        for (int c = 0; c < 4; ++c) acc[c] *= shrink;
        for (int t = 0; t < 64 && v0 + t < a.V; ++t) {
            const float q = __shfl(p, t);
            const T* w = (const T*)a.w + (v0 + t) * a.w_ld;
            for (int c = 0; c < 4; ++c)
                if (c * 64 + lane < a.D) acc[c] = fmaf(q, to_f32(w[c * 64 + lane]), acc[c]);
        }
    }
    const float base = m == -INFINITY ? 0.f : m, all = e + (on ? expf(mine - base) : 0.f);
    if (lane == 0) {
        if (lse != nullptr) lse[n] = base + logf(all);
        loss[n] = !on ? 0.f : mine == m ? log1pf(e) : (base - mine) + logf(all);
    }
    if (dx == nullptr) return;
    const float c_n = on ? a.scale * (a.row_scale != nullptr ? a.row_scale[n] : 1.f) : 0.f;
    for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < a.D)
            dx[n * dx_ld + c * 64 + lane] =
                (T)(on ? c_n * (acc[c] - e * to_f32(((const T*)a.w + label * a.w_ld)[c * 64 + lane])) / all : 0.f);
}

// one wave per vocabulary row
template <typename T>
__global__ __launch_bounds__(64 * VS_WAVES) void vocab_dw_kernel(VocabView a, const float* lse, T* dw, int64_t dw_ld, float* db) {
    const int64_t v = (int64_t)blockIdx.x * VS_WAVES + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (v >= a.V) return;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
    for (int n0 = 0; n0 < a.N; n0 += 64) {
        const int n = n0 + lane;
        const int label = n < a.N ? a.labels[n] : -1;
        const bool on = label >= 0 && label < a.V;
        float g = 0.f;
        if (on) {
            const float t = logit<T>(a, (const T*)a.x + n * a.x_ld, v) - lse[n];
            g = a.scale * (a.row_scale != nullptr ? a.row_scale[n] : 1.f) * (v == label ? expm1f(t) : expf(t));
        }
        sum += g;
        const uint64_t rows = __ballot(on);
        for (int t = 0; t < 64; ++t) {
            const float q = __shfl(g, t);
            if (!(rows >> t & 1)) continue;
            const T* x = (const T*)a.x + (n0 + t) * a.x_ld;
            for (int c = 0; c < 4; ++c)
                if (c * 64 + lane < a.D) acc[c] = fmaf(q, to_f32(x[c * 64 + lane]), acc[c]);
        }
    }
    for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < a.D) dw[v * dw_ld + c * 64 + lane] = (T)(acc[c]);
    sum = vs_sum(sum);
    if (db != nullptr && lane == 0) db[v] = sum;
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
static int check_sizes(int dtype, int N, int64_t V, int D) {
    DCTR_REQUIRE(dtype == DCTR_TYPE_F32 || dtype == DCTR_TYPE_BF16, "vocab softmax: unknown element type %d", dtype);
    DCTR_REQUIRE(N >= 0, "vocab softmax: %d rows", N);
    DCTR_REQUIRE(V >= 1 && V <= INT32_MAX, "vocab softmax: vocabulary of %lld (1..2^31-1)", (long long)V);
    DCTR_REQUIRE(D >= 8 && D <= 256 && D % 8 == 0, "vocab softmax: width %d (a multiple of 8, 8..256)", D);
    return DCTR_OK;
}

static int check_rows(const char* what, const void* p, int ld, int D, int elem) {
    DCTR_REQUIRE(p != nullptr, "vocab softmax: %s is null", what);
    DCTR_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((int64_t)ld * elem) % 16 == 0, "vocab softmax: rows of %s must be 16-byte aligned", what);
    DCTR_REQUIRE(ld >= D, "vocab softmax: row stride %d of %s is below %d", ld, what, D);
    return DCTR_OK;
}

static int64_t workspace_bytes(int, int64_t, int, int) { return 0; }

static int make_view(int dtype, const void* x, int x_ld, const void* w, int w_ld, const float* b, const int32_t* labels, int N, int64_t V, int D,
                     const float* row_scale, float scale, int train, const void* ws, size_t ws_bytes, VocabView* view) {
    DCTR_TRY(check_sizes(dtype, N, V, D));
    const int elem = dtype == DCTR_TYPE_F32 ? 4 : 2;
    if (N > 0) {
        DCTR_TRY(check_rows("x", x, x_ld, D, elem));
        DCTR_REQUIRE(labels != nullptr, "vocab softmax: labels are null");
    }
    DCTR_TRY(check_rows("w", w, w_ld, D, elem));
    DCTR_REQUIRE(std::isfinite(scale), "vocab softmax: scale is not finite");
    const int64_t need = workspace_bytes(N, V, D, train);
    DCTR_REQUIRE(need == 0 || (ws != nullptr && (int64_t)ws_bytes >= need), "vocab softmax: workspace of %lld bytes needed, %lld given",
                 (long long)need, ws != nullptr ? (long long)ws_bytes : 0ll);
    DCTR_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "vocab softmax: workspace must be 16-byte aligned");
    *view = VocabView{x, w, x_ld, w_ld, V, b, labels, row_scale, scale, N, D};
    return DCTR_OK;
}

}  // namespace dctr

using namespace dctr;

extern "C" {

int dctr_vocab_softmax_workspace_bytes(int dtype, int N, int64_t V, int D, int train, int64_t* bytes) {
    DCTR_REQUIRE(bytes != nullptr, "null out pointer");
    DCTR_TRY(check_sizes(dtype, N, V, D));
    *bytes = workspace_bytes(N, V, D, train);
    return DCTR_OK;
}

int dctr_vocab_softmax_fwd(int dtype, const void* d_x, int x_ld, const void* d_w, int w_ld, const float* d_b, const int32_t* d_labels, int N,
                           int64_t V, int D, const float* d_row_scale, float scale, float* d_loss, float* d_lse, void* d_dx, int dx_ld,
                           int32_t* d_status, void* d_workspace, size_t workspace_bytes, void* stream) {
    VocabView a;
    DCTR_TRY(make_view(dtype, d_x, x_ld, d_w, w_ld, d_b, d_labels, N, V, D, d_row_scale, scale, d_dx != nullptr, d_workspace, workspace_bytes, &a));
    if (N == 0) return DCTR_OK;
    DCTR_REQUIRE(d_loss != nullptr, "vocab softmax: loss is null");
    if (d_dx != nullptr) DCTR_TRY(check_rows("dx", d_dx, dx_ld, D, dtype == DCTR_TYPE_F32 ? 4 : 2));
    hipStream_t st = as_stream(stream);
    const int grid = ceil_div(N, VS_WAVES);
    if (dtype == DCTR_TYPE_F32)
        vocab_fwd_kernel<float><<<grid, 64 * VS_WAVES, 0, st>>>(a, d_loss, d_lse, (float*)d_dx, dx_ld, d_status);
    else
        vocab_fwd_kernel<__bf16><<<grid, 64 * VS_WAVES, 0, st>>>(a, d_loss, d_lse, (__bf16*)d_dx, dx_ld, d_status);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

int dctr_vocab_softmax_bwd_weights(int dtype, const void* d_x, int x_ld, const void* d_w, int w_ld, const float* d_b, const int32_t* d_labels, int N,
                                   int64_t V, int D, const float* d_row_scale, float scale, const float* d_lse, void* d_dw, int dw_ld, float* d_db,
                                   void* d_workspace, size_t workspace_bytes, void* stream) {
    VocabView a;
    DCTR_TRY(make_view(dtype, d_x, x_ld, d_w, w_ld, d_b, d_labels, N, V, D, d_row_scale, scale, 1, d_workspace, workspace_bytes, &a));
    DCTR_REQUIRE(N == 0 || d_lse != nullptr, "vocab softmax: lse is null");
    DCTR_TRY(check_rows("dw", d_dw, dw_ld, D, dtype == DCTR_TYPE_F32 ? 4 : 2));
    hipStream_t st = as_stream(stream);
    const int grid = ceil_div(V, VS_WAVES);
    if (dtype == DCTR_TYPE_F32)
        vocab_dw_kernel<float><<<grid, 64 * VS_WAVES, 0, st>>>(a, d_lse, (float*)d_dw, dw_ld, d_db);
    else
        vocab_dw_kernel<__bf16><<<grid, 64 * VS_WAVES, 0, st>>>(a, d_lse, (__bf16*)d_dw, dw_ld, d_db);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

}  // extern "C"
