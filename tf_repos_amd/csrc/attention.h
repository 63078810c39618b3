// Ragged multi-head attention of queries over another sequence's keys, with a learned bias per bucket of the distance between them:
// what the entry points check once and the kernels of attention*.hip share.
//
// Segment b owns query rows [q_offsets[b], q_offsets[b+1]) and key rows [k_offsets[b], k_offsets[b+1]); query i of it stands at
// position q_start[b] + i among the keys 0, 1, 2, ...  With h a query head and g = h / (heads / kv_heads) the key head it reads:
//     s_ij = scale <q_i, k_j> + T[bucket(j - q_start[b] - i), h]         bucket(d) = number of boundaries <= d
//     p_ij = softmax over the keys j that query i sees (key_keep[j] != 0; j <= q_start[b] + i when causal)
//     o_i  = sum_j p_ij v_j                lse_i = log sum_j exp(s_ij)   (no key seen: o_i = 0, lse_i = -inf)
// and for the gradient do of o:
//     dv_j = sum_ih p_ij do_i     ds_ij = p_ij (<do_i, v_j> - <do_i, o_i>)      dT[u, h] = sum over the pairs of bucket u of ds_ij
//     dq_i = scale sum_j ds_ij k_j                dk_j = scale sum_ih ds_ij q_i
#pragma once
#include <algorithm>
#include <type_traits>

#include "seq_mma.h"

namespace dctr {

struct RelBuckets {                                     // passed by value: a captured graph keeps what it was captured with
    int32_t n;                                          // 0: no bias
    int32_t edge[DCTR_MAX_REL_BUCKETS];                 // n - 1 ascending, then INT32_MAX; bucket(d) = #{u : edge[u] <= d}
};

struct AttnView {
    const void *q, *k, *v;
    int64_t q_ld, k_ld, v_ld;                           // row strides in elements
    const int32_t *q_off, *k_off, *q_start;             // q_start may be null (0)
    const uint8_t* keep;                                // may be null (every key)
    const float* bias;                                  // [n_buckets, heads]
    int64_t total_q, total_k;
    int32_t n_seg, heads, group, dim, max_q, max_k, causal;
    float scale;
    RelBuckets rel;
};

struct Segment { int64_t q0, k0; int nq, nk, start; };

__device__ __forceinline__ int64_t cut_to(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// A segment's rows, kept inside the arrays whatever the offsets say (the forward reports the ones that had to be cut, see flag_segment).
__device__ __forceinline__ Segment load_segment(const AttnView& a, int b) {
    Segment s;
    s.q0 = cut_to(a.q_off[b], 0, a.total_q);
    s.k0 = cut_to(a.k_off[b], 0, a.total_k);
    s.nq = (int)cut_to(cut_to(a.q_off[b + 1], s.q0, a.total_q) - s.q0, 0, a.max_q);
    s.nk = (int)cut_to(cut_to(a.k_off[b + 1], s.k0, a.total_k) - s.k0, 0, a.max_k);
    s.start = a.q_start != nullptr ? (int)cut_to(a.q_start[b], -DCTR_MAX_POSITION, DCTR_MAX_POSITION) : 0;
    return s;
}

__device__ __forceinline__ int segment_keys(const AttnView& a, int b) {
    const int64_t k0 = cut_to(a.k_off[b], 0, a.total_k);
    return (int)cut_to(cut_to(a.k_off[b + 1], k0, a.total_k) - k0, 0, a.max_k);
}

__device__ __forceinline__ bool segment_is_bad(const AttnView& a, int b) {
    const int q0 = a.q_off[b], q1 = a.q_off[b + 1], k0 = a.k_off[b], k1 = a.k_off[b + 1];
    const int st = a.q_start != nullptr ? a.q_start[b] : 0;
    return q0 < 0 || q1 < q0 || q1 > a.total_q || (int64_t)q1 - q0 > a.max_q || k0 < 0 || k1 < k0 || k1 > a.total_k ||
           (int64_t)k1 - k0 > a.max_k || st < -DCTR_MAX_POSITION || st > DCTR_MAX_POSITION;
}
__device__ __forceinline__ void flag_segment(const AttnView& a, int b, int32_t* status) {
    if (status != nullptr && segment_is_bad(a, b)) { status[0] = 1; status[1] = b; }
}

// Operand kind: float arrays in planes (seq_mma.h) up to heads of 64; wider ones' planes pass the registers of the backward and the shared memory
// of the forms whose waves have tiles of their own.
template <typename T, int DP>
using AttnKind = std::conditional_t<std::is_same_v<T, float> && DP <= 64, Split, T>;
template <typename T, int DP>
constexpr int attn_width = Mma<AttnKind<T, DP>>::BYTES * DP;           // bytes of a row in a tile

// The bias of one tile of scores.  Distances below the first boundary all share bucket 0, those from the last boundary on the last bucket: only
// a tile that reaches between the two ("near") looks values up, any other adds one number.  Tables hold log2(e) x the bias (the kernels'
// exponents are base 2) and reach REL_PAD distances past either boundary, so that a near tile's lookups need no clamp.
constexpr int REL_PAD = 128;                            // > keys + queries of a tile

__device__ __forceinline__ bool near_tile(const RelBuckets& r, int dmin, int dmax) { return r.n > 1 && dmax >= r.edge[0] && dmin < r.edge[r.n - 2]; }
// bucket of every distance of a tile that is not near
__device__ __forceinline__ int far_bucket(const RelBuckets& r, int dmin) { return r.n > 1 && dmin >= r.edge[r.n - 2] ? r.n - 1 : 0; }

// bucket of distance d; the edges come by scalar loads, one compare each for the whole wave
__device__ __forceinline__ int bucket_of(const RelBuckets& r, int d) {
    int n = 0;
    for (int u = 0; u + 1 < r.n; u += 8)
#pragma unroll
        for (int v = 0; v < 8; ++v) n += r.edge[u + v] <= d;
    return n;
}
__device__ __forceinline__ int rel_reach(const RelBuckets& r) { return r.n > 1 ? r.edge[r.n - 2] - r.edge[0] + 2 * REL_PAD : 0; }

// The entries of such a table that distances in [dmin, dmax] can ask for: short lists do without the rest.
struct RelRange { int lo, hi; };
__device__ __forceinline__ RelRange rel_range(const RelBuckets& r, int64_t dmin, int64_t dmax) {
    const int reach = rel_reach(r);
    if (reach == 0) return {0, 0};
    const int64_t zero = (int64_t)REL_PAD - r.edge[0];
    return {(int)cut_to(dmin + zero, 0, reach), (int)cut_to(dmax + zero + 1, 0, reach)};
}

// Keys that are not kept, as numbers to add to a tile's scores (0, -inf): one read for four keys and no vector work beyond the fma that is there.
__device__ __forceinline__ f32x4 hidden4(const float* hidden, int k, int i) {      // rows of registers 4 i .. 4 i + 3 of block k
    return *reinterpret_cast<const f32x4*>(hidden + 32 * k + 8 * i + 4 * ((threadIdx.x >> 5) & 1));
}

// log2(e) x a head's bias of the two far buckets, read once: a load within the tile loop would wait for the tiles under way
struct FarBias { float before, behind; };
__device__ __forceinline__ FarBias far_bias(const AttnView& a, int h) {
    FarBias f{0.f, 0.f};
    if (a.rel.n > 0) f = {LOG2E * a.bias[h], LOG2E * a.bias[(int64_t)(a.rel.n - 1) * a.heads + h]};
    return f;
}

// Item (segment, head, block of its rows) of a launch whose blocks of rows go slowest: the first of every segment, then the second, ...  Consecutive
// workgroups go to the eight XCDs in turn; the segments move on by one a round, or a long one among short ones would have all its work on one XCD
// (16 segments x 2 heads: 441 us against 139).
struct Item { int head, seg, nth; };
__device__ __forceinline__ Item item_of(int item, int heads, int n_seg) {
    const int nth = item / heads / n_seg;
    return {item % heads, (item / heads % n_seg + nth) % n_seg, nth};
}

inline int rel_reach(const dctr_attention* a) {         // entries of a table over distances
    return a->n_buckets > 1 ? a->boundaries[a->n_buckets - 2] - a->boundaries[0] + 2 * REL_PAD : 0;
}

// Items (32 rows of a segment and head) that are many and short go to a wave each, without barriers or joins; fewer or longer ones share a
// block's waves.  (f32 heads wider than 64 would spill; a wave's own bias tables have to fit beside the tiles.)
inline bool attn_solo(const dctr_attention* a, int64_t items) {
    return items >= 1024 && a->max_k <= 512 && !(a->dtype == DCTR_TYPE_F32 && a->head_dim > 64) &&
           a->n_buckets * std::min(a->heads / a->kv_heads, 32) <= 1024 && rel_reach(a) <= 512;
}

// ---- launchers (attention_fwd.hip, attention_bwd.hip): DP = 32, 64 or 128 by head_dim
// The forward's form for few query rows a key head (splits = 0: the other form).  An item's keys are cut every `each` tiles, into `splits` at most;
// chunks: no more pairs of segment and cut than these, of segments that do not overlap.
struct AttnSplit { int row_blocks, splits, each, chunks; bool solo; };
AttnSplit attn_split(const dctr_attention* a);
int64_t attn_fwd_blocks(const dctr_attention* a);         // of the call's largest launch
int64_t attn_fwd_workspace(const dctr_attention* a);      // bytes
int attn_fwd(const dctr_attention* a, const AttnView& v, void* out, int64_t out_ld, float* lse, int32_t* status, float* ws, hipStream_t st);

struct AttnGrads {
    const void* out; int64_t out_ld;
    const float* lse;
    const void* dout; int64_t dout_ld;
    void* dq; int64_t dq_ld;
    void* dk; int64_t dk_ld;
    void* dv; int64_t dv_ld;
    float* dbias;                                       // may be null
};
int64_t attn_bwd_blocks(const dctr_attention* a);
int64_t attn_bwd_workspace(const dctr_attention* a);
int attn_bwd(const dctr_attention* a, const AttnView& v, const AttnGrads& x, float* ws, hipStream_t st);

}  // namespace dctr
