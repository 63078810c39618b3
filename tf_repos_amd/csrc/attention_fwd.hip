// Forward of the ragged cross attention (attention.h: formulas; seq_mma.h: the matrix blocks).  One pass over the keys with a running maximum
// and sum: S^T = K Q^T puts a query's scores into one lane pair, so the softmax statistics are a number a lane and P feeds O^T += V^T P from
// the registers it lies in.  Two forms:
//   rows   4 waves of 32 queries of one head share 64-key tiles (double-buffered; the next tile's loads run under the products)
//   split  32 rows = (query, head of the key head's group) pairs; every wave takes its own 32-key tiles, waves and, for long histories, blocks
//          split the keys and join their (maximum, sum, weighted sum): few queries still use the whole chip, and shared key heads are read once
#include <cmath>

#include "attention.h"

namespace dctr {

// A wave's finished row: the lane pair's halves hold alternating groups of four columns.
template <typename T, typename M, int DP>
__device__ __forceinline__ void write_rows(const AttnView& a, const Softmax<M, DP>& o, int64_t qrow, int h, T* out, int64_t out_ld, float* lse) {
    const int half = (threadIdx.x >> 5) & 1;
    const float l = both_sum(o.l), inv = l == 0.f ? 0.f : 1.f / l;             // (0: no key was seen)
    if (lse != nullptr && half == 0) lse[qrow * a.heads + h] = l == 0.f ? -INFINITY : LN2 * (o.m + log2f(l));
    T* to = out + qrow * out_ld + (int64_t)h * a.dim + 4 * half;
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * k + 8 * i < a.dim)
                Mma<M>::store4(to + 32 * k + 8 * i, o.acc[k][4 * i] * inv, o.acc[k][4 * i + 1] * inv, o.acc[k][4 * i + 2] * inv, o.acc[k][4 * i + 3] * inv);
}

// ---- row form ------------------------------------------------------------------------------------------------------------------------
// 32 rows a wave, 128 a block, whose waves share the tiles of K and V (two buffers, loaded straight into shared memory).  Bound by the softmax's vector
// work and the power that it and the matrix unit draw together: 16 segments of 1024 x 1024, 8 heads, bf16: 713 TF/s at 128 wide (96 us), 538 at 64
// (64 us); f32 in planes at 64 170 TF/s (202 us), f32 instructions at 128 98 (704 us).  Of few and uneven segments the longest list's chain of tiles is
// what takes the time: 2.2 us a tile of 64 keys at 128 wide.
constexpr int ROWS_THREADS = 256;
template <typename T, int DP>
constexpr int rows_keys = attn_width<T, DP> <= 256 ? 64 : 32;           // keys of a tile

template <typename T, int DP>
__global__ __launch_bounds__(ROWS_THREADS, (attn_width<T, DP> <= 384 ? 2 : 1)) void attn_rows_kernel(AttnView a, T* out, int64_t out_ld, float* lse, int32_t* status,
                                                                                                            int row_blocks) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using M = AttnKind<T, DP>;
    using S = typename Mma<M>::Store;
    constexpr int ROWS_KEYS = rows_keys<T, DP>, NB = ROWS_KEYS / 32, TILE = ROWS_KEYS * Tile<M, DP>::STRIDE;
    S *kt = reinterpret_cast<S*>(lds), *vt = kt + 2 * TILE;
    float* hidden = reinterpret_cast<float*>(vt + 2 * TILE);            // [buffer][ROWS_KEYS]
    float* lut = hidden + 2 * ROWS_KEYS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // last row blocks of every head first: under a causal mask they are the longest, and each compute unit begins with one of them
    const Item it = item_of(blockIdx.x, a.heads, a.n_seg);
    const int h = it.head, b = it.seg, rb = row_blocks - 1 - it.nth;
    const Segment s = load_segment(a, b);
    if (rb == 0 && h == 0 && tid == 0) flag_segment(a, b, status);
    const int row0 = rb * 128;
    if (row0 >= s.nq) return;
    const int wrow = row0 + wave * 32, row = wrow + (lane & 31);
    const int chunks = a.dim / Tile<M, DP>::PER;
    const float scale = fabsf(a.scale) * LOG2E;

    RowFrags<M, DP> q;
    q.load((const T*)a.q + (s.q0 + row) * a.q_ld + (int64_t)h * a.dim, chunks, row < s.nq);
    if (a.scale < 0.f) q.negate();                                      // the running maximum is taken before the scale

    const T* K = (const T*)a.k + s.k0 * a.k_ld + (int64_t)(h / a.group) * a.dim;
    const T* V = (const T*)a.v + s.k0 * a.v_ld + (int64_t)(h / a.group) * a.dim;
    int keys = s.nk;                                                    // of this block
    if (a.causal) keys = max(0, min(keys, s.start + min(row0 + 128, s.nq)));
    const int tiles = (keys + ROWS_KEYS - 1) / ROWS_KEYS;
    const bool busy = wrow < s.nq;
    const int wend = a.causal ? s.start + min(wrow + 32, s.nq) : keys;  // keys from here on are hidden from the whole wave

    Softmax<M, DP> o;
    Loader<M, DP, ROWS_KEYS, ROWS_THREADS> ks, vs;
    uint8_t kept = 1;
    uint64_t bits = 0;
    auto fetch = [&](int j0, int buf) {
        ks.fetch(kt + buf * TILE, K, a.k_ld, j0, s.nk, chunks, tid);
        vs.fetch(vt + buf * TILE, V, a.v_ld, j0, s.nk, chunks, tid);
        kept = lane < ROWS_KEYS && j0 + lane < s.nk ? (a.keep != nullptr ? a.keep[s.k0 + j0 + lane] : 1) : 0;
    };
    auto land = [&](int buf) {
        bits = __ballot(kept != 0);
        if (tid < ROWS_KEYS) hidden[buf * ROWS_KEYS + tid] = kept != 0 ? 0.f : -INFINITY;
        ks.land(kt + buf * TILE, tid, bits);
        vs.land(vt + buf * TILE, tid, bits);
    };
    if (tiles > 0) fetch(0, 0);
    const RelRange range = rel_range(a.rel, (int64_t)0 - s.start - (row0 + 127), (int64_t)tiles * ROWS_KEYS - 1 - s.start - row0);      // (under the first loads)
    for (int u = range.lo + tid; u < range.hi; u += ROWS_THREADS) lut[u] = LOG2E * a.bias[bucket_of(a.rel, a.rel.edge[0] - REL_PAD + u) * a.heads + h];
    FarBias fars = far_bias(a, h);
    q.wait();
    settle(fars.before);
    settle(fars.behind);
    if (tiles > 0) land(0);
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
        const int j0 = t * ROWS_KEYS;
        const uint64_t now = bits;
        if (t + 1 < tiles) fetch(j0 + ROWS_KEYS, (t + 1) & 1);
        if (busy && j0 < wend) {
            const S* kb = kt + (t & 1) * TILE;
            f32x16 sc[NB];
#pragma unroll
            for (int k = 0; k < NB; ++k) sc[k] = scores<M, DP, (attn_width<T, DP> > 192)>(kb, 32 * k, q);
            const int d0 = j0 - s.start - wrow;                         // distance of the tile's first key from the wave's first query
            const bool near = near_tile(a.rel, d0 - 31, d0 + ROWS_KEYS - 1);
            const float far = near ? 0.f : far_bucket(a.rel, d0 - 31) > 0 ? fars.behind : fars.before;
            const bool cut = a.causal && d0 + ROWS_KEYS - 1 > 0;
            float c = scale, add = far;
            if (near || cut) {
                uint64_t seen = now;
                if (cut) {
                    const int last = row + s.start - j0;                // last key of the tile that this query sees
                    seen &= last < 0 ? 0ull : last >= 63 ? ~0ull : (2ull << last) - 1;
                }
                seen = lane_bits(seen);
                const float* tab = lut + (near ? d0 - (lane & 31) + 4 * (lane >> 5) - a.rel.edge[0] + REL_PAD : 0);
#pragma unroll
                for (int k = 0; k < NB; ++k)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = 32 * k + reg_row(r);
                        const float x = fmaf(sc[k][r], scale, near ? tab[at] : far);
                        sc[k][r] = (seen >> at & 1) ? x : -INFINITY;
                    }
                c = 1.f;
                add = 0.f;
            } else if (now != ~0ull >> (64 - ROWS_KEYS)) {
                const float* hide = hidden + (t & 1) * ROWS_KEYS;
#pragma unroll
                for (int k = 0; k < NB; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 x = hidden4(hide, k, i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[k][4 * i + j] = fmaf(sc[k][4 * i + j], scale, x[j]);
                    }
                c = 1.f;
            }
            o.template step<NB>(sc, c, add);
            o.template weigh<NB>(vt + (t & 1) * TILE, sc);
        }
        if (t + 1 < tiles) land((t + 1) & 1);
        __syncthreads();
    }
    if (row < s.nq) write_rows<T, M, DP>(a, o, s.q0 + row, h, out, out_ld, lse);
}

// ---- split form, solo form -----------------------------------------------------------------------------------------------------------
// An item is 32 (query, head of the group) rows of a segment and key head.  Split: the block's waves, and the blocks of an item, share its keys.
// Solo: a wave has an item to itself, nothing to join and nobody to wait for -- for short lists in number.
// One query an item (serving) reads each key once: 48 histories of up to 16384 keys, 64 MB, 21 us (3.0 TB/s) and 5.3 for the join, the rest the launch
// and the first loads; a single short item takes 6 us, which is the latency of four dependent reads and the code's own first fetch.
constexpr int SPLIT_KEYS = 32, SPLIT_TILES = 16;                       // keys of a wave's tile, tiles below which an item is not split
// shared memory: 4 waves' K and V tiles, in whose place the waves' results meet (rows of DP + 4 floats: no two rows start at the same bank)
template <typename T, int DP>
struct SplitLds {
    static constexpr size_t tiles = 4 * 2 * SPLIT_KEYS * attn_width<T, DP>, join = 4 * 32 * (DP + 4) * sizeof(float);
    static constexpr size_t first = tiles > join ? tiles : join, stats = 4 * 32 * 2 * sizeof(float);        // statistics, or (while the tiles last) hidden keys
};

template <typename T, int DP>
__device__ __forceinline__ void finish_row(const AttnView& a, int64_t qrow, int h, int tid, float m, float l, const float (&o)[DP / 8], T* out,
                                           int64_t out_ld, float* lse) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int d0 = (tid & 7) * (DP / 8);
    if (lse != nullptr && (tid & 7) == 0) lse[qrow * a.heads + h] = l == 0.f ? -INFINITY : LN2 * (m + log2f(l));
    T* to = out + qrow * out_ld + (int64_t)h * a.dim + d0;
#pragma unroll
    for (int d = 0; d < DP / 8; d += 4)
        if (d0 + d < a.dim) Mma<T>::store4(to + d, o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
}

// Tiles of an item's keys
__device__ __forceinline__ int item_tiles(const AttnView& a, const Segment& s, int rb) {
    int keys = s.nk;
    if (a.causal) keys = max(0, min(keys, s.start + min(rb * 32 + 31, s.nq * a.group - 1) / a.group + 1));
    return (keys + SPLIT_KEYS - 1) / SPLIT_KEYS;
}

// Which segment and which of its cuts chunk c is: a wave counts the segments' cuts, 64 segments at a time.  (A grid of segments x cuts of the
// longest one would mostly start blocks without work: 3072 for 340 of work in a batch of 48 histories of 1..16384 keys, 57 us against 24.)
// Offsets that descend make segments overlap, and the grid's chunks would not do for all of their cuts: from such a place on, a segment is one cut
// (each: tiles of a cut).
__device__ __forceinline__ bool find_chunk(const AttnView& a, const AttnSplit& cut, int c, int* b, int* sp, int* each) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    bool broken = false;
    for (int b0 = 0; b0 < a.n_seg; b0 += 64) {
        int mine = 0;
        bool descends = false;
        if (b0 + lane < a.n_seg) {
            mine = max(1, (segment_keys(a, b0 + lane) + cut.each * SPLIT_KEYS - 1) / (cut.each * SPLIT_KEYS));
            descends = a.k_off[b0 + lane + 1] < a.k_off[b0 + lane];
        }
        const uint64_t down = __ballot(descends), upto_me = ~0ull >> (63 - lane);
        if (mine > 0 && (broken || (down & upto_me) != 0)) mine = 1;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o);
            if (lane >= o) upto += x;
        }
        const uint64_t past = __ballot(before + upto > c);
        if (past != 0) {
            const int at = __ffsll((unsigned long long)past) - 1;
            *b = b0 + at;
            *sp = c - before - __shfl(upto - mine, at);
            *each = broken || (down & (~0ull >> (63 - at))) != 0 ? 1 << 24 : cut.each;         // (> the tiles of DCTR_MAX_POSITION keys)
            return true;
        }
        before += __shfl(upto, 63);
        broken = broken || down != 0;
    }
    return false;
}

// part: [item][split][32][DP + 2] (weighted sum, maximum, sum), then [item] how many of an item's are written; not used when there is one split
template <typename T, int DP, bool SOLO>
__global__ __launch_bounds__(256, (attn_width<T, DP> <= 128 ? 3 : attn_width<T, DP> <= 192 ? 2 : 1)) void attn_split_kernel(AttnView a, T* out, int64_t out_ld, float* lse, int32_t* status, float* part,
                                                                                              AttnSplit cut) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using L = SplitLds<T, DP>;
    using M = AttnKind<T, DP>;
    using S = typename Mma<M>::Store;
    constexpr int TILE = SPLIT_KEYS * Tile<M, DP>::STRIDE, STEP = SOLO ? 1 : 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kv_heads = a.heads / a.group;
    S* kt = reinterpret_cast<S*>(lds) + wave * 2 * TILE;
    S* vt = kt + TILE;
    float* stats = reinterpret_cast<float*>(lds + L::first);
    float* hidden = stats + wave * 64;                                  // (in the statistics' place)
    const int64_t items = (int64_t)cut.row_blocks * kv_heads * a.n_seg, at_item = SOLO ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    int rb, g, b, sp = 0, item, each = cut.each;
    if (SOLO) {                                                         // (row block slowest: a block's waves are alike long)
        item = (int)min(at_item, items - 1);
        const Item it = item_of(item, kv_heads, a.n_seg);
        g = it.head, b = it.seg, rb = it.nth;
    } else if (cut.splits == 1) {
        item = (int)at_item;
        rb = item % cut.row_blocks, g = item / cut.row_blocks % kv_heads, b = item / cut.row_blocks / kv_heads;
    } else {
        rb = blockIdx.x % cut.row_blocks, g = blockIdx.x / cut.row_blocks % kv_heads;
        if (!find_chunk(a, cut, blockIdx.x / cut.row_blocks / kv_heads, &b, &sp, &each)) return;
        item = (b * kv_heads + g) * cut.row_blocks + rb;
    }
    const Segment s = load_segment(a, b);
    if (rb == 0 && g == 0 && sp == 0 && (SOLO ? lane : tid) == 0) flag_segment(a, b, status);
    const int rows = s.nq * a.group, r0 = rb * 32;
    const int tiles = item_tiles(a, s, rb), t0 = sp * each, t1 = cut.splits == 1 ? tiles : min(tiles, t0 + each);
    const bool none = r0 >= rows || (SOLO && at_item >= items);
    if (!SOLO && (none || (sp > 0 && t0 >= tiles))) return;
    if (!SOLO && cut.splits > 1 && sp == 0 && tid == 0)
        reinterpret_cast<int32_t*>(part + items * cut.splits * 32 * (DP + 2))[item] = max(1, (tiles + each - 1) / each);
    const int r = r0 + (lane & 31), i = r / a.group, hg = r % a.group, h = g * a.group + hg;
    const int chunks = a.dim / Tile<M, DP>::PER;
    const float scale = fabsf(a.scale) * LOG2E;

    RowFrags<M, DP> q;
    q.load((const T*)a.q + (s.q0 + i) * a.q_ld + (int64_t)h * a.dim, chunks, !none && r < rows);
    if (a.scale < 0.f) q.negate();

    const T* K = (const T*)a.k + s.k0 * a.k_ld + (int64_t)g * a.dim;
    const T* V = (const T*)a.v + s.k0 * a.v_ld + (int64_t)g * a.dim;
    const int i0 = r0 / a.group, i1 = min(r0 + 31, rows - 1) / a.group;
    Softmax<M, DP> o;
    Staged<M, DP, SPLIT_KEYS, 64> ks, vs;
    uint8_t kept = 0;
    auto fetch = [&](int j0) {
        ks.fetch(kt, K, a.k_ld, j0, s.nk, chunks, lane);
        vs.fetch(vt, V, a.v_ld, j0, s.nk, chunks, lane);
        kept = lane < SPLIT_KEYS && j0 + lane < s.nk ? (a.keep != nullptr ? a.keep[s.k0 + j0 + lane] : 1) : 0;
    };
    int t = SOLO ? (none ? t1 : 0) : t0 + wave;
    if (t < t1) fetch(t * SPLIT_KEYS);

    // Bias, under the first loads: bucket of a distance, then its value for the row's head (an item's rows have min(group, 32) different ones).
    const int wide = min(a.group, 32), col = a.group <= 32 ? hg : r - r0, reach = rel_reach(a.rel);
    int32_t* lut = reinterpret_cast<int32_t*>(stats + 4 * 32 * 2);
    float* table = reinterpret_cast<float*>(lut + reach) + (SOLO ? wave * a.rel.n * wide : 0);      // [n_buckets][wide]
    for (int u = SOLO ? lane : tid; u < a.rel.n * wide; u += SOLO ? 64 : 256)
        table[u] = LOG2E * a.bias[u / wide * a.heads + g * a.group + (a.group <= 32 ? u % wide : (r0 + u % wide) % a.group)];
    // (SOLO's waves fill one table for the whole range)
    const RelRange range = SOLO ? RelRange{0, reach} : rel_range(a.rel, (int64_t)t0 * SPLIT_KEYS - s.start - i1, (int64_t)t1 * SPLIT_KEYS - 1 - s.start - i0);
    if (SOLO || near_tile(a.rel, t0 * SPLIT_KEYS - s.start - i1, t1 * SPLIT_KEYS - 1 - s.start - i0))
        for (int u = range.lo + tid; u < range.hi; u += 256) lut[u] = bucket_of(a.rel, a.rel.edge[0] - REL_PAD + u) * wide;
    if (a.rel.n > 0) __syncthreads();
    if (SOLO && none) return;
    for (; t < t1; t += STEP) {
        const int j0 = t * SPLIT_KEYS;
        const uint64_t now = __ballot(kept != 0);
        // the tile is this wave's own: its reads of the last step are behind these writes in program order
        __builtin_amdgcn_wave_barrier();
        ks.land(kt, lane, now);
        vs.land(vt, lane, now);
        if (lane < SPLIT_KEYS) hidden[lane] = kept != 0 ? 0.f : -INFINITY;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (t + STEP < t1) fetch((t + STEP) * SPLIT_KEYS);
        f32x16 sc[1];
        sc[0] = scores<M, DP, (attn_width<T, DP> > 192)>(kt, 0, q);
        const int dmin = j0 - s.start - i1, dmax = j0 + SPLIT_KEYS - 1 - s.start - i0;
        const bool near = near_tile(a.rel, dmin, dmax);
        const float far = a.rel.n > 0 && !near ? table[far_bucket(a.rel, dmin) * wide + col] : 0.f;
        const bool hide = a.causal && dmax > 0;
        float c = scale, add = far;
        if (near || hide) {
            uint64_t seen = now;
            if (hide) {
                const int last = i + s.start - j0;
                seen &= last < 0 ? 0ull : last >= 63 ? ~0ull : (2ull << last) - 1;
            }
            seen = lane_bits(seen);
            const int32_t* at = lut + (near ? j0 - s.start - min(i, i1) + 4 * (lane >> 5) - a.rel.edge[0] + REL_PAD : 0);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = fmaf(sc[0][e], scale, near ? table[at[reg_row(e)] + col] : far);
                sc[0][e] = (seen >> reg_row(e) & 1) ? x : -INFINITY;
            }
            c = 1.f;
            add = 0.f;
        } else if (now != 0xFFFFFFFFull) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 x = hidden4(hidden, 0, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[0][4 * i + j] = fmaf(sc[0][4 * i + j], scale, x[j]);
            }
            c = 1.f;
        }
        o.template step<1>(sc, c, add);
        o.template weigh<1>(vt, sc);
    }

    if (SOLO) {
        if (r < rows) write_rows<T, M, DP>(a, o, s.q0 + i, h, out, out_ld, lse);
        return;
    }
    float m, sum, w[DP / 8];
    join_waves<M, DP>(o, reinterpret_cast<float*>(lds), stats, m, sum, w);
    const int mine = r0 + (tid >> 3);
    if (cut.splits == 1) {
        if (mine < rows) finish_row<T, DP>(a, s.q0 + mine / a.group, g * a.group + mine % a.group, tid, m, sum, w, out, out_ld, lse);
        return;
    }
    float* to = part + (((int64_t)item * cut.splits + sp) * 32 + (tid >> 3)) * (DP + 2);
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) to[(tid & 7) * (DP / 8) + d] = w[d];
    if ((tid & 7) == 0) { to[DP] = m; to[DP + 1] = sum; }
}

// one wave a row: the splits' statistics by lanes, their sums one split after the other
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnView a, T* out, int64_t out_ld, float* lse, const float* part, AttnSplit cut) {
    const int lane = threadIdx.x & 63, kv_heads = a.heads / a.group, item = blockIdx.x >> 3, r = (blockIdx.x & 7) * 4 + (threadIdx.x >> 6);
    const int rb = item % cut.row_blocks, g = item / cut.row_blocks % kv_heads, b = item / cut.row_blocks / kv_heads;
    const int splits = reinterpret_cast<const int32_t*>(part + (int64_t)cut.row_blocks * kv_heads * a.n_seg * cut.splits * 32 * (DP + 2))[item];
    const Segment s = load_segment(a, b);
    const int mine = rb * 32 + r;
    if (mine >= s.nq * a.group) return;
    const int64_t step = 32 * (DP + 2);
    const float* p = part + ((int64_t)item * cut.splits * 32 + r) * (DP + 2);
    float m = -INFINITY;
    for (int n = lane; n < splits; n += 64) m = fmaxf(m, p[n * step + DP]);
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    constexpr int PER = DP > 64 ? 2 : 1;
    const int d0 = lane * PER < DP ? lane * PER : 0;
    float l = 0.f, o[PER] = {};
    for (int n0 = 0; n0 < splits; n0 += 64) {
        const int n = n0 + lane;
        const float f = n < splits ? exp2f(p[n * step + DP] - base) : 0.f;
        if (n < splits) l = fmaf(p[n * step + DP + 1], f, l);
        const int many = min(64, splits - n0);
        for (int k = 0; k < many; k += 8) {                             // eight loads under way (the last ones again where there are fewer)
            float w[8], x[8][PER];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int n1 = min(n0 + k + e, splits - 1);
                w[e] = k + e < many ? __shfl(f, k + e) : 0.f;
#pragma unroll
                for (int d = 0; d < PER; ++d) x[e][d] = p[n1 * step + d0 + d];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int d = 0; d < PER; ++d) o[d] = fmaf(x[e][d], w[e], o[d]);
        }
    }
    l = wave_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t qrow = s.q0 + mine / a.group;
    const int h = g * a.group + mine % a.group;
    if (lse != nullptr && lane == 0) lse[qrow * a.heads + h] = l == 0.f ? -INFINITY : LN2 * (m + log2f(l));
#pragma unroll
    for (int d = 0; d < PER; ++d)
        if (lane * PER + d < a.dim) out[qrow * out_ld + (int64_t)h * a.dim + lane * PER + d] = (T)(o[d] * inv);
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
static int padded(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

// Row form or the others.  Blocks of 128 rows that are too few for the compute units lose by two to three times to the split form, few rows sooner
// (4 segments of 96 x 2000, heads of 64: 49 us against 19; of 512 x 2000: 49 against 24; but 1 of 2048 x 2048, 8 heads of 128: 67 against 129).  Where
// there are enough, sharing the tiles pays from 128 rows on (64 segments of 128 x 300: 16.4 us against 20.4), for bf16 heads wider than 64 from 32 on
// (96 x 300: 19 against 27; narrower heads: 14..17 both).
static bool row_form(const dctr_attention* a, int64_t rows) {
    const int64_t blocks = (a->total_q / 128 + a->n_seg) * a->heads, items = (rows + 31) / 32 * a->kv_heads * a->n_seg;
    if (blocks < (rows <= 128 ? 256 : 100) && items <= 4096) return false;
    return rows >= 128 || (rows > 32 && a->dtype == DCTR_TYPE_BF16 && a->head_dim > 64);
}

AttnSplit attn_split(const dctr_attention* a) {
    const int64_t rows = (int64_t)a->max_q * (a->heads / a->kv_heads);
    AttnSplit c{0, 0, 0, 0, false};
    if (row_form(a, rows)) return c;
    c.row_blocks = (int)((rows + 31) / 32);
    c.splits = 1;
    const int64_t items = (int64_t)c.row_blocks * a->kv_heads * a->n_seg, tiles = (a->max_k + SPLIT_KEYS - 1) / SPLIT_KEYS;
    c.solo = attn_solo(a, items);
    if (c.solo || items == 0 || items > 4096) return c;
    // cuts of 512 keys (4 tiles a wave: about 1 us each, after 5 us for a block's start and its join), longer ones where there would be more than 8192
    // parts (136 MB of heads of 128, 69 of 64, 36 of 32)
    const int64_t most = std::min<int64_t>((tiles + SPLIT_TILES - 1) / SPLIT_TILES, std::max<int64_t>(1, 8192 / items));
    if (most <= 1) return c;
    c.each = (int)((tiles + most - 1) / most);
    c.splits = (int)((tiles + c.each - 1) / c.each);
    c.chunks = (int)std::min<int64_t>((int64_t)c.splits * a->n_seg, a->total_k / ((int64_t)c.each * SPLIT_KEYS) + a->n_seg);
    return c;
}

template <typename T, int DP>
static int launch_fwd(const dctr_attention* a, const AttnView& v, void* out, int64_t out_ld, float* lse, int32_t* status, float* ws, hipStream_t st) {
    const AttnSplit cut = attn_split(a);
    const size_t table = sizeof(float) * a->n_buckets * std::min(v.group, 32), lut = sizeof(float) * rel_reach(a);
    if (cut.splits == 0) {
        const int row_blocks = ceil_div(a->max_q, 128);
        const int64_t blocks = (int64_t)row_blocks * a->heads * a->n_seg;
        const size_t lds = 4 * rows_keys<T, DP> * attn_width<T, DP> + (2 * rows_keys<T, DP> + rel_reach(a)) * sizeof(float);
        attn_rows_kernel<T, DP><<<(unsigned)blocks, ROWS_THREADS, lds, st>>>(v, (T*)out, out_ld, lse, status, row_blocks);
        DCTR_LAUNCH_CHECK();
        return DCTR_OK;
    }
    const int64_t items = (int64_t)cut.row_blocks * a->kv_heads * a->n_seg;
    if (items == 0) return DCTR_OK;
    using L = SplitLds<T, DP>;
    constexpr bool wide = sizeof(T) == 4 && DP > 64;                    // (attn_solo: never)
    if (cut.solo)
        attn_split_kernel<T, DP, !wide><<<ceil_div(items, 4), 256, L::first + L::stats + lut + 4 * table, st>>>(v, (T*)out, out_ld, lse, status, ws, cut);
    else
        attn_split_kernel<T, DP, false><<<(unsigned)(cut.splits > 1 ? items / a->n_seg * cut.chunks : items), 256, L::first + L::stats + lut + table, st>>>(v, (T*)out, out_ld, lse, status, ws, cut);
    DCTR_LAUNCH_CHECK();
    if (cut.splits > 1) {
        attn_join_kernel<T, DP><<<(unsigned)(items * 8), 256, 0, st>>>(v, (T*)out, out_ld, lse, ws, cut);
        DCTR_LAUNCH_CHECK();
    }
    return DCTR_OK;
}

template <typename T>
static int by_width(const dctr_attention* a, const AttnView& v, void* out, int64_t out_ld, float* lse, int32_t* status, float* ws, hipStream_t st) {
    switch (padded(a->head_dim)) {
        case 32: return launch_fwd<T, 32>(a, v, out, out_ld, lse, status, ws, st);
        case 64: return launch_fwd<T, 64>(a, v, out, out_ld, lse, status, ws, st);
        default: return launch_fwd<T, 128>(a, v, out, out_ld, lse, status, ws, st);
    }
}

int64_t attn_fwd_blocks(const dctr_attention* a) {
    const AttnSplit cut = attn_split(a);
    if (cut.splits == 0) return (int64_t)ceil_div(a->max_q, 128) * a->heads * a->n_seg;
    const int64_t items = (int64_t)cut.row_blocks * a->kv_heads * a->n_seg;
    return cut.solo ? (items + 3) / 4 : cut.splits > 1 ? std::max((int64_t)cut.row_blocks * a->kv_heads * cut.chunks, items * 8) : items;
}

int64_t attn_fwd_workspace(const dctr_attention* a) {
    const AttnSplit cut = attn_split(a);
    return cut.splits > 1 ? (int64_t)cut.row_blocks * a->kv_heads * a->n_seg * (cut.splits * 32 * (padded(a->head_dim) + 2) + 1) * (int64_t)sizeof(float) : 0;
}

int attn_fwd(const dctr_attention* a, const AttnView& v, void* out, int64_t out_ld, float* lse, int32_t* status, float* ws, hipStream_t st) {
    return a->dtype == DCTR_TYPE_F32 ? by_width<float>(a, v, out, out_ld, lse, status, ws, st) : by_width<__bf16>(a, v, out, out_ld, lse, status, ws, st);
}

}  // namespace dctr
