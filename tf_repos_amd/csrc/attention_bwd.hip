// Backward of the ragged cross attention (attention.h: formulas; seq_mma.h: the matrix blocks): scores and p are formed again from lse, nothing
// of size queries x keys is stored.  Two kernels, each summing in registers over the axis that it walks, so no atomics meet in memory:
//   query side  S^T = K Q^T and dP^T = V dO^T by 32 queries a wave, dQ^T += K^T dS^T; delta = <do, out> on the way, kept for the key side;
//               the bias gradient's sums over a tile's diagonals
//   key side    S = Q K^T and dP = dO V^T by 32 keys a wave, over the queries of every head of the group: dV^T += dO^T P, dK^T += Q^T dS
#include <cmath>

#include "attention.h"

namespace dctr {

constexpr int BWD_THREADS = 256;

// keys of a query-side tile: QW waves share the rows' work, 4 / QW the tile's keys
template <typename T, int DP, int QW>
struct QuerySide {
    static constexpr int KW = 4 / QW, NB = QW == 4 && sizeof(T) * DP <= 256 ? 2 : 1, KEYS = 32 * NB * KW, BUFS = QW == 4 ? 2 : 1;
    static constexpr int TILE = KEYS * DP, ROWS = 32 * QW;
    static constexpr size_t tiles = 2 * BUFS * TILE * sizeof(T), join = QW == 1 ? 4 * 32 * (DP + 4) * sizeof(float) : 0;
    static constexpr size_t first = tiles > join ? tiles : join;
};

// Sums of ds by distance.  A near tile adds every element to its distance's cell: of one half-wave and register no two lanes (queries) share a
// distance, so each half of each wave has cells of its own and the order of every cell's sum is the program's.
__device__ __forceinline__ void lds_add(float* cell, float x) { __hip_atomic_fetch_add(cell, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }

// part: [head][segment * row_blocks + row block][n_buckets] shares of the bias gradient, or null; delta [total_q, heads]
template <typename T, int DP, int QW>
__global__ __launch_bounds__(BWD_THREADS, (sizeof(T) * DP <= 128 ? 2 : 1)) void attn_bwd_q_kernel(AttnView a, const T* out, int64_t out_ld, const float* lse, const T* dout, int64_t dout_ld,
                                                                 T* dq, int64_t dq_ld, float* delta, float* part, int row_blocks) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using Q = QuerySide<T, DP, QW>;
    constexpr int NB = Q::NB, TILE = Q::TILE;
    // For bf16 <do, out> is off by the rounding of `out`, an error that all of a row's ds share.  The walk sums p dp over every key, which is the
    // same number unrounded, and P K besides: dq is put right with (rounded - unrounded) P K at the end, the key side and the bias gradient take
    // the unrounded one.  (Measured: the relative error of dq and dk 0.0030 -> 0.0023 at 777 x 1531 x 128.)
    constexpr bool ROUNDED = sizeof(T) == 2;
    T *kt = reinterpret_cast<T*>(lds), *vt = kt + Q::BUFS * TILE;
    float* lut = reinterpret_cast<float*>(lds + Q::first);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int rb = blockIdx.x % row_blocks, h = blockIdx.x / row_blocks % a.heads, b = blockIdx.x / row_blocks / a.heads;
    const Segment s = load_segment(a, b);
    const int row0 = rb * Q::ROWS;
    float* share = part != nullptr ? part + ((int64_t)h * a.n_seg * row_blocks + (int64_t)b * row_blocks + rb) * a.rel.n : nullptr;
    if (row0 >= s.nq) {
        if (share != nullptr)
            for (int u = tid; u < a.rel.n; u += BWD_THREADS) share[u] = 0.f;
        return;
    }
    const int wrow = row0 + 32 * (wave % QW), row = wrow + (lane & 31), first_key = 32 * NB * (wave / QW);
    const int chunks = a.dim / Tile<T, DP>::PER;
    const float scale = a.scale * LOG2E;
    const int reach = rel_reach(a.rel);
    float* cells = lut + reach;                                         // [4 waves][2 halves][reach], then 2 x 4 far sums
    float* mine = cells + (2 * wave + half) * reach;

    RowFrags<T, DP> q, go;
    q.load((const T*)a.q + (s.q0 + row) * a.q_ld + (int64_t)h * a.dim, chunks, row < s.nq);
    go.load(dout + (s.q0 + row) * dout_ld + (int64_t)h * a.dim, chunks, row < s.nq);
    float dl = 0.f, minus_lse = -INFINITY;                              // (a row that saw nothing: p = 2^-inf = 0)
    {
        RowFrags<T, DP> o;
        o.load(out + (s.q0 + row) * out_ld + (int64_t)h * a.dim, chunks, row < s.nq);
#pragma unroll
        for (int c = 0; c < RowFrags<T, DP>::STEPS; ++c)
#pragma unroll
            for (int e = 0; e < Tile<T, DP>::PER; ++e) dl = fmaf(to_f32(go.c[c][e]), to_f32(o.c[c][e]), dl);
        dl = both_sum(dl);
        if (row < s.nq) {
            const float L = lse[(s.q0 + row) * a.heads + h];
            if (L != -INFINITY) minus_lse = -LOG2E * L;
            if (!ROUNDED && wave < QW && half == 0) delta[(s.q0 + row) * a.heads + h] = dl;
        }
    }

    const T* K = (const T*)a.k + s.k0 * a.k_ld + (int64_t)(h / a.group) * a.dim;
    const T* V = (const T*)a.v + s.k0 * a.v_ld + (int64_t)(h / a.group) * a.dim;
    int keys = s.nk;
    if (a.causal) keys = max(0, min(keys, s.start + min(row0 + Q::ROWS, s.nq)));
    const int tiles = (keys + Q::KEYS - 1) / Q::KEYS;
    const bool busy = wrow < s.nq;
    const int wend = a.causal ? s.start + min(wrow + 32, s.nq) : keys;

    f32x16 acc[DP / 32] = {}, pk[ROUNDED ? DP / 32 : 1] = {};
    float far_ds[2] = {0.f, 0.f}, far_p[2] = {0.f, 0.f}, pdp = 0.f;     // [below the first boundary, from the last one on]
    Staged<T, DP, Q::KEYS, BWD_THREADS> ks, vs;
    uint64_t bits[2] = {0, 0};                                          // kept keys of the tile
    uint8_t kept[2] = {0, 0};
    auto fetch = [&](int j0) {
        ks.fetch(K, a.k_ld, j0, s.nk, chunks, tid);
        vs.fetch(V, a.v_ld, j0, s.nk, chunks, tid);
#pragma unroll
        for (int w = 0; w < (Q::KEYS + 63) / 64; ++w) {
            const int j = j0 + 64 * w + lane;
            kept[w] = 64 * w + lane < Q::KEYS && j < s.nk ? (a.keep != nullptr ? a.keep[s.k0 + j] : 1) : 0;
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int w = 0; w < (Q::KEYS + 63) / 64; ++w) bits[w] = __ballot(kept[w] != 0);
        ks.store_kept(kt + buf * TILE, tid, bits);
        vs.store_kept(vt + buf * TILE, tid, bits);
    };
    // p and dp of this wave's part of the tile at j0; returns whether the tile is near, `side` its far side otherwise
    auto pair = [&](const T* kb, const T* vb, int j0, uint64_t now, f32x16 (&p)[NB], f32x16 (&dp)[NB], int& cell, int& side) {
        const int d0 = j0 + first_key - s.start - wrow;                 // the part's first key from the wave's first query
        const bool near = near_tile(a.rel, d0 - 31, d0 + 32 * NB - 1);
        const int fb = a.rel.n > 0 && !near ? far_bucket(a.rel, d0 - 31) : 0;
        const float far = (a.rel.n > 0 && !near ? LOG2E * a.bias[fb * a.heads + h] : 0.f);
        side = fb > 0;
        cell = near ? d0 - (lane & 31) + 4 * half - a.rel.edge[0] + REL_PAD : 0;
        const bool cut = a.causal && d0 + 32 * NB - 1 > 0;
        uint64_t seen = now;
        if (cut) {
            const int last = row + s.start - j0 - first_key;
            seen &= last < 0 ? 0ull : last >= 63 ? ~0ull : (2ull << last) - 1;
        }
        const bool hide = __any((uint32_t)(seen >> (32 * (NB - 1))) != ~0u || (uint32_t)seen != ~0u);
        seen = lane_bits(seen);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            p[k] = scores<T, DP>(kb, first_key + 32 * k, q);
            dp[k] = scores<T, DP>(vb, first_key + 32 * k, go);
        }
        if (near || hide) {
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 32 * k + reg_row(r);
                    const float x = fmaf(p[k][r], scale, near ? lut[cell + at] : far) + minus_lse;
                    p[k][r] = (seen >> at & 1) ? __builtin_amdgcn_exp2f(x) : 0.f;
                }
        } else {
            const float off = far + minus_lse;
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) p[k][r] = __builtin_amdgcn_exp2f(fmaf(p[k][r], scale, off));
        }
        return near;
    };
    auto part_bits = [&](const uint64_t (&w)[2]) { return first_key < 64 ? w[0] >> first_key : w[1] >> (first_key - 64); };
    // one walk over the tiles; `second`: only the near ones, for their cells
    auto walk = [&](bool second) {
        int t = 0;
        if (second) {                                                   // tiles before this one are far for every row of the block
            const int64_t from = (int64_t)a.rel.edge[0] + s.start + row0 - (Q::KEYS - 1);
            t = from <= 0 ? 0 : (int)min((int64_t)tiles, from / Q::KEYS);
        }
        int last = tiles;
        if (second) {
            const int64_t to = (int64_t)a.rel.edge[a.rel.n - 2] + s.start + row0 + Q::ROWS - 1;      // (`near` goes by whole waves too)
            last = to <= 0 ? 0 : (int)min((int64_t)tiles, (to + Q::KEYS - 1) / Q::KEYS);
        }
        if (t >= last) return;
        __syncthreads();
        fetch(t * Q::KEYS);
        if (!second) {                                                  // under the first tile's loads
            for (int u = tid; u < reach; u += BWD_THREADS) lut[u] = LOG2E * a.bias[bucket_of(a.rel, a.rel.edge[0] - REL_PAD + u) * a.heads + h];
            if (part != nullptr)
                for (int u = tid; u < 8 * reach; u += BWD_THREADS) cells[u] = 0.f;
        }
        store(0);
        __syncthreads();
        for (int n = 0; t < last; ++t, ++n) {
            const int j0 = t * Q::KEYS, buf = Q::BUFS == 2 ? n & 1 : 0;
            const uint64_t now = part_bits(bits);
            if (t + 1 < last) fetch(j0 + Q::KEYS);
            if (busy && j0 + first_key < wend) {
                const T *kb = kt + buf * TILE, *vb = vt + buf * TILE;
                f32x16 p[NB], dp[NB];
                int cell, side;
                const bool near = pair(kb, vb, j0, now, p, dp, cell, side);
                if (!second) {
                    if (ROUNDED || (part != nullptr && !near)) {
                        float x = 0.f, y = 0.f;
#pragma unroll
                        for (int k = 0; k < NB; ++k)
#pragma unroll
                            for (int r = 0; r < 16; ++r) { x = fmaf(p[k][r], dp[k][r], x); y += p[k][r]; }
                        pdp += x;
                        if (!near) { far_ds[side] += x; far_p[side] += y; }
                    }
#pragma unroll
                    for (int k = 0; k < NB; ++k) {
                        if (ROUNDED) {
                            const auto w = Mma<T>::pack(p[k]);
#pragma unroll
                            for (int d = 0; d < DP / 32; ++d)
                                pk[ROUNDED ? d : 0] = Mma<T>::template weigh<DP>(kb, first_key + 32 * k, 32 * d, w, pk[ROUNDED ? d : 0]);
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) p[k][r] *= dp[k][r] - dl;
                        if (!ROUNDED && part != nullptr && near)
#pragma unroll
                            for (int r = 0; r < 16; ++r) lds_add(mine + cell + 32 * k + reg_row(r), p[k][r]);
                        const auto w = Mma<T>::pack(p[k]);
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d) acc[d] = Mma<T>::template weigh<DP>(kb, first_key + 32 * k, 32 * d, w, acc[d]);
                    }
                } else if (near) {
#pragma unroll
                    for (int k = 0; k < NB; ++k)
#pragma unroll
                        for (int r = 0; r < 16; ++r) lds_add(mine + cell + 32 * k + reg_row(r), p[k][r] * (dp[k][r] - dl));
                }
            }
            if (Q::BUFS == 1) __syncthreads();
            if (t + 1 < last) store(Q::BUFS == 2 ? (n + 1) & 1 : 0);
            __syncthreads();
        }
    };
    walk(false);

    if (ROUNDED) {
        float exact = both_sum(pdp);
        if (QW == 1) {                                                  // the waves hold different keys of the same rows
            float* meet = reinterpret_cast<float*>(lds);
            __syncthreads();
            if (half == 0) meet[wave * 32 + lane] = exact;
            __syncthreads();
            exact = (meet[lane & 31] + meet[32 + (lane & 31)]) + (meet[64 + (lane & 31)] + meet[96 + (lane & 31)]);
        }
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] += (dl - exact) * pk[ROUNDED ? d : 0];
        dl = exact;
        if (wave < QW && half == 0 && row < s.nq) delta[(s.q0 + row) * a.heads + h] = dl;
    }
    if (part != nullptr) {
        if (ROUNDED && a.rel.n > 1) walk(true);                         // the near tiles again, for their distances' sums
        float* fars = cells + 8 * reach;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float x = fmaf(-dl, far_p[side], far_ds[side]);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
            if (lane == 0) fars[4 * side + wave] = x;
        }
        __syncthreads();
        // every distance's eight cells, then a wave a bucket
        if (tiles > 0)
            for (int u = tid; u < reach; u += BWD_THREADS) {
                float x = cells[u];
#pragma unroll
                for (int w = 1; w < 8; ++w) x += cells[w * reach + u];
                cells[u] = x;
            }
        __syncthreads();
        for (int u = wave; u < a.rel.n; u += 4) {
            float x = 0.f;
            if (reach > 0 && tiles > 0) {
                const int lo = u == 0 ? 0 : a.rel.edge[u - 1] - a.rel.edge[0] + REL_PAD, hi = u + 1 == a.rel.n ? reach : a.rel.edge[u] - a.rel.edge[0] + REL_PAD;
                for (int d = lo + lane; d < hi; d += 64) x += cells[d];
                x = wave_sum(x);
            }
            if (u == 0) x += (fars[0] + fars[1]) + (fars[2] + fars[3]);
            if (u > 0 && u + 1 == a.rel.n) x += (fars[4] + fars[5]) + (fars[6] + fars[7]);
            if (lane == 0) share[u] = x;
        }
    }

    if (QW == 1) {                                                      // the four waves' sums meet
        float* join = reinterpret_cast<float*>(lds);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<f32x4*>(join + (wave * 32 + (lane & 31)) * (DP + 4) + 32 * k + 8 * e + 4 * half) =
                    f32x4{acc[k][4 * e], acc[k][4 * e + 1], acc[k][4 * e + 2], acc[k][4 * e + 3]};
        __syncthreads();
        const int r = tid >> 3, d0 = (tid & 7) * (DP / 8);
        if (row0 + r >= s.nq) return;
        T* to = dq + (s.q0 + row0 + r) * dq_ld + (int64_t)h * a.dim + d0;
#pragma unroll
        for (int d = 0; d < DP / 8; d += 4) {
            if (d0 + d >= a.dim) break;
            f32x4 x = *reinterpret_cast<f32x4*>(join + r * (DP + 4) + d0 + d);
#pragma unroll
            for (int w = 1; w < 4; ++w) x += *reinterpret_cast<f32x4*>(join + (w * 32 + r) * (DP + 4) + d0 + d);
            x *= a.scale;
            Mma<T>::store4(to + d, x[0], x[1], x[2], x[3]);
        }
        return;
    }
    if (row >= s.nq) return;
    T* to = dq + (s.q0 + row) * dq_ld + (int64_t)h * a.dim + 4 * half;
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * k + 8 * i < a.dim)
                Mma<T>::store4(to + 32 * k + 8 * i, acc[k][4 * i] * a.scale, acc[k][4 * i + 1] * a.scale, acc[k][4 * i + 2] * a.scale,
                               acc[k][4 * i + 3] * a.scale);
}

// One block a head, behind the key side's blocks: thread = (slice of the shares, bucket), slices added in order.
struct BiasShares { const float* part; int64_t shares; float* dbias; };
__device__ __forceinline__ void sum_shares(const BiasShares& x, int n, int heads, int h, float* red) {
    const int slices = BWD_THREADS / n, u = threadIdx.x % n, sl = threadIdx.x / n;
    float y = 0.f;
    if (sl < slices) {
        const float* p = x.part + (int64_t)h * x.shares * n + u;
#pragma unroll 8
        for (int64_t i = sl; i < x.shares; i += slices) y += p[i * n];
    }
    red[threadIdx.x] = y;
    __syncthreads();
    if (sl == 0) {
        for (int w = 1; w < slices; ++w) y += red[w * n + u];
        x.dbias[u * heads + h] = y;
    }
}

// ---- key side ------------------------------------------------------------------------------------------------------------------------
template <typename T, int DP>
struct KeySide {
    static constexpr int QT = sizeof(T) * DP <= 256 ? 64 : 32, TILE = QT * DP;      // queries of a tile
    static constexpr size_t tiles = 2 * 2 * TILE * sizeof(T), stats = 2 * 2 * QT * sizeof(float);
};

template <typename T, int DP>
__global__ __launch_bounds__(BWD_THREADS, (sizeof(T) * DP <= 128 ? 2 : 1)) void attn_bwd_kv_kernel(AttnView a, const float* lse, const float* delta, const T* dout, int64_t dout_ld, T* dk,
                                                                  int64_t dk_ld, T* dv, int64_t dv_ld, int key_blocks, BiasShares shares, int blocks) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using Kd = KeySide<T, DP>;
    constexpr int QT = Kd::QT, TILE = Kd::TILE;
    T *qt = reinterpret_cast<T*>(lds), *gt = qt + 2 * TILE;
    float* stats = reinterpret_cast<float*>(lds + Kd::tiles);           // [buffer][-log2(e) lse, delta][QT]
    float* lut = reinterpret_cast<float*>(lds + Kd::tiles + Kd::stats);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, kv_heads = a.heads / a.group;
    if ((int)blockIdx.x >= blocks) {
        sum_shares(shares, a.rel.n, a.heads, blockIdx.x - blocks, stats);
        return;
    }
    const int kb = blockIdx.x % key_blocks, g = blockIdx.x / key_blocks % kv_heads, b = blockIdx.x / key_blocks / kv_heads;
    const Segment s = load_segment(a, b);
    const int key0 = kb * 128;
    if (key0 >= s.nk) return;
    const int wkey = key0 + wave * 32, key = wkey + (lane & 31);
    const int chunks = a.dim / Tile<T, DP>::PER;
    const float scale = a.scale * LOG2E;
    const int reach = rel_reach(a.rel);
    int32_t* buckets = reinterpret_cast<int32_t*>(lut + reach);         // of every distance
    for (int u = tid; u < reach; u += BWD_THREADS) buckets[u] = bucket_of(a.rel, a.rel.edge[0] - REL_PAD + u);
    const bool on = key < s.nk && (a.keep == nullptr || a.keep[s.k0 + key] != 0);
    RowFrags<T, DP> k, v;
    k.load((const T*)a.k + (s.k0 + key) * a.k_ld + (int64_t)g * a.dim, chunks, on);
    v.load((const T*)a.v + (s.k0 + key) * a.v_ld + (int64_t)g * a.dim, chunks, on);
    const bool all_on = __all(on);
    const bool busy = __any(on);

    // queries that see one of the block's keys: [first, nq)
    const int first = a.causal ? max(0, key0 - s.start) / QT : 0;
    const int tiles = max(0, (s.nq + QT - 1) / QT - first);
    f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
    Staged<T, DP, QT, BWD_THREADS> qs, gs;
    float lv = -INFINITY, dv_ = 0.f;
    auto fetch = [&](int h, int i0) {
        qs.fetch((const T*)a.q + s.q0 * a.q_ld + (int64_t)h * a.dim, a.q_ld, i0, s.nq, chunks, tid);
        gs.fetch(dout + s.q0 * dout_ld + (int64_t)h * a.dim, dout_ld, i0, s.nq, chunks, tid);
        lv = -INFINITY;
        dv_ = 0.f;
        if (tid < QT && i0 + tid < s.nq) {
            const float L = lse[(s.q0 + i0 + tid) * a.heads + h];
            lv = L == -INFINITY ? -INFINITY : -LOG2E * L;               // p = 2^-inf = 0 for a row that saw nothing, and behind the last row
            dv_ = delta[(s.q0 + i0 + tid) * a.heads + h];
        }
    };
    auto store = [&](int buf) {
        qs.store(qt + buf * TILE, tid);
        gs.store(gt + buf * TILE, tid);
        if (tid < QT) {
            stats[buf * 2 * QT + tid] = lv;
            stats[buf * 2 * QT + QT + tid] = dv_;
        }
    };
    for (int h = g * a.group; h < (g + 1) * a.group; ++h) {
        if (tiles == 0) break;
        __syncthreads();
        fetch(h, first * QT);
        for (int u = tid; u < reach; u += BWD_THREADS) lut[u] = LOG2E * a.bias[buckets[u] * a.heads + h];
        store(0);
        __syncthreads();
        for (int t = 0; t < tiles; ++t) {
            const int i0 = (first + t) * QT;
            if (t + 1 < tiles) fetch(h, i0 + QT);
            const T *qb = qt + (t & 1) * TILE, *gb = gt + (t & 1) * TILE;
            const float* st = stats + (t & 1) * 2 * QT;
            if (busy)
#pragma unroll
                for (int n = 0; n < QT / 32; ++n) {
                    const int r0 = i0 + 32 * n;
                    if (r0 >= s.nq) break;
                    const int d0 = wkey - s.start - r0;                 // the wave's first key from the step's first query
                    if (a.causal && d0 - 31 > 0) continue;              // its last query is before the wave's first key
                    const bool near = near_tile(a.rel, d0 - 31, d0 + 31);
                    const float far = a.rel.n > 0 && !near ? LOG2E * a.bias[far_bucket(a.rel, d0 - 31) * a.heads + h] : 0.f;
                    const bool cut = a.causal && d0 + 31 > 0;
                    f32x16 p = scores<T, DP>(qb, 32 * n, k), dp = scores<T, DP>(gb, 32 * n, v);
                    f32x4 ml[4], dl[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ml[i] = *reinterpret_cast<const f32x4*>(st + 32 * n + 8 * i + 4 * half);
                        dl[i] = *reinterpret_cast<const f32x4*>(st + QT + 32 * n + 8 * i + 4 * half);
                    }
                    if (near || cut || !all_on) {
                        const int from = key - s.start - r0;            // first query of the step that sees the key
                        uint32_t seen = !on ? 0u : !cut || from <= 0 ? ~0u : from > 31 ? 0u : ~0u << from;
                        seen >>= 4 * half;
                        const float* tab = lut + (near ? key - s.start - r0 - 4 * half - 27 - a.rel.edge[0] + REL_PAD : 0);
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float x = fmaf(p[r], scale, near ? tab[27 - reg_row(r)] : far) + ml[r >> 2][r & 3];
                            p[r] = (seen >> reg_row(r) & 1) ? __builtin_amdgcn_exp2f(x) : 0.f;
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], scale, far + ml[r >> 2][r & 3]));
                    }
                    const auto wp = Mma<T>::pack(p);
#pragma unroll
                    for (int r = 0; r < 16; ++r) p[r] *= dp[r] - dl[r >> 2][r & 3];
                    const auto wd = Mma<T>::pack(p);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) {
                        av[d] = Mma<T>::template weigh<DP>(gb, 32 * n, 32 * d, wp, av[d]);
                        ak[d] = Mma<T>::template weigh<DP>(qb, 32 * n, 32 * d, wd, ak[d]);
                    }
                }
            if (t + 1 < tiles) store((t + 1) & 1);
            __syncthreads();
        }
    }
    if (key >= s.nk) return;
    if (!on) {                                                          // (0, also where an infinite dout has met the zeros in its place)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) ak[d] = av[d] = f32x16{};
    }
    T* tk = dk + (s.k0 + key) * dk_ld + (int64_t)g * a.dim + 4 * half;
    T* tv = dv + (s.k0 + key) * dv_ld + (int64_t)g * a.dim + 4 * half;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * d + 8 * i < a.dim) {
                Mma<T>::store4(tk + 32 * d + 8 * i, ak[d][4 * i] * a.scale, ak[d][4 * i + 1] * a.scale, ak[d][4 * i + 2] * a.scale, ak[d][4 * i + 3] * a.scale);
                Mma<T>::store4(tv + 32 * d + 8 * i, av[d][4 * i], av[d][4 * i + 1], av[d][4 * i + 2], av[d][4 * i + 3]);
            }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
static int padded(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }
// Rows of a query-side block: short query lists leave three of four row waves idle, so there the waves share the keys instead (not for f32
// heads wider than 64, whose 128-key tiles do not fit the shared memory).
static bool few_rows(const dctr_attention* a) { return a->max_q <= 64 && !(a->dtype == DCTR_TYPE_F32 && a->head_dim > 64); }
static int row_blocks_of(const dctr_attention* a) { return ceil_div(a->max_q, few_rows(a) ? 32 : 128); }

// delta, then the bias gradient's shares
int64_t attn_bwd_workspace(const dctr_attention* a) {
    return 4 * (round_up(a->total_q * a->heads, 4) + (int64_t)a->heads * a->n_seg * row_blocks_of(a) * a->n_buckets);
}

template <typename T, int DP, int QW>
static int launch_q(const dctr_attention* a, const AttnView& v, const void* out, int64_t out_ld, const float* lse, const void* dout, int64_t dout_ld,
                    void* dq, int64_t dq_ld, float* delta, float* part, hipStream_t st) {
    const int row_blocks = row_blocks_of(a);
    const int64_t blocks = (int64_t)row_blocks * a->heads * a->n_seg;
    DCTR_REQUIRE(blocks <= INT32_MAX, "attention: too many blocks for one launch");
    if (blocks == 0) return DCTR_OK;
    const size_t lds = QuerySide<T, DP, QW>::first + sizeof(float) * (9 * rel_reach(a) + 8);
    attn_bwd_q_kernel<T, DP, QW><<<(unsigned)blocks, BWD_THREADS, lds, st>>>(v, (const T*)out, out_ld, lse, (const T*)dout, dout_ld, (T*)dq, dq_ld, delta, part,
                                                                             row_blocks);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

template <typename T, int DP>
static int launch_bwd(const dctr_attention* a, const AttnView& v, const AttnGrads& x, float* ws, hipStream_t st) {
    float *delta = ws, *part = x.dbias != nullptr ? ws + round_up(a->total_q * a->heads, 4) : nullptr;
    constexpr bool wide = sizeof(T) == 4 && DP > 64;
    if (!wide && few_rows(a))
        DCTR_TRY((launch_q<T, DP, wide ? 4 : 1>(a, v, x.out, x.out_ld, x.lse, x.dout, x.dout_ld, x.dq, x.dq_ld, delta, part, st)));
    else
        DCTR_TRY((launch_q<T, DP, 4>(a, v, x.out, x.out_ld, x.lse, x.dout, x.dout_ld, x.dq, x.dq_ld, delta, part, st)));
    const int key_blocks = ceil_div(a->max_k, 128);
    const int64_t blocks = (int64_t)key_blocks * a->kv_heads * a->n_seg;
    DCTR_REQUIRE(blocks + a->heads <= INT32_MAX, "attention: too many blocks for one launch");
    const int sums = part != nullptr ? a->heads : 0;
    if (blocks + sums == 0) return DCTR_OK;
    const size_t lds = KeySide<T, DP>::tiles + std::max<size_t>(KeySide<T, DP>::stats, BWD_THREADS * sizeof(float)) + sizeof(float) * 2 * rel_reach(a);
    attn_bwd_kv_kernel<T, DP><<<(unsigned)(blocks + sums), BWD_THREADS, lds, st>>>(v, x.lse, delta, (const T*)x.dout, x.dout_ld, (T*)x.dk, x.dk_ld, (T*)x.dv,
                                                                                   x.dv_ld, key_blocks,
                                                                                   BiasShares{part, (int64_t)a->n_seg * row_blocks_of(a), x.dbias}, (int)blocks);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

template <typename T>
static int by_width(const dctr_attention* a, const AttnView& v, const AttnGrads& x, float* ws, hipStream_t st) {
    switch (padded(a->head_dim)) {
        case 32: return launch_bwd<T, 32>(a, v, x, ws, st);
        case 64: return launch_bwd<T, 64>(a, v, x, ws, st);
        default: return launch_bwd<T, 128>(a, v, x, ws, st);
    }
}

int attn_bwd(const dctr_attention* a, const AttnView& v, const AttnGrads& x, float* ws, hipStream_t st) {
    return a->dtype == DCTR_TYPE_F32 ? by_width<float>(a, v, x, ws, st) : by_width<__bf16>(a, v, x, ws, st);
}

}  // namespace dctr
