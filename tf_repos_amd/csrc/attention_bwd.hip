// Backward of the ragged cross attention (attention.h: formulas; seq_mma.h: the matrix blocks): scores and p are formed again from lse, nothing
// of size queries x keys is stored.  Two kernels, each summing in registers over the axis that it walks, so no atomics meet in memory:
//   query side  S^T = K Q^T and dP^T = V dO^T by 32 queries a wave, dQ^T += K^T dS^T; delta = <do, out> on the way, kept for the key side;
//               the bias gradient's sums over a tile's diagonals
//   key side    S = Q K^T and dP = dO V^T by 32 keys a wave, over the queries of every head of the group: dV^T += dO^T P, dK^T += Q^T dS
// p and ds are rounded to bf16 for the second products of bf16 arrays, half a step each, as the results are; everything that is summed is f32.  Where a
// wave has items or tiles of its own and heads are up to 64 wide, ds (and p on the key side) keep what is rounded off as a second plane (FINE): rounding them
// makes sqrt(2) times the error of rounding the results, and small calls scatter above that, but wait for latencies more than for the matrix unit (bf16
// with gradients, 512 x (<= 40 x 200), 4 heads of 16: 70 -> 72 us; 300 x (<= 40 x 90), 8 heads of 64: 66 -> 71; wider heads would spill).
// Measured on 16 segments of 1024 x 1024, 8 heads, bf16: query side 92 us at 64 wide (747 TF/s of its four products) and 235 at 128 (584), key side 98
// (703) and 240 (573): at 128 the accumulators leave one wave a SIMD, whose exponents then run beside nothing.  f32 in planes at 64: 272 and 428 us.
// 512 segments of up to 40 x 200, 4 heads of 16, f32 with a bias: 37 and 35 us, the latency of each wave's few tiles and of its bias tables.
#include <cmath>

#include "attention.h"

namespace dctr {

constexpr int BWD_THREADS = 256;

// -log2(e) lse, the addend of a row's exponents: -inf where there is nothing to form again.  A row that saw nothing has lse = -inf.  One that saw only keys of
// biases like -1e9 has an lse whose last place is worth more than its weights (2^-24 of 1e7 is 0.6): exponents off by whole units, up to
// infinite weights, would reach the gradients of every key it sees, so it passes on none.
constexpr float LEAST_LSE = -1e7f;
__device__ __forceinline__ float minus_log2(float lse) { return lse < LEAST_LSE ? -INFINITY : -LOG2E * lse; }

// Query-side forms: ROWS a block's waves take 32 rows each and share 64-key tiles; SPLIT the waves take 32-key tiles of their own of the same 32
// rows and add up at the end; SOLO a wave has 32 rows to itself.
enum { ROWS = 0, SPLIT = 1, SOLO = 2 };

template <typename T, int DP, int FORM>
struct QuerySide {
    using M = AttnKind<T, DP>;
    static constexpr int NB = FORM == ROWS && attn_width<T, DP> <= 256 ? 2 : 1, KEYS = 32 * NB, BUFS = FORM == ROWS || sizeof(T) == 2 ? 2 : 1, THREADS = FORM == ROWS ? 256 : 64;
    static constexpr int HIDDEN = (FORM == ROWS ? 1 : 4) * BUFS * KEYS, TILE = KEYS * Tile<M, DP>::STRIDE, ITEM_ROWS = FORM == ROWS ? 128 : 32;
    static constexpr size_t tiles = (FORM == ROWS ? 1 : 4) * 2 * BUFS * KEYS * attn_width<T, DP>, join = FORM == SPLIT ? 4 * 32 * (DP + 4) * sizeof(float) : 0;
    static constexpr size_t first = tiles > join ? tiles : join;
};

// Sums of a 32 x 32 block of ds by distance, into the wave's cells (`cells`: that of the block's first key and first query).  A block's rows go to
// shared memory each shifted by its own number, so that equal distances stand in one column; the columns' sums are then added to the cells.  16 queries
// at a time: 16 x 48 floats, of which a row always writes the same 32 and the rest stays zero.  (Float atomics to the cells took 64 and more cycles an
// instruction: 104 us of a 254 us pass over 8 x 2048 causal steps, 8 heads.)  The order of every sum is the program's.
constexpr int SKEW = 16 * 48;
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ void add_diagonals(float* skew, const f32x16& x, float* cells) {
    const int lane = threadIdx.x & 63, half = lane >> 5, row = lane & 15, quad = lane & 15, group = lane >> 4;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        wave_order();
        if ((group & 1) == pass) {
            float* to = skew + row * 47 + 15 + 4 * half;
#pragma unroll
            for (int r = 0; r < 16; ++r) to[reg_row(r)] = x[r];
        }
        wave_order();
        f32x4 sum = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += *reinterpret_cast<const f32x4*>(skew + (4 * group + j) * 48 + 4 * min(quad, 11));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const Halves y = row_pair(sum[e]);
            sum[e] = both_sum(y.lo + y.hi);
        }
        const float mine = group == 0 ? sum[0] : group == 1 ? sum[1] : group == 2 ? sum[2] : sum[3];
        const int c = 4 * quad + group;
        if (c < 47) cells[c - 15 - 16 * pass] += mine;
    }
}

// part: [head][segment * row_blocks + row block][n_buckets] shares of the bias gradient, or null; delta [total_q, heads]
template <typename T, int DP, int FORM>
__global__ __launch_bounds__(BWD_THREADS, (attn_width<T, DP> <= 192 || (FORM == ROWS && attn_width<T, DP> == 384) ? 2 : 1)) void attn_bwd_q_kernel(AttnView a, const T* out, int64_t out_ld, const float* lse, const T* dout, int64_t dout_ld,
                                                                 T* dq, int64_t dq_ld, float* delta, float* part, int row_blocks) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using Q = QuerySide<T, DP, FORM>;
    constexpr int NB = Q::NB, TILE = Q::TILE;
    // For bf16 <do, out> is off by the rounding of `out`, an error that all of a row's ds share.  The walk sums p dp over every key, which is the
    // same number unrounded, and P K besides: dq is put right with (rounded - unrounded) P K at the end, the key side and the bias gradient take
    // the unrounded one.  (Measured: the relative error of dq and dk 0.0030 -> 0.0023 at 777 x 1531 x 128.)
    using M = AttnKind<T, DP>;
    using S = typename Mma<M>::Store;
    constexpr bool ROUNDED = Mma<M>::ROUNDS;
    constexpr bool OWN = FORM != ROWS;                                  // tiles of a wave's own
    constexpr bool FINE = ROUNDED && OWN && DP <= 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    S* kt = reinterpret_cast<S*>(lds) + (OWN ? wave * 2 * Q::BUFS * TILE : 0);
    S* vt = kt + Q::BUFS * TILE;
    const int64_t items = (int64_t)row_blocks * a.heads * a.n_seg, at_item = FORM == SOLO ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    const int item = (int)min(at_item, items - 1);
    // Row block slowest.  ROWS, SPLIT: the last first, which a causal mask makes the longest; SOLO: a block's waves are alike long.
    const Item it = item_of(item, a.heads, a.n_seg);
    const int h = it.head, b = it.seg, rb = FORM == SOLO ? it.nth : row_blocks - 1 - it.nth;
    const Segment s = load_segment(a, b);
    const int row0 = rb * Q::ITEM_ROWS;
    float* share = part != nullptr ? part + ((int64_t)h * a.n_seg * row_blocks + (int64_t)b * row_blocks + rb) * a.rel.n : nullptr;
    if (at_item >= items) return;                                       // (the forms that share have no such block)
    if (row0 >= s.nq) {
        if (share != nullptr)
            for (int u = FORM == SOLO ? lane : tid; u < a.rel.n; u += FORM == SOLO ? 64 : BWD_THREADS) share[u] = 0.f;
        return;
    }
    // one wave: what it wrote is what it reads, in program order; a block: a barrier
    auto meet = [&] {
        if (OWN) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
        }
    };
    const int wrow = row0 + (OWN ? 0 : 32 * wave), row = wrow + (lane & 31);
    const int chunks = a.dim / Tile<M, DP>::PER;
    const float scale = a.scale * LOG2E;
    const int reach = rel_reach(a.rel);
    // skewed blocks, a wave each; SOLO: every wave's own table and cells; else one table, [4 waves][reach] cells; 2 x 4 far sums
    float* hidden = reinterpret_cast<float*>(lds + Q::first) + (OWN ? wave * Q::BUFS * Q::KEYS : 0);     // [buffer][KEYS]
    float* skew = reinterpret_cast<float*>(lds + Q::first) + Q::HIDDEN + wave * SKEW;
    float* lut = reinterpret_cast<float*>(lds + Q::first) + Q::HIDDEN + 4 * SKEW + (FORM == SOLO ? wave * 2 * reach : 0);
    float* cells = lut + reach;
    float* mine = cells + (FORM == SOLO ? 0 : wave * reach);
    const int loader = OWN ? lane : tid;

    // The matrix unit's sums of bf16 products lean to one side by a small part of a half step.  A row's <do, out> does not share that lean, so the bias
    // gradient would add it up over thousands of rows (relative error 1.8e-6 over 512 segments of 40 x 200 by 4 heads of 16): every other row has its dO
    // negated and dP's sign turned back, which leaves 3e-7.  (bf16 arrays: delta comes from the same dP, below.)
    const float sign = ROUNDED || !(lane & 1) ? 1.f : -1.f;
    RowFrags<M, DP> q, go;
    q.load((const T*)a.q + (s.q0 + row) * a.q_ld + (int64_t)h * a.dim, chunks, row < s.nq);
    go.load(dout + (s.q0 + row) * dout_ld + (int64_t)h * a.dim, chunks, row < s.nq);
    float dl = 0.f, minus_lse = -INFINITY;                              // (a row that saw nothing: p = 2^-inf = 0)
    {
        RowFrags<M, DP> o;
        o.load(out + (s.q0 + row) * out_ld + (int64_t)h * a.dim, chunks, row < s.nq);
#pragma unroll
        for (int c = 0; c < RowFrags<M, DP>::STEPS; ++c) dl = Mma<M>::product(go.c[c], o.c[c], dl);
        dl = both_sum(dl);
        if (!ROUNDED && (lane & 1)) go.negate();
        if (row < s.nq) {
            minus_lse = minus_log2(lse[(s.q0 + row) * a.heads + h]);
            if (!ROUNDED && (FORM != SPLIT || wave == 0) && half == 0) delta[(s.q0 + row) * a.heads + h] = dl;
        }
    }

    const T* K = (const T*)a.k + s.k0 * a.k_ld + (int64_t)(h / a.group) * a.dim;
    const T* V = (const T*)a.v + s.k0 * a.v_ld + (int64_t)(h / a.group) * a.dim;
    int keys = s.nk;
    if (a.causal) keys = max(0, min(keys, s.start + min(row0 + Q::ITEM_ROWS, s.nq)));
    const int tiles = (keys + Q::KEYS - 1) / Q::KEYS;
    const RelRange range = rel_range(a.rel, (int64_t)0 - s.start - (row0 + Q::ITEM_ROWS - 1), (int64_t)tiles * Q::KEYS - 1 - s.start - row0);
    const bool busy = wrow < s.nq;
    const int wend = a.causal ? s.start + min(wrow + 32, s.nq) : keys;

    FarBias fars = far_bias(a, h);
    f32x16 acc[DP / 32] = {}, pk[ROUNDED ? DP / 32 : 1] = {};
    float far_ds[2] = {0.f, 0.f}, far_p[2] = {0.f, 0.f}, pdp = 0.f;     // [below the first boundary, from the last one on]
    std::conditional_t<Q::BUFS == 2, Loader<M, DP, Q::KEYS, Q::THREADS>, Staged<M, DP, Q::KEYS, Q::THREADS>> ks, vs;
    uint64_t bits = 0;                                                  // kept keys of the tile
    uint8_t kept = 0;
    auto fetch = [&](int j0, int buf) __attribute__((always_inline)) {
        ks.fetch(kt + buf * TILE, K, a.k_ld, j0, s.nk, chunks, loader);
        vs.fetch(vt + buf * TILE, V, a.v_ld, j0, s.nk, chunks, loader);
        kept = lane < Q::KEYS && j0 + lane < s.nk ? (a.keep != nullptr ? a.keep[s.k0 + j0 + lane] : 1) : 0;
    };
    auto land = [&](int buf) __attribute__((always_inline)) {
        bits = __ballot(kept != 0);
        if (loader < Q::KEYS) hidden[buf * Q::KEYS + loader] = kept != 0 ? 0.f : -INFINITY;
        ks.land(kt + buf * TILE, loader, bits);
        vs.land(vt + buf * TILE, loader, bits);
    };
    // cell of the distance between a block's first key and the wave's first query
    auto block_cell = [&](int key) { return key - s.start - wrow - a.rel.edge[0] + REL_PAD; };
    // p and dp of the tile at j0; returns whether it is near, `side` its far side otherwise
    auto pair = [&](const S* kb, const S* vb, const float* hide, int j0, uint64_t now, f32x16 (&p)[NB], f32x16 (&dp)[NB], int& cell, int& side) {
        const int d0 = j0 - s.start - wrow;                             // the tile's first key from the wave's first query
        const bool near = near_tile(a.rel, d0 - 31, d0 + 32 * NB - 1);
        const int fb = a.rel.n > 0 && !near ? far_bucket(a.rel, d0 - 31) : 0;
        const float far = near ? 0.f : fb > 0 ? fars.behind : fars.before;
        side = fb > 0;
        cell = near ? d0 - (lane & 31) + 4 * half - a.rel.edge[0] + REL_PAD : 0;
        const bool cut = a.causal && d0 + 32 * NB - 1 > 0;
        uint64_t seen = now;
        if (cut) {
            const int last = row + s.start - j0;
            seen &= last < 0 ? 0ull : last >= 63 ? ~0ull : (2ull << last) - 1;
        }
        seen = lane_bits(seen);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            p[k] = scores<M, DP, (attn_width<T, DP> > 192)>(kb, 32 * k, q);
            dp[k] = scores<M, DP, (attn_width<T, DP> > 192)>(vb, 32 * k, go);
        }
        if (near || cut) {
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 32 * k + reg_row(r);
                    const float x = fmaf(p[k][r], scale, near ? lut[cell + at] : far) + minus_lse;
                    p[k][r] = (seen >> at & 1) ? __builtin_amdgcn_exp2f(x) : 0.f;
                }
        } else if (now != ~0ull >> (64 - Q::KEYS)) {
            const float off = far + minus_lse;
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 x = hidden4(hide, k, i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[k][4 * i + j] = __builtin_amdgcn_exp2f(fmaf(p[k][4 * i + j], scale, x[j]) + off);
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
    // one walk over the tiles; `second`: only the near ones, for their cells
    auto walk = [&](bool second) __attribute__((always_inline)) {
        int t = 0, last = tiles;
        if (second) {                                                   // tiles before and behind these are far for every row of the block
            const int64_t from = (int64_t)a.rel.edge[0] + s.start + row0 - (Q::KEYS - 1);
            const int64_t to = (int64_t)a.rel.edge[a.rel.n - 2] + s.start + row0 + Q::ITEM_ROWS - 1;      // (`near` goes by whole waves too)
            t = from <= 0 ? 0 : (int)min((int64_t)tiles, from / Q::KEYS);
            last = to <= 0 ? 0 : (int)min((int64_t)tiles, (to + Q::KEYS - 1) / Q::KEYS);
        }
        constexpr int STEP = FORM == SPLIT ? 4 : 1;
        if (FORM == SPLIT) t += wave;
        meet();
        if (t < last) fetch(t * Q::KEYS, 0);
        if (!second) {                                                  // under the first tile's loads
            for (int u = range.lo + (FORM == SOLO ? lane : tid); u < range.hi; u += FORM == SOLO ? 64 : BWD_THREADS)
                lut[u] = LOG2E * a.bias[bucket_of(a.rel, a.rel.edge[0] - REL_PAD + u) * a.heads + h];
            if (part != nullptr)
                for (int u = range.lo + lane; u < range.hi; u += 64) mine[u] = 0.f;
            if (part != nullptr && reach > 0)
                for (int u = lane; u < SKEW; u += 64) skew[u] = 0.f;
            if (FORM == SPLIT) __syncthreads();
            q.wait();
            go.wait();
            settle(minus_lse);
            settle(dl);
            settle(fars.before);
            settle(fars.behind);
        }
        if (t < last) land(0);
        meet();
        for (int n = 0; t < last; t += STEP, ++n) {
            const int j0 = t * Q::KEYS, buf = Q::BUFS == 2 ? n & 1 : 0;
            const uint64_t now = bits;
            if (t + STEP < last) fetch(j0 + STEP * Q::KEYS, Q::BUFS == 2 ? (n + 1) & 1 : 0);
            if (busy && j0 < wend) {
                const S *kb = kt + buf * TILE, *vb = vt + buf * TILE;
                f32x16 p[NB], dp[NB];
                int cell, side;
                const bool near = pair(kb, vb, hidden + buf * Q::KEYS, j0, now, p, dp, cell, side);
                if (!second) {
                    if (ROUNDED) {
                        float x[2] = {0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < NB; ++k)
#pragma unroll
                            for (int r = 0; r < 16; ++r) x[r & 1] = fmaf(p[k][r], dp[k][r], x[r & 1]);
                        pdp += x[0] + x[1];
                        if (part != nullptr && !near) {
                            float y[2] = {0.f, 0.f};
#pragma unroll
                            for (int k = 0; k < NB; ++k)
#pragma unroll
                                for (int r = 0; r < 16; ++r) y[r & 1] += p[k][r];
                            far_ds[0] += side ? 0.f : x[0] + x[1];
                            far_ds[1] += side ? x[0] + x[1] : 0.f;
                            far_p[0] += side ? 0.f : y[0] + y[1];
                            far_p[1] += side ? y[0] + y[1] : 0.f;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < NB; ++k) {
                        if (ROUNDED) {
                            const auto w = Mma<M>::pack(p[k]);
#pragma unroll
                            for (int d = 0; d < DP / 32; ++d)
                                pk[ROUNDED ? d : 0] = Mma<M>::template weigh<DP>(kb, 32 * k, 32 * d, w, pk[ROUNDED ? d : 0]);
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) p[k][r] *= ROUNDED ? dp[k][r] - dl : fmaf(dp[k][r], sign, -dl);
                        if (!ROUNDED && part != nullptr) {
                            if (near) {
                                add_diagonals(skew, p[k], mine + block_cell(j0 + 32 * k));
                            } else {
                                float x[2] = {0.f, 0.f};
#pragma unroll
                                for (int r = 0; r < 16; ++r) x[r & 1] += p[k][r];
                                far_ds[0] += side ? 0.f : x[0] + x[1];
                                far_ds[1] += side ? x[0] + x[1] : 0.f;
                            }
                        }
                        const auto w = Mma<M>::pack(p[k]);
                        if constexpr (FINE) {
                            const auto rest = Mma<M>::pack_rest(p[k], w);
#pragma unroll
                            for (int d = 0; d < DP / 32; ++d) acc[d] = Mma<M>::template weigh<DP>(kb, 32 * k, 32 * d, rest, acc[d]);
                        }
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d) acc[d] = Mma<M>::template weigh<DP>(kb, 32 * k, 32 * d, w, acc[d]);
                    }
                } else if (near) {
#pragma unroll
                    for (int k = 0; k < NB; ++k) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) p[k][r] *= ROUNDED ? dp[k][r] - dl : fmaf(dp[k][r], sign, -dl);
                        add_diagonals(skew, p[k], mine + block_cell(j0 + 32 * k));
                    }
                }
            }
            if (Q::BUFS == 1) meet();
            if (t + STEP < last) land(Q::BUFS == 2 ? (n + 1) & 1 : 0);
            meet();
        }
    };
    walk(false);

    if (ROUNDED) {
        float exact = both_sum(pdp);
        if (FORM == SPLIT) {                                            // the waves hold different keys of the same rows
            float* sums = reinterpret_cast<float*>(lds);
            __syncthreads();
            if (half == 0) sums[wave * 32 + lane] = exact;
            __syncthreads();
            exact = (sums[lane & 31] + sums[32 + (lane & 31)]) + (sums[64 + (lane & 31)] + sums[96 + (lane & 31)]);
            __syncthreads();
        }
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] += (dl - exact) * pk[ROUNDED ? d : 0];
        dl = exact;
        if ((FORM != SPLIT || wave == 0) && half == 0 && row < s.nq) delta[(s.q0 + row) * a.heads + h] = dl;
    }
    if (part != nullptr) {
        if (ROUNDED && a.rel.n > 1) walk(true);                         // the near tiles again, for their distances' sums
        // the outer buckets: the far tiles' sums and the wave's own cells of the near ones
        float far_sum[2];
#pragma unroll
        for (int side = 0; side < 2; ++side) far_sum[side] = ROUNDED ? fmaf(-dl, far_p[side], far_ds[side]) : far_ds[side];
        const int inner = REL_PAD, outer = reach - REL_PAD;             // cells [inner, outer) are of the buckets between
        wave_order();
        for (int u = range.lo + lane; u < min(range.hi, inner); u += 64) far_sum[0] += mine[u];
        for (int u = max(range.lo, outer) + lane; u < range.hi; u += 64) far_sum[1] += mine[u];
#pragma unroll
        for (int side = 0; side < 2; ++side) far_sum[side] = wave_sum(far_sum[side]);
        const int lo = max(range.lo, inner), hi = min(range.hi, outer);
        if (FORM != SOLO) {
            float* both = cells + 4 * reach;
            if (lane == 0) {
                both[wave] = far_sum[0];
                both[4 + wave] = far_sum[1];
            }
            __syncthreads();
            far_sum[0] = (both[0] + both[1]) + (both[2] + both[3]);
            far_sum[1] = (both[4] + both[5]) + (both[6] + both[7]);
            for (int u = lo + tid; u < hi; u += BWD_THREADS)
                cells[u] = (cells[u] + cells[reach + u]) + (cells[2 * reach + u] + cells[3 * reach + u]);
            __syncthreads();
        }
        if (FORM == SOLO ? lane == 0 : tid == 0) {
            share[0] = far_sum[0];
            if (a.rel.n > 1) share[a.rel.n - 1] = far_sum[1];
        }
        // sixteen lanes a bucket
        for (int u0 = FORM == SOLO ? 1 : 1 + 4 * wave; u0 < a.rel.n - 1; u0 += FORM == SOLO ? 4 : 16) {
            int edge[5];
#pragma unroll
            for (int i = 0; i < 5; ++i) edge[i] = min(a.rel.edge[min(u0 - 1 + i, a.rel.n - 2)] - a.rel.edge[0] + REL_PAD, hi);
            const int g = lane >> 4;
            const int from = max(lo, g == 0 ? edge[0] : g == 1 ? edge[1] : g == 2 ? edge[2] : edge[3]), to = g == 0 ? edge[1] : g == 1 ? edge[2] : g == 2 ? edge[3] : edge[4];
            float x = 0.f;
            for (int d = from + (lane & 15); d < to; d += 16) x += cells[d];
            x = row_sum(x);
            if ((lane & 15) == 0 && u0 + g < a.rel.n - 1) share[u0 + g] = x;
        }
    }

    if (FORM == SPLIT) {                                                // the four waves' sums meet
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
            Mma<M>::store4(to + d, x[0], x[1], x[2], x[3]);
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
                Mma<M>::store4(to + 32 * k + 8 * i, acc[k][4 * i] * a.scale, acc[k][4 * i + 1] * a.scale, acc[k][4 * i + 2] * a.scale,
                               acc[k][4 * i + 3] * a.scale);
}

// One block a head, before the key side's blocks: thread = (slice of the shares, bucket), slices added in order.
struct BiasShares { const float* part; int64_t shares; float* dbias; };
__device__ __forceinline__ void sum_shares(const BiasShares& x, int n, int heads, int h, float* red) {
    const int slices = BWD_THREADS / n, u = threadIdx.x % n, sl = threadIdx.x / n;
    double y = 0.;                                                      // (thousands of shares)
    if (sl < slices) {
        const float* p = x.part + (int64_t)h * x.shares * n + u;
#pragma unroll 8
        for (int64_t i = sl; i < x.shares; i += slices) y += p[i * n];
    }
    red[threadIdx.x] = (float)y;
    __syncthreads();
    if (sl == 0) {
        for (int w = 1; w < slices; ++w) y += red[w * n + u];
        x.dbias[u * heads + h] = (float)y;
    }
}

// ---- key side ------------------------------------------------------------------------------------------------------------------------
// Key-side forms: KEY_ROWS a block's waves take 32 keys each and share the tiles of queries; KEY_SPLIT the waves take 32-query tiles of their own for
// the same 32 keys and add up at the end; KEY_SOLO a wave has 32 keys to itself.
enum { KEY_ROWS = 0, KEY_SPLIT = 1, KEY_SOLO = 2 };
template <typename T, int DP, int FORM>
struct KeySide {
    using M = AttnKind<T, DP>;
    static constexpr bool OWN = FORM != KEY_ROWS;
    static constexpr int QT = !OWN && attn_width<T, DP> <= 256 ? 64 : 32, TILE = QT * Tile<M, DP>::STRIDE, THREADS = OWN ? 64 : 256;      // queries of a tile
    static constexpr int BUFS = !OWN || sizeof(T) == 2 ? 2 : 1;         // (planes pass through registers: there the other waves cover the loads)
    static constexpr size_t tiles = (OWN ? 4 : 1) * 2 * BUFS * QT * attn_width<T, DP>, stats = (OWN ? 4 : 1) * BUFS * 2 * QT * sizeof(float);
    static_assert(FORM != KEY_SPLIT || tiles >= 4 * 32 * (DP + 4) * sizeof(float), "the waves' sums meet in the tiles' place");
};

template <typename T, int DP, int FORM>
__global__ __launch_bounds__(BWD_THREADS, (attn_width<T, DP> <= 192 ? 2 : 1)) void attn_bwd_kv_kernel(AttnView a, const float* lse, const float* delta, const T* dout,
                                                                                                   int64_t dout_ld, T* dk, int64_t dk_ld, T* dv, int64_t dv_ld,
                                                                                                   int key_blocks, BiasShares shares, int sums) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    using Kd = KeySide<T, DP, FORM>;
    using M = AttnKind<T, DP>;
    using S = typename Mma<M>::Store;
    constexpr int QT = Kd::QT, TILE = Kd::TILE, BUFS = Kd::BUFS, STEP = FORM == KEY_SPLIT ? 4 : 1;
    constexpr bool OWN = Kd::OWN, FINE = Mma<M>::ROUNDS && OWN && DP <= 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, kv_heads = a.heads / a.group, loader = OWN ? lane : tid;
    S* qt = reinterpret_cast<S*>(lds) + (OWN ? wave * 2 * BUFS * TILE : 0);
    S* gt = qt + BUFS * TILE;
    float* stats = reinterpret_cast<float*>(lds + Kd::tiles) + (OWN ? wave * BUFS * 2 * QT : 0);  // [buffer][-log2(e) lse, delta][QT]
    if ((int)blockIdx.x < sums) {                                       // (first: behind the others they would be the launch's tail)
        sum_shares(shares, a.rel.n, a.heads, blockIdx.x, reinterpret_cast<float*>(lds));
        return;
    }
    const int block = blockIdx.x - sums;
    const int64_t items = (int64_t)key_blocks * kv_heads * a.n_seg, at_item = FORM == KEY_SOLO ? (int64_t)block * 4 + wave : block;
    if (at_item >= items) return;                                       // (KEY_SOLO has no barriers)
    const Item it = item_of((int)at_item, kv_heads, a.n_seg);           // (under a causal mask the first key blocks are the longest)
    const int g = it.head, b = it.seg, kb = it.nth;
    const Segment s = load_segment(a, b);
    const int key0 = kb * (OWN ? 32 : 128);
    if (key0 >= s.nk) return;
    const int wkey = key0 + (OWN ? 0 : wave * 32), key = wkey + (lane & 31);
    const int chunks = a.dim / Tile<M, DP>::PER;
    const float scale = a.scale * LOG2E;
    const int reach = rel_reach(a.rel), first_u = OWN ? lane : tid, step_u = Kd::THREADS;
    float* lut = reinterpret_cast<float*>(lds + Kd::tiles + Kd::stats) + (OWN ? wave * 2 * reach : 0);
    int32_t* buckets = reinterpret_cast<int32_t*>(lut + reach);         // of every distance
    auto meet = [&] {
        if (OWN) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
        }
    };
    const bool on = key < s.nk && (a.keep == nullptr || a.keep[s.k0 + key] != 0);
    RowFrags<M, DP> k, v;
    k.load((const T*)a.k + (s.k0 + key) * a.k_ld + (int64_t)g * a.dim, chunks, on);
    v.load((const T*)a.v + (s.k0 + key) * a.v_ld + (int64_t)g * a.dim, chunks, on);
    const bool busy = __any(on);

    // queries that see one of the block's keys: [first, nq)
    const int first = a.causal ? max(0, key0 - s.start) / QT : 0;
    const int tiles = max(0, (s.nq + QT - 1) / QT - first);
    const RelRange range = rel_range(a.rel, (int64_t)key0 - s.start - ((int64_t)(first + tiles) * QT - 1), (int64_t)key0 + (OWN ? 31 : 127) - s.start - (int64_t)first * QT);
    for (int u = range.lo + first_u; u < range.hi; u += step_u) buckets[u] = bucket_of(a.rel, a.rel.edge[0] - REL_PAD + u);
    f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
    std::conditional_t<BUFS == 2, Loader<M, DP, QT, Kd::THREADS>, Staged<M, DP, QT, Kd::THREADS>> qs, gs;
    float lv = -INFINITY, dv_ = 0.f;                                    // as loaded: nothing waits for them before the tile lands
    auto fetch = [&](int h, int i0, int buf) {
        qs.fetch(qt + buf * TILE, (const T*)a.q + s.q0 * a.q_ld + (int64_t)h * a.dim, a.q_ld, i0, s.nq, chunks, loader);
        gs.fetch(gt + buf * TILE, dout + s.q0 * dout_ld + (int64_t)h * a.dim, dout_ld, i0, s.nq, chunks, loader);
        lv = -INFINITY;
        dv_ = 0.f;
        if (loader < QT && i0 + loader < s.nq) {
            lv = lse[(s.q0 + i0 + loader) * a.heads + h];
            dv_ = delta[(s.q0 + i0 + loader) * a.heads + h];
        }
    };
    auto land = [&](int i0, int buf) {
        qs.land(qt + buf * TILE, loader, first_rows(s.nq - i0));
        gs.land(gt + buf * TILE, loader, first_rows(s.nq - i0));
        if (loader < QT) {
            stats[buf * 2 * QT + loader] = minus_log2(lv);              // p = 2^-inf = 0 for a row that saw nothing, and behind the last row
            stats[buf * 2 * QT + QT + loader] = dv_;
        }
    };
    for (int h = g * a.group; h < (g + 1) * a.group; ++h) {
        if (tiles == 0) break;
        int t = FORM == KEY_SPLIT ? wave : 0;
        meet();
        if (t < tiles) fetch(h, (first + t) * QT, 0);
        for (int u = range.lo + first_u; u < range.hi; u += step_u) lut[u] = LOG2E * a.bias[buckets[u] * a.heads + h];
        FarBias fars = far_bias(a, h);
        k.wait();
        v.wait();
        settle(fars.before);
        settle(fars.behind);
        if (t < tiles) land((first + t) * QT, 0);
        meet();
        for (int turn = 0; t < tiles; t += STEP, ++turn) {
            const int i0 = (first + t) * QT, then = i0 + STEP * QT, buf = BUFS == 2 ? turn & 1 : 0;
            const bool more = t + STEP < tiles;
            if (BUFS == 2 && more) fetch(h, then, buf ^ 1);
            const S *qb = qt + buf * TILE, *gb = gt + buf * TILE;
            const float* st = stats + buf * 2 * QT;
            if (busy)
#pragma unroll
                for (int n = 0; n < QT / 32; ++n) {
                    const int r0 = i0 + 32 * n;
                    if (r0 >= s.nq) break;
                    const int d0 = wkey - s.start - r0;                 // the wave's first key from the step's first query
                    if (a.causal && d0 - 31 > 0) continue;              // its last query is before the wave's first key
                    const bool near = near_tile(a.rel, d0 - 31, d0 + 31);
                    const float far = !on ? -INFINITY : near ? 0.f : far_bucket(a.rel, d0 - 31) > 0 ? fars.behind : fars.before;      // a key: a lane
                    const bool cut = a.causal && d0 + 31 > 0;
                    f32x16 p = scores<M, DP, (attn_width<T, DP> > 192)>(qb, 32 * n, k), dp = scores<M, DP>(gb, 32 * n, v);
                    f32x4 ml[4], dl[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ml[i] = *reinterpret_cast<const f32x4*>(st + 32 * n + 8 * i + 4 * half);
                        dl[i] = *reinterpret_cast<const f32x4*>(st + QT + 32 * n + 8 * i + 4 * half);
                    }
                    if (near || cut) {
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
                    const auto wp = Mma<M>::pack(p);
                    if constexpr (FINE) {
                        const auto rest = Mma<M>::pack_rest(p, wp);
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d) {
                            av[d] = Mma<M>::template weigh<DP>(gb, 32 * n, 32 * d, rest, av[d]);
                            av[d] = Mma<M>::template weigh<DP>(gb, 32 * n, 32 * d, wp, av[d]);
                        }
                        __builtin_amdgcn_sched_barrier(0);              // (p's planes are done with before ds's are made: registers)
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) p[r] *= dp[r] - dl[r >> 2][r & 3];
                    const auto wd = Mma<M>::pack(p);
                    if constexpr (FINE) {
                        const auto rest = Mma<M>::pack_rest(p, wd);
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d) ak[d] = Mma<M>::template weigh<DP>(qb, 32 * n, 32 * d, rest, ak[d]);
                    }
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) {
                        if constexpr (!FINE) av[d] = Mma<M>::template weigh<DP>(gb, 32 * n, 32 * d, wp, av[d]);
                        ak[d] = Mma<M>::template weigh<DP>(qb, 32 * n, 32 * d, wd, ak[d]);
                    }
                }
            if (BUFS == 1) meet();
            if (more) {
                if (BUFS == 1) fetch(h, then, 0);
                land(then, BUFS == 2 ? buf ^ 1 : 0);
            }
            meet();
        }
    }
    if (!on) {                                                          // (0, also where an infinite dout has met the zeros in its place)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) ak[d] = av[d] = f32x16{};
    }
    if (FORM == KEY_SPLIT) {                                            // the four waves' sums meet, dk's and then dv's
        float* join = reinterpret_cast<float*>(lds);
        const int r = tid >> 3, c0 = (tid & 7) * (DP / 8);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x16& x = which == 0 ? ak[d] : av[d];
                    *reinterpret_cast<f32x4*>(join + (wave * 32 + (lane & 31)) * (DP + 4) + 32 * d + 8 * e + 4 * half) =
                        f32x4{x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]};
                }
            __syncthreads();
            if (key0 + r < s.nk) {
                const float by = which == 0 ? a.scale : 1.f;
                T* to = (which == 0 ? dk + (s.k0 + key0 + r) * dk_ld : dv + (s.k0 + key0 + r) * dv_ld) + (int64_t)g * a.dim + c0;
#pragma unroll
                for (int d = 0; d < DP / 8; d += 4) {
                    if (c0 + d >= a.dim) break;
                    f32x4 x = *reinterpret_cast<f32x4*>(join + r * (DP + 4) + c0 + d);
#pragma unroll
                    for (int w = 1; w < 4; ++w) x += *reinterpret_cast<f32x4*>(join + (w * 32 + r) * (DP + 4) + c0 + d);
                    x *= by;
                    Mma<T>::store4(to + d, x[0], x[1], x[2], x[3]);
                }
            }
        }
        return;
    }
    if (key >= s.nk) return;
    T* tk = dk + (s.k0 + key) * dk_ld + (int64_t)g * a.dim + 4 * half;
    T* tv = dv + (s.k0 + key) * dv_ld + (int64_t)g * a.dim + 4 * half;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * d + 8 * i < a.dim) {
                Mma<M>::store4(tk + 32 * d + 8 * i, ak[d][4 * i] * a.scale, ak[d][4 * i + 1] * a.scale, ak[d][4 * i + 2] * a.scale, ak[d][4 * i + 3] * a.scale);
                Mma<M>::store4(tv + 32 * d + 8 * i, av[d][4 * i], av[d][4 * i + 1], av[d][4 * i + 2], av[d][4 * i + 3]);
            }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
static int padded(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }
// Which form: a wave to an item where they are many and short; else rows where those blocks fill the chip, or the waves share an item's other side
// (key side, 16 segments of up to 777 x 1531, 8 heads of 128 over 2: 106 blocks of rows, 194 us against 139; 4 of 1024 x 1024, 8 heads: 288 blocks,
// a training pass of 176 us against 216).
// (f32 heads wider than 64 have the rows form only, as bias tables beyond 256 distances between first and last boundary: registers, shared memory.)
static bool rows_only(const dctr_attention* a) { return (a->dtype == DCTR_TYPE_F32 && a->head_dim > 64) || rel_reach(a) > 512; }
static int query_form(const dctr_attention* a) {
    if (rows_only(a)) return ROWS;
    if (a->max_q <= 64 && attn_solo(a, (int64_t)ceil_div(a->max_q, 32) * a->heads * a->n_seg)) return SOLO;
    return a->max_q <= 64 || (a->total_q / 128 + a->n_seg) * a->heads < 100 ? SPLIT : ROWS;
}
static int key_form(const dctr_attention* a) {
    if (rows_only(a)) return KEY_ROWS;
    if (a->max_q <= 128 && attn_solo(a, (int64_t)ceil_div(a->max_k, 32) * a->kv_heads * a->n_seg)) return KEY_SOLO;
    return (a->total_k / 128 + a->n_seg) * a->kv_heads < 200 ? KEY_SPLIT : KEY_ROWS;
}
static int row_blocks_of(const dctr_attention* a) { return ceil_div(a->max_q, query_form(a) == ROWS ? 128 : 32); }

int64_t attn_bwd_blocks(const dctr_attention* a) {
    const int keys = key_form(a);
    const int64_t q = (int64_t)row_blocks_of(a) * a->heads * a->n_seg, k = (int64_t)ceil_div(a->max_k, keys == KEY_ROWS ? 128 : 32) * a->kv_heads * a->n_seg;
    return std::max(query_form(a) == SOLO ? (q + 3) / 4 : q, (keys == KEY_SOLO ? (k + 3) / 4 : k) + a->heads);
}

// delta, then the bias gradient's shares
int64_t attn_bwd_workspace(const dctr_attention* a) {
    return 4 * (round_up(a->total_q * a->heads, 4) + (int64_t)a->heads * a->n_seg * row_blocks_of(a) * a->n_buckets);
}

template <typename T, int DP, int FORM>
static int launch_q(const dctr_attention* a, const AttnView& v, const AttnGrads& x, float* delta, float* part, hipStream_t st) {
    const int row_blocks = row_blocks_of(a);
    const int64_t items = (int64_t)row_blocks * a->heads * a->n_seg, blocks = FORM == SOLO ? (items + 3) / 4 : items;
    if (blocks == 0) return DCTR_OK;
    const size_t lds = QuerySide<T, DP, FORM>::first + sizeof(float) * (QuerySide<T, DP, FORM>::HIDDEN + 4 * SKEW + (FORM == SOLO ? 8 : 5) * rel_reach(a) + 8);
    attn_bwd_q_kernel<T, DP, FORM><<<(unsigned)blocks, BWD_THREADS, lds, st>>>(v, (const T*)x.out, x.out_ld, x.lse, (const T*)x.dout, x.dout_ld, (T*)x.dq, x.dq_ld,
                                                                               delta, part, row_blocks);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

template <typename T, int DP, int FORM>
static int launch_kv(const dctr_attention* a, const AttnView& v, const AttnGrads& x, const float* delta, const float* part, hipStream_t st) {
    using Kd = KeySide<T, DP, FORM>;
    const int key_blocks = ceil_div(a->max_k, Kd::OWN ? 32 : 128), sums = part != nullptr ? a->heads : 0;
    const int64_t items = (int64_t)key_blocks * a->kv_heads * a->n_seg, blocks = FORM == KEY_SOLO ? (items + 3) / 4 : items;
    if (blocks + sums == 0) return DCTR_OK;
    const size_t lds = std::max(Kd::tiles + Kd::stats + sizeof(float) * (Kd::OWN ? 8 : 2) * rel_reach(a), BWD_THREADS * sizeof(float));
    attn_bwd_kv_kernel<T, DP, FORM><<<(unsigned)(blocks + sums), BWD_THREADS, lds, st>>>(
        v, x.lse, delta, (const T*)x.dout, x.dout_ld, (T*)x.dk, x.dk_ld, (T*)x.dv, x.dv_ld, key_blocks,
        BiasShares{part, (int64_t)a->n_seg * row_blocks_of(a), x.dbias}, sums);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

template <typename T, int DP>
static int launch_bwd(const dctr_attention* a, const AttnView& v, const AttnGrads& x, float* ws, hipStream_t st) {
    float *delta = ws, *part = x.dbias != nullptr ? ws + round_up(a->total_q * a->heads, 4) : nullptr;
    constexpr bool wide = sizeof(T) == 4 && DP > 64;                    // (ROWS only)
    const int form = query_form(a);
    if (form == ROWS || wide)
        DCTR_TRY((launch_q<T, DP, ROWS>(a, v, x, delta, part, st)));
    else if (form == SPLIT)
        DCTR_TRY((launch_q<T, DP, wide ? ROWS : SPLIT>(a, v, x, delta, part, st)));
    else
        DCTR_TRY((launch_q<T, DP, wide ? ROWS : SOLO>(a, v, x, delta, part, st)));
    const int keys = key_form(a);
    if (keys == KEY_ROWS || wide) return launch_kv<T, DP, KEY_ROWS>(a, v, x, delta, part, st);
    if (keys == KEY_SPLIT) return launch_kv<T, DP, wide ? KEY_ROWS : KEY_SPLIT>(a, v, x, delta, part, st);
    return launch_kv<T, DP, wide ? KEY_ROWS : KEY_SOLO>(a, v, x, delta, part, st);
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
