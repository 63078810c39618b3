// Softmax cross entropy over a large vocabulary from the hidden rows and the vocabulary's table: the [N, V] logits exist a tile at a time, in
// registers (seq_mma.h).
//     z_nv = <x_n, w_v> + b_v        lse_n = log sum_v exp(z_nv)        loss_n = lse_n - z_n,label(n)
//     g_nv = c_n (exp(z_nv - lse_n) - [v = label(n)]),  c_n = scale row_scale_n (0 for a row without a label)
//     dx_n = sum_v g_nv w_v          dw_v = sum_n g_nv x_n              db_v = sum_n g_nv
// The forward's sums leave the label out and add it at the end: with e the sum of the others, 1 - p_label = e / (e + exp(z_label - m)) has
// no cancellation however sure the model is, nor has loss = log1p(e) where the label is the row's largest.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "seq_mma.h"

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

constexpr int VS_THREADS = 256;

// ---- forward: the same pass as an attention whose keys and values are both the table --------------------------------------------------
// What a split of the vocabulary leaves for every row, the label's column left out: maximum (base 2), sum, weighted sum of table rows.
struct VocabParts {
    float *m, *e, *acc;             // [splits][N], [splits][N], [splits][N][DP]
    int splits;
    int64_t each;                   // vocabulary rows of a split, a multiple of the tile
};

// Operand kind: float arrays in planes (seq_mma.h) up to 128 wide, beyond that the planes of 32 rows and their accumulators pass the registers.
template <typename T, int DP>
using VocabKind = std::conditional_t<std::is_same_v<T, float> && DP <= 128, Split, T>;

template <typename T, int DP>
struct VocabTile {
    using M = VocabKind<T, DP>;
    static constexpr int WIDTH = Mma<M>::BYTES * DP, ROWS = WIDTH <= 384 ? 64 : 32, NB = ROWS / 32, SIZE = ROWS * Tile<M, DP>::STRIDE;
    static constexpr size_t bytes = (size_t)ROWS * WIDTH;
    static constexpr bool LEAD = WIDTH == 512;                          // bf16 of 256, a wave a SIMD (rows of 2048 x 100000: 3 % longer without; f32 the same)
};

// Bias and hidden columns (behind the table, the row's label) of a wave's 32 rows' scores against NB * 32 table rows from v0 on; returns the factor
// that is left to the exponent.  `bt`: log2(e) b of the tile's rows, in shared memory, or null.
template <int NB>
__device__ __forceinline__ float adjust(f32x16 (&s)[NB], const float* bt, int64_t v0, int64_t v1, int64_t label) {
    const int half = (threadIdx.x >> 5) & 1;
    const int64_t own = label - v0;
    const bool hide = v0 + 32 * NB > v1 || __any(own >= 0 && own < 32 * NB);
    if (bt == nullptr && !hide) return LOG2E;
    uint64_t seen = v1 - v0 >= 64 ? ~0ull : (1ull << (v1 - v0)) - 1;
    if (own >= 0 && own < 64) seen &= ~(1ull << own);
    seen = lane_bits(seen);
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 add = bt != nullptr ? *reinterpret_cast<const f32x4*>(bt + 32 * k + 8 * i + 4 * half) : f32x4{};
#pragma unroll
            for (int j = 0; j < 4; ++j) s[k][4 * i + j] = fmaf(s[k][4 * i + j], LOG2E, add[j]);
        }
    if (hide) {
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[k][r] = (seen >> (32 * k + reg_row(r)) & 1) ? s[k][r] : -INFINITY;
    }
    return 1.f;
}

template <typename M, int DP, bool DX>
__device__ __forceinline__ void write_parts(const VocabParts& p, int sp, int N, int64_t n, bool on, const Softmax<M, DP>& o) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const float e = both_sum(o.l);
    if (!on) return;
    const int64_t at = (int64_t)sp * N + n;
    if (half == 0) { p.m[at] = o.m; p.e[at] = e; }
    if (DX)
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(p.acc + at * DP + 32 * k + 8 * i + 4 * half) =
                    f32x4{o.acc[k][4 * i], o.acc[k][4 * i + 1], o.acc[k][4 * i + 2], o.acc[k][4 * i + 3]};
}

// 4 waves of 32 rows share the table's tiles, three buffers: while a tile is weighed, the scores of the next one are formed under its exponents and
// the one after that is on its way.  Bound by the matrix unit and the exponents beside it: bf16 2048 x 1000000 x 64 with dx 697 us (752 TF/s of its two
// products), 2048 x 100000 x 256 342 us (613: one wave a SIMD); f32 in planes 4096 x 117581 x 64 without dx, the whole call: 379 us (163 TF/s; a large
// f32 matrix product of the library runs at 153).
template <typename T, int DP, bool DX>
__global__ __launch_bounds__(VS_THREADS, (VocabTile<T, DP>::WIDTH <= (DX ? 384 : 512) ? 2 : 1)) void vocab_rows_kernel(VocabView a, VocabParts p, int row_blocks) {
    extern __shared__ __attribute__((aligned(TILE_ALIGN))) char lds[];
    using Ti = VocabTile<T, DP>;
    using M = VocabKind<T, DP>;
    using S = typename Mma<M>::Store;
    constexpr int NB = Ti::NB;
    // (not where a second step's scores are what takes the kernel past two waves a SIMD: bf16 of 128, 213 us against 166 at 1024 x 100000)
    constexpr bool AHEAD = !(DX && Ti::WIDTH == 256);
    S* tiles = reinterpret_cast<S*>(lds);
    float* bias = reinterpret_cast<float*>(tiles + 3 * Ti::SIZE);                       // [3][ROWS]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rb = blockIdx.x % row_blocks, sp = blockIdx.x / row_blocks;
    const int64_t n = (int64_t)rb * 128 + wave * 32 + (lane & 31), v0 = sp * p.each, v1 = min(a.V, v0 + p.each);
    const int chunks = a.D / Tile<M, DP>::PER;
    const bool on = n < a.N, busy = rb * 128 + wave * 32 < a.N;
    RowFrags<M, DP> x;
    x.load((const T*)a.x + n * a.x_ld, chunks, on);
    int label = on ? a.labels[n] : -1;
    Softmax<M, DP> o;
    Loader<M, DP, Ti::ROWS, VS_THREADS> ws;
    float bv = 0.f;
    auto fetch = [&](int64_t v, int buf) {
        ws.fetch(tiles + buf * Ti::SIZE, (const T*)a.w, a.w_ld, v, v1, chunks, tid);
        if (a.b != nullptr && tid < Ti::ROWS) bv = v + tid < v1 ? LOG2E * a.b[v + tid] : 0.f;
    };
    auto land = [&](int64_t v, int buf) {
        ws.land(tiles + buf * Ti::SIZE, tid, first_rows(v1 - v));
        if (a.b != nullptr && tid < Ti::ROWS) bias[buf * Ti::ROWS + tid] = bv;
    };
    x.wait();
    settle(label);
    if (v0 < v1) {                                                                      // (rows behind v1 are zeros)
        fetch(v0, 0);
        land(v0, 0);
        fetch(v0 + Ti::ROWS, 1);
        land(v0 + Ti::ROWS, 1);
    }
    __syncthreads();
    f32x16 sc[NB];
    if (AHEAD) {
#pragma unroll
        for (int k = 0; k < NB; ++k) sc[k] = scores<M, DP, VocabTile<T, DP>::LEAD>(tiles, 32 * k, x);
    }
    int now = 0;
    for (int64_t v = v0; v < v1; v += Ti::ROWS) {
        const int next = now == 2 ? 0 : now + 1, then = next == 2 ? 0 : next + 1;
        const bool more = v + 2 * Ti::ROWS < v1;
        if (more) fetch(v + 2 * Ti::ROWS, then);
        if (busy) {
            if (!AHEAD) {
#pragma unroll
                for (int k = 0; k < NB; ++k) sc[k] = scores<M, DP, VocabTile<T, DP>::LEAD>(tiles + now * Ti::SIZE, 32 * k, x);
            }
            const float c = adjust<NB>(sc, a.b != nullptr ? bias + now * Ti::ROWS : nullptr, v, v1, label);
            const float off = o.template raise<NB>(sc, c, 0.f);
            f32x16 ahead[NB];
            if (AHEAD) {
#pragma unroll
                for (int k = 0; k < NB; ++k) ahead[k] = scores<M, DP, VocabTile<T, DP>::LEAD>(tiles + next * Ti::SIZE, 32 * k, x);
            }
            o.template weights<NB>(sc, c, off);
            if (DX) o.template weigh<NB>(tiles + now * Ti::SIZE, sc);

            if (AHEAD) {
#pragma unroll
                for (int k = 0; k < NB; ++k) sc[k] = ahead[k];
            }
        }
        if (more) land(v + 2 * Ti::ROWS, then);
        __syncthreads();
        now = next;
    }
    write_parts<M, DP, DX>(p, sp, a.N, n, on, o);
}

// Up to 32 rows: every wave takes tiles of its own, the four join before they leave their part.
template <typename T, int DP>
struct FewLds {
    static constexpr size_t tiles = 4 * 32 * (size_t)VocabTile<T, DP>::WIDTH, join = 4 * 32 * (DP + 4) * sizeof(float), first = tiles > join ? tiles : join;
    static constexpr size_t all = first + 4 * 32 * 2 * sizeof(float) + 4 * 32 * sizeof(float);      // + statistics + bias
};
template <typename T, int DP, bool DX>
__global__ __launch_bounds__(VS_THREADS, (VocabTile<T, DP>::WIDTH <= 256 ? 2 : 1)) void vocab_few_kernel(VocabView a, VocabParts p) {
    extern __shared__ __attribute__((aligned(TILE_ALIGN))) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sp = blockIdx.x;
    using M = VocabKind<T, DP>;
    using S = typename Mma<M>::Store;
    S* tile = reinterpret_cast<S*>(lds) + wave * 32 * Tile<M, DP>::STRIDE;
    float* stats = reinterpret_cast<float*>(lds + FewLds<T, DP>::first);
    float* bias = stats + 4 * 32 * 2 + wave * 32;
    const int64_t n = lane & 31, v0 = sp * p.each, v1 = min(a.V, v0 + p.each);
    const int chunks = a.D / Tile<M, DP>::PER;
    const bool on = n < a.N;
    RowFrags<M, DP> x;
    x.load((const T*)a.x + n * a.x_ld, chunks, on);
    const int64_t label = on ? a.labels[n] : -1;
    Softmax<M, DP> o;
    Staged<M, DP, 32, 64> ws;
    float bv = 0.f;
    auto fetch = [&](int64_t v) {
        ws.fetch(tile, (const T*)a.w, a.w_ld, v, v1, chunks, lane);
        if (a.b != nullptr && lane < 32) bv = v + lane < v1 ? LOG2E * a.b[v + lane] : 0.f;
    };
    int64_t v = v0 + 32 * wave;
    if (v < v1) fetch(v);
    for (; v < v1; v += 128) {
        __builtin_amdgcn_wave_barrier();
        ws.land(tile, lane, ~0ull);
        if (a.b != nullptr && lane < 32) bias[lane] = bv;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (v + 128 < v1) fetch(v + 128);
        f32x16 sc[1] = {scores<M, DP, VocabTile<T, DP>::LEAD>(tile, 0, x)};
        const float c = adjust<1>(sc, a.b != nullptr ? bias : nullptr, v, v1, label);
        o.template step<1>(sc, c, 0.f);
        if (DX) o.template weigh<1>(tile, sc);
    }
    if (DX) {
        float m, e, w[DP / 8];
        join_waves<M, DP>(o, reinterpret_cast<float*>(lds), stats, m, e, w);
        const int row = threadIdx.x >> 3, part = threadIdx.x & 7;
        if (row >= a.N) return;
        const int64_t at = (int64_t)sp * a.N + row;
        if (part == 0) { p.m[at] = m; p.e[at] = e; }
#pragma unroll
        for (int d = 0; d < DP / 8; d += 4) *reinterpret_cast<f32x4*>(p.acc + at * DP + part * (DP / 8) + d) = f32x4{w[d], w[d + 1], w[d + 2], w[d + 3]};
        return;
    }
    const float e = both_sum(o.l);
    if (lane < 32) {
        stats[(wave * 32 + lane) * 2] = o.m;
        stats[(wave * 32 + lane) * 2 + 1] = e;
    }
    __syncthreads();
    if ((int)threadIdx.x >= a.N) return;
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, stats[(k * 32 + threadIdx.x) * 2]);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = fmaf(stats[(k * 32 + threadIdx.x) * 2 + 1], exp2f(stats[(k * 32 + threadIdx.x) * 2] - (m == -INFINITY ? 0.f : m)), sum);
    p.m[(int64_t)sp * a.N + threadIdx.x] = m;
    p.e[(int64_t)sp * a.N + threadIdx.x] = sum;
}

// Joins the splits and adds the label's column: one block a row (and every gridDim.x-th one behind it), thread = (4 columns, slice of the splits) for dx.
constexpr int JOIN_BLOCKS = 1 << 22;                    // of the launch: there are more rows than one can have blocks
template <typename T, int DP, bool DX>
__device__ __forceinline__ void vocab_join_row(const VocabView& a, const VocabParts& p, float* loss, float* lse, T* dx, int64_t dx_ld, int32_t* status, int64_t n,
                                               float (&red)[3][4], f32x4 (&cols)[VS_THREADS]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int label = a.labels[n];
    const bool on = label >= 0 && label < a.V;
    if (label >= a.V && tid == 0 && status != nullptr) { status[0] = 1; status[1] = label; }
    const T* x = (const T*)a.x + n * a.x_ld;
    const T* w = (const T*)a.w + (on ? label : 0) * a.w_ld;
    float z = on && tid < a.D ? to_f32(x[tid]) * to_f32(w[tid]) : 0.f, m = -INFINITY;
    for (int s = tid; s < p.splits; s += VS_THREADS) m = fmaxf(m, p.m[(int64_t)s * a.N + n]);
    z = wave_sum(z);
    m = wave_max(m);
    if (lane == 0) { red[0][wave] = z; red[1][wave] = m; }
    __syncthreads();
    z = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    const float mine = on ? LOG2E * (a.b != nullptr ? z + a.b[label] : z) : -INFINITY;           // the label's logit, base 2
    m = fmaxf(mine, fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3])));
    const float base = m == -INFINITY ? 0.f : m;
    float e = 0.f;
    for (int s = tid; s < p.splits; s += VS_THREADS) e = fmaf(p.e[(int64_t)s * a.N + n], exp2f(p.m[(int64_t)s * a.N + n] - base), e);
    e = wave_sum(e);
    if (lane == 0) red[2][wave] = e;
    f32x4 acc = {};
    constexpr int COLS = DP / 4, SLICES = VS_THREADS / COLS;
    const int col = tid % COLS * 4, slice = tid / COLS;
    if (DX && on)
#pragma unroll 4
        for (int s = slice; s < p.splits; s += SLICES)
            acc += exp2f(p.m[(int64_t)s * a.N + n] - base) * *reinterpret_cast<const f32x4*>(p.acc + ((int64_t)s * a.N + n) * DP + col);
    if (DX) cols[tid] = acc;
    __syncthreads();
    e = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    const float all = e + (on ? exp2f(mine - base) : 0.f);
    if (tid == 0) {
        if (lse != nullptr) lse[n] = LN2 * base + logf(all);
        loss[n] = !on ? 0.f : mine == m ? log1pf(e) : LN2 * (base - mine) + logf(all);
    }
    if (!DX || slice > 0 || col >= a.D) return;
    for (int s = 1; s < SLICES; ++s) acc += cols[s * COLS + tid];
    const float c = on ? a.scale * (a.row_scale != nullptr ? a.row_scale[n] : 1.f) : 0.f;
    float to[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) to[d] = on ? c * (acc[d] - e * to_f32(w[col + d])) / all : 0.f;
    Mma<T>::store4(dx + n * dx_ld + col, to[0], to[1], to[2], to[3]);
}
template <typename T, int DP, bool DX>
__global__ __launch_bounds__(VS_THREADS) void vocab_join_kernel(VocabView a, VocabParts p, float* loss, float* lse, T* dx, int64_t dx_ld, int32_t* status) {
    __shared__ float red[3][4];
    __shared__ f32x4 cols[VS_THREADS];
    for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
        vocab_join_row<T, DP, DX>(a, p, loss, lse, dx, dx_ld, status, n, red, cols);
        __syncthreads();                                                // (the next row's sums go where this one's are read)
    }
}

// ---- dw, db: 32 table rows a wave, over the rows of x ---------------------------------------------------------------------------------
// bf16 2048 x 1000000 x 64: 600 us (874 TF/s of two products); 2048 x 100000 x 256: 352 us (596).  f32 in planes 1024 x 117581 x 64: 178 us (173 TF/s).
// With more than one split (a short vocabulary): part [splits][V][DP], part_b [splits][V], joined by vocab_dw_join_kernel.
// (bf16 of 256: two waves a SIMD at the price of 13 spilled registers take 2048 x 100000 in 0.73 of the time; the rows kernel would spill 110 and take 1.2 times its)
template <typename T, int DP>
__global__ __launch_bounds__(VS_THREADS, (VocabTile<T, DP>::WIDTH <= 256 || VocabTile<T, DP>::WIDTH == 512 ? 2 : 1)) void vocab_dw_kernel(VocabView a, const float* lse, T* dw, int64_t dw_ld, float* db, float* part, float* part_b,
                                                              int splits, int each, int table_blocks) {
    extern __shared__ __attribute__((aligned(TILE_ALIGN))) char lds[];
    using Ti = VocabTile<T, DP>;
    using M = VocabKind<T, DP>;
    using S = typename Mma<M>::Store;
    S* tiles = reinterpret_cast<S*>(lds);
    float* stats = reinterpret_cast<float*>(tiles + 2 * Ti::SIZE);                      // [2][-log2(e) lse, row scale, label][ROWS]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int tb = blockIdx.x % table_blocks, sp = blockIdx.x / table_blocks;
    const int64_t w0 = (int64_t)tb * 128 + wave * 32, v = w0 + (lane & 31);
    const int chunks = a.D / Tile<M, DP>::PER, n0 = sp * each, n1 = min(a.N, n0 + each);
    const bool on = v < a.V;
    RowFrags<M, DP> w;
    w.load((const T*)a.w + v * a.w_ld, chunks, on);
    float bv = on && a.b != nullptr ? LOG2E * a.b[v] : 0.f;
    w.wait();
    settle(bv);
    f32x16 acc[DP / 32] = {};
    float sum = 0.f;
    Loader<M, DP, Ti::ROWS, VS_THREADS> xs;
    float lv = 0.f, cv = 0.f;
    int label = -1;
    auto fetch = [&](int n, int buf) {
        xs.fetch(tiles + buf * Ti::SIZE, (const T*)a.x, a.x_ld, n, n1, chunks, tid);
        const int r = n + lane;                                                         // (every wave: the rows' bits)
        const bool there = lane < Ti::ROWS && r < n1;
        label = there ? a.labels[r] : -1;                                               // (all looked at on landing: nothing waits here)
        lv = there ? lse[r] : 0.f;
        if (a.row_scale != nullptr) cv = there ? a.row_scale[r] : 0.f;
    };
    auto land = [&](int buf) {
        const bool labelled = label >= 0 && label < a.V;
        xs.land(tiles + buf * Ti::SIZE, tid, __ballot(labelled));
        if (wave == 0 && lane < Ti::ROWS) {
            float* st = stats + buf * 3 * Ti::ROWS + lane;
            st[0] = labelled ? -LOG2E * lv : -INFINITY;                                 // no label: p = 2^-inf = 0
            st[Ti::ROWS] = labelled ? cv : 0.f;
            reinterpret_cast<int32_t*>(st)[2 * Ti::ROWS] = labelled ? label : -1;
        }
    };
    if (n0 < n1) {
        fetch(n0, 0);
        land(0);
    }
    __syncthreads();
    int buf = 0;
    for (int n = n0; n < n1; n += Ti::ROWS, buf ^= 1) {
        const bool more = n + Ti::ROWS < n1;
        if (more) fetch(n + Ti::ROWS, buf ^ 1);
        const S* xt = tiles + buf * Ti::SIZE;
        const float* st = stats + buf * 3 * Ti::ROWS;
        const int32_t* lt = reinterpret_cast<const int32_t*>(st) + 2 * Ti::ROWS;
        const int64_t there = lane < Ti::ROWS ? (int64_t)lt[lane] - w0 : -1;
        const bool hot = __any(there >= 0 && there < 32);                               // a row's label is one of the wave's table rows
#pragma unroll
        for (int k = 0; k < Ti::NB; ++k) {
            f32x16 p = scores<M, DP>(xt, 32 * k, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 ml = *reinterpret_cast<const f32x4*>(st + 32 * k + 8 * i + 4 * half);
#pragma unroll
                for (int j = 0; j < 4; ++j) p[4 * i + j] = __builtin_amdgcn_exp2f(fmaf(p[4 * i + j], LOG2E, ml[j] + bv));
            }
            if (hot) {
#pragma unroll
                for (int r = 0; r < 16; ++r) p[r] -= lt[32 * k + reg_row(r) + 4 * half] == v ? 1.f : 0.f;
            }
            if (a.row_scale != nullptr) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 c = *reinterpret_cast<const f32x4*>(st + Ti::ROWS + 32 * k + 8 * i + 4 * half);
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[4 * i + j] *= c[j];
                }
            }
            if (db != nullptr) {
                float part4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 16; ++r) part4[r & 3] += p[r];
                sum += (part4[0] + part4[1]) + (part4[2] + part4[3]);
            }
            weigh_all<M, DP>(xt, 32 * k, Mma<M>::pack(p), acc);
        }
        if (more) land(buf ^ 1);
        __syncthreads();
    }
    sum = both_sum(sum);
    if (!on) return;
    if (splits > 1) {
        const int64_t at = (int64_t)sp * a.V + v;
        if (db != nullptr && half == 0) part_b[at] = sum;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(part + at * DP + 32 * d + 8 * i + 4 * half) =
                    f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
        return;
    }
    if (db != nullptr && half == 0) db[v] = a.scale * sum;
    T* to = dw + v * dw_ld + 4 * half;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * d + 8 * i < a.D)
                Mma<M>::store4(to + 32 * d + 8 * i, a.scale * acc[d][4 * i], a.scale * acc[d][4 * i + 1], a.scale * acc[d][4 * i + 2],
                               a.scale * acc[d][4 * i + 3]);
}

// thread = 4 columns of a table row
template <typename T, int DP>
__global__ __launch_bounds__(VS_THREADS) void vocab_dw_join_kernel(VocabView a, T* dw, int64_t dw_ld, float* db, const float* part, const float* part_b,
                                                                   int splits) {
    const int64_t at = (int64_t)blockIdx.x * VS_THREADS + threadIdx.x, v = at / (DP / 4);
    const int d = (int)(at % (DP / 4)) * 4;
    if (v >= a.V) return;
    if (db != nullptr && d == 0) {
        float x = 0.f;
        for (int s = 0; s < splits; ++s) x += part_b[(int64_t)s * a.V + v];
        db[v] = a.scale * x;
    }
    if (d >= a.D) return;
    f32x4 x = {};
    for (int s = 0; s < splits; ++s) x += *reinterpret_cast<const f32x4*>(part + ((int64_t)s * a.V + v) * DP + d);
    x *= a.scale;
    Mma<T>::store4(dw + v * dw_ld + d, x[0], x[1], x[2], x[3]);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
static int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

struct VocabPlan { bool few; int row_blocks, splits; int64_t each; };
// Splits of the vocabulary: two blocks a compute unit, no split below 256 rows of the table.
static VocabPlan plan_fwd(int N, int64_t V) {
    VocabPlan p;
    p.few = N <= 32;
    p.row_blocks = p.few ? 1 : ceil_div(N, 128);
    const int64_t want = (512 + p.row_blocks - 1) / p.row_blocks, cut = std::min(want, (V + 255) / 256);
    p.each = round_up((V + cut - 1) / cut, 64);
    p.splits = (int)((V + p.each - 1) / p.each);
    return p;
}
struct VocabWPlan { int table_blocks, splits, each; };
// Splits of the rows: a vocabulary of fewer than 512 blocks of 128 rows leaves compute units idle.
static VocabWPlan plan_dw(int N, int64_t V) {
    VocabWPlan p;
    p.table_blocks = ceil_div(V, 128);
    const int64_t want = std::max<int64_t>(1, 512 / p.table_blocks), most = std::max(1, ceil_div(N, 256));
    const int64_t cut = std::min(want, most);
    p.each = (int)std::max<int64_t>(64, round_up((N + cut - 1) / cut, 64));
    p.splits = std::max(1, ceil_div(N, p.each));
    return p;
}

static int64_t workspace_bytes(int N, int64_t V, int D, int train) {
    const VocabPlan f = plan_fwd(N, V);
    const int64_t rows = (int64_t)f.splits * N, stats = round_up(2 * rows, 4);
    int64_t floats = stats + (train ? rows * padded(D) : 0);
    if (train) {
        const VocabWPlan w = plan_dw(N, V);
        if (w.splits > 1) floats = std::max(floats, (int64_t)w.splits * V * (padded(D) + 1));
    }
    return floats * (int64_t)sizeof(float);
}

template <typename T, int DP, bool DX>
static int launch_fwd(const VocabView& a, float* loss, float* lse, void* dx, int64_t dx_ld, int32_t* status, float* ws, hipStream_t st) {
    const VocabPlan f = plan_fwd(a.N, a.V);
    const int64_t rows = (int64_t)f.splits * a.N;
    const VocabParts p{ws, ws + rows, ws + round_up(2 * rows, 4), f.splits, f.each};
    if (f.few)
        vocab_few_kernel<T, DP, DX><<<f.splits, VS_THREADS, FewLds<T, DP>::all, st>>>(a, p);
    else
        vocab_rows_kernel<T, DP, DX><<<(unsigned)(f.row_blocks * f.splits), VS_THREADS,
                                       3 * (VocabTile<T, DP>::bytes + VocabTile<T, DP>::ROWS * sizeof(float)), st>>>(a, p, f.row_blocks);
    DCTR_LAUNCH_CHECK();
    vocab_join_kernel<T, DP, DX><<<std::min(a.N, JOIN_BLOCKS), VS_THREADS, 0, st>>>(a, p, loss, lse, (T*)dx, dx_ld, status);
    DCTR_LAUNCH_CHECK();
    return DCTR_OK;
}

template <typename T, int DP>
static int launch_dw(const VocabView& a, const float* lse, void* dw, int64_t dw_ld, float* db, float* ws, hipStream_t st) {
    const VocabWPlan w = plan_dw(a.N, a.V);
    float *part = ws, *part_b = ws + (int64_t)w.splits * a.V * DP;
    const size_t lds = 2 * (VocabTile<T, DP>::bytes + 3 * VocabTile<T, DP>::ROWS * sizeof(float));
    vocab_dw_kernel<T, DP><<<(unsigned)(w.table_blocks * w.splits), VS_THREADS, lds, st>>>(a, lse, (T*)dw, dw_ld, db, part, part_b, w.splits, w.each,
                                                                                           w.table_blocks);
    DCTR_LAUNCH_CHECK();
    if (w.splits > 1) {
        vocab_dw_join_kernel<T, DP><<<ceil_div(a.V * (DP / 4), VS_THREADS), VS_THREADS, 0, st>>>(a, (T*)dw, dw_ld, db, part, part_b, w.splits);
        DCTR_LAUNCH_CHECK();
    }
    return DCTR_OK;
}

template <typename T, int DP>
static int fwd(const VocabView& a, float* loss, float* lse, void* dx, int64_t dx_ld, int32_t* status, float* ws, hipStream_t st) {
    return dx != nullptr ? launch_fwd<T, DP, true>(a, loss, lse, dx, dx_ld, status, ws, st)
                         : launch_fwd<T, DP, false>(a, loss, lse, dx, dx_ld, status, ws, st);
}

#define VOCAB_BY_WIDTH(T, D, FN, ...)                     \
    switch (padded(D)) {                                  \
        case 32: return FN<T, 32>(__VA_ARGS__);           \
        case 64: return FN<T, 64>(__VA_ARGS__);           \
        case 128: return FN<T, 128>(__VA_ARGS__);         \
        default: return FN<T, 256>(__VA_ARGS__);          \
    }

static int check_sizes(int dtype, int N, int64_t V, int D) {
    DCTR_REQUIRE(dtype == DCTR_TYPE_F32 || dtype == DCTR_TYPE_BF16, "vocab softmax: unknown element type %d", dtype);
    DCTR_REQUIRE(N >= 0 && N <= 1 << 30, "vocab softmax: %d rows (0..2^30)", N);              // (row numbers and the tile behind the last stay in 32 bits)
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
    float* ws = (float*)d_workspace;
    if (dtype == DCTR_TYPE_F32) VOCAB_BY_WIDTH(float, D, fwd, a, d_loss, d_lse, d_dx, dx_ld, d_status, ws, st)
    VOCAB_BY_WIDTH(__bf16, D, fwd, a, d_loss, d_lse, d_dx, dx_ld, d_status, ws, st)
}

int dctr_vocab_softmax_bwd_weights(int dtype, const void* d_x, int x_ld, const void* d_w, int w_ld, const float* d_b, const int32_t* d_labels, int N,
                                   int64_t V, int D, const float* d_row_scale, float scale, const float* d_lse, void* d_dw, int dw_ld, float* d_db,
                                   void* d_workspace, size_t workspace_bytes, void* stream) {
    VocabView a;
    DCTR_TRY(make_view(dtype, d_x, x_ld, d_w, w_ld, d_b, d_labels, N, V, D, d_row_scale, scale, 1, d_workspace, workspace_bytes, &a));
    DCTR_REQUIRE(N == 0 || d_lse != nullptr, "vocab softmax: lse is null");
    DCTR_REQUIRE(V <= 128 * MAX_BLOCKS, "vocab softmax: vocabulary of %lld (gradients: at most %lld)", (long long)V, (long long)(128 * MAX_BLOCKS));   // (a block 128 rows)
    DCTR_TRY(check_rows("dw", d_dw, dw_ld, D, dtype == DCTR_TYPE_F32 ? 4 : 2));
    hipStream_t st = as_stream(stream);
    float* ws = (float*)d_workspace;
    if (dtype == DCTR_TYPE_F32) VOCAB_BY_WIDTH(float, D, launch_dw, a, d_lse, d_dw, dw_ld, d_db, ws, st)
    VOCAB_BY_WIDTH(__bf16, D, launch_dw, a, d_lse, d_dw, dw_ld, d_db, ws, st)
}

}  // extern "C"
