// Matrix-core building blocks of the sequence operators (attention*.hip, vocab_softmax.hip), for float and bfloat16 operands alike.
//
// Every product is one of two, on 32 x 32 output blocks, f32 accumulators (16 a lane):
//   scores    S[m, n] = sum_d A[m, d] B[n, d]    A: 32 rows of a tile in shared memory, B: 32 rows held in registers (RowFrags)
//   weighted  O[d, n] += sum_m A[m, d] P[m, n]   A: the same kind of tile read by columns, P: the scores' block after softmax or its gradient
// Lane l of an output block holds column n = l & 31 and rows 8 i + 4 (l >> 5) + j for i, j in 0..3 (register 4 i + j).  P enters the second
// product AS IT LIES in those registers: a matrix instruction sums over its inner index in any order as long as both operands agree, so the
// columns of the tile are read in the order in which the registers hold the rows.  No value crosses lanes between the two products, and a
// row statistic of n (softmax maximum, sum) is one number a lane, shared by lanes l and l ^ 32 only.
//
// Tiles: DP (a power of two >= the row's width, the rest zero) elements a row, 16-byte chunk c of row r at chunk c ^ swz(r).  A row read takes
// one chunk of 32 consecutive rows, a column read (ds_read_b64_tr_b16) 64 bytes of 4 consecutive rows: swz spreads both over all 64 banks.
#pragma once
#include <hip/hip_bf16.h>

#include "common.h"

namespace dctr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }

// Both halves' values of a column: lo = lane l & 31's, hi = lane (l & 31) + 32's
struct Halves { float lo, hi; };
__device__ __forceinline__ Halves halves(float x) {
    const uint32_t a = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const uint32_t lo = r[0], hi = r[1];                // (a bit cast straight from r[1] reads r[0])
    return {__uint_as_float(lo), __uint_as_float(hi)};
}
__device__ __forceinline__ float both_max(float x) { const Halves h = halves(x); return fmaxf(h.lo, h.hi); }
__device__ __forceinline__ float both_sum(float x) { const Halves h = halves(x); return h.lo + h.hi; }

// row of register r within its 32-row block
__device__ __forceinline__ constexpr int reg_row(int r) { return 8 * (r >> 2) + (r & 3); }      // + 4 * (lane >> 5)

// The lane, for the addresses of a tile's reads.  At the widest rows the compiler would keep every address of the loop in a register of its own
// and spill the accumulators for them: there it is told nothing, and forms them again a tile (one exclusive or each).
template <int DP>
__device__ __forceinline__ int tile_lane() {
    int l = threadIdx.x & 63;
    if (DP > 128) asm volatile("" : "+v"(l));
    return l;
}

template <typename T, int DP>
struct Tile {
    static constexpr int CHUNKS = DP * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T);
    static __device__ __forceinline__ int swz(int r) {
        if (sizeof(T) == 2) {
            if (CHUNKS == 4) return (r >> 2) & 3;
            if (CHUNKS == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
            return (r & 3) << 2 | ((r >> 2) & 3);
        }
        if (CHUNKS == 8) return (r >> 1) & 7;
        return ((r >> 2) & 1) << 3 | ((r >> 3) & 1) << 2 | (r & 3);
    }
    static __device__ __forceinline__ int at(int r, int c) { return r * DP + (c ^ swz(r)) * PER; }
};

// One 16-byte chunk a lane: 16 (bf16) or 8 (f32) columns of 32 rows.
template <typename T> struct Mma;

template <> struct Mma<__bf16> {
    using Chunk = bf16x8;
    struct Weights { bf16x8 w[2]; };                    // a 32-row block of P, rounded to bf16: half a step of 2^-8 relative a weight
    static __device__ __forceinline__ f32x16 dot(Chunk a, Chunk b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Weights pack(const f32x16& p) {
        Weights r;
#pragma unroll
        for (int i = 0; i < 16; ++i) r.w[i >> 3][i & 7] = (__bf16)p[i];
        return r;
    }
    template <int DP>
    static __device__ __forceinline__ f32x16 weigh(const __bf16* tile, int row0, int col0, const Weights& p, f32x16 acc) {
        const int l = tile_lane<DP>(), row = row0 + 4 * (l >> 5) + ((l & 15) >> 2), col = col0 + 16 * ((l >> 4) & 1) + 4 * (l & 3);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf16x8 a;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = row + 16 * s + 8 * half;
                const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + Tile<__bf16, DP>::at(r, col >> 3) + (col & 7)));
                const bf16x4 b = __builtin_bit_cast(bf16x4, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[4 * half + j] = b[j];
            }
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, p.w[s], acc, 0, 0, 0);
        }
        return acc;
    }
    static __device__ __forceinline__ Chunk negate(Chunk a) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = -a[i];
        return a;
    }
    static __device__ __forceinline__ void store4(__bf16* p, float a, float b, float c, float d) {
        bf16x4 v;
        v[0] = (__bf16)a; v[1] = (__bf16)b; v[2] = (__bf16)c; v[3] = (__bf16)d;
        *reinterpret_cast<bf16x4*>(p) = v;
    }
};

template <> struct Mma<float> {
    using Chunk = f32x4;
    struct Weights { f32x16 w; };
    static __device__ __forceinline__ f32x16 dot(Chunk a, Chunk b, f32x16 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Weights pack(const f32x16& p) { return {p}; }
    template <int DP>
    static __device__ __forceinline__ f32x16 weigh(const float* tile, int row0, int col0, const Weights& p, f32x16 acc) {
        const int l = tile_lane<DP>(), row = row0 + 4 * (l >> 5), col = col0 + (l & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(tile[Tile<float, DP>::at(row + reg_row(r), col >> 2) + (col & 3)], p.w[r], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ Chunk negate(Chunk a) { return -a; }
    static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d}; }
};

// 32 rows in registers, one a lane (both halves together hold a row's chunks): the B operand of the scores
template <typename T, int DP>
struct RowFrags {
    static constexpr int STEPS = Tile<T, DP>::CHUNKS / 2;
    typename Mma<T>::Chunk c[STEPS];
    __device__ __forceinline__ void load(const T* row, int chunks, bool on) {          // `on`: the row exists; the rest is zero
        const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            c[s] = typename Mma<T>::Chunk{};
            if (on && 2 * s + g < chunks) c[s] = *reinterpret_cast<const typename Mma<T>::Chunk*>(row + (2 * s + g) * Tile<T, DP>::PER);
        }
    }
    __device__ __forceinline__ void negate() {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) c[s] = Mma<T>::negate(c[s]);
    }
};

// S of tile rows [row0, row0 + 32) against held rows
template <typename T, int DP>
__device__ __forceinline__ f32x16 scores(const T* tile, int row0, const RowFrags<T, DP>& held) {
    const int l = tile_lane<DP>(), row = row0 + (l & 31), g = l >> 5;
    f32x16 s = {};
#pragma unroll
    for (int k = 0; k < RowFrags<T, DP>::STEPS; ++k)
        s = Mma<T>::dot(*reinterpret_cast<const typename Mma<T>::Chunk*>(tile + Tile<T, DP>::at(row, 2 * k + g)), held.c[k], s);
    return s;
}

// ROWS rows of an array on their way into a tile, by THREADS threads: fetched into registers while the tile before is in use
template <typename T, int DP, int ROWS, int THREADS>
struct Staged {
    static constexpr int CHUNKS = Tile<T, DP>::CHUNKS, N = ROWS * CHUNKS / THREADS;
    static_assert(N >= 1 && ROWS * CHUNKS % THREADS == 0, "a tile is a whole number of chunks a thread");
    f32x4 v[N];
    // rows [first, first + ROWS) of those below `end`; the rest is zero
    __device__ __forceinline__ void fetch(const T* base, int64_t ld, int64_t first, int64_t end, int chunks, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * THREADS, r = at / CHUNKS, c = at % CHUNKS;
            v[i] = f32x4{};
            if (first + r < end && c < chunks) v[i] = *reinterpret_cast<const f32x4*>(base + (first + r) * ld + c * Tile<T, DP>::PER);
        }
    }
    // rows whose bit is not set become zero, whatever the array holds there
    __device__ __forceinline__ void store(T* tile, int tid, uint64_t rows = ~0ull) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * THREADS, r = at / CHUNKS, c = at % CHUNKS;
            *reinterpret_cast<f32x4*>(tile + Tile<T, DP>::at(r, c)) = (rows >> r & 1) ? v[i] : f32x4{};
        }
    }
};

// bits of 64 consecutive tile rows as register r of 32-row block `blk` sees them: bit reg_row(r) + 32 blk of the shifted word
__device__ __forceinline__ uint64_t lane_bits(uint64_t rows) { return rows >> (4 * ((threadIdx.x >> 5) & 1)); }

// Running softmax of a wave's 32 columns: m (base 2) and this half's share of the sum, the weighted sum as O^T blocks.
template <typename T, int DP>
struct Softmax {
    float m = -INFINITY, l = 0.f;
    f32x16 acc[DP / 32] = {};

    // Takes one 32 x NB*32 step's scores: t = fma(s, c, b), hidden entries -inf already where c = 1, b = 0.  Returns the weights in s.
    // The running maximum moves only when a score passes it by 2^8: weights up to 256 lose nothing in either type, and most steps
    // then skip the rescaling of the accumulators.
    template <int NB>
    __device__ __forceinline__ void step(f32x16 (&s)[NB], float c, float b) {
        float top = s[0][0];
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[k][r]);
        top = both_max(fmaf(top, c, b));
        if (__any(top > m + 8.f)) {
            const float mn = fmaxf(m, top), shrink = exp2f(m - (mn == -INFINITY ? 0.f : mn));
            l *= shrink;
#pragma unroll
            for (int k = 0; k < DP / 32; ++k) {
                acc[k] *= shrink;
                if (DP > 64) __builtin_amdgcn_sched_barrier(0);         // one block at a time: accumulators live in the other register file there
            }
            m = mn;
        }
        const float off = b - (m == -INFINITY ? 0.f : m);
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[k][r] = __builtin_amdgcn_exp2f(fmaf(s[k][r], c, off));
                part[r & 3] += s[k][r];
            }
        l += (part[0] + part[1]) + (part[2] + part[3]);
    }
    template <int NB>
    __device__ __forceinline__ void weigh(const T* tile, const f32x16 (&p)[NB]) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const auto w = Mma<T>::pack(p[k]);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) acc[d] = Mma<T>::template weigh<DP>(tile, 32 * k, 32 * d, w, acc[d]);
        }
    }
};

// The results of a block's four waves on the same 32 rows meet in shared memory: `join` 4 x 32 rows of DP + 4 floats (no two rows start at the
// same bank), `stats` 4 x 32 pairs (maximum, sum).  Afterwards thread t holds row t / 8's maximum, sum and columns [t % 8 * DP/8, + DP/8).
template <typename T, int DP>
__device__ __forceinline__ void join_waves(const Softmax<T, DP>& o, float* join, float* stats, float& m, float& l, float (&w)[DP / 8]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = tid >> 3;
    __syncthreads();                                                    // every wave is done with the tiles
    const float sum = both_sum(o.l);
    if (lane < 32) {
        stats[(wave * 32 + lane) * 2] = o.m;
        stats[(wave * 32 + lane) * 2 + 1] = sum;
    }
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *reinterpret_cast<f32x4*>(join + (wave * 32 + (lane & 31)) * (DP + 4) + 32 * k + 8 * e + 4 * (lane >> 5)) =
                f32x4{o.acc[k][4 * e], o.acc[k][4 * e + 1], o.acc[k][4 * e + 2], o.acc[k][4 * e + 3]};
    __syncthreads();
    m = -INFINITY;
#pragma unroll
    for (int n = 0; n < 4; ++n) m = fmaxf(m, stats[(n * 32 + row) * 2]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) w[d] = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const float f = exp2f(stats[(n * 32 + row) * 2] - base);
        l = fmaf(stats[(n * 32 + row) * 2 + 1], f, l);
#pragma unroll
        for (int d = 0; d < DP / 8; d += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(join + (n * 32 + row) * (DP + 4) + (tid & 7) * (DP / 8) + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[d + e] = fmaf(x[e], f, w[d + e]);
        }
    }
}

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

}  // namespace dctr
