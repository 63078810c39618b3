// Matrix-core building blocks of the sequence operators (attention*.hip, vocab_softmax.hip).  Operand kinds M:
//   __bf16   bfloat16 arrays
//   Split    float arrays, every element as three bfloat16 planes x = h + m + l (3 x 8 significand bits: exact) and the six leading plane products
//            in f32 on the bf16 pipe: what is dropped is below 2^-25 of an element product.  The f32 matrix instructions run at the vector
//            units' rate, 1/16 of the bf16 pipe's, and hold the vector units up meanwhile
//   float    float arrays on the f32 matrix instructions: where the planes' registers do not suffice
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
#include <type_traits>

#include <hip/hip_bf16.h>

#include "common.h"

namespace dctr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;           // of 256 threads: a grid's dimension has fewer than 2^32 threads

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
// and spill the accumulators for them: there it is told nothing, and forms them again a tile, one exclusive or each (flipped; from row, chunk and
// swizzle anew they were four instructions each, half of all of a wave that shares its SIMD with no other).
template <int DP>
__device__ __forceinline__ int tile_lane() {
    int l = threadIdx.x & 63;
    if (DP > 128) asm volatile("" : "+v"(l));
    return l;
}

// p with some of the bits flipped that its offset in a row of a tile takes (rows of a power of two bytes, the tile at a multiple of it)
template <typename S>
__device__ __forceinline__ const S* flipped(const S* p, int bits) {
    typedef __attribute__((address_space(3))) const S lds_S;
    return (const S*)(lds_S*)(uintptr_t)((uint32_t)(uintptr_t)(lds_S*)p ^ (uint32_t)bits);
}
constexpr int TILE_ALIGN = 1024;                        // of shared memory that holds tiles of rows this wide

struct Split {};
template <typename M> struct Mma;

template <typename M, int DP>
struct Tile {
    using S = typename Mma<M>::Store;
    static constexpr int PER = 16 / (int)sizeof(S), CHUNKS = DP / PER, STRIDE = DP * Mma<M>::PLANES;      // a row: its planes one after the other
    static __device__ __forceinline__ int swz(int r) {
        if (sizeof(S) == 2) {
            if (CHUNKS == 4) return (r >> 2) & 3;
            if (CHUNKS == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
            return (r & 3) << 2 | ((r >> 2) & 3);
        }
        if (CHUNKS == 8) return (r >> 1) & 7;
        return ((r >> 2) & 1) << 3 | ((r >> 3) & 1) << 2 | (r & 3);
    }
    static __device__ __forceinline__ int at(int r, int c) { return r * STRIDE + (c ^ swz(r)) * PER; }
};

// 32 (rows) x 16 columns of a bf16 plane, transposed: the lane's column, rows 4 (lane >> 5) + {0..3} and + 8
template <typename M, int DP>
__device__ __forceinline__ bf16x8 column_chunk(const __bf16* tile, int row, int col) {
    bf16x8 a;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + Tile<M, DP>::at(row + 8 * half, col >> 3) + (col & 7)));
        const bf16x4 b = __builtin_bit_cast(bf16x4, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[4 * half + j] = b[j];
    }
    return a;
}

template <> struct Mma<__bf16> {
    using Global = __bf16;                              // element of the arrays
    using Store = __bf16;                               // element of a tile
    static constexpr int PLANES = 1, BYTES = 2;         // of an element in a tile or held row
    static constexpr bool ROUNDS = true;                // the weights are rounded
    using Chunk = bf16x8;                               // one 16-byte chunk a lane: 16 columns of 32 rows
    struct Weights { bf16x8 w[2]; };                    // a 32-row block of P, rounded to bf16: half a step of 2^-8 relative a weight
    static __device__ __forceinline__ Chunk load(const Global* p) { return *reinterpret_cast<const Chunk*>(p); }
    static __device__ __forceinline__ f32x16 dot(const Store* a, Chunk b, f32x16 c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(a), b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Weights pack(const f32x16& p) {
        Weights r;
#pragma unroll
        for (int i = 0; i < 16; ++i) r.w[i >> 3][i & 7] = (__bf16)p[i];
        return r;
    }
    static __device__ __forceinline__ Weights pack_rest(f32x16 p, const Weights& first) {       // what pack has rounded off, exact to 2^-17 of a weight
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] -= (float)first.w[i >> 3][i & 7];
        return pack(p);
    }
    template <int DP>
    static __device__ __forceinline__ f32x16 weigh(const __bf16* tile, int row0, int col0, const Weights& p, f32x16 acc) {
        const int l = tile_lane<DP>(), row = row0 + 4 * (l >> 5) + ((l & 15) >> 2), col = col0 + 16 * ((l >> 4) & 1) + 4 * (l & 3);
#pragma unroll
        for (int s = 0; s < 2; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(column_chunk<__bf16, DP>(tile, row + 16 * s, col), p.w[s], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ Chunk negate(Chunk a) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = -a[i];
        return a;
    }
    static __device__ __forceinline__ float product(Chunk a, Chunk b, float c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = fmaf((float)a[i], (float)b[i], c);
        return c;
    }
    static __device__ __forceinline__ void store4(__bf16* p, float a, float b, float c, float d) {
        bf16x4 v;
        v[0] = (__bf16)a; v[1] = (__bf16)b; v[2] = (__bf16)c; v[3] = (__bf16)d;
        *reinterpret_cast<bf16x4*>(p) = v;
    }
};

template <> struct Mma<float> {
    using Global = float;
    using Store = float;
    static constexpr int PLANES = 1, BYTES = 4;
    static constexpr bool ROUNDS = false;
    using Chunk = f32x4;                                // 8 columns of 32 rows
    struct Weights { f32x16 w; };
    static __device__ __forceinline__ Chunk load(const Global* p) { return *reinterpret_cast<const Chunk*>(p); }
    static __device__ __forceinline__ f32x16 dot(const Store* p, Chunk b, f32x16 c, int) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p);
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
    static __device__ __forceinline__ float product(Chunk a, Chunk b, float c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = fmaf(a[i], b[i], c);
        return c;
    }
    static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d}; }
};

struct Planes { bf16x8 h, m, l; };
// x = h + m + l, each the nearest bf16 of what is left: the subtractions are exact
__device__ __forceinline__ Planes planes_of(const float (&x)[8]) {
    Planes p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        p.h[i] = (__bf16)x[i];
        const float r = x[i] - (float)p.h[i];
        p.m[i] = (__bf16)r;
        p.l[i] = (__bf16)(r - (float)p.m[i]);
    }
    return p;
}
// the six products, smallest first
__device__ __forceinline__ f32x16 six(const Planes& a, const Planes& b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b.m, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.l, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.m, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.h, c, 0, 0, 0);
}

template <> struct Mma<Split> {
    using Global = float;
    using Store = __bf16;
    static constexpr int PLANES = 3, BYTES = 6;
    static constexpr bool ROUNDS = false;
    using Chunk = Planes;                               // 16 columns of 32 rows
    struct Weights { Planes w[2]; };
    static __device__ __forceinline__ Chunk load(const Global* p) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(p + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
        }
        return planes_of(x);
    }
    static __device__ __forceinline__ f32x16 dot(const Store* a, const Chunk& b, f32x16 c, int plane) {
        return six(Planes{*reinterpret_cast<const bf16x8*>(a), *reinterpret_cast<const bf16x8*>(a + plane), *reinterpret_cast<const bf16x8*>(a + 2 * plane)}, b, c);
    }
    static __device__ __forceinline__ Weights pack(const f32x16& p) {
        Weights r;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[8 * s + i];
            r.w[s] = planes_of(x);
        }
        return r;
    }
    template <int DP>
    static __device__ __forceinline__ f32x16 weigh(const __bf16* tile, int row0, int col0, const Weights& p, f32x16 acc) {
        const int l = tile_lane<DP>(), row = row0 + 4 * (l >> 5) + ((l & 15) >> 2), col = col0 + 16 * ((l >> 4) & 1) + 4 * (l & 3);
#pragma unroll
        for (int s = 0; s < 2; ++s)
            acc = six(Planes{column_chunk<Split, DP>(tile, row + 16 * s, col), column_chunk<Split, DP>(tile + DP, row + 16 * s, col),
                             column_chunk<Split, DP>(tile + 2 * DP, row + 16 * s, col)}, p.w[s], acc);
        return acc;
    }
    static __device__ __forceinline__ Chunk negate(Chunk a) {
        a.h = Mma<__bf16>::negate(a.h);
        a.m = Mma<__bf16>::negate(a.m);
        a.l = Mma<__bf16>::negate(a.l);
        return a;
    }
    static __device__ __forceinline__ float product(const Chunk& a, const Chunk& b, float c) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            c = fmaf(((float)a.h[i] + (float)a.m[i]) + (float)a.l[i], ((float)b.h[i] + (float)b.m[i]) + (float)b.l[i], c);
        return c;
    }
    static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d}; }
};

// Waits for a value's load here and not at its first use: within a loop that wait would hold up the tile loads under way (which the compiler does
// not see) on every turn.
__device__ __forceinline__ void settle(float& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void settle(int& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void settle(f32x4& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void settle(bf16x8& x) {
    f32x4 y = __builtin_bit_cast(f32x4, x);
    settle(y);
    x = __builtin_bit_cast(bf16x8, y);
}
__device__ __forceinline__ void settle(Planes& x) { settle(x.h); settle(x.m); settle(x.l); }

// 32 rows in registers, one a lane (both halves together hold a row's chunks): the B operand of the scores
template <typename M, int DP>
struct RowFrags {
    using T = typename Mma<M>::Global;
    static constexpr int STEPS = Tile<M, DP>::CHUNKS / 2;
    typename Mma<M>::Chunk c[STEPS];
    __device__ __forceinline__ void load(const T* row, int chunks, bool on) {          // `on`: the row exists; the rest is zero
        const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            c[s] = typename Mma<M>::Chunk{};
            if (on && 2 * s + g < chunks) c[s] = Mma<M>::load(row + (2 * s + g) * Tile<M, DP>::PER);
        }
    }
    __device__ __forceinline__ void negate() {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) c[s] = Mma<M>::negate(c[s]);
    }
    __device__ __forceinline__ void wait() {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) settle(c[s]);
    }
};

// S of tile rows [row0, row0 + 32) against held rows.  LEAD: four reads of the tile before the first product and one behind each from there on.
// For kernels of one wave a SIMD, which nothing else covers: the compiler spares registers there and has each read waited for.
template <typename M, int DP, bool LEAD = false>
__device__ __forceinline__ f32x16 scores(const typename Mma<M>::Store* tile, int row0, const RowFrags<M, DP>& held) {
    static_assert(DP <= 128 || Mma<M>::PLANES == 1, "a row's bytes are a power of two");
    const int l = tile_lane<DP>(), row = row0 + (l & 31), g = l >> 5;
    const auto* first = tile + Tile<M, DP>::at(row, g);
    f32x16 s = {};
#pragma unroll
    for (int k = 0; k < RowFrags<M, DP>::STEPS; ++k) {
        if constexpr (DP > 128)
            s = Mma<M>::dot(flipped(first, 32 * k), held.c[k], s, DP);
        else
            s = Mma<M>::dot(tile + Tile<M, DP>::at(row, 2 * k + g), held.c[k], s, DP);
    }
    if constexpr (LEAD) {
        constexpr int P = Mma<M>::PLANES, PRODUCTS = P == 3 ? 6 : sizeof(typename Mma<M>::Store) == 2 ? 1 : 4;
        constexpr int AHEAD = RowFrags<M, DP>::STEPS < 4 ? RowFrags<M, DP>::STEPS : 4;
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * P, 0);
#pragma unroll
        for (int k = 0; k < RowFrags<M, DP>::STEPS; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
            if (k + AHEAD < RowFrags<M, DP>::STEPS) __builtin_amdgcn_sched_group_barrier(0x100, P, 0);
        }
    }
    return s;
}

// O of tile rows [row0, row0 + 32) with a block of weights, every column
template <typename M, int DP>
__device__ __forceinline__ void weigh_all(const typename Mma<M>::Store* tile, int row0, const typename Mma<M>::Weights& w, f32x16 (&acc)[DP / 32]) {
    if constexpr (DP > 128 && std::is_same_v<M, __bf16>) {
        const int l = tile_lane<DP>(), row = row0 + 4 * (l >> 5) + ((l & 15) >> 2);
        const __bf16* first = tile + Tile<M, DP>::at(row, 2 * ((l >> 4) & 1) + ((l & 3) >> 1)) + 4 * (l & 1);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf16x8 a;
#pragma unroll
                for (int half = 0; half < 2; ++half) {                  // (rows + 8: swz differs in the bit of two chunks)
                    const __bf16* at = flipped(first, 64 * d + 32 * half) + (16 * s + 8 * half) * Tile<M, DP>::STRIDE;
                    const bf16x4 b = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[4 * half + j] = b[j];
                }
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w.w[s], acc[d], 0, 0, 0);
            }
    } else {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Mma<M>::template weigh<DP>(tile, row0, 32 * d, w, acc[d]);
    }
}

// ROWS rows of an array on their way into a tile, by THREADS threads: fetched into registers while the tile before is in use
template <typename M, int DP, int ROWS, int THREADS>
struct Staged {
    using T = typename Mma<M>::Global;
    using S = typename Mma<M>::Store;
    static constexpr int CHUNKS = Tile<M, DP>::CHUNKS, PER = Tile<M, DP>::PER, N = ROWS * CHUNKS / THREADS, LOADS = PER * (int)sizeof(T) / 16;
    static_assert(N >= 1 && ROWS * CHUNKS % THREADS == 0, "a tile is a whole number of chunks a thread");
    f32x4 v[N][LOADS];
    // rows [first, first + ROWS) of those below `end`; the rest is zero
    __device__ __forceinline__ void fetch(S*, const T* base, int64_t ld, int64_t first, int64_t end, int chunks, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * THREADS, r = at / CHUNKS, c = at % CHUNKS;
            const bool on = first + r < end && c < chunks;
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                v[i][j] = f32x4{};
                if (on) v[i][j] = *reinterpret_cast<const f32x4*>(base + (first + r) * ld + c * PER + j * (16 / (int)sizeof(T)));
            }
        }
    }
    // rows whose bit is not set become zero, whatever the array holds there
    __device__ __forceinline__ void land(S* tile, int tid, uint64_t rows) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * THREADS, r = at / CHUNKS, c = at % CHUNKS;
            const bool on = rows >> r & 1;
            S* to = tile + Tile<M, DP>::at(r, c);
            if constexpr (LOADS == 1) {
                *reinterpret_cast<f32x4*>(to) = on ? v[i][0] : f32x4{};
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = on ? v[i][e >> 2][e & 3] : 0.f;
                const Planes p = planes_of(x);
                *reinterpret_cast<bf16x8*>(to) = p.h;
                *reinterpret_cast<bf16x8*>(to + DP) = p.m;
                *reinterpret_cast<bf16x8*>(to + 2 * DP) = p.l;
            }
        }
    }
};

// The same straight into the tile (no registers: held back there, the compiler parks them in the accumulator file and waits for the loads to do
// so).  A wave's load fills 64 consecutive 16-byte slots, so the swizzle is in the addresses that it reads.  Rows behind the end are read as the
// last one and columns behind the row's width as its last chunk: the first become zero on landing, the second meet zeros in the held rows.
template <typename M, int DP, int ROWS, int THREADS>
struct Direct {
    using T = typename Mma<M>::Global;
    static constexpr int CHUNKS = Tile<M, DP>::CHUNKS, PER = Tile<M, DP>::PER, N = ROWS * CHUNKS / THREADS;
    static_assert(N >= 1 && ROWS * CHUNKS % THREADS == 0 && THREADS % 64 == 0 && Mma<M>::PLANES == 1, "a wave's load is 64 slots of a tile of one plane");
    __device__ __forceinline__ void fetch(T* tile, const T* base, int64_t ld, int64_t first, int64_t end, int chunks, int tid) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");              // this wave's reads of what the tile held are answered (others': a barrier ago)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * THREADS, r = at / CHUNKS, c = (at % CHUNKS) ^ Tile<M, DP>::swz(r);
            const int64_t row = first + r < end ? first + r : end - 1;
            const T* from = base + row * ld + (c < chunks ? c : chunks - 1) * PER;
            const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) T*)(tile + (at & ~63) * PER);
            uint32_t m0;                                                // (kept: the register is the compiler's)
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                         : "=&s"(m0) : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(from) : "memory");
        }
    }
    // to be called before the barrier behind which the tile is read; rows whose bit is not set become zero
    __device__ __forceinline__ void land(T* tile, int tid, uint64_t rows) const {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if ((rows | (ROWS < 64 ? ~0ull << (ROWS & 63) : 0)) == ~0ull) return;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * THREADS;
            if (!(rows >> (at / CHUNKS) & 1)) *reinterpret_cast<f32x4*>(tile + at * PER) = f32x4{};
        }
    }
};

template <typename M, int DP, int ROWS, int THREADS>
struct Loader : std::conditional_t<Mma<M>::PLANES == 1, Direct<M, DP, ROWS, THREADS>, Staged<M, DP, ROWS, THREADS>> {};

__device__ __forceinline__ uint64_t first_rows(int64_t n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// bits of 64 consecutive tile rows as register r of 32-row block `blk` sees them: bit reg_row(r) + 32 blk of the shifted word
__device__ __forceinline__ uint64_t lane_bits(uint64_t rows) { return rows >> (4 * ((threadIdx.x >> 5) & 1)); }

// Running softmax of a wave's 32 columns: m (base 2) and this half's share of the sum, the weighted sum as O^T blocks.
template <typename M, int DP>
struct Softmax {
    float m = -INFINITY, l = 0.f;
    f32x16 acc[DP / 32] = {};

    // The running maximum takes in one 32 x NB*32 step's scores, t = fma(s, c, b); returns b - maximum for weights().
    // It moves only when a score passes it by 2^8: weights up to 256 lose nothing in either type, and most steps then skip the rescaling of
    // the accumulators.
    template <int NB>
    __device__ __forceinline__ float raise(const f32x16 (&s)[NB], float c, float b) {
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
        return b - (m == -INFINITY ? 0.f : m);
    }
    // s becomes the weights 2^(s c + off), whose sum l takes in
    template <int NB>
    __device__ __forceinline__ void weights(f32x16 (&s)[NB], float c, float off) {
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
    __device__ __forceinline__ void step(f32x16 (&s)[NB], float c, float b) { weights<NB>(s, c, raise<NB>(s, c, b)); }
    template <int NB>
    __device__ __forceinline__ void weigh(const typename Mma<M>::Store* tile, const f32x16 (&p)[NB]) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            weigh_all<M, DP>(tile, 32 * k, Mma<M>::pack(p[k]), acc);
        }
    }
};

// The results of a block's four waves on the same 32 rows meet in shared memory: `join` 4 x 32 rows of DP + 4 floats (no two rows start at the
// same bank), `stats` 4 x 32 pairs (maximum, sum).  Afterwards thread t holds row t / 8's maximum, sum and columns [t % 8 * DP/8, + DP/8).
template <typename M, int DP>
__device__ __forceinline__ void join_waves(const Softmax<M, DP>& o, float* join, float* stats, float& m, float& l, float (&w)[DP / 8]) {
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

// Sums and maxima over 16 lanes (a DPP row: pairs, quads, mirrored halves) and over a wave; every lane has the result
template <int CTRL>
__device__ __forceinline__ float from_lane(float x) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ Halves row_pair(float x) {
    const uint32_t a = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return {__uint_as_float(lo), __uint_as_float(hi)};
}
__device__ __forceinline__ float row_sum(float x) {
    x += from_lane<0xB1>(x);
    x += from_lane<0x4E>(x);
    x += from_lane<0x141>(x);
    return x + from_lane<0x140>(x);
}
__device__ __forceinline__ float wave_sum(float x) {
    const Halves h = row_pair(row_sum(x));
    return both_sum(h.lo + h.hi);
}
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, from_lane<0xB1>(x));
    x = fmaxf(x, from_lane<0x4E>(x));
    x = fmaxf(x, from_lane<0x141>(x));
    x = fmaxf(x, from_lane<0x140>(x));
    const Halves h = row_pair(x);
    return both_max(fmaxf(h.lo, h.hi));
}

}  // namespace dctr
