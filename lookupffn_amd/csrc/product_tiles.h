// Products of 16-bit numbers in tiles that eight wavefronts share, for kernels whose operands are large arrays.
//
// A workgroup forms BM x BN results, sums over STEP numbers at a time: both operands' steps are copied from memory to LDS without passing a register, into one of two
// buffers, while the products of the other are formed (v_mfma_f32_32x32x16, fp32 sums).  An operand lies in memory either with the summed index along its rows (Along) or
// with the summed index from row to row (Across); the latter is read from LDS by the transposing read, so that nothing is ever transposed in memory.
// 256 x 256: a step is 64 KB and 2061 clocks of products at the peak rate, its LDS reads 1536, its copies 32 bytes a clock.
//
// A float is two half-precision terms in two planes (split_mfma.h): a step has 32 numbers of each plane and three products.
#pragma once

#include "rows16.h"
#include "split_mfma.h"

namespace product_tiles {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint4 lds_word_t;

constexpr int STEP = 64;          // numbers of a row in LDS: 128 bytes

// How operands are multiplied.
struct BF16 {
    static constexpr int PLANES = 1;
    static __device__ __forceinline__ f32x16_t mma(uint4 a, uint4 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return BF16Row::pack2(a, b); }
};
struct F16 {
    static constexpr int PLANES = 1;
    static __device__ __forceinline__ f32x16_t mma(uint4 a, uint4 b, f32x16_t c) { return mfma_f16(a, b, c); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return F16Row::pack2(a, b); }
};
struct F32Two : F16 {
    static constexpr int PLANES = 2;
};

__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)), lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    return (uint64_t)hi << 32 | lo;
}

// 16 bytes a lane from memory straight to LDS, the wavefront's 1 KB together at lds_byte.  Inline assembly, so that the compiler does not wait for the copy
// before LDS reads of the other buffer; whoever reads waits (arrived) and has a barrier.  M0 is put back: the compiler reserves it.
__device__ __forceinline__ void copy_to_lds(const char *base, uint32_t lane_offset, uint32_t lds_byte) {
    uint32_t saved_m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved_m0)
                 : "v"(lane_offset), "s"(base), "s"(lds_byte)
                 : "memory");
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_byte_of(const void *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p; }

// An array [rows, columns] of 16-bit numbers, `stride` bytes a row, the second plane `plane` bytes behind the first.  rows and columns (a multiple of 8) are those that may
// be read: what lies beyond is read as its nearest neighbour, and the other operand has zeros there, or the result is not stored.
struct Source {
    const char *at;
    int64_t stride, plane;
    int rows, columns;
};

// ROWS rows of a tile, the sum along them.  16-byte piece p of row r is at piece p ^ (r / 2 % 8), so that the 16 lanes of an LDS read that have the same piece
// of 16 rows meet every bank once.
template <int ROWS, int THREADS, int PLANES>
struct Along {
    static constexpr int WORDS = ROWS * 8, SHARE = WORDS / THREADS, K = STEP / PLANES;
    static_assert(WORDS % THREADS == 0 && THREADS % 64 == 0 && (THREADS / 8) % 16 == 0, "whole wavefronts, a thread's rows turned alike");
    const char *base;
    int64_t plane;
    uint32_t offset[SHARE];       // of the thread's rows, from base
    int k, last;                  // first number of the thread's piece in a step; the last piece that may be read

    // rows from `row`, which is less than s.rows; a tile's rows lie within 32 bits
    __device__ __forceinline__ Along(const Source &s, int row) {
        base = (const char *)uniform((uint64_t)(s.at + row * s.stride));
        const int tid = threadIdx.x, r = tid / 8, piece = (tid % 8) ^ (r / 2 % 8);
        plane = PLANES == 2 && piece >= 4 ? s.plane : 0;
        k = piece % (8 / PLANES) * 8;
        last = s.columns - 8;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) offset[i] = uint32_t(min(r + i * (THREADS / 8), s.rows - 1 - row) * s.stride);
    }
    __device__ __forceinline__ void begin(int step, uint32_t lds) const {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 * 1024), column = min(step * K + k, last) * 2;
        if constexpr (PLANES == 1) {
#pragma unroll
            for (int i = 0; i < SHARE; ++i) copy_to_lds(base, offset[i] + column, lds + wave + i * THREADS * 16);
        } else {
#pragma unroll
            for (int i = 0; i < SHARE; ++i) copy_to_lds_far(base + plane + offset[i] + column, lds + wave + i * THREADS * 16);
        }
    }
    static __device__ __forceinline__ void copy_to_lds_far(const char *at, uint32_t lds_byte) {
        uint32_t saved_m0;
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                     : "=&s"(saved_m0)
                     : "v"(at), "s"(lds_byte)
                     : "memory");
    }
    struct Reader {
        uint32_t at[4];
        __device__ __forceinline__ Reader(int first_row) {
            const int lane = threadIdx.x % 64, r = first_row + lane % 32, half = lane / 32;
#pragma unroll
            for (int c = 0; c < 4; ++c) at[c] = (r * 8 + ((2 * c + half) ^ (r / 2 % 8))) * 16;
        }
        // rows first_row + 32 b + lane % 32, numbers 16 c + 8 (lane / 32) ... + 7 of the row in LDS
        __device__ __forceinline__ uint4 operand(uint32_t lds, int b, int c) const {
            return __builtin_bit_cast(uint4, *(const lds_word_t *)(uintptr_t)(lds + at[c] + b * 32 * 128));
        }
    };
};

// COLUMNS columns of a tile, the sum from row to row.  16-byte piece p of row r is at piece p ^ 4 (r % 4), so that the four rows that a transposing read takes of 32
// columns meet every bank once.
template <int COLUMNS, int THREADS, int PLANES>
struct Across {
    static constexpr int PIECES = COLUMNS / 8, WORDS = STEP * PIECES, SHARE = WORDS / THREADS, K = STEP / PLANES;
    static_assert(PIECES >= 16 && WORDS % THREADS == 0 && THREADS % PIECES == 0 && (THREADS / PIECES) % 4 == 0, "a thread's rows turned alike");
    const char *base;
    int64_t stride, plane;
    int last_row, row, column;    // bytes

    // columns from `column0`, which is less than s.columns
    __device__ __forceinline__ Across(const Source &s, int column0) {
        base = (const char *)uniform((uint64_t)(s.at + int64_t(column0) * 2));
        stride = s.stride, plane = s.plane, last_row = s.rows - 1;
        const int tid = threadIdx.x;
        row = tid / PIECES;
        column = min((tid % PIECES ^ 4 * (row % 4)) * 8, s.columns - 8 - column0) * 2;
    }
    __device__ __forceinline__ void begin(int step, uint32_t lds) const {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 * 1024);
        // the step's rows lie within 32 bits of its first one
        const int first = step * K;
        const char *from = base + first * stride;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
            const int r = row + i * (THREADS / PIECES);
            // (a plane's rows are a multiple of the rows that a pass of all threads takes: uniform)
            const char *const of = PLANES == 2 && i * (THREADS / PIECES) >= K ? from + plane : from;
            const int in_plane = PLANES == 2 && i * (THREADS / PIECES) >= K ? r - K : r;
            copy_to_lds(of, uint32_t(min(in_plane, last_row - first) * stride) + column, lds + wave + i * THREADS * 16);
        }
    }
    struct Reader {
        uint32_t at[4];           // by d % 4
        __device__ __forceinline__ Reader(int first_column) {
            const int lane = threadIdx.x % 64, half = lane / 32, r = lane % 16 / 4, d0 = first_column / 32;
            const int piece = 2 * (lane / 16 % 2) + lane % 4 / 2;
#pragma unroll
            for (int d = 0; d < 4; ++d) at[d] = (8 * half + r) * COLUMNS * 2 + ((4 * (d0 + d) + piece) ^ 4 * r) * 16 + lane % 2 * 8;
        }
        // columns first_column + 32 b + lane % 32, rows 16 c + 8 (lane / 32) ... + 7 in LDS
        __device__ __forceinline__ uint4 operand(uint32_t lds, int b, int c) const {
            const uint2 lo = transposed(lds + at[b] + 16 * c * COLUMNS * 2), hi = transposed(lds + at[b] + (16 * c + 4) * COLUMNS * 2);
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        // Of 16 lanes' 8 bytes, lanes 4 i .. 4 i + 3 having 16 numbers of row i: lane j gets the four rows' number j.
        static __device__ __forceinline__ uint2 transposed(uint32_t at) {
            typedef __attribute__((address_space(3))) i16x4_t lds_t;
            return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)(uintptr_t)at));
        }
    };
};

// Results of a wavefront: 32 x 32 blocks, [i][j] of A's rows 32 i and B's columns 32 j from its first ones; element e of a lane is row mfma_row(e, lane / 32), column lane % 32.
template <int MB, int NB>
struct Sums {
    f32x16_t v[MB][NB];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) v[i][j][e] = 0.f;
    }
};

// Adds the products of steps first .. end - 1.  lds: two buffers of (A's + B's words) each.  of_b(operand) is shown B's operands.
template <typename F, int MB, int NB, typename A, typename B, typename OfB>
__device__ __forceinline__ void multiply(Sums<MB, NB> &sums, const A &a, const B &b, const typename A::Reader &ra, const typename B::Reader &rb, uint32_t lds, int first,
                                         int end, OfB &&of_b) {
    constexpr uint32_t BUFFER = (A::WORDS + B::WORDS) * 16;
    if (first >= end) return;
    a.begin(first, lds);
    b.begin(first, lds + A::WORDS * 16);
    uint32_t now = lds;
    for (int s = first; s < end; ++s) {
        arrived();
        __syncthreads();                  // everyone's copies are there, and nobody reads the other buffer any more
        const uint32_t next = lds + (now == lds ? BUFFER : 0);
        if (s + 1 < end) {
            a.begin(s + 1, next);
            b.begin(s + 1, next + A::WORDS * 16);
        }
        if constexpr (F::PLANES == 1) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint4 fa[MB], fb[NB];
#pragma unroll
                for (int i = 0; i < MB; ++i) fa[i] = ra.operand(now, i, c);
#pragma unroll
                for (int j = 0; j < NB; ++j) fb[j] = rb.operand(now + A::WORDS * 16, j, c);
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    of_b(j, fb[j]);
#pragma unroll
                    for (int i = 0; i < MB; ++i) sums.v[i][j] = F::mma(fa[i], fb[j], sums.v[i][j]);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint4 fa[2][MB], fb[2][NB];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
#pragma unroll
                    for (int i = 0; i < MB; ++i) fa[p][i] = ra.operand(now, i, 2 * p + c);
#pragma unroll
                    for (int j = 0; j < NB; ++j) fb[p][j] = rb.operand(now + A::WORDS * 16, j, 2 * p + c);
                }
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    of_b(j, fb[1][j]);
                    of_b(j, fb[0][j]);
                }
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int i = 0; i < MB; ++i) sums.v[i][j] = F::mma(fa[1][i], fb[0][j], sums.v[i][j]);
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int i = 0; i < MB; ++i) sums.v[i][j] = F::mma(fa[0][i], fb[1][j], sums.v[i][j]);
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int i = 0; i < MB; ++i) sums.v[i][j] = F::mma(fa[0][i], fb[0][j], sums.v[i][j]);
            }
        }
        now = next;
    }
    __syncthreads();                      // the buffers are free
}

}  // namespace product_tiles
