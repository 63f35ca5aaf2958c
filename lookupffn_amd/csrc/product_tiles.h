// Products of 16-bit numbers in tiles that eight wavefronts share, for kernels whose operands are large arrays.
//
// A workgroup forms BM x BN results, sums over STEP numbers at a time: both operands' steps are copied from memory to LDS without passing a register, into one of two
// buffers, while the products of the other are formed (v_mfma_f32_32x32x16, fp32 sums).  An operand lies in memory either with the summed index along its rows (Along) or
// with the summed index from row to row (Across); the latter is read from LDS by the transposing read, so that nothing is ever transposed in memory.
// 256 x 256: a step is 64 KB and 2061 clocks of products at the peak rate, its LDS reads 1536, its copies 32 bytes a clock.
//
// A float is two half-precision terms (split_mfma.h), "planes" of an operand: a step has 32 numbers of each plane and three products.  In memory a row's planes take turns, 32 numbers each, so
// that a step reads whole lines (two arrays one behind the other: logits of 385 tokens, 32003 x 520, 57 us instead of 47, of 9 tokens, 50265 x 840, 100 instead of 71).
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

// An array [rows, columns] of 16-bit numbers, or of two planes' in turns, `stride` bytes a row.  rows and columns (a multiple of 8, of two planes of 32) are those that may
// be read: what lies beyond is read as its nearest neighbour, and the other operand has zeros there, or the result is not stored.
struct Source {
    const char *at;
    int64_t stride;
    int rows, columns;
};

// Where a number of the first plane is in a row, in bytes; the second's is 64 further.
template <int PLANES>
__host__ __device__ __forceinline__ constexpr int64_t byte_of(int64_t column) {
    return PLANES == 1 ? column * 2 : column / 32 * 128 + column % 32 * 2;
}

// ROWS rows of a tile, the sum along them.  16-byte piece p of row r is at piece p ^ (r / 2 % 8), so that the 16 lanes of an LDS read that have the same piece
// of 16 rows meet every bank once.
template <int ROWS, int THREADS, int PLANES>
struct Along {
    static constexpr int WORDS = ROWS * 8, SHARE = WORDS / THREADS, K = STEP / PLANES;
    static_assert(WORDS % THREADS == 0 && THREADS % 64 == 0 && (THREADS / 8) % 16 == 0, "whole wavefronts, a thread's rows turned alike");
    const char *base;
    uint32_t offset[SHARE];       // of the thread's rows, from base
    int k, last;                  // bytes: the thread's piece in a step; the last piece that may be read

    // rows from `row`, which is less than s.rows; a tile's rows lie within 32 bits
    __device__ __forceinline__ Along(const Source &s, int row) {
        base = (const char *)uniform((uint64_t)(s.at + row * s.stride));
        const int tid = threadIdx.x, r = tid / 8;
        k = ((tid % 8) ^ (r / 2 % 8)) * 16;
        last = s.columns * 2 * PLANES - 16;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) offset[i] = uint32_t(min(r + i * (THREADS / 8), s.rows - 1 - row) * s.stride);
    }
    // the thread's i-th piece of a step
    __device__ __forceinline__ void begin(int step, uint32_t lds, int i) const {
        const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64 * 1024) + i * THREADS * 16;
        copy_to_lds(base, offset[i] + min(step * (STEP * 2) + k, last), to);
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
    int64_t stride;
    int last_row, row, column;    // bytes

    // columns from `column0`, which is less than s.columns
    __device__ __forceinline__ Across(const Source &s, int column0) {
        base = (const char *)uniform((uint64_t)(s.at + byte_of<PLANES>(column0)));
        stride = s.stride, last_row = s.rows - 1;
        const int tid = threadIdx.x;
        row = tid / PIECES;
        column = (int)byte_of<PLANES>(min((tid % PIECES ^ 4 * (row % 4)) * 8, s.columns - 8 - column0));
    }
    // the thread's i-th piece of a step
    __device__ __forceinline__ void begin(int step, uint32_t lds, int i) const {
        const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64 * 1024) + i * THREADS * 16;
        // the step's rows lie within 32 bits of its first one (a step that is behind the last row reads that)
        const int first = min(step * K, last_row), r = row + i * (THREADS / PIECES);
        const char *from = base + first * stride;
        // (a plane's rows are a multiple of the rows that a pass of all threads takes: uniform)
        const bool second = PLANES == 2 && i * (THREADS / PIECES) >= K;
        copy_to_lds(second ? from + 64 : from, uint32_t(min(second ? r - K : r, last_row - first) * (int)stride) + column, to);
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

// The products of one tile after the other.  The steps of all tiles are one stream: while a step's products are formed the next one is there, and the one behind it is on its way, also where
// it is the next tile's, so that a tile's first products have their operands when the last tile's results are done with.  (While those are, all eight wavefronts are at it and no products are
// formed: for the loss's logits 8700 clocks a tile, of 29100 at 512 columns, for their gradients 12400 of 33000.)  In a step four chunks of operands are read from
// LDS, each while the products of the chunk before are formed; with the last one in registers the buffer is free: the one barrier of a step stands there, before the last chunk's products.
// Every tile has at least two steps.
template <typename F, int MB, int NB, typename A, typename B>
struct Stream {
    static constexpr uint32_t OF_B = A::WORDS * 16, BUFFER = (A::WORDS + B::WORDS) * 16, LDS = 2 * BUFFER;
    const typename A::Reader ra;
    const typename B::Reader rb;
    uint32_t now, other;                 // buffers: of the step that is next to be multiplied, and of the one behind it

    __device__ __forceinline__ Stream(uint32_t lds, int row_a, int row_b) : ra(row_a), rb(row_b), now(lds), other(lds + BUFFER) {}

    static constexpr int COPIES = A::SHARE + B::SHARE, READS = MB + NB, PRODUCTS = MB * NB;
    static __device__ __forceinline__ void copy(const A &a, const B &b, int step, uint32_t buffer, int n) {
        if (n < A::SHARE) a.begin(step, buffer, n);
        else b.begin(step, buffer + OF_B, n - A::SHARE);
    }
    static __device__ __forceinline__ void copy(const A &a, const B &b, int step, uint32_t buffer) {
#pragma unroll
        for (int n = 0; n < COPIES; ++n) copy(a, b, step, buffer, n);
    }
    // the first tile's first two steps
    __device__ __forceinline__ void prime(const A &a, const B &b, int first) const {
        copy(a, b, first, now);
        copy(a, b, first + 1, other);
        arrived();
        __syncthreads();
    }
    static __device__ __forceinline__ void landed() { arrived(); }
    // Nothing is on its way any more, and nobody reads the buffers.
    static __device__ __forceinline__ void done() {
        arrived();
        __syncthreads();
    }
    // Adds the products of steps first .. end - 1 of (of_a, of_b); behind them those from next_first of (next_a, next_b) are brought, which become of_a and of_b (behind the last tile
    // any steps that can be read, and done()).  seen(j, operand) is shown B's operands; beside() is called once, for copies that come with the next tile's first step.  Between two tiles the
    // caller waits (landed) for what is on its way, before it stores anything: the second tile's first step does not wait, so that the stores have that long.
    template <typename Seen, typename Beside>
    __device__ __forceinline__ void multiply(Sums<MB, NB> &sums, A &of_a, B &of_b, int first, int end, const A &next_a, const B &next_b, int next_first, Seen &&seen,
                                             Beside &&beside) {
        // chunk c: of one plane, numbers 16 c .. of both; of two, numbers 16 (c / 2) .., of A the second terms and then the first, of B the first and then the second
        constexpr bool TWO = F::PLANES == 2;
        uint4 fa[2][MB], fb[2][NB];
        // the n-th read of a chunk's operands, in the order in which the products want them
        auto read = [&](uint32_t buffer, int c, int n) {
            const int part_a = TWO ? (c % 2 == 0 ? 2 : 0) + c / 2 : c, part_b = TWO ? (c % 2 == 0 ? 0 : 2) + c / 2 : c;
            if (n == 0) fb[c % 2][0] = rb.operand(buffer + OF_B, 0, part_b);
            else if (n <= MB) fa[c % 2][n - 1] = ra.operand(buffer, n - 1, part_a);
            else fb[c % 2][n - MB] = rb.operand(buffer + OF_B, n - MB, part_b);
        };
        auto read_all = [&](uint32_t buffer, int c) {
#pragma unroll
            for (int n = 0; n < READS; ++n) read(buffer, c, n);
        };
        // a chunk's products, between(n) behind the n-th; nothing is moved across
        auto form = [&](int c, auto &&between) {
#pragma unroll
            for (int n = 0; n < PRODUCTS; ++n) {
                const int i = n % MB, j = n / MB;
                if (i == 0) seen(j, fb[c % 2][j]);
                sums.v[i][j] = F::mma(fa[c % 2][i], fb[c % 2][j], sums.v[i][j]);
                between(n);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // of two planes, the product of both first terms: B's are those of the chunk before, whose place the next chunk's take
        auto form_first = [&](int c) {
            if (TWO && c % 2 == 1) {
#pragma unroll
                for (int n = 0; n < PRODUCTS; ++n) sums.v[n % MB][n / MB] = F::mma(fa[1][n % MB], fb[0][n / MB], sums.v[n % MB][n / MB]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        read_all(now, 0);
        int ahead = 2;
        for (int s = first; s < end; ++s) {
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                form_first(c);
                form(c, [&](int n) {
#pragma unroll
                    for (int r = n * READS / PRODUCTS; r < (n + 1) * READS / PRODUCTS; ++r) read(now, c + 1, r);
                });
            }
            if (s > first) arrived();
            lds_barrier();                       // the next step is there, and nobody reads this one any more
            form_first(3);
            if (s + 2 == end) {
                of_a = next_a;
                of_b = next_b;
                ahead = next_first - end + 2;
                beside();
            }
            form(3, [&](int n) {
#pragma unroll
                for (int r = n * READS / PRODUCTS; r < (n + 1) * READS / PRODUCTS; ++r) read(other, 0, r);            // (behind the last step: read again later)
#pragma unroll
                for (int r = n * COPIES / PRODUCTS; r < (n + 1) * COPIES / PRODUCTS; ++r) copy(of_a, of_b, s + ahead, now, r);
            });
            const uint32_t swap = now;
            now = other;
            other = swap;
        }
    }
};

}  // namespace product_tiles
