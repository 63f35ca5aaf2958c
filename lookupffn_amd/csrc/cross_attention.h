// What the forward and backward kernels of the attention to an encoder's states share: operands, tiles in LDS, the products.
//
// Everything is formed of v_mfma_f32_32x32x16 products with fp32 sums.  A wavefront has 32 columns (queries, or keys where their gradients are
// formed) of every product, whose operand stays in its registers; the 32 rows come from tiles in LDS that the workgroup's four wavefronts share.  A
// result element's row is 8 (e / 4) + 4 (lane / 32) + e % 4, its column lane % 32, so that what follows of a column stays in two lanes, and
// the results are, where they are, the next product's operand: its sum runs over the tile's rows in the order the lanes hold them, and
// the tile, read down its columns in that order by the transposing LDS read, is the other operand.
//
// bfloat16 and half numbers are operands as they are.  A float is two half-precision terms (split_mfma.h), three products for one, in the backward and in forward
// calls with work enough to pay for a launch that looks for the longest rows of every batch and key head: by them the numbers that pass are scaled (powers of two)
// to half's range, those that stand each row by its own.  A number that passes is held to 2^-22 of itself, or to 2^-36 of the longest row of its head where that
// is more, any other to 2^-22.  Elsewhere a float is three bfloat16 terms of 8 bits each, which together are it (the exponent range is the same, so nothing has to be
// scaled), and of the nine products six are formed, those of at least 2^-16: what is left out, second times third terms, is at most 2^-22 of the product.  (Two terms for three, 16 x 512 x 512
// x 12 x 64: forward 77 us to 54 and 10 for the look, queries' gradients 111 to 78, keys' 159 to 113.)
#pragma once

#include "rows16.h"
#include "split_mfma.h"

typedef _Float16 ca_f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 ca_bf16x8_t __attribute__((ext_vector_type(8)));
typedef short ca_i16x4_t __attribute__((ext_vector_type(4)));
typedef float ca_f32x16_t __attribute__((ext_vector_type(16)));

namespace cross_attention {

constexpr int WG = 256, WAVES = 4;
constexpr int ROWS = 32;                  // columns of a wavefront's products
constexpr int TILE = WAVES * ROWS;        // of a workgroup's
constexpr int BLOCK = 64;                 // steps whose masks are looked at together
constexpr float LOG2E = 1.4426950408889634f;

// An operand: 8 numbers along the sum, in PLANES terms.
template <int PLANES>
struct Frag {
    uint4 p[PLANES];
};

// Eight fp32 numbers as three bfloat16 terms: exact.  The first is cut off (rounded, the largest numbers would pass the range), the second, below 2^-7 of the first's
// power of two, rounded to the nearest, so that the third is at most 2^-16 of it, of either sign (cut off as well, 2^-15, always towards zero: within 1 % of the time,
// and twice as much left out).
__device__ __forceinline__ void split3(const float (&v)[8], uint4 (&t)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            // (the upper halves of both; of the third term nothing is left below them)
            w[k][i] = k == 1 ? BF16Row::pack2(a, b) : __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
            if (k < 2) {
                a -= __uint_as_float(w[k][i] << 16);
                b -= __uint_as_float(w[k][i] & 0xFFFF0000u);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) t[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}

// f of a lane's number and of that of the lane 32 away, on the vector ALU (an LDS permute is waited for).
template <typename T>
__device__ __forceinline__ float of_both_halves(float v, T &&f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

struct BF16 {
    static constexpr int PLANES = 1, BYTES = 2;
    static constexpr bool SCALED = false;
    static constexpr float LIFT = 0.f;                 // added to the exponents of the softmax's weights
    static __device__ __forceinline__ ca_f32x16_t mma(const Frag<1> &a, const Frag<1> &b, ca_f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ca_bf16x8_t, a.p[0]), __builtin_bit_cast(ca_bf16x8_t, b.p[0]), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag<1> operand(const float (&v)[8]) { return {{BF16Row::pack(v)}}; }
    // 8 numbers in memory and what a thread holds of them on their way
    struct Raw {
        uint4 u;
    };
    static __device__ __forceinline__ Raw load(const char *p) { return {*reinterpret_cast<const uint4 *>(p)}; }
    static __device__ __forceinline__ Raw zero() { return {make_uint4(0, 0, 0, 0)}; }
    static __device__ __forceinline__ Frag<1> operand(const Raw &r, float) { return {{r.u}}; }
    static __device__ __forceinline__ void unpack(const Raw &r, float (&v)[8]) { BF16Row::unpack(r.u, v); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return BF16Row::pack2(a, b); }
    static __device__ __forceinline__ float rounded(float a) { return (float)(__bf16)a; }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(BF16Row::pack2(a, b), BF16Row::pack2(c, d));
    }
};

struct F16 {
    static constexpr int PLANES = 1, BYTES = 2;
    static constexpr bool SCALED = false;
    // A weight of the softmax is at most 1 and one of many keys' small: held 2^8 times larger (2^14 in the backward), so that half's normal numbers reach down
    // to 2^-22 of the largest.
    static constexpr float LIFT = 8.f;
    static __device__ __forceinline__ ca_f32x16_t mma(const Frag<1> &a, const Frag<1> &b, ca_f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ca_f16x8_t, a.p[0]), __builtin_bit_cast(ca_f16x8_t, b.p[0]), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag<1> operand(const float (&v)[8]) { return {{F16Row::pack(v)}}; }
    typedef BF16::Raw Raw;
    static __device__ __forceinline__ Raw load(const char *p) { return BF16::load(p); }
    static __device__ __forceinline__ Raw zero() { return BF16::zero(); }
    static __device__ __forceinline__ Frag<1> operand(const Raw &r, float) { return {{r.u}}; }
    static __device__ __forceinline__ void unpack(const Raw &r, float (&v)[8]) { F16Row::unpack(r.u, v); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return F16Row::pack2(a, b); }
    static __device__ __forceinline__ float rounded(float a) { return (float)(_Float16)a; }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(F16Row::pack2(a, b), F16Row::pack2(c, d));
    }
};

struct F32 {
    static constexpr int PLANES = 3, BYTES = 4;
    static constexpr bool SCALED = false;
    static constexpr float LIFT = 0.f;
    static __device__ __forceinline__ ca_f32x16_t mma(const Frag<3> &a, const Frag<3> &b, ca_f32x16_t c) {
        auto one = [&](int i, int j) {
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ca_bf16x8_t, a.p[i]), __builtin_bit_cast(ca_bf16x8_t, b.p[j]), c, 0, 0, 0);
        };
        one(2, 0), one(0, 2), one(1, 1), one(1, 0), one(0, 1), one(0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag<3> operand(const float (&v)[8]) {
        Frag<3> f;
        split3(v, f.p);
        return f;
    }
    struct Raw {
        float4 u[2];
    };
    static __device__ __forceinline__ Raw load(const char *p) {
        return {{reinterpret_cast<const float4 *>(p)[0], reinterpret_cast<const float4 *>(p)[1]}};
    }
    static __device__ __forceinline__ Raw zero() { return {{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)}}; }
    static __device__ __forceinline__ void unpack(const Raw &r, float (&v)[8]) {
        v[0] = r.u[0].x, v[1] = r.u[0].y, v[2] = r.u[0].z, v[3] = r.u[0].w, v[4] = r.u[1].x, v[5] = r.u[1].y, v[6] = r.u[1].z, v[7] = r.u[1].w;
    }
    static __device__ __forceinline__ Frag<3> operand(const Raw &r, float) {
        float v[8];
        unpack(r, v);
        return operand(v);
    }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
        *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
    }
    static __device__ __forceinline__ float rounded(float a) { return a; }
};

// What sums are multiplied with on their way out: a number, or, where sums are scaled to half's range, a number and a power of two that a float may not have.
struct Factor {
    float by;
    int exponent;
};
__device__ __forceinline__ float times(float v, float by) { return v * by; }
__device__ __forceinline__ float times(float v, const Factor &f) { return __builtin_amdgcn_ldexpf(v * f.by, f.exponent); }
template <typename F>
__device__ __forceinline__ auto factor(float by, int exponent) {
    if constexpr (F::SCALED) return Factor{by, exponent};
    else return __builtin_amdgcn_ldexpf(by, exponent);
}

// The columns 32 d + 8 g + 4 half .. + 3 of a lane's row (half = lane / 32) to memory, by d and g; `row` where the lane's row begins, all lanes together.  Of 16-bit
// results the lanes of a row exchange four columns of two groups, so that each has eight that lie together and stores 16 bytes.
// rest: where what the rounding takes goes, or null.
template <typename F, int DB, typename S>
__device__ __forceinline__ void store_row(const ca_f32x16_t (&o)[DB], const S &by, char *row, bool live, int columns, int half, char *rest = nullptr) {
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        if constexpr (F::BYTES == 4) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = 32 * d + 8 * g + 4 * half;
                if (live && col < columns)
                    F::store4(row + col * F::BYTES, times(o[d][4 * g], by), times(o[d][4 * g + 1], by), times(o[d][4 * g + 2], by), times(o[d][4 * g + 3], by));
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = times(o[d][4 * g + e], by);
                auto put = [&](char *to) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // the upper lanes' first four columns and the lower lanes' last four change places
                        const auto swapped = __builtin_amdgcn_permlane32_swap(F::pack2(t[2 * e], t[2 * e + 1]), F::pack2(t[4 + 2 * e], t[4 + 2 * e + 1]), false, false);
                        w[e] = swapped[0], w[2 + e] = swapped[1];
                    }
                    const int col = 32 * d + 8 * (g + half);
                    if (live && col < columns) *reinterpret_cast<uint4 *>(to + col * 2) = make_uint4(w[0], w[1], w[2], w[3]);
                };
                put(row);
                if (rest) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e] -= F::rounded(t[e]);
                    put(rest);
                }
            }
        }
    }
}

// A tile of KT rows of DP numbers in LDS, PLANES terms of 16 bits, DP / 8 pieces of 16 bytes a row.  The pieces of a row are turned by its number, so
// that the 16 rows that an operand's read takes of one piece, and the 4 rows x 64 bytes that half a transposing read takes, are on different banks.
template <typename F, int DP, int KT>
struct Tile {
    static constexpr int PIECES = DP / 8, PLANE = KT * PIECES, SIZE = F::PLANES * PLANE;     // in 16-byte words
    static constexpr int SHARE = PLANE / WG;                                                 // pieces a thread brings
    typedef __attribute__((address_space(3))) const char *lds_bytes;
    typedef uint32_t word_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) const word_t *lds_words;
    static __host__ __device__ __forceinline__ constexpr int turned(int row) {
        if constexpr (DP == 32) return (row >> 2) & 3;
        else if constexpr (DP == 64) return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
        else return (row & 3) << 2 | ((row >> 2) & 3);
    }
    static __device__ __forceinline__ int at(int row, int piece) { return row * PIECES + (piece ^ turned(row)); }
    static __device__ __forceinline__ void put(uint4 *lds, int row, int piece, const typename F::Raw &raw, float scale) {
        const Frag<F::PLANES> f = F::operand(raw, scale);
#pragma unroll
        for (int p = 0; p < F::PLANES; ++p) lds[p * PLANE + at(row, piece)] = f.p[p];
    }

    // Where a lane reads, as byte addresses in LDS: of a tile at 0, block of 32 rows (16 where the sum is over rows) 0, term 0; what
    // else there is to a place is a constant of the instruction.
    struct Reader {
        uint32_t row[DP / 16], lo[DP / 32], hi[DP / 32];
        __device__ __forceinline__ explicit Reader(const uint4 *lds, int lane) {
            const uint32_t base = (uint32_t)(uintptr_t)(lds_bytes)lds;
            const int r = lane & 31, half = lane >> 5;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) row[c] = base + at(r, 2 * c + half) * 16;
            const int first = 4 * half + ((lane & 15) >> 2), piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), byte = 8 * (lane & 1);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                lo[d] = base + at(first, 4 * d + piece) * 16 + byte;
                hi[d] = base + at(first + 8, 4 * d + piece) * 16 + byte;
            }
        }
        // operand of the 32 rows from 32 b, 16 columns `chunk`, of the tile at `tile` (in 16-byte words)
        __device__ __forceinline__ Frag<F::PLANES> rows(int tile, int b, int chunk) const {
            Frag<F::PLANES> f;
#pragma unroll
            for (int p = 0; p < F::PLANES; ++p) f.p[p] = __builtin_bit_cast(uint4, *(lds_words)(uintptr_t)(row[chunk] + (tile + p * PLANE + b * 32 * PIECES) * 16));
            return f;
        }
        // operand of the tile's columns 32 d + lane % 32 with the sum over its rows 16 c + 4 half + {0 .. 3, 8 .. 11}: the order in which
        // a lane has the elements 8 (c % 2) .. + 7 of a result of the rows from 32 (c / 2)
        __device__ __forceinline__ Frag<F::PLANES> columns(int tile, int c, int d) const {
            Frag<F::PLANES> f;
#pragma unroll
            for (int p = 0; p < F::PLANES; ++p) {
                const uint32_t off = (tile + p * PLANE + c * 16 * PIECES) * 16;
                const uint2 a = transposed(lo[d] + off), b = transposed(hi[d] + off);
                f.p[p] = make_uint4(a.x, a.y, b.x, b.y);
            }
            return f;
        }
    };

    // Of 16 lanes' 8 bytes, lanes 4 i .. 4 i + 3 having 16 numbers of row i: lane j gets the four rows' number j.
    static __device__ __forceinline__ uint2 transposed(uint32_t at) {
        typedef __attribute__((address_space(3))) ca_i16x4_t lds_t;
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)(uintptr_t)at));
    }
};

// fp32 numbers in two half-precision terms.  SCALED: what comes from memory is multiplied by a power of two.
struct F32Two {
    static constexpr int PLANES = 2, BYTES = 4;
    static constexpr bool SCALED = true;
    static constexpr float LIFT = F16::LIFT;
    static __device__ __forceinline__ ca_f32x16_t mma(const Frag<2> &a, const Frag<2> &b, ca_f32x16_t c) {
        c = mfma_f16(a.p[1], b.p[0], c);
        c = mfma_f16(a.p[0], b.p[1], c);
        return mfma_f16(a.p[0], b.p[0], c);
    }
    static __device__ __forceinline__ Frag<2> operand(const float (&v)[8]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = split_hi(v[2 * i], v[2 * i + 1], 1.f);
            l[i] = split_rest(v[2 * i], v[2 * i + 1], h[i]);
        }
        return {{make_uint4(h[0], h[1], h[2], h[3]), make_uint4(l[0], l[1], l[2], l[3])}};
    }
    typedef F32::Raw Raw;
    static __device__ __forceinline__ Raw load(const char *p) { return F32::load(p); }
    static __device__ __forceinline__ Raw zero() { return F32::zero(); }
    static __device__ __forceinline__ void unpack(const Raw &r, float (&v)[8]) { F32::unpack(r, v); }
    static __device__ __forceinline__ Frag<2> operand(const Raw &r, float scale) {
        float v[8];
        unpack(r, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= scale;
        return operand(v);
    }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) { F32::store4(p, a, b, c, d); }
    static __device__ __forceinline__ float rounded(float a) { return a; }
};

// Largest over an aligned group of lanes, as lane_group_sum; from groups to the wavefront.
template <int LANES>
__device__ __forceinline__ float lane_group_max(float v) {
    if constexpr (LANES > 1) v = fmaxf(v, lane_xor<1>(v));
    if constexpr (LANES > 2) v = fmaxf(v, lane_xor<2>(v));
    if constexpr (LANES > 4) v = fmaxf(v, lane_xor<4>(v));
    if constexpr (LANES > 8) v = fmaxf(v, lane_xor<8>(v));
    return v;
}
template <int LANES>
__device__ __forceinline__ float over_groups_max(float v) {
    if constexpr (LANES <= 4) v = fmaxf(v, lane_xor<4>(v));
    if constexpr (LANES <= 8) v = fmaxf(v, lane_xor<8>(v));
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}

// log2 of a row's length, LANES lanes a row, 8 columns a lane; -infinity where there is nothing but zeros, or no length.  (By way of the largest number's
// power of two: squares would leave fp32's range.)
template <int LANES>
__device__ __forceinline__ float row_level(const float (&v)[8]) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
    most = lane_group_max<LANES>(most);
    const int e = int(__float_as_uint(most) >> 23) - 127;
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = __builtin_amdgcn_ldexpf(v[i], -e);
        squares = fmaf(x, x, squares);
    }
    squares = lane_group_sum<LANES>(squares);
    return most > 0.f && is_finite(squares) ? (float)e + 0.5f * __builtin_amdgcn_logf(squares) : -INFINITY;
}
constexpr int LEVEL_ROWS = 128;           // rows of a workgroup that looks for the longest: those of a group of lanes are asked for together
constexpr int level_lanes(int columns) { return columns <= 32 ? 4 : columns <= 64 ? 8 : 16; }

// Largest of the `tiles` levels of a batch and key head (every lane's); -infinity of none.
__device__ __forceinline__ float longest(const float *levels, int64_t bh, int tiles) {
    if (tiles == 0) return -INFINITY;
    const float *const l = levels + bh * tiles;
    const int lane = threadIdx.x & 63;
    float most = l[min(lane, tiles - 1)];
    for (int i = lane + 64; i < tiles; i += 64) most = fmaxf(most, l[i]);
    most = fmaxf(most, lane_xor<1>(most));
    most = fmaxf(most, lane_xor<2>(most));
    most = fmaxf(most, lane_xor<4>(most));
    most = fmaxf(most, lane_xor<8>(most));
    most = fmaxf(most, lane_xor<16>(most));
    most = fmaxf(most, lane_xor<32>(most));
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(most)));
}
// The power of two that takes rows of at most that length below 2^14.
__device__ __forceinline__ int exponent_for(float level) { return level == -INFINITY ? 0 : min(max(13 - (int)ceilf(level), -126), 126); }

// Factors that a lane is about to multiply with, and that span fp32's range, as fp32 numbers in two terms of half precision: times 2^n for the lane, which falls where
// one of them passes 2^15 (by 2^3 more than it has to: the next ones are of like size), and takes its sums along.  So a lane's sums are as near as their largest
// term has them, however small it is: by one power for all lanes the keys' gradients of a key to which little attends were left with a few bits.
template <int DB>
__device__ __forceinline__ void fit(ca_f32x16_t &t, int &n, ca_f32x16_t (&sums)[DB]) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(t[e]));
    most = of_both_halves(most, [](float x, float y) { return fmaxf(x, y); });
    const int at_most = 141 - int(__float_as_uint(most) >> 23);
    if (__any(at_most < n)) {
        const int to = at_most < n ? at_most - 3 : n;
        const float by = __builtin_amdgcn_ldexpf(1.f, to - n);
        n = to;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) sums[d][e] *= by;
    }
    const float by = __builtin_amdgcn_ldexpf(1.f, n);
#pragma unroll
    for (int e = 0; e < 16; ++e) t[e] *= by;
}
constexpr int FIT_FIRST = 126;            // n before there are any

// N products, product i with the operand that load(i) reads from LDS, AHEAD operands asked for ahead of the one that is used: left to itself the compiler asks for
// one, waits for it, and asks for the next (keys' gradients of 4 x 2048 to 4096 x 16 x 128 bfloat16, in pairs: see there).
template <typename F, int N, bool ORDERED = true, typename L, typename M>
__device__ __forceinline__ void products(L &&load, M &&multiply) {
    if constexpr (!ORDERED) {
        static_for<N>([&](auto i) { multiply(i, load(i)); });
        return;
    }
    constexpr int MOST = F::PLANES == 1 ? 4 : 2, AHEAD = N < MOST ? N : MOST, ORDER = 0x406;        // (what may pass: the vector and scalar ALU)
    Frag<F::PLANES> f[AHEAD];
    static_for<AHEAD>([&](auto i) { f[i] = load(i); });
    __builtin_amdgcn_sched_barrier(ORDER);
    static_for<N>([&](auto i) {
        multiply(i, f[i % AHEAD]);
        __builtin_amdgcn_sched_barrier(ORDER);
        if constexpr (i + AHEAD < N) {
            f[i % AHEAD] = load(std::integral_constant<int, i + AHEAD>{});
            __builtin_amdgcn_sched_barrier(ORDER);
        }
    });
}

// A wavefront's own 32 rows straight from memory in operand layout: of 16 columns the lane's row, 8 of them by half, zeros beyond the row.  fp32 numbers in two
// terms are scaled to half's range, every row by a power of two of its own: -> its exponent.
template <typename F, int CHUNKS>
__device__ __forceinline__ int own_rows(const char *row, bool live, int half, int pieces, Frag<F::PLANES> (&out)[CHUNKS]) {
    typename F::Raw raw[CHUNKS];
    float most = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int piece = 2 * c + half;
        raw[c] = live && piece < pieces ? F::load(row + piece * 8 * F::BYTES) : F::zero();
        if constexpr (F::SCALED) {
            float v[8];
            F::unpack(raw[c], v);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
        }
    }
    int exponent = 0;
    if constexpr (F::SCALED) {
        most = of_both_halves(most, [](float x, float y) { return fmaxf(x, y); });
        if (most > 0.f && is_finite(most)) exponent = min(max(140 - int(__float_as_uint(most) >> 23), -126), 126);          // to 2^13 and more
    }
    const float scale = F::SCALED ? __builtin_amdgcn_ldexpf(1.f, exponent) : 1.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) out[c] = F::operand(raw[c], scale);
    return exponent;
}

// Division of numbers below 2^31 by one that the host knows (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994): the compiler's takes
// thirty instructions, this one three.
struct Divisor {
    uint32_t by, multiplier, shift;
    Divisor() = default;
    explicit Divisor(uint32_t d) : by(d), multiplier(0), shift(0) {
        while ((1u << shift) < d) ++shift;
        multiplier = uint32_t((((uint64_t(1) << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, multiplier) + n) >> shift; }
};

// Queries of the heads that share a key head are rows of one matrix: row r is token r / group, head h' * group + r % group.
struct Rows {
    const char *base;                     // of the batch and the key head's first query head
    int64_t token, head;                  // strides in bytes
    Divisor group;
    __device__ __forceinline__ const char *at(int r) const {
        const int t = group.quotient(r);
        return base + t * token + (r - t * group.by) * head;
    }
};

// Bit j of a step's word: key step * KT + j takes part.  words[i]: of step first + i.  All wavefronts of a workgroup call it together; a barrier is theirs to have.
template <int KT>
__device__ __forceinline__ void look_at_masks(uint64_t *words, const uint8_t *mask, int64_t first, int64_t steps, int64_t keys) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 4
    for (int n = 0; n < BLOCK / WAVES; ++n) {
        const int i = n * WAVES + wave;
        const int64_t key = (first + i) * KT + lane;
        const bool in = first + i < steps && lane < KT && key < keys;
        const uint64_t w = __ballot(in && (!mask || mask[key] != 0));
        if (lane == 0) words[i] = w;
    }
}

__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    // (the builtin's result is signed)
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)), lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    return (uint64_t)hi << 32 | lo;
}

// 16 bytes a lane from memory straight to LDS, the wavefront's 1 KB together at lds_byte_addr.  Inline assembly, so that the compiler does not wait for the
// copy before LDS reads of the other buffer; whoever reads waits (arrived) and has a barrier.  M0 is put back: the compiler
// reserves it and does not honour a clobber declaration of it.
__device__ __forceinline__ void copy_to_lds(const char *base, uint32_t lane_offset, uint32_t lds_byte_addr) {
    uint32_t saved_m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved_m0)
                 : "v"(lane_offset), "s"(base), "s"(lds_byte_addr)
                 : "memory");
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Brings the rows of two arrays, tile by tile, into a buffer of two tiles: numbers of 16 bits as they are, by copies that pass no register; fp32 numbers
// through registers, where they are split.  begin(): asked for; end(): there, after the barrier that follows.
template <typename F, int DP, int KT>
struct Feed {
    typedef Tile<F, DP, KT> T;
    static constexpr int ROWS_APART = WG / T::PIECES;         // of a thread's pieces
    static_assert(T::turned(ROWS_APART) == 0 || T::SHARE == 1, "a thread's pieces are turned alike");
    uint4 *lds;
    uint32_t lds_byte;
    float scale_a = 1.f, scale_b = 1.f;   // of numbers that are split
    int row, piece;                       // of the thread's first piece; the piece is that of memory
    typename F::Raw raw[F::PLANES == 1 ? 1 : 2 * T::SHARE];

    __device__ __forceinline__ Feed(uint4 *at, int pieces) : lds(at) {
        const int tid = threadIdx.x;
        row = tid / T::PIECES;
        piece = tid % T::PIECES;
        if constexpr (F::PLANES == 1) {
            lds_byte = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)at + (tid >> 6) * 1024;
            piece ^= T::turned(row);
        }
        column = (piece < pieces ? piece : 0) * 8 * F::BYTES;         // (what is beyond the columns meets zeros or is not stored)
    }
    // Piece i of a thread is at a + offset_a(row), b + offset_b(row) of tile row `row`.
    template <typename A, typename B>
    __device__ __forceinline__ void begin(int buf, const char *a, const char *b, A &&offset_a, B &&offset_b) {
#pragma unroll
        for (int i = 0; i < T::SHARE; ++i) {
            const int r = row + i * ROWS_APART;
            const uint32_t from_a = offset_a(r, i) + column, from_b = offset_b(r, i) + column;
            if constexpr (F::PLANES == 1) {
                const uint32_t to = lds_byte + (buf * 2 * T::SIZE + i * WG) * 16;
                copy_to_lds(a, from_a, __builtin_amdgcn_readfirstlane(to));
                copy_to_lds(b, from_b, __builtin_amdgcn_readfirstlane(to + T::SIZE * 16));
            } else {
                raw[2 * i] = F::load(a + from_a);
                raw[2 * i + 1] = F::load(b + from_b);
            }
        }
    }
    __device__ __forceinline__ void end(int buf) {
        if constexpr (F::PLANES == 1) {
            arrived();
        } else {
            uint4 *const to = lds + buf * 2 * T::SIZE;
#pragma unroll
            for (int i = 0; i < T::SHARE; ++i) {
                T::put(to, row + i * ROWS_APART, piece, raw[2 * i], scale_a);
                T::put(to + T::SIZE, row + i * ROWS_APART, piece, raw[2 * i + 1], scale_b);
            }
        }
    }

private:
    uint32_t column;
};

// The keys and values of a step: those that take no part are the step's first that does once more (their weights are zero, and what they hold is
// not looked at).  Every step that is asked for has one.
template <typename F, int DP, int KT>
struct KeyFeed : Feed<F, DP, KT> {
    const char *k, *v;
    int64_t k_stride, v_stride;           // bytes; 64 of either fit in 32 bits
    __device__ __forceinline__ KeyFeed(uint4 *at, int pieces, const char *k, const char *v, int64_t ks, int64_t vs)
        : Feed<F, DP, KT>(at, pieces), k(k), v(v), k_stride(ks), v_stride(vs) {}
    __device__ __forceinline__ void begin(int buf, int64_t step, uint64_t word) {
        constexpr uint64_t FULL = ~0ull >> (64 - KT);
        const char *const kp = k + step * KT * k_stride, *const vp = v + step * KT * v_stride;
        const uint32_t ks = (uint32_t)k_stride, vs = (uint32_t)v_stride;
        if (word == FULL) {
            Feed<F, DP, KT>::begin(buf, kp, vp, [&](int r, int) { return r * ks; }, [&](int r, int) { return r * vs; });
        } else {
            const int first = __builtin_ctzll(word);
            auto of = [&](int r) { return (uint32_t)(word >> r & 1 ? r : first); };
            Feed<F, DP, KT>::begin(buf, kp, vp, [&](int r, int) { return of(r) * ks; }, [&](int r, int) { return of(r) * vs; });
        }
    }
};

// Walks the steps of [begin, end) that have a key that takes part: compute(buffer, word) with the buffer as a constant, once behind each begin and end of the feed.
template <int KT, typename KF, typename C>
__device__ __forceinline__ void walk_keys(KF &feed, uint64_t *words, const uint8_t *mask, int64_t begin, int64_t end, int64_t keys, C &&compute) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int64_t first = begin; first < end; first += BLOCK) {
        look_at_masks<KT>(words, mask, first, end, keys);
        __syncthreads();
        uint64_t left = __ballot(words[lane] != 0);
        if (left) {
            uint64_t word, next = 0;
            int64_t step, coming = 0;
            auto ask = [&](int buf) {                    // for the next step, if there is one
                if (!left) return false;
                const int i = __builtin_ctzll(left);
                left &= left - 1;
                next = uniform(words[i]);
                coming = first + i;
                feed.begin(buf, coming, next);
                return true;
            };
            ask(0);
            feed.end(0);
            __syncthreads();
#pragma unroll 1
            for (;;) {
                word = next, step = coming;
                bool more = ask(1);
                compute(std::integral_constant<int, 0>{}, word, step);
                if (!more) break;
                feed.end(1);
                __syncthreads();
                word = next, step = coming;
                more = ask(0);
                compute(std::integral_constant<int, 1>{}, word, step);
                if (!more) break;
                feed.end(0);
                __syncthreads();
            }
        }
        __syncthreads();                  // the words and the buffers are free again
    }
}

// Where row `row` (of the queries that share key head kh, or with group 1 of the keys) of a batch is in [B, len, heads, columns]: its number of heads' rows.
__device__ __forceinline__ int64_t heads_row(int b, int kh, int row, int64_t len, int key_heads, const Divisor &group) {
    const int token = group.quotient(row);
    return ((b * len + token) * key_heads + kh) * group.by + (row - token * group.by);
}

// What a forward keeps for its backward beside the result: every row's level, and of 16-bit results what their rounding took, in the same format: delta, a sum
// of the result times its gradient, is what is left of ds where a query has few keys, and with the rounded result alone ds would be off by as much as by
// its own rounding and more (5 keys: 3.7e-3 of the queries' gradients in bfloat16 where a rounding is 1.7e-3).
struct Kept {
    float *levels;
    char *rest;
};
inline int64_t kept_bytes(int64_t rows, int64_t columns, int bytes) { return (rows * 4 + 15) / 16 * 16 + (bytes == 2 ? rows * columns * 2 : 0); }
inline Kept kept_at(void *p, int64_t rows, int bytes) {
    char *const at = static_cast<char *>(p);
    return {static_cast<float *>(p), at && bytes == 2 ? at + (rows * 4 + 15) / 16 * 16 : nullptr};
}

// Threads of a launch at most.
constexpr int64_t MOST_THREADS = UINT32_MAX;

// Which unit of work a workgroup has: neighbours (tiles that read the same keys) on one XCD.
struct Unit {
    int tile, split, bh, b, kh;
};
__device__ __forceinline__ Unit unit_of(uint32_t block, uint32_t blocks, const Divisor &tiles, const Divisor &splits, const Divisor &key_heads) {
    const uint32_t xcd = block & 7, per = blocks >> 3, rem = blocks & 7, unit = xcd * per + (xcd < rem ? xcd : rem) + (block >> 3);
    const uint32_t pair = tiles.quotient(unit), bh = splits.quotient(pair), b = key_heads.quotient(bh);
    return {int(unit - pair * tiles.by), int(pair - bh * splits.by), int(bh), int(b), int(bh - b * key_heads.by)};
}

}  // namespace cross_attention
