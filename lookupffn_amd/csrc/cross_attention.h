// What the forward and backward kernels of the attention to an encoder's states share: operands, tiles in LDS, the products.
//
// Everything is formed of v_mfma_f32_32x32x16 products with fp32 sums.  A wavefront has 32 columns (queries, or keys where their gradients are
// formed) of every product, whose operand stays in its registers; the 32 rows come from tiles in LDS that the workgroup's four wavefronts share.  A
// result element's row is 8 (e / 4) + 4 (lane / 32) + e % 4, its column lane % 32, so that what follows of a column stays in two lanes, and
// the results are, where they are, the next product's operand: its sum runs over the tile's rows in the order the lanes hold them, and
// the tile, read down its columns in that order by the transposing LDS read, is the other operand.
//
// bfloat16 and half numbers are operands as they are.  A float is taken as three bfloat16 terms of 8 bits each, which together are it (the
// exponent range is the same, so nothing has to be scaled), and of the nine products six are formed, those of at least 2^-16:
// what is left out is below 2^-22 of the product.
#pragma once

#include "rows16.h"

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

// Eight fp32 numbers as three bfloat16 terms by cutting off: exact.
__device__ __forceinline__ void split3(const float (&v)[8], uint4 (&t)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
            w[k][i] = __builtin_amdgcn_perm(y, x, 0x07060302);       // the upper halves of both
            if (k < 2) {
                a -= __uint_as_float(x & 0xFFFF0000u);
                b -= __uint_as_float(y & 0xFFFF0000u);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) t[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}

struct BF16 {
    static constexpr int PLANES = 1, BYTES = 2;
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
    static __device__ __forceinline__ Frag<1> operand(const Raw &r) { return {{r.u}}; }
    static __device__ __forceinline__ void unpack(const Raw &r, float (&v)[8]) { BF16Row::unpack(r.u, v); }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(BF16Row::pack2(a, b), BF16Row::pack2(c, d));
    }
};

struct F16 {
    static constexpr int PLANES = 1, BYTES = 2;
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
    static __device__ __forceinline__ Frag<1> operand(const Raw &r) { return {{r.u}}; }
    static __device__ __forceinline__ void unpack(const Raw &r, float (&v)[8]) { F16Row::unpack(r.u, v); }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(F16Row::pack2(a, b), F16Row::pack2(c, d));
    }
};

struct F32 {
    static constexpr int PLANES = 3, BYTES = 4;
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
    static __device__ __forceinline__ Frag<3> operand(const Raw &r) {
        float v[8];
        unpack(r, v);
        return operand(v);
    }
    static __device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
        *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
    }
};

// A tile of KT rows of DP numbers in LDS, PLANES terms of 16 bits, DP / 8 pieces of 16 bytes a row.  The pieces of a row are turned by its number, so
// that the 16 rows that an operand's read takes of one piece, and the 4 rows x 64 bytes that half a transposing read takes, are on different banks.
template <typename F, int DP, int KT>
struct Tile {
    static constexpr int PIECES = DP / 8, PLANE = KT * PIECES, SIZE = F::PLANES * PLANE;     // in 16-byte words
    static constexpr int SHARE = PLANE / WG;                                                 // pieces a thread brings
    static __device__ __forceinline__ int turned(int row) {
        if constexpr (DP == 32) return (row >> 2) & 3;
        else if constexpr (DP == 64) return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
        else return (row & 3) << 2 | ((row >> 2) & 3);
    }
    static __device__ __forceinline__ int at(int row, int piece) { return row * PIECES + (piece ^ turned(row)); }
    static __device__ __forceinline__ void put(uint4 *lds, int row, int piece, const typename F::Raw &raw) {
        const Frag<F::PLANES> f = F::operand(raw);
#pragma unroll
        for (int p = 0; p < F::PLANES; ++p) lds[p * PLANE + at(row, piece)] = f.p[p];
    }
    // operand of 32 of the tile's rows (the lane's is `row`), 16 columns `chunk`
    static __device__ __forceinline__ Frag<F::PLANES> rows(const uint4 *lds, int row, int chunk, int half) {
        Frag<F::PLANES> f;
#pragma unroll
        for (int p = 0; p < F::PLANES; ++p) f.p[p] = lds[p * PLANE + at(row, 2 * chunk + half)];
        return f;
    }
    // operand of 32 of the tile's columns (32 db + lane % 32) with the sum over its rows base + 4 half + {0 .. 3, 8 .. 11}: the order in which a lane
    // has the elements 8 c .. 8 c + 7 of a result, base = 32 x (its block of rows) + 16 c
    static __device__ __forceinline__ Frag<F::PLANES> columns(const uint4 *lds, int base, int db, int lane) {
        const int row = base + 4 * (lane >> 5) + ((lane & 15) >> 2), piece = 4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), byte = 8 * (lane & 1);
        Frag<F::PLANES> f;
#pragma unroll
        for (int p = 0; p < F::PLANES; ++p) {
            const auto lo = transposed(lds + p * PLANE + at(row, piece), byte), hi = transposed(lds + p * PLANE + at(row + 8, piece), byte);
            f.p[p] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        return f;
    }

private:
    // Of 16 lanes' 8 bytes, lanes 4 i .. 4 i + 3 having 16 numbers of row i: lane j gets the four rows' number j.
    static __device__ __forceinline__ uint2 transposed(const uint4 *word, int byte) {
        typedef __attribute__((address_space(3))) ca_i16x4_t lds_t;
        lds_t *const p = (lds_t *)(__attribute__((address_space(3))) char *)(reinterpret_cast<const char *>(word) + byte);
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
    }
};

// Operand layout of a wavefront's own 32 rows straight from memory: 16 columns `chunk` of the lane's row (8 of them, by half), zeros beyond the row.
template <typename F>
__device__ __forceinline__ Frag<F::PLANES> own_rows(const char *row, bool live, int chunk, int half, int pieces) {
    const int piece = 2 * chunk + half;
    return F::operand(live && piece < pieces ? F::load(row + piece * 8 * F::BYTES) : F::zero());
}

// Queries of the heads that share a key head are rows of one matrix: row r is token r / group, head h' * group + r % group.
struct Rows {
    const char *base;                     // of the batch and the key head's first query head
    int64_t token, head;                  // strides in bytes
    int group;
    __device__ __forceinline__ const char *at(int r) const {
        const int t = group == 1 ? r : r / group;
        return base + t * token + (r - t * group) * head;
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

// Where row `row` (of the queries that share key head kh, or with group 1 of the keys) of a batch is in [B, len, heads, columns]: its number of heads' rows.
__device__ __forceinline__ int64_t heads_row(int64_t b, int64_t kh, int row, int64_t len, int key_heads, int group) {
    const int token = group == 1 ? row : row / group;
    return ((b * len + token) * key_heads + kh) * group + (row - token * group);
}

// Which unit of work a workgroup has: neighbours (tiles that read the same keys) on one XCD.
__device__ __forceinline__ int64_t unit_of(int64_t block, int64_t blocks) {
    const int64_t xcd = block & 7, per = blocks >> 3, rem = blocks & 7;
    return xcd * per + (xcd < rem ? xcd : rem) + (block >> 3);
}

}  // namespace cross_attention
