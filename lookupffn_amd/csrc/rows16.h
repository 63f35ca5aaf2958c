// Rows of numbers in fp32, bfloat16 or half, 16 bytes at a time.
#pragma once

#include "lffn_common.h"

// Where a lane's 16 bytes are numbers of a format: N of them, to fp32 and back (one rounding, to the nearest).
struct F32Row {
    static constexpr int N = 4, BYTES = 4;
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[N]) {
        v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};

template <typename E>
struct Row16 {
    static constexpr int N = 8, BYTES = 2;
    typedef E pair_t __attribute__((ext_vector_type(2)));
    typedef float float_pair_t __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const float_pair_t v = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pair_t));
    }
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[N]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const pair_t p = __builtin_bit_cast(pair_t, w[i]);
            v[2 * i] = (float)p[0], v[2 * i + 1] = (float)p[1];
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
        return make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
    }
};
typedef Row16<__bf16> BF16Row;
typedef Row16<_Float16> F16Row;
