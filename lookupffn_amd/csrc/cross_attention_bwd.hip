// The backward of the attention to an encoder's states (cross_attention.h: operands and tiles).
//
//   delta_i = g_i . o_i;  p_ij = 2^(c s_ij - lse_i);  ds_ij = p_ij (g_i . v_j - delta_i)
//   grad v_j = sum_i p_ij g_i;  grad k_j = scale sum_i ds_ij q_i;  grad q_i = scale sum_j ds_ij k_j
// Three kernels: delta; the queries' gradients, a workgroup's 128 rows standing and the keys and values passing; the keys' and values', 128 keys
// standing and the rows with their gradients passing.  Scores and g . v are formed twice (seven products for five; once where a key head has 128 rows at most, in one
// kernel for both), for that every sum has one owner and a fixed order: no atomics, the same bits on every call.  Where there are too few standing rows or keys to fill
// the chip what passes is shared out over several workgroups, and a last kernel adds their sums.
//
// Half precision, and fp32 numbers in two terms of it: p is held 2^14 times larger (at most 2^14), ds times a power of two that takes 2 |g| |v|, of the
// longest rows of the batch and key head, which no ds exceeds, below 2^15: gradients of any size, and weights of many keys, stay among half's normal numbers.
// 16 bits: weights and ds are operands of one term, a rounding each beside the gradients' own (1.4 to 1.5 times that alone; two terms each would be ten products for seven).
// fp32 numbers are scaled by the longest rows of q, k, v and g in the same way, and p and ds once more by what a key's, or a query's, largest so far leaves
// of half's range (fit).
//
// Bound by the products where there are many rows and keys: 4 x 2048 x 4096 x 16 x 128 bfloat16 keys' gradients 645 us (0.85 PFLOP/s), queries' 375 (1.1), delta 13.
#include <algorithm>

#include "cross_attention.h"

using namespace cross_attention;

__attribute__((visibility("hidden"))) int lffn_internal_cross_attention_check(const lffn_cross_attention *a);

namespace {

constexpr float P_LIFT = 14.f;            // half precision, one term or two

struct BwdArgs {
    const char *q, *k, *v, *out, *rest, *g;
    const uint8_t *mask;
    const float *lse;
    char *gq, *gk, *gv;
    float *delta;                         // [B, key heads, rows]
    float *g_levels, *q_levels, *v_levels, *k_levels;                // log2 of the longest rows, [B, key heads, g_tiles or v_tiles]
    int32_t *single;                      // [B], with a mask: whether one key alone takes part
    float *part;                          // [splits, B, key heads, rows or keys, columns] (keys: of k, then of v)
    int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, mask_stride;         // strides in bytes
    int64_t keys, steps, split_steps, q_len;
    Divisor group, tile_by, split_by, heads, level_tiles; // query heads of a key head, standing tiles, shares of what passes, key heads, delta_kernel's tiles
    int64_t units;
    int batch_heads, key_heads, rows, tiles, splits, columns, g_tiles, v_tiles;
    float c, scale;
};

// How many keys of a sequence take part, as far as two: a workgroup looks at 4096 flags at a time and seldom at more.
__device__ __forceinline__ void look_for_a_single_key(const BwdArgs &a, int b) {
    constexpr int EACH = 16;
    const uint8_t *const mask = a.mask + b * a.mask_stride;
    int found = 0;
    for (int64_t first = threadIdx.x; first - threadIdx.x < a.keys && found < 2; first += EACH * WG) {
        uint8_t flag[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) flag[i] = mask[first + i * WG < a.keys ? first + i * WG : a.keys - 1];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) mine += first + i * WG < a.keys && flag[i] != 0;
        found += __syncthreads_count(mine > 0);
        found += __syncthreads_or(mine > 1);
    }
    if (threadIdx.x == 0) a.single[b] = found == 1;
}
// What the queries' and keys' gradients are multiplied with.  A key that takes part alone has all the weight, and ds is nothing; g . v and delta, summed in different orders,
// would leave their roundings.
__device__ __forceinline__ float gradient_scale(const BwdArgs &a, int b) { return (a.mask ? a.single[b] != 0 : a.keys == 1) ? 0.f : a.scale; }

// delta of every row; half precision: the longest rows of g and v as well; fp32 numbers in two terms: of q and k, too.  A lane has 8 columns, the rows of a group of lanes are
// asked for together.  Bound by memory: out, its rest and g (and v, q, k) once.  (Rows one after the other, 1024 a workgroup: 4 x 2048 rows of 16 x 128 bfloat16
// 65 us, so 13.)
template <typename F, int LANES, bool LEVELS>
__global__ __launch_bounds__(WG) void delta_kernel(BwdArgs a) {
    constexpr int APART = WG / LANES, EACH = LEVEL_ROWS / APART;
    const int lane = threadIdx.x % LANES, tiles = a.g_tiles + a.v_tiles;
    const bool on = lane * 8 < a.columns;
    const int col = on ? lane * 8 : 0;
    if (blockIdx.x >= (uint32_t)a.batch_heads * tiles) return look_for_a_single_key(a, blockIdx.x - (uint32_t)a.batch_heads * tiles);
    const int bh = a.level_tiles.quotient(blockIdx.x), b = a.heads.quotient(bh), kh = bh - b * a.key_heads, tile = blockIdx.x - bh * tiles;
    float most[2] = {-INFINITY, -INFINITY};             // of g and q, or v and k
    auto look = [&](int n, const typename F::Raw &r, bool live) {
        float v[8];
        F::unpack(on ? r : F::zero(), v);
        const float l = row_level<LANES>(v);
        if (live) most[n] = fmaxf(most[n], l);
    };
    if (tile < a.g_tiles) {
        typename F::Raw o[EACH], g[EACH], rest[F::BYTES == 2 ? EACH : 1], q[F::SCALED ? EACH : 1];
        const int first = tile * LEVEL_ROWS + threadIdx.x / LANES;
        const Rows rows{a.q + b * a.qb + kh * a.group.by * a.qh, a.qt, a.qh, a.group};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int row = min(first + i * APART, a.rows - 1);
            const int64_t at = (heads_row(b, kh, row, a.q_len, a.key_heads, a.group) * a.columns + col) * F::BYTES;
            o[i] = F::load(a.out + at);
            g[i] = F::load(a.g + at);
            if constexpr (F::BYTES == 2) rest[i] = F::load(a.rest + at);
            if constexpr (F::SCALED) q[i] = F::load(rows.at(row) + col * F::BYTES);
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            float dot = 0.f, u[8], v[8];
            F::unpack(o[i], u);
            F::unpack(g[i], v);
            if constexpr (F::BYTES == 2) {
                float w[8];
                F::unpack(rest[i], w);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] += w[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(u[e], v[e], dot);
            dot = lane_group_sum<LANES>(on ? dot : 0.f);
            const int row = first + i * APART;
            if (lane == 0 && row < a.rows) a.delta[int64_t(bh) * a.rows + row] = dot;
            if (LEVELS) look(0, g[i], true);            // (a row once more changes nothing)
            if constexpr (F::SCALED) look(1, q[i], true);
        }
    } else if (LEVELS) {
        typename F::Raw v[EACH], k[F::SCALED ? EACH : 1];
        bool live[EACH];
        const int64_t first = int64_t(tile - a.g_tiles) * LEVEL_ROWS + threadIdx.x / LANES;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int64_t key = first + i * APART, at = key < a.keys ? key : a.keys - 1;
            live[i] = !a.mask || a.mask[b * a.mask_stride + at] != 0;
            v[i] = F::load(a.v + b * a.vb + kh * a.vh + at * a.vt + col * F::BYTES);
            if constexpr (F::SCALED) k[i] = F::load(a.k + b * a.kb + kh * a.kh + at * a.kt + col * F::BYTES);
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            look(0, v[i], live[i]);
            if constexpr (F::SCALED) look(1, k[i], live[i]);
        }
    }
    if (LEVELS) {
        __shared__ float red[2][WAVES];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            most[n] = over_groups_max<LANES>(most[n]);
            if ((threadIdx.x & 63) == 0) red[n][threadIdx.x >> 6] = most[n];
        }
        __syncthreads();
        if (threadIdx.x < (F::SCALED ? 2 : 1)) {
            const float *const r = red[threadIdx.x];
            const float all = fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
            if (tile < a.g_tiles) (threadIdx.x ? a.q_levels : a.g_levels)[int64_t(bh) * a.g_tiles + tile] = all;
            else (threadIdx.x ? a.k_levels : a.v_levels)[int64_t(bh) * a.v_tiles + tile - a.g_tiles] = all;
        }
    }
}

// The powers of two that everything is multiplied with, as exponents: ds, and of fp32 numbers in two terms q, k, v and g.
struct Exponents {
    int ds, q, k, v, g;
};
template <typename F>
__device__ __forceinline__ Exponents exponents(const BwdArgs &a, int64_t bh) {
    Exponents e{};
    if constexpr (F::LIFT != 0.f) {
        const float g = longest(a.g_levels, bh, a.g_tiles), v = longest(a.v_levels, bh, a.v_tiles);
        if (g != -INFINITY && v != -INFINITY) e.ds = 14 - (int)ceilf(1.f + g + v);
        if constexpr (F::SCALED) {
            e.q = exponent_for(longest(a.q_levels, bh, a.g_tiles)), e.k = exponent_for(longest(a.k_levels, bh, a.v_tiles));
            e.v = exponent_for(v), e.g = exponent_for(g);
        }
    }
    return e;
}
__device__ __forceinline__ float power(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }

template <typename F, int DP, int KT>
__global__ __launch_bounds__(WG, F::PLANES == 1 && DP <= 64 ? 3 : F::PLANES == 1 || DP <= 64 ? 2 : 1) void query_gradient_kernel(BwdArgs a) {
    typedef Tile<F, DP, KT> T;
    typedef Frag<F::PLANES> Op;
    constexpr int CHUNKS = DP / 16, KB = KT / 32, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // [2][keys, values], words
    uint64_t *const words = reinterpret_cast<uint64_t *>(lds + 4 * T::SIZE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, half = lane >> 5;
    const Unit unit = unit_of(blockIdx.x, a.units, a.tile_by, a.split_by, a.heads);
    const int tile = unit.tile, split = unit.split, bh = unit.bh, b = unit.b, kh = unit.kh;
    const int pieces = a.columns / 8;
    const char *const kp = a.k + b * a.kb + kh * a.kh, *const vp = a.v + b * a.vb + kh * a.vh;
    const uint8_t *const mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int row = tile * TILE + wave * ROWS + r;
    const bool live = row < a.rows;

    KeyFeed<F, DP, KT> feed(lds, pieces, kp, vp, a.kt, a.vt);
    const typename T::Reader read(lds, lane);
    const int64_t out_row = heads_row(b, kh, live ? row : 0, a.q_len, a.key_heads, a.group) * a.columns * F::BYTES;
    const Exponents e2 = exponents<F>(a, bh);
    if constexpr (F::SCALED) feed.scale_a = power(e2.k), feed.scale_b = power(e2.v);
    Op fq[CHUNKS], fg[CHUNKS];
    const int eq = own_rows<F>(Rows{a.q + b * a.qb + kh * a.group.by * a.qh, a.qt, a.qh, a.group}.at(live ? row : 0), live, half, pieces, fq);
    const int eg = own_rows<F>(a.g + out_row, live, half, pieces, fg);
    const float f = power(e2.ds - eg - e2.v), by_c = __builtin_amdgcn_ldexpf(a.c, -(eq + e2.k));
    const float level = live ? a.lse[int64_t(bh) * a.rows + row] : INFINITY;
    const float delta = live ? __builtin_amdgcn_ldexpf(a.delta[int64_t(bh) * a.rows + row], e2.ds) : 0.f;
    ca_f32x16_t dq[DB] = {};
    int fitted = F::SCALED ? FIT_FIRST : 0;

    const bool wave_works = tile * TILE + wave * ROWS < a.rows;
    auto compute = [&](auto buf, uint64_t word, int64_t) {
        if (!wave_works) return;
        constexpr int KEYS = decltype(buf)::value * 2 * T::SIZE, VALUES = KEYS + T::SIZE;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            ca_f32x16_t s = {}, dp = {};
            products<F, 2 * CHUNKS>([&](auto i) { return read.rows(i % 2 ? VALUES : KEYS, kb, i / 2); }, [&](auto i, const Op &x) {
                if constexpr (i % 2) dp = F::mma(x, fg[i / 2], dp);
                else s = F::mma(x, fq[i / 2], s);
            });
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], by_c, -level)) * fmaf(dp[e], f, -delta);
            const uint32_t part = (uint32_t)(word >> (32 * kb));
            if (part != ~0u) {
                const uint32_t w = part >> (4 * half);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(w >> (8 * (e / 4) + e % 4) & 1)) s[e] = 0.f;
            }
            if constexpr (F::SCALED) fit(s, fitted, dq);
            Op ds[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = s[8 * c + e];
                ds[c] = F::operand(t);
            }
            products<F, 2 * DB>([&](auto i) { return read.columns(KEYS, 2 * kb + i / DB, i % DB); },
                                [&](auto i, const Op &x) { dq[i % DB] = F::mma(x, ds[i / DB], dq[i % DB]); });
        }
    };

    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;
    walk_keys<KT>(feed, words, mask, begin, end, a.keys, compute);
    const auto by = factor<F>(gradient_scale(a, b), -(e2.ds + e2.k + fitted));
    if (a.splits > 1) store_row<F32, DB>(dq, by, reinterpret_cast<char *>(a.part + ((int64_t(split) * a.batch_heads + bh) * a.rows + row) * a.columns), live, a.columns, half);
    else store_row<F, DB>(dq, by, a.gq + out_row, live, a.columns, half);
}

// All three gradients where the rows of a key head are 128 at most: they and their gradients stay in LDS, the keys pass 32 at a time, and of a step's keys
// every sum over the rows is there at once, so that scores and g . v are formed once (five products for seven) and keys and values read once.  A wavefront has 32
// rows: it forms their weights and ds with the step's keys, adds to their queries' gradients, and leaves both in LDS, turned round; then of the four tiles
// of 32 columns x 32 keys, two of values' and two of keys' gradients, each wavefront forms one.  What it formed is stored in the next step, so that no step waits for a store.
template <typename F>
__global__ __launch_bounds__(WG, 2) void gradients_kernel(BwdArgs a) {
    constexpr int DP = 64, KT = 32, CHUNKS = DP / 16, DB = DP / 32, OWN = TILE / 16;
    typedef Tile<F, DP, TILE> Own;
    typedef Tile<F, DP, KT> T;
    typedef Tile<F, KT, TILE> Turned;
    typedef Frag<1> Op;
    static_assert(F::PLANES == 1 && DB * 2 == WAVES, "a tile of the results a wavefront");
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // rows, their gradients, [2][keys, values], weights, ds, words
    constexpr int GRADIENTS_AT = Own::SIZE, PASSING = 2 * Own::SIZE, WEIGHTS = PASSING + 4 * T::SIZE, WORDS = WEIGHTS + 2 * Turned::SIZE;
    uint64_t *const words = reinterpret_cast<uint64_t *>(lds + WORDS);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, half = lane >> 5;
    const Unit unit = unit_of(blockIdx.x, a.units, a.tile_by, a.split_by, a.heads);
    const int split = unit.split, bh = unit.bh, b = unit.b, kh = unit.kh;
    const int pieces = a.columns / 8;
    const char *const kp = a.k + b * a.kb + kh * a.kh, *const vp = a.v + b * a.vb + kh * a.vh;
    const uint8_t *const mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;
    const int row = wave * ROWS + r;
    const bool live = row < a.rows, wave_works = wave * ROWS < a.rows;

    {
        const Rows rows{a.q + b * a.qb + kh * a.group.by * a.qh, a.qt, a.qh, a.group};
        const char *const gp = a.g + (b * a.q_len * a.key_heads + kh) * int64_t(a.group.by) * a.columns * F::BYTES;
        Feed<F, DP, TILE> own(lds, pieces);
        // (rows beyond the last are the last once more: their levels are infinite and so their weights zero)
        own.begin(0, rows.base, gp, [&](int at, int) { const int i = min(at, a.rows - 1), t = a.group.quotient(i); return t * (uint32_t)a.qt + (i - t * a.group.by) * (uint32_t)a.qh; },
                  [&](int at, int) {
                      const int i = min(at, a.rows - 1), t = a.group.quotient(i);
                      return (t * a.key_heads * a.group.by + (i - t * a.group.by)) * (uint32_t)(a.columns * F::BYTES);
                  });
        own.end(0);
    }
    // zeros for keys that take no part, and for the weights and ds of wavefronts without rows
    auto result = [&](int64_t key) { return ((b * a.keys + key) * a.key_heads + kh) * int64_t(a.columns * F::BYTES); };
    const uint4 zeros = make_uint4(0, 0, 0, 0);
    if (mask) {
        constexpr int EACH = 8, APART = WG / 8;
        const int64_t last = end * KT < a.keys ? end * KT : a.keys;
        const int piece = tid & 7;
        for (int64_t first = begin * KT + tid / 8; first < last; first += EACH * APART) {
            uint8_t flag[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) flag[i] = mask[first + i * APART < last ? first + i * APART : last - 1];
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int64_t key = first + i * APART;
                if (key < last && !flag[i] && piece < pieces) {
                    *reinterpret_cast<uint4 *>(a.gk + result(key) + piece * 16) = zeros;
                    *reinterpret_cast<uint4 *>(a.gv + result(key) + piece * 16) = zeros;
                }
            }
        }
    }
    if (!wave_works) {
#pragma unroll
        for (int i = 0; i < 2; ++i) lds[WEIGHTS + wave * 128 + i * 64 + lane] = zeros, lds[WEIGHTS + Turned::SIZE + wave * 128 + i * 64 + lane] = zeros;
    }
    __syncthreads();

    constexpr bool HALF = F::LIFT != 0.f;
    const Exponents e2 = exponents<F>(a, bh);
    const int of_delta = HALF ? e2.ds - int(P_LIFT) : 0;
    const float f = power(of_delta);
    const float level = live ? a.lse[int64_t(bh) * a.rows + row] - (HALF ? P_LIFT : 0.f) : INFINITY;
    const float delta = live ? __builtin_amdgcn_ldexpf(a.delta[int64_t(bh) * a.rows + row], of_delta) : 0.f;
    KeyFeed<F, DP, KT> feed(lds + PASSING, pieces, kp, vp, a.kt, a.vt);
    const typename T::Reader read(lds + PASSING, lane);
    const typename Own::Reader read_own(lds, lane);
    Op fq[CHUNKS], fg[CHUNKS];
    static_for<CHUNKS>([&](auto c) {      // (zeros beyond the columns, for what keys and values have there)
        const bool on = 2 * c + half < pieces;
        const Op q = read_own.rows(0, wave, c), g = read_own.rows(GRADIENTS_AT, wave, c);
        fq[c] = {{on ? q.p[0] : zeros}}, fg[c] = {{on ? g.p[0] : zeros}};
    });
    ca_f32x16_t dq[DB] = {}, sum[1] = {};

    // the wavefront's tile of the results
    const int d = wave & 1;
    const bool of_v = wave < 2;
    const typename Turned::Reader read_turned(lds + WEIGHTS + (of_v ? 0 : Turned::SIZE), lane);
    typename Own::Reader read_mine(lds + (of_v ? GRADIENTS_AT : 0), lane);
    read_mine.lo[0] = d ? read_mine.lo[1] : read_mine.lo[0], read_mine.hi[0] = d ? read_mine.hi[1] : read_mine.hi[0];
    const float by_q = __builtin_amdgcn_ldexpf(gradient_scale(a, b), -e2.ds), by = of_v ? (HALF ? power(-int(P_LIFT)) : 1.f) : by_q;
    char *const to = (of_v ? a.gv : a.gk) + d * 32 * F::BYTES;
    int64_t formed = -1;                  // the step that `sum` is of
    uint32_t formed_word = 0;
    auto store = [&]() {
        if (formed < 0) return;
        const bool in = formed_word >> r & 1;
        store_row<F, 1>(sum, by, to + result(formed * KT + (in ? r : 0)), in, a.columns - 32 * d, half);
    };
    auto compute = [&](auto buf, uint64_t word, int64_t step) {
        constexpr int KEYS = decltype(buf)::value * 2 * T::SIZE, VALUES = KEYS + T::SIZE;
        store();
        if (wave_works) {
            ca_f32x16_t s = {}, dp = {};
            products<F, 2 * CHUNKS>([&](auto i) { return read.rows(i % 2 ? VALUES : KEYS, 0, i / 2); }, [&](auto i, const Op &x) {
                if constexpr (i % 2) dp = F::mma(x, fg[i / 2], dp);
                else s = F::mma(x, fq[i / 2], s);
            });
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -level));
                dp[e] = s[e] * fmaf(dp[e], f, -delta);
            }
            if ((uint32_t)word != ~0u) {
                const uint32_t w = (uint32_t)word >> (4 * half);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(w >> (8 * (e / 4) + e % 4) & 1)) s[e] = 0.f, dp[e] = 0.f;
            }
            Op p[2], ds[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float t[8], u[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = s[8 * c + e], u[e] = dp[8 * c + e];
                p[c] = F::operand(t), ds[c] = F::operand(u);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint2 *const at = reinterpret_cast<uint2 *>(lds + WEIGHTS + Turned::at(row, 2 * c + i)) + half;
                    at[0] = i ? make_uint2(p[c].p[0].z, p[c].p[0].w) : make_uint2(p[c].p[0].x, p[c].p[0].y);
                    at[2 * Turned::SIZE] = i ? make_uint2(ds[c].p[0].z, ds[c].p[0].w) : make_uint2(ds[c].p[0].x, ds[c].p[0].y);
                }
            }
            products<F, 2 * DB>([&](auto i) { return read.columns(KEYS, i / DB, i % DB); },
                                [&](auto i, const Op &x) { dq[i % DB] = F::mma(x, ds[i / DB], dq[i % DB]); });
        }
        lds_barrier();                    // (copies on their way stay so)
        sum[0] = ca_f32x16_t{};
        Op x[OWN], y[OWN];
        static_for<OWN>([&](auto c) { x[c] = read_mine.columns(0, c, 0), y[c] = read_turned.columns(0, c, 0); });
        static_for<OWN>([&](auto c) { sum[0] = F::mma(x[c], y[c], sum[0]); });
        formed = step, formed_word = (uint32_t)word;
    };

    walk_keys<KT>(feed, words, mask, begin, end, a.keys, compute);
    store();
    if (a.splits > 1) store_row<F32, DB>(dq, by_q, reinterpret_cast<char *>(a.part + ((int64_t(split) * a.batch_heads + bh) * a.rows + row) * a.columns), live, a.columns, half);
    else store_row<F, DB>(dq, by_q, a.gq + heads_row(b, kh, live ? row : 0, a.q_len, a.key_heads, a.group) * a.columns * F::BYTES, live, a.columns, half);
}

template <typename F, int DP, int KT>
__global__ __launch_bounds__(WG, DP <= 64 ? 2 : 1) void key_gradient_kernel(BwdArgs a) {
    typedef Tile<F, DP, KT> T;
    typedef Frag<F::PLANES> Op;
    constexpr int CHUNKS = DP / 16, RB = KT / 32, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // [2][rows, their gradients], [2][levels, deltas]
    float *const levels = reinterpret_cast<float *>(lds + 4 * T::SIZE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, half = lane >> 5;
    const Unit unit = unit_of(blockIdx.x, a.units, a.tile_by, a.split_by, a.heads);
    const int tile = unit.tile, split = unit.split, bh = unit.bh, b = unit.b, kh = unit.kh;
    const int pieces = a.columns / 8;
    const int64_t key = int64_t(tile) * TILE + wave * ROWS + r;
    const bool in = key < a.keys;
    const int64_t at_key = in ? key : a.keys - 1;
    const Rows rows{a.q + b * a.qb + kh * a.group.by * a.qh, a.qt, a.qh, a.group};
    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;

    // (a masked key is read as any other: what it holds stays in its own column, which is not stored)
    const uint8_t flag = a.mask ? a.mask[b * a.mask_stride + at_key] : 1;
    constexpr bool HALF = F::LIFT != 0.f;
    const Exponents e2 = exponents<F>(a, bh);
    const int of_delta = HALF ? e2.ds - int(P_LIFT) : 0;
    Op fk[CHUNKS], fv[CHUNKS];
    const int ek = own_rows<F>(a.k + b * a.kb + kh * a.kh + at_key * a.kt, true, half, pieces, fk);
    const int ev = own_rows<F>(a.v + b * a.vb + kh * a.vh + at_key * a.vt, true, half, pieces, fv);
    const float f = power(of_delta - e2.g - ev), by_c = __builtin_amdgcn_ldexpf(a.c, -(e2.q + ek));

    // Rows beyond the last are the last once more: their levels are infinite and so their weights zero.  A step's addresses go by its first token; where
    // the heads that share a key divide KT they are the same for every step.
    Feed<F, DP, KT> feed(lds, pieces);
    if constexpr (F::SCALED) feed.scale_a = power(e2.q), feed.scale_b = power(e2.g);
    const typename T::Reader read(lds, lane);
    const bool even = KT % a.group.by == 0;
    const int64_t g_token = int64_t(a.key_heads) * a.group.by * a.columns * F::BYTES;
    const char *const gp = a.g + (b * a.q_len * g_token + kh * a.group.by * a.columns * F::BYTES);
    uint32_t q_offset[T::SHARE], g_offset[T::SHARE];
    float level = 0.f, delta = 0.f;
    auto ask = [&](int buf, int64_t step) {
        const int first = int(step) * KT, token = a.group.quotient(first);
        if (step == begin || !even || first + KT > a.rows) {
#pragma unroll
            for (int i = 0; i < T::SHARE; ++i) {
                const int row = min(first + feed.row + i * feed.ROWS_APART, a.rows - 1), t = a.group.quotient(row), h = row - t * a.group.by;
                q_offset[i] = (t - token) * (uint32_t)a.qt + h * (uint32_t)a.qh;
                g_offset[i] = (t - token) * (uint32_t)g_token + h * (uint32_t)(a.columns * F::BYTES);
            }
        }
        feed.begin(buf, rows.base + token * a.qt, gp + token * g_token, [&](int, int i) { return q_offset[i]; }, [&](int, int i) { return g_offset[i]; });
        // (nothing is made of the numbers here: that would wait for them, and for the copies)
        const int64_t of_row = int64_t(bh) * a.rows + min(first + tid % KT, a.rows - 1);
        level = a.lse[of_row];
        delta = a.delta[of_row];
    };
    auto placed = [&](int buf, int64_t step) {
        if (tid < KT) {
            const bool on = int(step) * KT + tid < a.rows;
            levels[buf * 2 * KT + tid] = on ? level - (HALF ? P_LIFT : 0.f) : INFINITY;
            levels[buf * 2 * KT + KT + tid] = on ? __builtin_amdgcn_ldexpf(delta, of_delta) : 0.f;
        }
        feed.end(buf);
    };

    ca_f32x16_t dk[DB] = {}, dv[DB] = {};
    int fitted_p = F::SCALED ? FIT_FIRST : 0, fitted_ds = fitted_p;
    auto compute = [&](auto buf) {
        constexpr int QUERIES = decltype(buf)::value * 2 * T::SIZE, GRADIENTS = QUERIES + T::SIZE;
        const float *const level = levels + decltype(buf)::value * 2 * KT + 4 * half, *const delta = level + KT;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            ca_f32x16_t s = {}, dp = {};
            products<F, 2 * CHUNKS>([&](auto i) { return read.rows(i % 2 ? GRADIENTS : QUERIES, rb, i / 2); }, [&](auto i, const Op &x) {
                if constexpr (i % 2) dp = F::mma(x, fv[i / 2], dp);
                else s = F::mma(x, fk[i / 2], s);
            });
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 l = *reinterpret_cast<const float4 *>(level + rb * 32 + 8 * g), d = *reinterpret_cast<const float4 *>(delta + rb * 32 + 8 * g);
                const float ls[4] = {l.x, l.y, l.z, l.w}, ds[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], by_c, -ls[e]));
                    s[4 * g + e] = p;
                    dp[4 * g + e] = p * fmaf(dp[4 * g + e], f, -ds[e]);
                }
            }
            if constexpr (F::SCALED) fit(s, fitted_p, dv), fit(dp, fitted_ds, dk);
            Op p[2], ds[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float t[8], u[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = s[8 * c + e], u[e] = dp[8 * c + e];
                p[c] = F::operand(t), ds[c] = F::operand(u);
            }
            products<F, 4 * DB>([&](auto i) { return read.columns(i % 2 ? QUERIES : GRADIENTS, 2 * rb + i / 2 / DB, i / 2 % DB); }, [&](auto i, const Op &x) {
                if constexpr (i % 2) dk[i / 2 % DB] = F::mma(x, ds[i / 2 / DB], dk[i / 2 % DB]);
                else dv[i / 2 % DB] = F::mma(x, p[i / 2 / DB], dv[i / 2 % DB]);
            });
        }
    };

    if (begin < end) ask(0, begin);
    const bool live = in && flag != 0, wave_works = __any(live), works = __syncthreads_or(live);
    if (begin < end) placed(0, begin);
    if (works && begin < end) {
        __syncthreads();
#pragma unroll 1
        for (int64_t step = begin;;) {
            bool more = ++step < end;
            if (more) ask(1, step);
            if (wave_works) compute(std::integral_constant<int, 0>{});
            if (!more) break;
            placed(1, step);
            __syncthreads();
            more = ++step < end;
            if (more) ask(0, step);
            if (wave_works) compute(std::integral_constant<int, 1>{});
            if (!more) break;
            placed(0, step);
            __syncthreads();
        }
    }
    if (!live) {
#pragma unroll
        for (int d = 0; d < DB; ++d) dk[d] = ca_f32x16_t{}, dv[d] = ca_f32x16_t{};
    }
    const auto by_k = factor<F>(gradient_scale(a, b), -(e2.ds + e2.q + fitted_ds)), by_v = factor<F>(1.f, (HALF ? -int(P_LIFT) : 0) - e2.g - fitted_p);
    if (a.splits > 1) {
        const int64_t all = int64_t(a.batch_heads) * a.keys, of = (split * all + bh * a.keys + key) * a.columns;
        store_row<F32, DB>(dk, by_k, reinterpret_cast<char *>(a.part + of), in, a.columns, half);
        store_row<F32, DB>(dv, by_v, reinterpret_cast<char *>(a.part + a.splits * all * a.columns + of), in, a.columns, half);
    } else {
        const int64_t at = ((b * a.keys + key) * a.key_heads + kh) * a.columns * F::BYTES;
        store_row<F, DB>(dk, by_k, a.gk + at, in, a.columns, half);
        store_row<F, DB>(dv, by_v, a.gv + at, in, a.columns, half);
    }
}

// The same with two wavefronts a block of 32 keys: one forms the weights and the values' gradient, the other ds and the keys' gradient, and the weights go from one
// to the other through LDS, in fp32.  Each has half of the operands and sums (128 columns: 96 registers for 192), so that two fit on a SIMD, the one's
// exponentials beside the other's products; with all in one wavefront a SIMD has one, which waits for itself (4 x 2048 to 4096 x 16 x 128 bfloat16: 758 us).
// Between two barriers: the weights' products with a step of 32 rows and the scores of the next one, whose rows are there, while those of the one after
// are on their way (three buffers).
template <typename F, int DP, int ROLE>
__device__ __forceinline__ void key_gradient_pairs(const BwdArgs &a, uint4 *const lds) {
    constexpr bool OF_V = ROLE == 0;
    constexpr int KT = 32, THREADS = 2 * WG, BUFFERS = 3, CHUNKS = DP / 16, DB = DP / 32;
    typedef Tile<F, DP, KT> T;
    typedef Frag<F::PLANES> Op;
    constexpr int SHARE = 2 * T::PLANE / THREADS;        // of the pieces of a step's rows and their gradients
    static_assert(SHARE >= 1 && T::PLANE % 64 == 0, "a wavefront's pieces are of one tile");
    float4 *const handed = reinterpret_cast<float4 *>(lds + BUFFERS * 2 * T::SIZE);
    float *const levels = reinterpret_cast<float *>(handed + BUFFERS * WAVES * 256);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), pair = wave & 3;
    const int r = lane & 31, half = lane >> 5;
    const Unit unit = unit_of(blockIdx.x, a.units, a.tile_by, a.split_by, a.heads);
    const int tile = unit.tile, split = unit.split, bh = unit.bh, b = unit.b, kh = unit.kh;
    const int pieces = a.columns / 8;
    const int64_t key = int64_t(tile) * TILE + pair * ROWS + r;
    const bool in = key < a.keys;
    const int64_t at_key = in ? key : a.keys - 1;
    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;
    // whether the tile's keys take part: every wavefront looks at all 128
    uint64_t flags[2] = {~0ull, ~0ull};
    if (a.mask) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t k = int64_t(tile) * TILE + 64 * i + lane;
            flags[i] = __ballot(a.mask[b * a.mask_stride + (k < a.keys ? k : a.keys - 1)] != 0 && k < a.keys);
        }
    }
    constexpr bool HALF = F::LIFT != 0.f;
    const Exponents e2 = exponents<F>(a, bh);
    const int of_delta = HALF ? e2.ds - int(P_LIFT) : 0;
    Op own[CHUNKS];                       // the weights' wavefront: keys; the other: values
    const int of_own = own_rows<F>(OF_V ? a.k + b * a.kb + kh * a.kh + at_key * a.kt : a.v + b * a.vb + kh * a.vh + at_key * a.vt, true, half, pieces, own);
    const float f = power(of_delta - e2.g - of_own), by_c = __builtin_amdgcn_ldexpf(a.c, -(e2.q + of_own));

    const Rows rows{a.q + b * a.qb + kh * a.group.by * a.qh, a.qt, a.qh, a.group};
    const int64_t g_token = int64_t(a.key_heads) * a.group.by * a.columns * F::BYTES;
    const char *const gp = a.g + (b * a.q_len * g_token + kh * a.group.by * a.columns * F::BYTES);
    typename F::Raw raw[F::PLANES == 1 ? 1 : SHARE];
    float level = 0.f, delta = 0.f;
    // piece i of the thread: of tile (0: rows, 1: gradients), row and place in memory
    auto piece_of = [&](int i, int &of, int &row, int &place) {
        const int p = tid + THREADS * i, q = p % T::PLANE;
        of = p / T::PLANE, row = q / T::PIECES, place = q % T::PIECES;
        if constexpr (F::PLANES == 1) place ^= T::turned(row);
    };
    auto ask = [&](int buf, int64_t step) {
        const int first = int(step) * KT, token = a.group.quotient(first);
        const char *const q_base = rows.base + token * a.qt, *const g_base = gp + token * g_token;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
            int of, at, place;
            piece_of(i, of, at, place);
            const int row = min(first + at, a.rows - 1), t = a.group.quotient(row), h = row - t * a.group.by;
            const uint32_t column = (place < pieces ? place : 0) * 8 * F::BYTES;
            const uint32_t offset = (t - token) * (of ? (uint32_t)g_token : (uint32_t)a.qt) + h * (of ? (uint32_t)(a.columns * F::BYTES) : (uint32_t)a.qh) + column;
            const bool of_g = __builtin_amdgcn_readfirstlane(of);
            const char *const base = of_g ? g_base : q_base;
            if constexpr (F::PLANES == 1) {
                const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + (buf * 2 * T::SIZE + i * THREADS + wave * 64) * 16;
                copy_to_lds(base, offset, __builtin_amdgcn_readfirstlane(to));
            } else {
                raw[i] = F::load(base + offset);
            }
        }
        const int64_t of_row = int64_t(bh) * a.rows + min(first + tid % KT, a.rows - 1);
        level = a.lse[of_row];
        delta = a.delta[of_row];
    };
    auto placed = [&](int buf, int64_t step) {
        if (tid < KT) {
            const bool on = int(step) * KT + tid < a.rows;
            levels[buf * 2 * KT + tid] = on ? level - (HALF ? P_LIFT : 0.f) : INFINITY;
            levels[buf * 2 * KT + KT + tid] = on ? __builtin_amdgcn_ldexpf(delta, of_delta) : 0.f;
        }
        if constexpr (F::PLANES == 1) {
            arrived();
        } else {
#pragma unroll
            for (int i = 0; i < SHARE; ++i) {
                int of, at, place;
                piece_of(i, of, at, place);
                T::put(lds + (buf * 2 + of) * T::SIZE, at, place, raw[i], power(of ? e2.g : e2.q));
            }
        }
    };

    const typename T::Reader read(lds, lane);
    ca_f32x16_t sums[DB] = {}, s;
    int fitted = F::SCALED ? FIT_FIRST : 0;
    Op p[2];
    // scores and weights, or g . v, of a step
    auto first_half = [&](auto buf) {
        constexpr int QUERIES = decltype(buf)::value * 2 * T::SIZE, GRADIENTS = QUERIES + T::SIZE;
        s = ca_f32x16_t{};
        if constexpr (OF_V) {
            products<F, CHUNKS>([&](auto i) { return read.rows(QUERIES, 0, i); }, [&](auto i, const Op &x) { s = F::mma(x, own[i], s); });
            float4 *const to = handed + (decltype(buf)::value * WAVES + pair) * 256 + lane;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 l = *reinterpret_cast<const float4 *>(levels + decltype(buf)::value * 2 * KT + 8 * g + 4 * half);
                const float ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], by_c, -ls[e]));
                to[g * 64] = make_float4(s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]);
            }
        } else {
            products<F, CHUNKS>([&](auto i) { return read.rows(GRADIENTS, 0, i); }, [&](auto i, const Op &x) { s = F::mma(x, own[i], s); });
        }
    };
    // the products with them
    auto second_half = [&](auto buf) {
        constexpr int QUERIES = decltype(buf)::value * 2 * T::SIZE, GRADIENTS = QUERIES + T::SIZE;
        if constexpr (!OF_V) {
            const float4 *const from = handed + (decltype(buf)::value * WAVES + pair) * 256 + lane;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 w = from[g * 64], d = *reinterpret_cast<const float4 *>(levels + decltype(buf)::value * 2 * KT + KT + 8 * g + 4 * half);
                const float ws[4] = {w.x, w.y, w.z, w.w}, ds[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g + e] = ws[e] * fmaf(s[4 * g + e], f, -ds[e]);
            }
        }
        if constexpr (F::SCALED) fit(s, fitted, sums);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = s[8 * c + e];
            p[c] = F::operand(t);
        }
        if constexpr (OF_V) {
            products<F, 2 * DB>([&](auto i) { return read.columns(GRADIENTS, i / DB, i % DB); },
                                [&](auto i, const Op &x) { sums[i % DB] = F::mma(x, p[i / DB], sums[i % DB]); });
        } else {
            products<F, 2 * DB>([&](auto i) { return read.columns(QUERIES, i / DB, i % DB); },
                                [&](auto i, const Op &x) { sums[i % DB] = F::mma(x, p[i / DB], sums[i % DB]); });
        }
    };

    if (begin < end) ask(0, begin);
    const bool live = in && (flags[pair >> 1] >> (32 * (pair & 1) + r) & 1), wave_works = __any(live), works = (flags[0] | flags[1]) != 0;
    if (begin < end) placed(0, begin);
    if (works && begin < end) {
        __syncthreads();
        if (begin + 1 < end) ask(1, begin + 1);
        if (wave_works) first_half(std::integral_constant<int, 0>{});
        int64_t step = begin;
        // a step whose scores are there: in buffer `now`, the next step's rows on their way to `next`
        auto body = [&](auto now, auto next, auto behind) {
            const bool more = step + 1 < end;
            if (more) placed(decltype(next)::value, step + 1);
            __syncthreads();
            if (step + 2 < end) ask(decltype(behind)::value, step + 2);
            if (wave_works) {
                second_half(now);
                if (more) first_half(next);
            }
            ++step;
            return more;
        };
        const std::integral_constant<int, 0> zero;
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
#pragma unroll 1
        while (body(zero, one, two) && body(one, two, zero) && body(two, zero, one)) {
        }
    }
    if (!live) {
#pragma unroll
        for (int d = 0; d < DB; ++d) sums[d] = ca_f32x16_t{};
    }
    const auto by = OF_V ? factor<F>(1.f, (HALF ? -int(P_LIFT) : 0) - e2.g - fitted) : factor<F>(gradient_scale(a, b), -(e2.ds + e2.q + fitted));
    if (a.splits > 1) {
        const int64_t all = int64_t(a.batch_heads) * a.keys, of = (split * all + bh * a.keys + key + (OF_V ? a.splits * all : 0)) * a.columns;
        store_row<F32, DB>(sums, by, reinterpret_cast<char *>(a.part + of), in, a.columns, half);
    } else {
        store_row<F, DB>(sums, by, (OF_V ? a.gv : a.gk) + ((b * a.keys + key) * a.key_heads + kh) * a.columns * F::BYTES, in, a.columns, half);
    }
}

template <typename F, int DP>
__global__ __launch_bounds__(2 * WG, 2) void key_gradient_pairs_kernel(BwdArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // [3][rows, their gradients], [3][4] weights, [3][levels, deltas]
    // (whole wavefronts go either way, and either way has the same barriers in the same order)
    if (__builtin_amdgcn_readfirstlane(threadIdx.x) < WG) key_gradient_pairs<F, DP, 0>(a, lds);
    else key_gradient_pairs<F, DP, 1>(a, lds);
}

// The splits' sums of a row as one, in a fixed order, four of them asked for together; `second` beside `part` where there are two arrays.  Four columns a lane; of
// more splits than four each wavefront of a workgroup adds a share (1 x 128 rows, 128 splits of 4096 keys x 4 x 64 bfloat16: 12.7 us in one share,
// 4.8 in four).
struct AddArgs {
    const float *part[2];
    char *out[2];
    int64_t all, len;                     // rows: [batch, heads of keys] x rows
    Divisor heads, group;
    int rows, splits, columns;
};
template <typename F, int SHARES>
__global__ __launch_bounds__(WG) void add_splits_kernel(AddArgs a) {
    constexpr int TOGETHER = 4;
    const int quads = a.columns / 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = SHARES == 1 ? int64_t(blockIdx.x) * WG + threadIdx.x : int64_t(blockIdx.x) * 64 + lane, last = a.all * quads - 1, at = (i < last ? i : last) / quads;
    const int col = int((i < last ? i : last) - at * quads) * 4;
    const float *const part = a.part[blockIdx.y] + at * a.columns + col;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int first = SHARES == 1 ? 0 : wave; first < a.splits; first += SHARES * TOGETHER) {
        float4 v[TOGETHER];
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n) v[n] = *reinterpret_cast<const float4 *>(part + min(first + n * SHARES, a.splits - 1) * a.all * a.columns);
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n)
            if (first + n * SHARES < a.splits) acc.x += v[n].x, acc.y += v[n].y, acc.z += v[n].z, acc.w += v[n].w;
    }
    if constexpr (SHARES > 1) {
        __shared__ float4 sums[SHARES][64];
        sums[wave][lane] = acc;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int n = 1; n < SHARES; ++n) {
            const float4 v = sums[n][lane];
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
    }
    if (i > last) return;
    const int bh = int(at / a.rows), b = a.heads.quotient(bh), kh = bh - b * a.heads.by;
    F::store4(a.out[blockIdx.y] + (heads_row(b, kh, int(at - int64_t(bh) * a.rows), a.len, a.heads.by, a.group) * a.columns + col) * F::BYTES, acc.x, acc.y, acc.z,
              acc.w);
}

// Which form of the keys' gradients heads of so many columns get.
constexpr bool in_pairs(int planes, int columns) { return columns > (planes == 1 ? 64 : 32); }

constexpr int64_t COMPUTE_UNITS = 256;    // standing tiles, and more: what passes is not shared out
constexpr int64_t WANTED = 512;           // workgroups at most, where there is enough to share out (a forward and backward of 3 x 500 x 1500 x 10 x 128 bfloat16 120 us, with up to
                                          // a tile's shares more 141)
constexpr int64_t LEAST_STEPS = 2;        // of a workgroup

// All gradients in one kernel: where a key head's rows fit in LDS beside what passes.  us of a forward and backward, the gradients in two kernels and in one, batch x
// rows x keys x key heads x columns: 64 x 128 x 512 x 8 x 64 half 116, 92 (the kernels alone 46 + 27, 45; at least 31 for its bytes); 64 x 32 91, 72; 64 x 1 71, 54;
// 16 x 128 x 512 x 12 x 64 bfloat16 67, 59; 256 x 128 x 128 x 8 x 64 163, 143; 4 x 128 x 4096 x 8 x 64 67, 53; 1 x 128 x 4096 x 4 x 64 38, 34.
constexpr bool in_one(int format, int64_t columns, int64_t rows) { return format != LFFN_ROWS_F32 && columns > 32 && columns <= 64 && rows <= TILE; }

// The large launches, two or one, and where the workspace's parts begin (in floats).
struct Plan {
    BwdArgs q{}, k{}, both{};
    bool fits = true;                     // every launch
    int64_t delta = 0, g_levels = 0, q_levels = 0, v_levels = 0, k_levels = 0, single = 0, part = 0, floats = 0;
};

void share_out(BwdArgs &a, int64_t standing, int64_t passing, int kt, int64_t batch_heads) {
    a.tiles = int((standing + TILE - 1) / TILE);
    a.steps = (passing + kt - 1) / kt;
    const int64_t tiles = batch_heads * a.tiles;
    int64_t splits = tiles > 0 && tiles < COMPUTE_UNITS ? WANTED / tiles : 1;
    if (splits > a.steps / LEAST_STEPS) splits = a.steps / LEAST_STEPS;
    if (splits < 1) splits = 1;
    a.split_steps = (a.steps + splits - 1) / splits;
    a.splits = a.split_steps ? int((a.steps + a.split_steps - 1) / a.split_steps) : 1;
    a.units = tiles * a.splits;
    a.tile_by = Divisor(a.tiles > 0 ? (uint32_t)a.tiles : 1), a.split_by = Divisor((uint32_t)a.splits);
}

Plan plan(const lffn_cross_attention &c) {
    Plan p;
    BwdArgs a{};
    const int64_t size = c.format == LFFN_ROWS_F32 ? 4 : 2, batch_heads = c.B * c.key_heads;
    const int kt = c.format == LFFN_ROWS_F32 && c.columns > 32 ? 32 : 64;
    a.q = static_cast<const char *>(c.q), a.k = static_cast<const char *>(c.k), a.v = static_cast<const char *>(c.v);
    a.mask = c.key_mask, a.mask_stride = c.mask_stride;
    a.qb = c.q_strides[0] * size, a.qt = c.q_strides[1] * size, a.qh = c.q_strides[2] * size;
    a.kb = c.k_strides[0] * size, a.kt = c.k_strides[1] * size, a.kh = c.k_strides[2] * size;
    a.vb = c.v_strides[0] * size, a.vt = c.v_strides[1] * size, a.vh = c.v_strides[2] * size;
    a.keys = c.k_len, a.q_len = c.q_len, a.batch_heads = (int)batch_heads;
    const int64_t group = c.heads / c.key_heads;
    a.key_heads = (int)c.key_heads, a.columns = (int)c.columns;
    a.rows = int(c.q_len * group);
    a.group = Divisor(group > 0 ? (uint32_t)group : 1), a.heads = Divisor((uint32_t)a.key_heads);
    a.c = c.scale * LOG2E, a.scale = c.scale;
    const bool levels = c.format != LFFN_ROWS_BF16, scaled = c.format == LFFN_ROWS_F32;
    a.g_tiles = (a.rows + LEVEL_ROWS - 1) / LEVEL_ROWS;
    a.v_tiles = levels ? int((a.keys + LEVEL_ROWS - 1) / LEVEL_ROWS) : 0;
    a.level_tiles = Divisor(a.g_tiles + a.v_tiles > 0 ? uint32_t(a.g_tiles + a.v_tiles) : 1);
    p.q = p.k = p.both = a;
    if (in_one(c.format, c.columns, a.rows)) share_out(p.both, a.rows, a.keys, 32, batch_heads);
    share_out(p.q, a.rows, a.keys, kt, batch_heads);
    share_out(p.k, a.keys, a.rows, in_pairs(c.format == LFFN_ROWS_F32 ? 2 : 1, int(c.columns)) ? 32 : kt, batch_heads);
    p.fits = std::max({p.q.units, 2 * p.k.units, p.both.units, batch_heads * (a.g_tiles + a.v_tiles) + c.B}) <= MOST_THREADS / WG;
    // (whole lines: parts that began 16 bytes into one were written in 47 us for 43, keys' gradients of 4 x 333 x 509 x 8 x 128 fp32)
    auto take = [&](int64_t floats) {
        const int64_t at = p.floats;
        p.floats += (floats + 63) / 64 * 64;
        return at;
    };
    p.delta = take(batch_heads * a.rows);
    p.g_levels = take(levels ? batch_heads * a.g_tiles : 0);
    p.q_levels = take(scaled ? batch_heads * a.g_tiles : 0);
    p.v_levels = take(batch_heads * a.v_tiles);
    p.k_levels = take(scaled ? batch_heads * a.v_tiles : 0);
    p.single = take(c.B);
    const int64_t of_q = p.q.splits > 1 ? p.q.splits * batch_heads * a.rows * a.columns : 0;
    const int64_t of_k = p.k.splits > 1 ? 2 * p.k.splits * batch_heads * a.keys * a.columns : 0;
    const int64_t of_both = p.both.splits > 1 ? p.both.splits * batch_heads * a.rows * a.columns : 0;
    p.part = take(std::max({of_q, of_k, of_both}));       // (one launch's are added up before the next begins)
    return p;
}

template <typename F>
void add_splits(const AddArgs &a, int arrays, hipStream_t stream) {
    const int64_t quads = a.all * (a.columns / 4);
    if (a.splits > 4) add_splits_kernel<F, WAVES><<<dim3((unsigned)((quads + 63) / 64), arrays), dim3(WG), 0, stream>>>(a);
    else add_splits_kernel<F, 1><<<dim3((unsigned)((quads + WG - 1) / WG), arrays), dim3(WG), 0, stream>>>(a);
}

template <typename F, int DP, int KT>
int launch(const Plan &p, hipStream_t stream) {
    constexpr bool LEVELS = F::LIFT != 0.f;
    const int64_t tiles = int64_t(p.q.batch_heads) * (p.q.g_tiles + p.q.v_tiles);
    const int64_t looks = p.q.mask ? p.q.batch_heads / p.q.key_heads : 0;               // for a single key, a workgroup a sequence
    if (tiles + looks > 0) delta_kernel<F, level_lanes(DP), LEVELS><<<dim3((unsigned)(tiles + looks)), dim3(WG), 0, stream>>>(p.q);
    auto add_queries = [&](const BwdArgs &q) {
        if (q.splits > 1)
            add_splits<F>({{q.part, nullptr}, {q.gq, nullptr}, int64_t(q.batch_heads) * q.rows, q.q_len, q.heads, q.group, q.rows, q.splits, q.columns}, 1, stream);
    };
    if constexpr (F::PLANES == 1 && DP == 64) {
        if (p.both.units > 0 && p.q.units > 0 && p.k.units > 0) {
            static LdsGrant granted;
            const size_t bytes = (2 * Tile<F, DP, TILE>::SIZE + 4 * Tile<F, DP, 32>::SIZE + 2 * Tile<F, 32, TILE>::SIZE) * 16 + BLOCK * 8;
            if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&gradients_kernel<F>), bytes, granted)) return LFFN_ERR_LAUNCH;
            gradients_kernel<F><<<dim3((unsigned)p.both.units), dim3(WG), bytes, stream>>>(p.both);
            add_queries(p.both);
            return lffn_launch_status();
        }
    }
    if (p.q.units > 0) {
        static LdsGrant granted;
        const size_t bytes = 4 * Tile<F, DP, KT>::SIZE * 16 + BLOCK * 8;
        if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&query_gradient_kernel<F, DP, KT>), bytes, granted)) return LFFN_ERR_LAUNCH;
        query_gradient_kernel<F, DP, KT><<<dim3((unsigned)p.q.units), dim3(WG), bytes, stream>>>(p.q);
        add_queries(p.q);
    }
    if (p.k.units > 0) {
        static LdsGrant granted;
        if constexpr (in_pairs(F::PLANES, DP)) {
            const size_t bytes = 3 * (2 * Tile<F, DP, 32>::SIZE * 16 + WAVES * 4096 + 2 * 32 * 4);
            if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&key_gradient_pairs_kernel<F, DP>), bytes, granted)) return LFFN_ERR_LAUNCH;
            key_gradient_pairs_kernel<F, DP><<<dim3((unsigned)p.k.units), dim3(2 * WG), bytes, stream>>>(p.k);
        } else {
            const size_t bytes = 4 * Tile<F, DP, KT>::SIZE * 16 + 4 * KT * 4;
            if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&key_gradient_kernel<F, DP, KT>), bytes, granted)) return LFFN_ERR_LAUNCH;
            key_gradient_kernel<F, DP, KT><<<dim3((unsigned)p.k.units), dim3(WG), bytes, stream>>>(p.k);
        }
        const BwdArgs &k = p.k;
        const int64_t all = int64_t(k.batch_heads) * k.keys;
        if (k.splits > 1)
            add_splits<F>({{k.part, k.part + k.splits * all * k.columns}, {k.gk, k.gv}, all, k.keys, k.heads, Divisor(1), (int)k.keys, k.splits, k.columns}, 2,
                          stream);
    }
    return lffn_launch_status();
}

template <typename F>
int launch(const Plan &p, hipStream_t stream) {
    if (p.q.columns <= 32) return launch<F, 32, 64>(p, stream);
    if (p.q.columns <= 64) return launch<F, 64, F::PLANES == 1 ? 64 : 32>(p, stream);
    return launch<F, 128, F::PLANES == 1 ? 64 : 32>(p, stream);
}

}  // namespace

extern "C" int lffn_cross_attention_bwd_workspace_bytes(const lffn_cross_attention *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    const Plan p = plan(*c);
    LFFN_REQUIRE(p.fits, LFFN_ERR_UNSUPPORTED);
    *bytes = p.floats * 4;
    return LFFN_OK;
}

extern "C" int lffn_cross_attention_bwd(const lffn_cross_attention *c, const void *out, const void *kept, const void *g_out, void *grad_q,
                                        void *grad_k, void *grad_v, void *workspace, int64_t workspace_bytes, void *stream) {
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    Plan p = plan(*c);
    LFFN_REQUIRE(p.fits, LFFN_ERR_UNSUPPORTED);
    if (p.q.units == 0 && p.k.units == 0) return LFFN_OK;
    LFFN_REQUIRE(p.q.units == 0 || (out && kept && g_out), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(p.k.units == 0 || (grad_k != nullptr) == (grad_v != nullptr), LFFN_ERR_BAD_ARG);
    if (!grad_q) p.q.units = 0;                            // not wanted
    if (!grad_k) p.k.units = 0;
    if (p.q.units == 0 && p.k.units == 0) return LFFN_OK;
    for (const void *t : {out, kept, g_out, (const void *)grad_q, (const void *)grad_k, (const void *)grad_v}) LFFN_REQUIRE(lffn_aligned16(t), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(p.floats == 0 || (workspace && lffn_aligned16(workspace) && workspace_bytes >= p.floats * 4), LFFN_ERR_BAD_ARG);
    float *const w = static_cast<float *>(workspace);
    const Kept k = kept_at(const_cast<void *>(kept), c->B * c->q_len * c->heads, c->format == LFFN_ROWS_F32 ? 4 : 2);
    for (BwdArgs *a : {&p.q, &p.k, &p.both}) {
        a->out = static_cast<const char *>(out), a->g = static_cast<const char *>(g_out), a->lse = k.levels, a->rest = k.rest;
        a->gq = static_cast<char *>(grad_q), a->gk = static_cast<char *>(grad_k), a->gv = static_cast<char *>(grad_v);
        a->delta = w + p.delta, a->g_levels = w + p.g_levels, a->q_levels = w + p.q_levels, a->v_levels = w + p.v_levels, a->k_levels = w + p.k_levels, a->part = w + p.part;
        a->single = reinterpret_cast<int32_t *>(w + p.single);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (c->format == LFFN_ROWS_F32) return launch<F32Two>(p, s);
    return c->format == LFFN_ROWS_BF16 ? launch<BF16>(p, s) : launch<F16>(p, s);
}
