// The backward of the attention to an encoder's states (cross_attention.h: operands and tiles).
//
//   delta_i = g_i . o_i;  p_ij = 2^(c s_ij - lse_i);  ds_ij = p_ij (g_i . v_j - delta_i)
//   grad v_j = sum_i p_ij g_i;  grad k_j = scale sum_i ds_ij q_i;  grad q_i = scale sum_j ds_ij k_j
// Three kernels: delta; the queries' gradients, a workgroup's 128 rows standing and the keys and values passing; the keys' and values', 128 keys
// standing and the rows with their gradients passing.  Scores and g . v are formed twice (seven products for five), for that every sum
// has one owner and a fixed order: no atomics, the same bits on every call.  Where there are too few standing rows or keys to fill
// the chip what passes is shared out over several workgroups, and a last kernel adds their sums.
//
// Half precision: p is held 2^14 times larger (at most 2^14), ds times a power of two that takes 2 |g| |v|, of the longest
// rows of the batch and key head, which no ds exceeds, below 2^15: gradients of any size, and weights of many keys, stay among half's normal numbers.
#include "cross_attention.h"

using namespace cross_attention;

__attribute__((visibility("hidden"))) int lffn_internal_cross_attention_check(const lffn_cross_attention *a);

namespace {

constexpr int NORM_ROWS = 1024;           // rows whose longest is looked for by one workgroup
constexpr float P_LIFT = 14.f;            // half precision

struct BwdArgs {
    const char *q, *k, *v, *out, *g;
    const uint8_t *mask;
    const float *lse;
    char *gq, *gk, *gv;
    float *delta, *g_norms, *v_norms;     // [B, key heads, rows]; squares of the longest rows: [B, key heads, tiles]
    float *part;                          // [splits, B, key heads, rows or keys, columns] (keys: of k, then of v)
    int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, mask_stride;         // strides in bytes
    int64_t keys, steps, split_steps, q_len, units;
    int batch_heads, key_heads, group, rows, tiles, splits, columns, g_tiles, v_tiles;
    float c, scale;
};

// Largest of v over the wavefront
__device__ __forceinline__ float wave_most(float v) {
    v = fmaxf(v, lane_xor<1>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, lane_xor<4>(v));
    v = fmaxf(v, lane_xor<8>(v));
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}

// delta of every row; half precision: the longest rows of g and v as well.  16 lanes a row, 8 columns a lane.
template <typename F, bool NORMS>
__global__ __launch_bounds__(WG) void delta_kernel(BwdArgs a) {
    const int lane = threadIdx.x & 15, col = lane * 8, tiles = a.g_tiles + a.v_tiles;
    const int64_t bh = blockIdx.x / tiles, b = bh / a.key_heads, kh = bh - b * a.key_heads;
    const int tile = int(blockIdx.x - bh * tiles);
    float most = 0.f;
    if (tile < a.g_tiles) {
        for (int row = tile * NORM_ROWS + threadIdx.x / 16; row < min(a.rows, (tile + 1) * NORM_ROWS); row += WG / 16) {
            float dot = 0.f, squares = 0.f;
            if (col < a.columns) {
                const int64_t at = (heads_row(b, kh, row, a.q_len, a.key_heads, a.group) * a.columns + col) * F::BYTES;
                float o[8], g[8];
                F::unpack(F::load(a.out + at), o);
                F::unpack(F::load(a.g + at), g);
#pragma unroll
                for (int i = 0; i < 8; ++i) dot = fmaf(o[i], g[i], dot), squares = fmaf(g[i], g[i], squares);
            }
            dot = lane_group_sum<16>(dot);
            if (NORMS) most = fmaxf(most, lane_group_sum<16>(squares));
            if (lane == 0) a.delta[bh * a.rows + row] = dot;
        }
    } else if (NORMS) {
        const int64_t begin = int64_t(tile - a.g_tiles) * NORM_ROWS, end = begin + NORM_ROWS < a.keys ? begin + NORM_ROWS : a.keys;
        for (int64_t key = begin + threadIdx.x / 16; key < end; key += WG / 16) {
            if (a.mask && a.mask[b * a.mask_stride + key] == 0) continue;        // (the 16 lanes alike)
            float squares = 0.f;
            if (col < a.columns) {
                float v[8];
                F::unpack(F::load(a.v + b * a.vb + kh * a.vh + key * a.vt + col * F::BYTES), v);
#pragma unroll
                for (int i = 0; i < 8; ++i) squares = fmaf(v[i], v[i], squares);
            }
            most = fmaxf(most, lane_group_sum<16>(squares));
        }
    }
    if (NORMS) {
        __shared__ float red[WAVES];
        most = wave_most(most);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
        __syncthreads();
        if (threadIdx.x == 0) {
            most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
            if (tile < a.g_tiles) a.g_norms[bh * a.g_tiles + tile] = most;
            else a.v_norms[bh * a.v_tiles + tile - a.g_tiles] = most;
        }
    }
}

// What ds is multiplied with, as an exponent; half precision alone.
template <typename F>
__device__ __forceinline__ int ds_exponent(const BwdArgs &a, int64_t bh) {
    if constexpr (F::LIFT == 0.f) return 0;
    float g = 0.f, v = 0.f;
    for (int i = threadIdx.x & 63; i < a.g_tiles; i += 64) g = fmaxf(g, a.g_norms[bh * a.g_tiles + i]);
    for (int i = threadIdx.x & 63; i < a.v_tiles; i += 64) v = fmaxf(v, a.v_norms[bh * a.v_tiles + i]);
    const float most = 2.f * sqrtf(wave_most(g)) * sqrtf(wave_most(v));
    const int e = int(__float_as_uint(most) >> 23) - 127;    // most < 2^(e + 1)
    return most > 0.f && e < 128 ? __builtin_amdgcn_readfirstlane(min(max(14 - e, -60), 60)) : 0;
}

// The sums of a standing row, or a split's part of them, to where they belong.
template <typename F, int DB>
__device__ __forceinline__ void store_sums(const ca_f32x16_t (&o)[DB], float by, char *out, float *part, int columns, int half) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int col = 32 * d + 8 * g + 4 * half;
            if (col >= columns) continue;
            const float t[4] = {o[d][4 * g] * by, o[d][4 * g + 1] * by, o[d][4 * g + 2] * by, o[d][4 * g + 3] * by};
            if (part) *reinterpret_cast<float4 *>(part + col) = make_float4(t[0], t[1], t[2], t[3]);
            else F::store4(out + col * F::BYTES, t[0], t[1], t[2], t[3]);
        }
}

template <typename F, int DP, int KT>
__global__ __launch_bounds__(WG, F::PLANES == 1 && DP <= 64 ? 2 : 1) void query_gradient_kernel(BwdArgs a) {
    typedef Tile<F, DP, KT> T;
    typedef Frag<F::PLANES> Op;
    constexpr int CHUNKS = DP / 16, KB = KT / 32, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // [2][keys, values], words
    uint64_t *const words = reinterpret_cast<uint64_t *>(lds + 4 * T::SIZE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, half = lane >> 5;
    const int64_t unit = unit_of(blockIdx.x, a.units);
    const int tile = unit % a.tiles, split = unit / a.tiles % a.splits;
    const int64_t bh = unit / a.tiles / a.splits, b = bh / a.key_heads, kh = bh - b * a.key_heads;
    const int pieces = a.columns / 8;
    const char *const kp = a.k + b * a.kb + kh * a.kh, *const vp = a.v + b * a.vb + kh * a.vh;
    const uint8_t *const mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int row = tile * TILE + wave * ROWS + r;
    const bool live = row < a.rows;

    typename F::Raw rk[T::SHARE], rv[T::SHARE];
    auto fetch = [&](int64_t step, uint64_t word) {
#pragma unroll
        for (int i = 0; i < T::SHARE; ++i) {
            const int p = tid + WG * i, key = p / T::PIECES, piece = p % T::PIECES;
            const bool in = (word >> key & 1) && piece < pieces;
            const int64_t at = step * KT + key;
            rk[i] = in ? F::load(kp + at * a.kt + piece * 8 * F::BYTES) : F::zero();
            rv[i] = in ? F::load(vp + at * a.vt + piece * 8 * F::BYTES) : F::zero();
        }
    };
    auto place = [&](int buf) {
        uint4 *const to = lds + buf * 2 * T::SIZE;
#pragma unroll
        for (int i = 0; i < T::SHARE; ++i) {
            const int p = tid + WG * i, key = p / T::PIECES, piece = p % T::PIECES;
            T::put(to, key, piece, rk[i]);
            T::put(to + T::SIZE, key, piece, rv[i]);
        }
    };

    const int64_t out_row = heads_row(b, kh, live ? row : 0, a.q_len, a.key_heads, a.group) * a.columns * F::BYTES;
    Op fq[CHUNKS], fg[CHUNKS];
    {
        const char *const p = Rows{a.q + b * a.qb + kh * a.group * a.qh, a.qt, a.qh, a.group}.at(live ? row : 0);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            fq[c] = own_rows<F>(p, live, c, half, pieces);
            fg[c] = own_rows<F>(a.g + out_row, live, c, half, pieces);
        }
    }
    const int lift = ds_exponent<F>(a, bh);
    const float f = __builtin_amdgcn_ldexpf(1.f, lift);
    const float level = live ? a.lse[bh * a.rows + row] : INFINITY, delta = live ? a.delta[bh * a.rows + row] * f : 0.f;
    ca_f32x16_t dq[DB] = {};

    auto compute = [&](int buf, uint64_t word) {
        const uint4 *const keys = lds + buf * 2 * T::SIZE, *const values = keys + T::SIZE;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            ca_f32x16_t s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                s = F::mma(T::rows(keys, kb * 32 + r, c, half), fq[c], s);
                dp = F::mma(T::rows(values, kb * 32 + r, c, half), fg[c], dp);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -level)) * fmaf(dp[e], f, -delta);
            const uint32_t part = (uint32_t)(word >> (32 * kb));
            if (part != ~0u) {
                const uint32_t w = part >> (4 * half);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(w >> (8 * (e / 4) + e % 4) & 1)) s[e] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = s[8 * c + e];
                const Op ds = F::operand(t);
#pragma unroll
                for (int d = 0; d < DB; ++d) dq[d] = F::mma(T::columns(keys, kb * 32 + c * 16, d, lane), ds, dq[d]);
            }
        }
    };

    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;
#pragma unroll 1
    for (int64_t first = begin; first < end; first += BLOCK) {
        look_at_masks<KT>(words, mask, first, end, a.keys);
        __syncthreads();
        uint64_t left = __ballot(words[lane] != 0);
        if (left) {
            int i = __builtin_ctzll(left), buf = 0;
            uint64_t word = uniform(words[i]);
            left &= left - 1;
            fetch(first + i, word);
            place(0);
            __syncthreads();
#pragma unroll 1
            for (;;) {
                const bool more = left != 0;
                uint64_t next = 0;
                if (more) {
                    i = __builtin_ctzll(left);
                    left &= left - 1;
                    next = uniform(words[i]);
                    fetch(first + i, next);
                }
                compute(buf, word);
                if (!more) break;
                place(buf ^ 1);
                __syncthreads();
                buf ^= 1;
                word = next;
            }
        }
        __syncthreads();                  // the words and the buffers are free again
    }
    if (!live) return;
    float *const part = a.splits > 1 ? a.part + (int64_t(split) * a.batch_heads * a.rows + bh * a.rows + row) * a.columns : nullptr;
    store_sums<F, DB>(dq, __builtin_amdgcn_ldexpf(a.scale, -lift), a.gq + out_row, part, a.columns, half);
}

template <typename F, int DP, int KT>
__global__ __launch_bounds__(WG, F::PLANES == 1 && DP <= 64 ? 2 : 1) void key_gradient_kernel(BwdArgs a) {
    typedef Tile<F, DP, KT> T;
    typedef Frag<F::PLANES> Op;
    constexpr int CHUNKS = DP / 16, RB = KT / 32, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // [2][rows, their gradients], [2][levels, deltas]
    float *const levels = reinterpret_cast<float *>(lds + 4 * T::SIZE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, half = lane >> 5;
    const int64_t unit = unit_of(blockIdx.x, a.units);
    const int tile = unit % a.tiles, split = unit / a.tiles % a.splits;
    const int64_t bh = unit / a.tiles / a.splits, b = bh / a.key_heads, kh = bh - b * a.key_heads;
    const int pieces = a.columns / 8;
    const int64_t key = int64_t(tile) * TILE + wave * ROWS + r;
    const bool in = key < a.keys, live = in && (!a.mask || a.mask[b * a.mask_stride + key] != 0);
    const Rows rows{a.q + b * a.qb + kh * a.group * a.qh, a.qt, a.qh, a.group};

    Op fk[CHUNKS], fv[CHUNKS];
    {
        const int64_t at = live ? key : 0;
        const char *const kp = a.k + b * a.kb + kh * a.kh + at * a.kt, *const vp = a.v + b * a.vb + kh * a.vh + at * a.vt;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            fk[c] = own_rows<F>(kp, live, c, half, pieces);
            fv[c] = own_rows<F>(vp, live, c, half, pieces);
        }
    }
    const bool wave_works = __any(live), works = __syncthreads_or(live);
    constexpr bool HALF = F::LIFT != 0.f;
    const int lift = ds_exponent<F>(a, bh);
    const float f = __builtin_amdgcn_ldexpf(1.f, HALF ? lift - int(P_LIFT) : 0);

    typename F::Raw rq[T::SHARE], rg[T::SHARE];
    float level = 0.f, delta = 0.f;
    auto fetch = [&](int64_t step) {
#pragma unroll
        for (int i = 0; i < T::SHARE; ++i) {
            const int p = tid + WG * i, piece = p % T::PIECES, row = int(step) * KT + p / T::PIECES;
            const bool on = row < a.rows && piece < pieces;
            rq[i] = on ? F::load(rows.at(row) + piece * 8 * F::BYTES) : F::zero();
            rg[i] = on ? F::load(a.g + (heads_row(b, kh, row, a.q_len, a.key_heads, a.group) * a.columns + piece * 8) * F::BYTES) : F::zero();
        }
        if (tid < KT) {
            const int row = int(step) * KT + tid;
            level = row < a.rows ? a.lse[bh * a.rows + row] - (HALF ? P_LIFT : 0.f) : INFINITY;
            delta = row < a.rows ? a.delta[bh * a.rows + row] * f : 0.f;
        }
    };
    auto place = [&](int buf) {
        uint4 *const to = lds + buf * 2 * T::SIZE;
#pragma unroll
        for (int i = 0; i < T::SHARE; ++i) {
            const int p = tid + WG * i, row = p / T::PIECES, piece = p % T::PIECES;
            T::put(to, row, piece, rq[i]);
            T::put(to + T::SIZE, row, piece, rg[i]);
        }
        if (tid < KT) {
            levels[buf * 2 * KT + tid] = level;
            levels[buf * 2 * KT + KT + tid] = delta;
        }
    };

    ca_f32x16_t dk[DB] = {}, dv[DB] = {};
    auto compute = [&](int buf) {
        const uint4 *const queries = lds + buf * 2 * T::SIZE, *const gradients = queries + T::SIZE;
        const float *const level = levels + buf * 2 * KT + 4 * half, *const delta = level + KT;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            ca_f32x16_t s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                s = F::mma(T::rows(queries, rb * 32 + r, c, half), fk[c], s);
                dp = F::mma(T::rows(gradients, rb * 32 + r, c, half), fv[c], dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 l = *reinterpret_cast<const float4 *>(level + rb * 32 + 8 * g), d = *reinterpret_cast<const float4 *>(delta + rb * 32 + 8 * g);
                const float ls[4] = {l.x, l.y, l.z, l.w}, ds[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], a.c, -ls[e]));
                    s[4 * g + e] = p;
                    dp[4 * g + e] = p * fmaf(dp[4 * g + e], f, -ds[e]);
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float t[8], u[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = s[8 * c + e], u[e] = dp[8 * c + e];
                const Op p = F::operand(t), ds = F::operand(u);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    dv[d] = F::mma(T::columns(gradients, rb * 32 + c * 16, d, lane), p, dv[d]);
                    dk[d] = F::mma(T::columns(queries, rb * 32 + c * 16, d, lane), ds, dk[d]);
                }
            }
        }
    };

    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;
    if (works && begin < end) {
        int buf = 0;
        fetch(begin);
        place(0);
        __syncthreads();
#pragma unroll 1
        for (int64_t step = begin;;) {
            const bool more = ++step < end;
            if (more) fetch(step);
            if (wave_works) compute(buf);
            if (!more) break;
            place(buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
    }
    if (!in) return;
    if (!live) {
#pragma unroll
        for (int d = 0; d < DB; ++d) dk[d] = ca_f32x16_t{}, dv[d] = ca_f32x16_t{};
    }
    const int64_t at = heads_row(b, kh, int(key), a.keys, a.key_heads, 1) * a.columns * F::BYTES, all = int64_t(a.batch_heads) * a.keys;
    float *const part = a.splits > 1 ? a.part + (int64_t(split) * all + bh * a.keys + key) * a.columns : nullptr;
    store_sums<F, DB>(dk, __builtin_amdgcn_ldexpf(a.scale, -lift), a.gk + at, part, a.columns, half);
    store_sums<F, DB>(dv, HALF ? 1.f / 16384.f : 1.f, a.gv + at, part ? part + a.splits * all * a.columns : nullptr, a.columns, half);
}

// The splits' sums of a row as one, in their order.  Four columns a lane.
template <typename F>
__global__ __launch_bounds__(WG) void add_splits_kernel(const float *part, char *out, int64_t all, int rows, int64_t len, int key_heads, int group,
                                                        int splits, int columns) {
    const int quads = columns / 4;
    const int64_t i = int64_t(blockIdx.x) * WG + threadIdx.x, at = i / quads;
    const int col = int(i - at * quads) * 4;
    if (at >= all) return;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
        const float4 v = *reinterpret_cast<const float4 *>(part + (s * all + at) * columns + col);
        acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    const int64_t bh = at / rows, b = bh / key_heads, kh = bh - b * key_heads;
    F::store4(out + (heads_row(b, kh, int(at - bh * rows), len, key_heads, group) * columns + col) * F::BYTES, acc.x, acc.y, acc.z, acc.w);
}

constexpr int64_t WANTED = 512;           // workgroups, where there is enough to share out
constexpr int64_t LEAST_STEPS = 2;        // of a workgroup

// The two large launches and where the workspace's parts begin (in floats).
struct Plan {
    BwdArgs q{}, k{};
    int64_t delta = 0, g_norms = 0, v_norms = 0, part = 0, floats = 0;
};

void share_out(BwdArgs &a, int64_t standing, int64_t passing, int kt, int64_t batch_heads) {
    a.tiles = int((standing + TILE - 1) / TILE);
    a.steps = (passing + kt - 1) / kt;
    const int64_t tiles = batch_heads * a.tiles;
    int64_t splits = tiles > 0 && tiles < WANTED ? (WANTED + tiles - 1) / tiles : 1;
    if (splits > a.steps / LEAST_STEPS) splits = a.steps / LEAST_STEPS;
    if (splits < 1) splits = 1;
    a.split_steps = (a.steps + splits - 1) / splits;
    a.splits = a.split_steps ? int((a.steps + a.split_steps - 1) / a.split_steps) : 1;
    a.units = tiles * a.splits;
}

Plan plan(const lffn_cross_attention &c) {
    Plan p;
    BwdArgs a{};
    const int64_t size = c.format == LFFN_ROWS_F32 ? 4 : 2, batch_heads = c.B * c.key_heads;
    const int kt = c.format == LFFN_ROWS_F32 && c.columns > 64 ? 32 : 64;
    a.q = static_cast<const char *>(c.q), a.k = static_cast<const char *>(c.k), a.v = static_cast<const char *>(c.v);
    a.mask = c.key_mask, a.mask_stride = c.mask_stride;
    a.qb = c.q_strides[0] * size, a.qt = c.q_strides[1] * size, a.qh = c.q_strides[2] * size;
    a.kb = c.k_strides[0] * size, a.kt = c.k_strides[1] * size, a.kh = c.k_strides[2] * size;
    a.vb = c.v_strides[0] * size, a.vt = c.v_strides[1] * size, a.vh = c.v_strides[2] * size;
    a.keys = c.k_len, a.q_len = c.q_len, a.batch_heads = (int)batch_heads;
    a.key_heads = (int)c.key_heads, a.group = int(c.heads / c.key_heads), a.columns = (int)c.columns;
    a.rows = int(c.q_len * a.group);
    a.c = c.scale * LOG2E, a.scale = c.scale;
    const bool norms = c.format == LFFN_ROWS_F16;
    a.g_tiles = (a.rows + NORM_ROWS - 1) / NORM_ROWS;
    a.v_tiles = norms ? int((a.keys + NORM_ROWS - 1) / NORM_ROWS) : 0;
    p.q = p.k = a;
    share_out(p.q, a.rows, a.keys, kt, batch_heads);
    share_out(p.k, a.keys, a.rows, kt, batch_heads);
    auto take = [&](int64_t floats) {
        const int64_t at = p.floats;
        p.floats += (floats + 3) / 4 * 4;
        return at;
    };
    p.delta = take(batch_heads * a.rows);
    p.g_norms = take(norms ? batch_heads * a.g_tiles : 0);
    p.v_norms = take(batch_heads * a.v_tiles);
    const int64_t of_q = p.q.splits > 1 ? p.q.splits * batch_heads * a.rows * a.columns : 0;
    const int64_t of_k = p.k.splits > 1 ? 2 * p.k.splits * batch_heads * a.keys * a.columns : 0;
    p.part = take(of_q > of_k ? of_q : of_k);             // (one launch's are added up before the next begins)
    return p;
}

template <typename F>
void add_splits(const float *part, char *out, const BwdArgs &a, int rows, int64_t len, int group, hipStream_t stream) {
    const int64_t all = int64_t(a.batch_heads) * rows;
    add_splits_kernel<F><<<dim3((unsigned)((all * (a.columns / 4) + WG - 1) / WG)), dim3(WG), 0, stream>>>(part, out, all, rows, len, a.key_heads,
                                                                                                     group, a.splits, a.columns);
}

template <typename F, int DP, int KT>
int launch(const Plan &p, hipStream_t stream) {
    constexpr bool NORMS = F::LIFT != 0.f;
    const int64_t tiles = int64_t(p.q.batch_heads) * (p.q.g_tiles + p.q.v_tiles);
    if (tiles > 0) delta_kernel<F, NORMS><<<dim3((unsigned)tiles), dim3(WG), 0, stream>>>(p.q);
    if (p.q.units > 0) {
        static LdsGrant granted;
        const size_t bytes = 4 * Tile<F, DP, KT>::SIZE * 16 + BLOCK * 8;
        if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&query_gradient_kernel<F, DP, KT>), bytes, granted)) return LFFN_ERR_LAUNCH;
        query_gradient_kernel<F, DP, KT><<<dim3((unsigned)p.q.units), dim3(WG), bytes, stream>>>(p.q);
        if (p.q.splits > 1) add_splits<F>(p.q.part, p.q.gq, p.q, p.q.rows, p.q.q_len, p.q.group, stream);
    }
    if (p.k.units > 0) {
        static LdsGrant granted;
        const size_t bytes = 4 * Tile<F, DP, KT>::SIZE * 16 + 4 * KT * 4;
        if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&key_gradient_kernel<F, DP, KT>), bytes, granted)) return LFFN_ERR_LAUNCH;
        key_gradient_kernel<F, DP, KT><<<dim3((unsigned)p.k.units), dim3(WG), bytes, stream>>>(p.k);
        if (p.k.splits > 1) {
            const int64_t one = int64_t(p.k.splits) * p.k.batch_heads * p.k.keys * p.k.columns;
            add_splits<F>(p.k.part, p.k.gk, p.k, (int)p.k.keys, p.k.keys, 1, stream);
            add_splits<F>(p.k.part + one, p.k.gv, p.k, (int)p.k.keys, p.k.keys, 1, stream);
        }
    }
    return lffn_launch_status();
}

template <typename F>
int launch(const Plan &p, hipStream_t stream) {
    if (p.q.columns <= 32) return launch<F, 32, 64>(p, stream);
    if (p.q.columns <= 64) return launch<F, 64, 64>(p, stream);
    return launch<F, 128, F::PLANES == 1 ? 64 : 32>(p, stream);
}

}  // namespace

extern "C" int lffn_cross_attention_bwd_workspace_bytes(const lffn_cross_attention *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    *bytes = plan(*c).floats * 4;
    return LFFN_OK;
}

extern "C" int lffn_cross_attention_bwd(const lffn_cross_attention *c, const void *out, const float *lse, const void *g_out, void *grad_q,
                                        void *grad_k, void *grad_v, void *workspace, int64_t workspace_bytes, void *stream) {
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    Plan p = plan(*c);
    if (p.q.units == 0 && p.k.units == 0) return LFFN_OK;
    LFFN_REQUIRE(p.q.units == 0 || (out && lse && g_out), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(p.k.units == 0 || (grad_k != nullptr) == (grad_v != nullptr), LFFN_ERR_BAD_ARG);
    if (!grad_q) p.q.units = 0;                            // not wanted
    if (!grad_k) p.k.units = 0;
    if (p.q.units == 0 && p.k.units == 0) return LFFN_OK;
    for (const void *t : {out, g_out, (const void *)grad_q, (const void *)grad_k, (const void *)grad_v}) LFFN_REQUIRE(lffn_aligned16(t), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(p.floats == 0 || (workspace && lffn_aligned16(workspace) && workspace_bytes >= p.floats * 4), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(p.q.units <= INT32_MAX && p.k.units <= INT32_MAX &&
                     int64_t(p.q.batch_heads) * (p.q.g_tiles + p.q.v_tiles) <= INT32_MAX, LFFN_ERR_UNSUPPORTED);
    float *const w = static_cast<float *>(workspace);
    for (BwdArgs *a : {&p.q, &p.k}) {
        a->out = static_cast<const char *>(out), a->g = static_cast<const char *>(g_out), a->lse = lse;
        a->gq = static_cast<char *>(grad_q), a->gk = static_cast<char *>(grad_k), a->gv = static_cast<char *>(grad_v);
        a->delta = w + p.delta, a->g_norms = w + p.g_norms, a->v_norms = w + p.v_norms, a->part = w + p.part;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (c->format == LFFN_ROWS_F32) return launch<F32>(p, s);
    return c->format == LFFN_ROWS_BF16 ? launch<BF16>(p, s) : launch<F16>(p, s);
}
