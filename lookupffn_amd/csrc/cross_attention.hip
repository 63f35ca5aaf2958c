// softmax(scale q k^T) v of queries against an encoder's states: the forward kernels (cross_attention.h: operands and tiles).
//
// A workgroup has 128 rows (queries of the heads that share a key head), 32 a wavefront, and walks the keys 64 at a time with the running maximum and
// sum of a softmax taken in one pass.  Keys and values are fetched a step ahead and lie in LDS as in memory, in two buffers; scores are
// formed as keys x queries, weights times values as (values turned round) x weights.  Steps without a key that takes part are left out, masked
// keys and values are the step's first that takes part once more.  Where there are too few rows to fill the chip the keys are shared out over several workgroups,
// whose results a second kernel joins.
//
// Bound by the products where there are many rows, else by memory.  4 x 2048 rows x 4096 keys x 16 heads x 128 columns bfloat16 300 us, 0.92 PFLOP/s of the 1.26 that a
// large product reaches; 32 x 512 x 512 x 12 x 64 fp32 95 and 21 for the look at keys and values; one row of 32 heads on 4 x 16384 keys x 8 x 128 bfloat16, an eighth of
// them masked, 52 us, 4.5 TB/s, and 5 for the join.
#include "cross_attention.h"

using namespace cross_attention;

namespace {

struct FwdArgs {
    const char *q, *k, *v;
    const uint8_t *mask;
    char *out, *rest;                     // rest: null, or where what the rounding takes goes
    float *lse, *part, *part_lse;         // parts: [splits, B, key heads, rows(, columns)]
    float *k_levels, *v_levels;           // fp32 numbers in two terms: log2 of the longest rows, [B, key heads, level_tiles]
    int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, mask_stride;         // strides in bytes
    int64_t keys, steps, split_steps, q_len;
    Divisor group, tiles, split_by, heads, level_by;     // query heads of a key head, tiles of rows, shares of the keys, key heads, level_tiles
    int key_heads, rows, row_tiles, splits, columns, units;
    int level_tiles;
    int few_waves;                        // few_rows_kernel's wavefronts, 0: not the one
    float c;                              // scale log2 e
};

// few_rows_kernel: rows at most.  us, few_rows_kernel and cross_attention_kernel: 16 x 512 keys x 12 heads x 64 half, 1 row 7.8, 13.5; 4 x 16384 x 8 x 128 bfloat16,
// 1 row 59, 56, 2 rows 61, 60, 4 rows 69, 61; 64 x 512 x 16 x 64 bfloat16, 1 row 31, 36, 4 rows 49, 36; fp32 32 x 2048 x 16 x 64, 1 row 100, 123, 8 x 1024 x 8 x 128, 4 rows
// 20, 40, 32 x 1024 x 12 x 64, 3 rows 53, 64.
constexpr int few_rows(bool f32) { return f32 ? 4 : 2; }
constexpr int FEW_WAVES = 16;             // wavefronts of a workgroup at most,
constexpr int FEW_TOGETHER = 2;           // keys of a group of lanes asked for together
constexpr float SLACK = 6.f;              // how far (powers of two) a row's largest score may outgrow the one that its sums go by

// Four columns of a result, and what their rounding takes.
template <typename F>
__device__ __forceinline__ void store_result(const FwdArgs &a, int64_t at, const float4 &v) {
    F::store4(a.out + at, v.x, v.y, v.z, v.w);
    if (a.rest) F::store4(a.rest + at, v.x - F::rounded(v.x), v.y - F::rounded(v.y), v.z - F::rounded(v.z), v.w - F::rounded(v.w));
}

template <int LANES>
__device__ __forceinline__ float level_of(const F32::Raw &r, bool on) {
    float v[8];
    F32::unpack(on ? r : F32::zero(), v);
    return row_level<LANES>(v);
}

// log2 of the longest of 128 keys that take part, and of their values.  Bound by memory: both once.
template <int LANES>
__global__ __launch_bounds__(WG) void levels_kernel(FwdArgs a) {
    constexpr int APART = WG / LANES, EACH = LEVEL_ROWS / APART;
    __shared__ float red[2][WAVES];
    const int lane = threadIdx.x % LANES, col = lane * 8 < a.columns ? lane * 8 : 0;
    const bool on = lane * 8 < a.columns;
    const int bh = a.level_by.quotient(blockIdx.x), b = a.heads.quotient(bh), kh = bh - b * a.key_heads, tile = blockIdx.x - bh * a.level_tiles;
    F32::Raw k[EACH], v[EACH];
    bool live[EACH];
    const int64_t first = int64_t(tile) * LEVEL_ROWS + threadIdx.x / LANES;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t key = first + i * APART, at = key < a.keys ? key : a.keys - 1;
        live[i] = !a.mask || a.mask[b * a.mask_stride + at] != 0;
        k[i] = F32::load(a.k + b * a.kb + kh * a.kh + at * a.kt + col * 4);
        v[i] = F32::load(a.v + b * a.vb + kh * a.vh + at * a.vt + col * 4);
    }
    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const float lk = level_of<LANES>(k[i], on), lv = level_of<LANES>(v[i], on);
        if (live[i]) most[0] = fmaxf(most[0], lk), most[1] = fmaxf(most[1], lv);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        most[n] = over_groups_max<LANES>(most[n]);
        if ((threadIdx.x & 63) == 0) red[n][threadIdx.x >> 6] = most[n];
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const float *const r = red[threadIdx.x];
        (threadIdx.x ? a.v_levels : a.k_levels)[blockIdx.x] = fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
    }
}

template <typename F, int DP, int KT>
__global__ __launch_bounds__(WG, F::PLANES <= 2 && DP <= 64 ? 3 : DP <= 64 || F::PLANES <= 2 ? 2 : 1) void cross_attention_kernel(FwdArgs a) {
    typedef Tile<F, DP, KT> T;
    typedef Frag<F::PLANES> Op;
    constexpr int CHUNKS = DP / 16, KB = KT / 32, DB = DP / 32;
    extern __shared__ __attribute__((aligned(16))) uint4 lds[];           // [2][keys, values], words
    uint64_t *const words = reinterpret_cast<uint64_t *>(lds + 4 * T::SIZE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, half = lane >> 5;
    const Unit unit = unit_of(blockIdx.x, a.units, a.tiles, a.split_by, a.heads);
    const int tile = unit.tile, split = unit.split, bh = unit.bh, b = unit.b, kh = unit.kh;
    const int pieces = a.columns / 8;
    const Rows rows{a.q + b * a.qb + kh * a.group.by * a.qh, a.qt, a.qh, a.group};
    const char *const kp = a.k + b * a.kb + kh * a.kh, *const vp = a.v + b * a.vb + kh * a.vh;
    const uint8_t *const mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int row = tile * TILE + wave * ROWS + r;

    KeyFeed<F, DP, KT> feed(lds, pieces, kp, vp, a.kt, a.vt);
    const typename T::Reader read(lds, lane);
    Op fq[CHUNKS];
    float by_c = a.c;                     // what takes scores to powers of two
    int of_v = 0;                         // and values to what they are, as an exponent
    {
        const bool live = row < a.rows;
        const char *const p = rows.at(live ? row : 0);
        const int eq = own_rows<F>(p, live, half, pieces, fq);
        if constexpr (F::SCALED) {
            // keys and values by the longest of theirs
            const int ek = exponent_for(longest(a.k_levels, bh, a.level_tiles)), ev = exponent_for(longest(a.v_levels, bh, a.level_tiles));
            feed.scale_a = __builtin_amdgcn_ldexpf(1.f, ek);
            feed.scale_b = __builtin_amdgcn_ldexpf(1.f, ev);
            by_c = fmaxf(__builtin_amdgcn_ldexpf(a.c, -(eq + ek)), 0x1p-126f);       // (not zero, by which -infinity is no number: scores of nothing either way)
            of_v = -ev;
        }
    }
    ca_f32x16_t o[DB] = {};
    float most = -INFINITY, sum = 0.f;

    const bool wave_works = tile * TILE + wave * ROWS < a.rows;
    auto compute = [&](auto buf, uint64_t word, int64_t) {
        if (!wave_works) return;
        constexpr int KEYS = decltype(buf)::value * 2 * T::SIZE, VALUES = KEYS + T::SIZE;
        ca_f32x16_t s[KB] = {};
        products<F, KB * CHUNKS, F::PLANES == 1>([&](auto i) { return read.rows(KEYS, i % KB, i / KB); },
                                 [&](auto i, const Op &k) { s[i % KB] = F::mma(k, fq[i / KB], s[i % KB]); });
        constexpr uint64_t FULL = ~0ull >> (64 - KT);
        if (word != FULL) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const uint32_t w = (uint32_t)(word >> (32 * kb)) >> (4 * half);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(w >> (8 * (e / 4) + e % 4) & 1)) s[kb][e] = -INFINITY;
            }
        }
        float now = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) now = fmaxf(now, s[kb][e]);
        now = of_both_halves(now, [](float x, float y) { return fmaxf(x, y); });
        if (__any((now - most) * by_c > SLACK)) {             // (the first step's is: most is -infinity; -infinity - itself is no number, and not above)
            const float to = fmaxf(most, now), by = most == to ? 1.f : __builtin_amdgcn_exp2f(most * by_c - to * by_c);
            sum *= by;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= by;
            most = to;
        }
        const float less = (most == -INFINITY ? 0.f : most) * by_c - F::LIFT;
        // A step's weights are added up by themselves: one after the other onto the sum of all keys so far, each rounded as that is, 16384 of them left a row 9.8e-7
        // off, so 3.6e-7.  (In as many sums as cost no time: two for four 4096 x 16384 x 8 x 72 fp32 942 us, 953; 4 x 2048 x 4096 x 16 x 128 bfloat16 313, 310.)
        float of_step[F::PLANES == 1 ? 2 : 4] = {};
        Op p[2 * KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kb][e] = __builtin_amdgcn_exp2f(fmaf(s[kb][e], by_c, -less));
                of_step[e % (F::PLANES == 1 ? 2 : 4)] += s[kb][e];
            }
            // (16 bits: weights of one term, a rounding each of either sign beside the result's one: 1.4 times its error; two terms would be three products for two)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = s[kb][8 * c + e];
                p[2 * kb + c] = F::operand(t);
            }
        }
        if constexpr (F::PLANES == 1) sum += of_step[0] + of_step[1];
        else sum += (of_step[0] + of_step[1]) + (of_step[2] + of_step[3]);
        products<F, 2 * KB * DB, F::PLANES == 1>([&](auto i) { return read.columns(VALUES, i / DB, i % DB); },
                                 [&](auto i, const Op &v) { o[i % DB] = F::mma(v, p[i / DB], o[i % DB]); });
    };

    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.steps ? begin + a.split_steps : a.steps;
    walk_keys<KT>(feed, words, mask, begin, end, a.keys, compute);

    sum = of_both_halves(sum, [](float x, float y) { return x + y; });
    const auto inverse = factor<F>(sum == 0.f ? 0.f : 1.f / sum, of_v);     // a query without keys: zeros
    const float level = sum == 0.f ? INFINITY : (most == -INFINITY ? 0.f : most) * by_c - F::LIFT + __builtin_amdgcn_logf(sum);
    const bool live = row < a.rows;
    const int64_t at = int64_t(bh) * a.rows + row;
    if (a.splits > 1) {
        const int64_t of = int64_t(split) * (a.units / (a.splits * a.row_tiles)) * a.rows + at;
        if (live && half == 0) a.part_lse[of] = level;
        store_row<F32, DB>(o, inverse, reinterpret_cast<char *>(a.part + of * a.columns), live, a.columns, half);
        return;
    }
    if (a.lse && live && half == 0) a.lse[at] = level;
    const int64_t of = heads_row(b, kh, row, a.q_len, a.key_heads, a.group) * a.columns * F::BYTES;
    store_row<F, DB>(o, inverse, a.out + of, live, a.columns, half, a.rest ? a.rest + of : nullptr);
}

// A row or two for a key head (fp32: up to four): single tokens, with the heads that share it.  On the vector ALU, which keeps up with the memory here (a number of a key or value
// is one multiply-add a row) and needs neither tiles nor barriers: G lanes have a key and its value, 16 bytes a lane, 64 / G keys a wavefront and FEW_TOGETHER of them
// asked for at a time, so that a short call waits for memory once and its code is short (a launch fetches it anew).  Every group of lanes has a softmax of
// its own keys; groups and wavefronts are joined at the end.  Up to sixteen wavefronts a workgroup, so that 512 keys need no second kernel to join shares.
template <typename R, typename F, int G, int RN>
__global__ __launch_bounds__(64 * FEW_WAVES, RN == 1 ? 8 : 4) void few_rows_kernel(FwdArgs a) {
    constexpr int N = R::N, KEYS = 64 / G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, group = lane / G, j = lane % G;
    const Unit unit = unit_of(blockIdx.x, a.units, a.tiles, a.split_by, a.heads);
    const int split = unit.split, bh = unit.bh, b = unit.b, kh = unit.kh;
    const bool on = j * N < a.columns;
    const int64_t column = on ? j * 16 : 0;
    const char *const kp = a.k + b * a.kb + kh * a.kh + column, *const vp = a.v + b * a.vb + kh * a.vh + column;
    const uint8_t *const mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int64_t begin = split * a.split_steps, end = begin + a.split_steps < a.keys ? begin + a.split_steps : a.keys;      // (steps of one key)
    const int64_t first = begin + wave * (KEYS * FEW_TOGETHER) + group;

    // Whether a step's keys take part is asked for a step ahead of them: a wavefront does not ask for keys of which none does, but for its first, which wait for
    // nothing: 8 x 1 to 16384 of 16384 x 8 x 128 bfloat16 104 us, so 88.  (Keys and values a step ahead, too: 70 registers, so that a compute unit has one workgroup of 16 wavefronts for two, 256 x 512 x 16 x 64 half 94 us, so 107.)
    uint4 k[FEW_TOGETHER], v[FEW_TOGETHER];
    bool live[FEW_TOGETHER], next[FEW_TOGETHER];
    const int64_t apart = waves * (KEYS * FEW_TOGETHER);
    auto look = [&](int64_t from, bool (&live)[FEW_TOGETHER]) {
#pragma unroll
        for (int u = 0; u < FEW_TOGETHER; ++u) {
            const int64_t key = from + u * KEYS;
            live[u] = key < end && (!mask || mask[key] != 0);
        }
    };
    auto fetch = [&](int64_t from) {
#pragma unroll
        for (int u = 0; u < FEW_TOGETHER; ++u) {
            const int64_t key = from + u * KEYS, at = key < end ? key : end - 1;
            k[u] = *reinterpret_cast<const uint4 *>(kp + at * a.kt);
            v[u] = *reinterpret_cast<const uint4 *>(vp + at * a.vt);
        }
    };
    if (begin < end) {
        fetch(first);
        look(first, live);
        look(first + apart, next);
    }
    float q[RN][N], acc[RN][N] = {}, most[RN], sum[RN] = {};
    const Rows rows{a.q + b * a.qb + kh * a.group.by * a.qh + column, a.qt, a.qh, a.group};
#pragma unroll
    for (int r = 0; r < RN; ++r) {
        most[r] = -INFINITY;
        R::unpack(*reinterpret_cast<const uint4 *>(rows.at(r < a.rows ? r : 0)), q[r]);
#pragma unroll
        for (int e = 0; e < N; ++e) q[r][e] = on ? q[r][e] * a.c : 0.f;
    }
#pragma unroll 1
    for (int64_t at = first; at - group < end; at += apart) {
        float s[RN][FEW_TOGETHER];
#pragma unroll
        for (int u = 0; u < FEW_TOGETHER; ++u) {
            float x[N];
            R::unpack(k[u], x);
#pragma unroll
            for (int r = 0; r < RN; ++r) {
                float dot = 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) dot = fmaf(q[r][e], on ? x[e] : 0.f, dot);
                s[r][u] = live[u] ? lane_group_sum<G>(dot) : -INFINITY;
            }
        }
        float w[RN][FEW_TOGETHER];
#pragma unroll
        for (int r = 0; r < RN; ++r) {
            float now = most[r];
#pragma unroll
            for (int u = 0; u < FEW_TOGETHER; ++u) now = fmaxf(now, s[r][u]);
            const float less = now == -INFINITY ? 0.f : now, by = most[r] == now ? 1.f : __builtin_amdgcn_exp2f(most[r] - less);
            sum[r] *= by;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[r][e] *= by;
#pragma unroll
            for (int u = 0; u < FEW_TOGETHER; ++u) {
                w[r][u] = __builtin_amdgcn_exp2f(s[r][u] - less);
                sum[r] += w[r][u];
            }
            most[r] = now;
        }
#pragma unroll
        for (int u = 0; u < FEW_TOGETHER; ++u) {
            float x[N];
            R::unpack(v[u], x);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float value = live[u] ? x[e] : 0.f;                // (whatever is there)
#pragma unroll
                for (int r = 0; r < RN; ++r) acc[r][e] = fmaf(w[r][u], value, acc[r][e]);
            }
        }
        bool one = false;
#pragma unroll
        for (int u = 0; u < FEW_TOGETHER; ++u) live[u] = next[u], one |= next[u];
        if (__any(one)) fetch(at + apart);
        look(at + 2 * apart, next);
    }

    __shared__ float2 of_wave[FEW_WAVES][RN];            // largest score, sum of weights
    __shared__ float4 sums[FEW_WAVES][RN][G * N / 4];
    auto over_groups = [](float x, auto &&f) {
        if constexpr (G <= 4) x = f(x, lane_xor<4>(x));
        if constexpr (G <= 8) x = f(x, lane_xor<8>(x));
        if constexpr (G <= 16) x = f(x, lane_xor<16>(x));
        return f(x, lane_xor<32>(x));
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto plus = [](float x, float y) { return x + y; };
#pragma unroll
    for (int r = 0; r < RN; ++r) {
        const float all = over_groups(most[r], larger), by = most[r] == all ? 1.f : __builtin_amdgcn_exp2f(most[r] - all);
        const float total = over_groups(sum[r] * by, plus);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[r][e] = over_groups(acc[r][e] * by, plus);
        if (lane == 0) of_wave[wave][r] = make_float2(all, total);
        if (group == 0) {
#pragma unroll
            for (int e = 0; e < N; e += 4) sums[wave][r][(j * N + e) / 4] = make_float4(acc[r][e], acc[r][e + 1], acc[r][e + 2], acc[r][e + 3]);
        }
    }
    __syncthreads();
    // The wavefronts' sums as one, a group of 16 lanes four columns, a lane a wavefront (a lane all of them: 16 x 512 x 12 x 64 half 8.2 us for 7.8, 77 keys 4.4 for 4.2)
    for (int i = threadIdx.x / FEW_WAVES; i < RN * (G * N / 4); i += blockDim.x / FEW_WAVES) {
        const int r = i / (G * N / 4), quad = i % (G * N / 4), col = quad * 4, n = threadIdx.x % FEW_WAVES;
        if (r >= a.rows || col >= a.columns) continue;
        const float2 m = n < waves ? of_wave[n][r] : make_float2(-INFINITY, 0.f);
        const float4 x = n < waves ? sums[n][r][quad] : make_float4(0.f, 0.f, 0.f, 0.f);
        float all = m.x;
        all = larger(all, lane_xor<1>(all));
        all = larger(all, lane_xor<2>(all));
        all = larger(all, lane_xor<4>(all));
        all = larger(all, lane_xor<8>(all));
        const float by = m.x == all ? 1.f : __builtin_amdgcn_exp2f(m.x - all), total = lane_group_sum<FEW_WAVES>(by * m.y);
        const float4 o = make_float4(lane_group_sum<FEW_WAVES>(by * x.x), lane_group_sum<FEW_WAVES>(by * x.y), lane_group_sum<FEW_WAVES>(by * x.z),
                                     lane_group_sum<FEW_WAVES>(by * x.w));
        if (n != 0) continue;
        const float inverse = total == 0.f ? 0.f : 1.f / total, level = total == 0.f ? INFINITY : all + __builtin_amdgcn_logf(total);
        const int64_t at = int64_t(bh) * a.rows + r;
        if (a.splits > 1) {
            const int64_t of = int64_t(split) * (a.units / a.splits) * a.rows + at;
            if (quad == 0) a.part_lse[of] = level;
            *reinterpret_cast<float4 *>(a.part + of * a.columns + col) = make_float4(o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse);
        } else {
            if (quad == 0 && a.lse) a.lse[at] = level;
            store_result<F>(a, (heads_row(b, kh, r, a.q_len, a.key_heads, a.group) * a.columns + col) * F::BYTES,
                            make_float4(o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse));
        }
    }
}

// The splits' results of a row as one: weights 2^(level - largest level).  Four columns a lane, a fourth of the splits a wavefront, four of them asked for
// together; of few splits all by one thread.  (One thread for all, one split after the other: 16 splits of 128 rows x 128 columns 14.6 us, so 4.8; 2 splits of
// 32000 rows x 64 columns, a wavefront each 11.2, one thread 6.)
template <typename F, int SHARES>
__global__ __launch_bounds__(WG) void join_kernel(FwdArgs a, int64_t all_rows) {
    constexpr int TOGETHER = 4;
    const int quads = a.columns / 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = SHARES == 1 ? int64_t(blockIdx.x) * WG + threadIdx.x : int64_t(blockIdx.x) * 64 + lane, last = all_rows * quads - 1, at = (i < last ? i : last) / quads;
    const int col = int((i < last ? i : last) - at * quads) * 4;
    float most = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int first = SHARES == 1 ? 0 : wave; first < a.splits; first += SHARES * TOGETHER) {
        float l[TOGETHER], now = most;
        float4 v[TOGETHER];
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n) {
            const int64_t s = min(first + n * SHARES, a.splits - 1);
            l[n] = a.part_lse[s * all_rows + at];
            v[n] = *reinterpret_cast<const float4 *>(a.part + (s * all_rows + at) * a.columns + col);
        }
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n) {
            if (first + n * SHARES >= a.splits || l[n] == INFINITY) l[n] = -INFINITY, v[n] = make_float4(0.f, 0.f, 0.f, 0.f);      // (no key that takes part)
            now = fmaxf(now, l[n]);
        }
        const float less = now == -INFINITY ? 0.f : now, by = __builtin_amdgcn_exp2f(most - less);
        sum *= by;
        acc.x *= by, acc.y *= by, acc.z *= by, acc.w *= by;
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n) {
            const float w = __builtin_amdgcn_exp2f(l[n] - less);
            sum += w;
            acc.x = fmaf(w, v[n].x, acc.x), acc.y = fmaf(w, v[n].y, acc.y), acc.z = fmaf(w, v[n].z, acc.z), acc.w = fmaf(w, v[n].w, acc.w);
        }
        most = now;
    }
    float less = most == -INFINITY ? 0.f : most;
    if constexpr (SHARES > 1) {
        __shared__ float4 sums[SHARES][64];
        __shared__ float2 weights[SHARES][64];           // largest level, sum of weights
        sums[wave][lane] = acc;
        weights[wave][lane] = make_float2(most, sum);
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int w = 1; w < SHARES; ++w) most = fmaxf(most, weights[w][lane].x);
        less = most == -INFINITY ? 0.f : most;
        sum = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < SHARES; ++w) {
            const float2 m = weights[w][lane];
            const float4 v = sums[w][lane];
            const float by = __builtin_amdgcn_exp2f(m.x - less);
            sum = fmaf(by, m.y, sum);
            acc.x = fmaf(by, v.x, acc.x), acc.y = fmaf(by, v.y, acc.y), acc.z = fmaf(by, v.z, acc.z), acc.w = fmaf(by, v.w, acc.w);
        }
    }
    if (i > last) return;
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    const int bh = int(at / a.rows), b = a.heads.quotient(bh), kh = bh - b * a.key_heads, row = int(at - int64_t(bh) * a.rows);
    if (a.lse && col == 0) a.lse[at] = sum == 0.f ? INFINITY : less + __builtin_amdgcn_logf(sum);
    store_result<F>(a, (heads_row(b, kh, row, a.q_len, a.key_heads, a.group) * a.columns + col) * F::BYTES,
                    make_float4(acc.x * by, acc.y * by, acc.z * by, acc.w * by));
}

}  // namespace

__attribute__((visibility("hidden"))) int lffn_internal_cross_attention_check(const lffn_cross_attention *a) {
    LFFN_REQUIRE(a, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->B >= 0 && a->q_len >= 0 && a->k_len >= 0 && a->heads >= 0 && a->key_heads >= 1 && a->columns >= 1, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->heads % a->key_heads == 0 && a->format >= 0 && a->format <= 2, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->scale > 0.f && a->scale <= 3.4e38f, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->columns % 8 == 0 && a->columns <= 128, LFFN_ERR_UNSUPPORTED);
    const int64_t size = a->format == LFFN_ROWS_F32 ? 4 : 2;
    for (int d = 0; d < 3; ++d)
        for (const int64_t s : {a->q_strides[d], a->k_strides[d], a->v_strides[d]})
            LFFN_REQUIRE(s >= 0 && s * size % 16 == 0, LFFN_ERR_BAD_ARG);
    // (the kernels address a tile's rows, of the heads that share a key head, by 32 bits)
    const int64_t far = int64_t(1) << 32, group = a->heads / a->key_heads;
    LFFN_REQUIRE(a->k_strides[1] * size < far / 64 && a->v_strides[1] * size < far / 64 && a->q_strides[1] * size < far / 128 &&
                     (group <= 1 || a->q_strides[2] * size <= (far / 4 - 1) / group), LFFN_ERR_UNSUPPORTED);
    const bool no_rows = a->B == 0 || a->q_len == 0 || a->heads == 0, no_keys = a->B == 0 || a->k_len == 0;
    LFFN_REQUIRE((a->q || no_rows) && ((a->k && a->v) || no_keys) && a->mask_stride >= 0, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(lffn_aligned16(a->q) && lffn_aligned16(a->k) && lffn_aligned16(a->v), LFFN_ERR_BAD_ARG);
    const int64_t most = int64_t(1) << 30;
    LFFN_REQUIRE(a->heads <= 65536 && a->key_heads <= 65536 && a->q_len < most && a->k_len < most && a->B < most, LFFN_ERR_UNSUPPORTED);
    // (with no query head there may be key heads all the same; 2^32 of batches and heads times 2^23 tiles of keys is a number yet)
    const int64_t rows = a->q_len * group;
    LFFN_REQUIRE(rows < most && a->B * a->key_heads <= (int64_t(1) << 40) / (rows > 256 ? rows : 256), LFFN_ERR_UNSUPPORTED);
    return LFFN_OK;
}

namespace {

constexpr int64_t COMPUTE_UNITS = 256;    // a tile each and more: the keys are not shared out,
constexpr int64_t WANTED = 512;           // workgroups at most, where there are keys enough to share out (two a compute unit: up to a tile's shares more, 3 x 500 rows x 1500
                                          // keys x 10 x 128 bfloat16 32 us, so 43)
// but where a compute unit has little more than one tile (it has room for two or three) and the keys are so many that the join is little beside them.  us, whole and in
// shares, rows x keys x heads x columns: half 4000 x 4000 x 8 x 64 75, 64; x 6000 109, 79; x 12 heads 84, 78; x 15 heads 93, 108; 2 x 2000 x 2000 x 8 x 64 41, 43, x 3000
// 57, 50; 4000 x 4000 x 8 x 32 63, 45; bfloat16 4000 x 8000 x 8 x 128 195, 163; fp32 4000 x 4000 x 8 x 64 144, 128, x 128 241, 251.
constexpr int64_t MANY_KEYS = 2816;
constexpr int64_t MOST_TILES = 400, MANY_WANTED = 768;
// Where one wavefront of a tile's four has rows more tiles stand beside each other: 20 x 24 x 6571 x 12 x 16 half 70, 44; 32 x 8 x 2000 x 12 x 64 bfloat16 56, 45; 16 x 20 x
// 3000 x 8 x 128 half 49, 51; 4 x 16 x 8000 x 8 x 64 bfloat16 (16 shares, 32) 19, 23; 24 x 4 x 2877 x 12 x 64 half 49 with two shares, with three, more than stand beside each
// other, 62.
constexpr int64_t ONE_WAVE_KEYS = 1536, ONE_WAVE_LEAST = 192, ONE_WAVE_MOST = 512;
constexpr int64_t one_wave_wanted(int64_t columns) { return columns <= 32 ? 1024 : 768; }
constexpr int64_t LEAST_STEPS = 2;        // of a workgroup

// fp32: from where two terms of half precision are faster, with the look at keys and values that they take.  us, three terms and two, batch x rows x keys x heads x
// columns: 1 x 512 x 512 x 12 x 64 22, 27; 8 x 512 x 512 x 8 x 32 22, 23; 8 x 256 x 256 x 8 x 128 42, 35; 4 x 512 x 512 x 12 x 64 39, 37; 1 x 1024 x 1024 x 8 x 128 54, 42;
// 16 x 4096 x 77 x 8 x 64 109, 100; fewer rows: 16 x 128 x 512 x 12 x 64 37, 42; 64 x 128 x 512 x 12 x 64 94, 98; 32 x 64 x 1024 x 8 x 64 59, 67.
constexpr int64_t TWO_LEAST_ROWS = 256;   // of a key head
constexpr double TWO_LEAST_PRODUCTS = 5e8;        // multiply-adds of scores
constexpr int64_t FEW_WANTED = 4096;      // few_rows_kernel: wavefronts

// Lanes that have a key in few_rows_kernel.
int lanes_of_a_key(const lffn_cross_attention &c) {
    const int lanes = int(c.columns) * (c.format == LFFN_ROWS_F32 ? 4 : 2) / 16;
    return lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
}

// Fills sizes in; the workspace's bytes, or -1: too many tiles.
int64_t plan(const lffn_cross_attention &c, FwdArgs &a) {
    const int64_t size = c.format == LFFN_ROWS_F32 ? 4 : 2;
    const int kt = c.format == LFFN_ROWS_F32 && c.columns > 32 ? 32 : 64;
    a.q = static_cast<const char *>(c.q), a.k = static_cast<const char *>(c.k), a.v = static_cast<const char *>(c.v);
    a.mask = c.key_mask, a.mask_stride = c.mask_stride;
    a.qb = c.q_strides[0] * size, a.qt = c.q_strides[1] * size, a.qh = c.q_strides[2] * size;
    a.kb = c.k_strides[0] * size, a.kt = c.k_strides[1] * size, a.kh = c.k_strides[2] * size;
    a.vb = c.v_strides[0] * size, a.vt = c.v_strides[1] * size, a.vh = c.v_strides[2] * size;
    a.keys = c.k_len, a.q_len = c.q_len;
    const int64_t group = c.heads / c.key_heads;
    a.key_heads = (int)c.key_heads, a.columns = (int)c.columns;
    a.rows = int(c.q_len * group);
    a.row_tiles = (a.rows + TILE - 1) / TILE;
    a.steps = (c.k_len + kt - 1) / kt;
    a.c = c.scale * LOG2E;
    const int64_t tiles = c.B * c.key_heads * a.row_tiles;
    int64_t splits = tiles > 0 && tiles < COMPUTE_UNITS ? WANTED / tiles : 1;
    if (splits > a.steps / LEAST_STEPS) splits = a.steps / LEAST_STEPS;
    if (tiles >= COMPUTE_UNITS && tiles < MOST_TILES && c.k_len >= MANY_KEYS && (c.format != LFFN_ROWS_F32 || c.columns <= 64)) splits = MANY_WANTED / tiles;
    if (a.rows <= ROWS && c.columns <= 64 && tiles >= ONE_WAVE_LEAST && tiles < ONE_WAVE_MOST && c.k_len >= ONE_WAVE_KEYS) splits = one_wave_wanted(c.columns) / tiles;
    if (a.rows <= few_rows(c.format == LFFN_ROWS_F32)) {
        const int64_t at_once = 64 / lanes_of_a_key(c) * FEW_TOGETHER, rounds = (c.k_len + at_once - 1) / at_once;
        a.few_waves = int(rounds < 1 ? 1 : rounds < FEW_WAVES ? rounds : FEW_WAVES);
        a.steps = c.k_len;
        splits = tiles > 0 ? FEW_WANTED / (tiles * a.few_waves) : 1;
        if (splits > rounds / a.few_waves) splits = rounds / a.few_waves;
    }
    if (splits < 1) splits = 1;
    // fp32 numbers in two terms: where the products that this saves cost more than the look at keys and values
    const bool two = c.format == LFFN_ROWS_F32 && !a.few_waves && a.rows >= TWO_LEAST_ROWS &&
                     (double)tiles * TILE * (double)c.k_len * (double)c.columns >= TWO_LEAST_PRODUCTS;
    a.level_tiles = two ? int((c.k_len + LEVEL_ROWS - 1) / LEVEL_ROWS) : 0;
    a.level_by = Divisor(a.level_tiles > 0 ? (uint32_t)a.level_tiles : 1);
    a.split_steps = (a.steps + splits - 1) / splits;
    a.splits = a.split_steps ? int((a.steps + a.split_steps - 1) / a.split_steps) : 1;
    a.group = Divisor(group > 0 ? (uint32_t)group : 1), a.heads = Divisor((uint32_t)a.key_heads);
    a.tiles = Divisor(a.row_tiles > 0 ? (uint32_t)a.row_tiles : 1), a.split_by = Divisor((uint32_t)a.splits);
    if (tiles > MOST_THREADS / (a.few_waves ? 64 * a.few_waves : WG) / a.splits) return -1;
    a.units = int(tiles * a.splits);
    const int64_t batch_heads = c.B * c.key_heads;
    if (batch_heads * a.level_tiles > MOST_THREADS / WG) return -1;
    return (2 * batch_heads * a.level_tiles + (a.splits > 1 ? a.splits * batch_heads * a.rows * (a.columns + 1) : 0)) * 4;
}

template <typename F>
void join(const FwdArgs &a, hipStream_t stream) {
    const int64_t rows = int64_t(a.units / (a.splits * a.row_tiles)) * a.rows, quads = rows * (a.columns / 4);
    if (a.splits > 4) join_kernel<F, WAVES><<<dim3((unsigned)((quads + 63) / 64)), dim3(WG), 0, stream>>>(a, rows);
    else join_kernel<F, 1><<<dim3((unsigned)((quads + WG - 1) / WG)), dim3(WG), 0, stream>>>(a, rows);
}

template <typename F, typename R, int G>
int launch_few(const FwdArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned)a.units), block(64 * a.few_waves);
    if (a.rows == 1) few_rows_kernel<R, F, G, 1><<<grid, block, 0, stream>>>(a);
    else if (a.rows == 2) few_rows_kernel<R, F, G, 2><<<grid, block, 0, stream>>>(a);
    else if constexpr (few_rows(F::BYTES == 4) > 2) few_rows_kernel<R, F, G, 4><<<grid, block, 0, stream>>>(a);
    if (a.splits > 1) join<F>(a, stream);
    return lffn_launch_status();
}

template <typename F, typename R>
int launch_few(const FwdArgs &a, int lanes, hipStream_t stream) {
    switch (lanes) {
        case 4: return launch_few<F, R, 4>(a, stream);
        case 8: return launch_few<F, R, 8>(a, stream);
        case 16: return launch_few<F, R, 16>(a, stream);
        default: if constexpr (R::N == 4) return launch_few<F, R, 32>(a, stream);
    }
    return LFFN_ERR_UNSUPPORTED;          // (16-bit heads have at most 128 columns)
}

template <typename F, int DP, int KT>
int launch(const FwdArgs &a, hipStream_t stream) {
    static LdsGrant granted;
    const size_t bytes = 4 * Tile<F, DP, KT>::SIZE * 16 + BLOCK * 8;
    if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&cross_attention_kernel<F, DP, KT>), bytes, granted)) return LFFN_ERR_LAUNCH;
    cross_attention_kernel<F, DP, KT><<<dim3((unsigned)a.units), dim3(WG), bytes, stream>>>(a);
    if (a.splits > 1) join<F>(a, stream);
    return lffn_launch_status();
}

template <typename F>
int launch(const FwdArgs &a, hipStream_t stream) {
    if (a.columns <= 32) return launch<F, 32, 64>(a, stream);
    if (a.columns <= 64) return launch<F, 64, F::PLANES == 1 ? 64 : 32>(a, stream);
    return launch<F, 128, F::PLANES == 1 ? 64 : 32>(a, stream);
}

}  // namespace

extern "C" int lffn_cross_attention_workspace_bytes(const lffn_cross_attention *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    FwdArgs a{};
    *bytes = plan(*c, a);
    LFFN_REQUIRE(*bytes >= 0, LFFN_ERR_UNSUPPORTED);
    return LFFN_OK;
}

extern "C" int lffn_cross_attention_kept_bytes(const lffn_cross_attention *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    *bytes = kept_bytes(c->B * c->q_len * c->heads, c->columns, c->format == LFFN_ROWS_F32 ? 4 : 2);
    return LFFN_OK;
}

extern "C" int lffn_cross_attention_fwd(const lffn_cross_attention *c, void *out, void *kept, void *workspace, int64_t workspace_bytes,
                                        void *stream) {
    if (const int rc = lffn_internal_cross_attention_check(c)) return rc;
    FwdArgs a{};
    const int64_t bytes = plan(*c, a);
    LFFN_REQUIRE(bytes >= 0, LFFN_ERR_UNSUPPORTED);
    if (a.units == 0) return LFFN_OK;
    LFFN_REQUIRE(out && lffn_aligned16(out) && lffn_aligned16(kept), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(bytes == 0 || (workspace && lffn_aligned16(workspace) && workspace_bytes >= bytes), LFFN_ERR_BAD_ARG);
    const Kept k = kept_at(kept, c->B * c->q_len * c->heads, c->format == LFFN_ROWS_F32 ? 4 : 2);
    a.out = static_cast<char *>(out), a.lse = k.levels, a.rest = k.rest;
    // (parts first: they are read 16 bytes at a time)
    float *at = static_cast<float *>(workspace);
    const int64_t batch_heads = c->B * c->key_heads;
    if (a.splits > 1) {
        a.part = at;
        a.part_lse = at + a.splits * batch_heads * a.rows * a.columns;
        at = a.part_lse + a.splits * batch_heads * a.rows;
    }
    if (a.level_tiles) a.k_levels = at, a.v_levels = at + batch_heads * a.level_tiles;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.few_waves) {
        const int lanes = lanes_of_a_key(*c);
        if (c->format == LFFN_ROWS_F32) return launch_few<F32, F32Row>(a, lanes, s);
        return c->format == LFFN_ROWS_BF16 ? launch_few<BF16, BF16Row>(a, lanes, s) : launch_few<F16, F16Row>(a, lanes, s);
    }
    if (a.level_tiles) {
        const dim3 grid((unsigned)(batch_heads * a.level_tiles)), block(WG);
        const int lanes = level_lanes(a.columns);
        if (lanes == 4) levels_kernel<4><<<grid, block, 0, s>>>(a);
        else if (lanes == 8) levels_kernel<8><<<grid, block, 0, s>>>(a);
        else levels_kernel<16><<<grid, block, 0, s>>>(a);
        return launch<F32Two>(a, s);
    }
    if (c->format == LFFN_ROWS_F32) return launch<F32>(a, s);
    return c->format == LFFN_ROWS_BF16 ? launch<BF16>(a, s) : launch<F16>(a, s);
}
