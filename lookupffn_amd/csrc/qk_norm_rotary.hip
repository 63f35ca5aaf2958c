// Norms of queries and keys for each head with the rotation to their positions in the same pass, and its backward.
//
//   y = x r w,  r = 1 / sqrt(mean(x^2) + eps);  of a pair (a, b) of columns and its angle t:  (a cos t - b sin t, b cos t + a sin t).
// Backward: h = the gradient turned back by t;  grad w = sum h x r;  grad x = r (h w - x r mean(h w x r)).  r is formed again from x: to
// keep it would take a launch's write and read for what two instructions a number give.
//
// Bound by memory: x in and y out, or x and the gradient in and x's gradient out, once each.  A row is held by a group of lanes, each with two 16-byte
// vectors whose columns are each other's partners, so that the rotation stays in the lane; sine and cosine of a lane's columns (fp32: two
// to four times a 16-bit row's bytes) are read once for several heads of a token.  Queries and keys are one launch: the workgroups
// of one follow those of the other.
// 16384 tokens of 12 + 12 heads of 64, fp32: 35.5 us for 201 MB; 2 x 32768 tokens of 8 heads of 64, half: forward 32 us for 134 MB, backward 44 for 201 and
// 4 for the weights' partial sums (a copy moves 5.1 TB/s).
#include "rows16.h"

namespace {

constexpr int WG = 256;
constexpr int BWD_WORKGROUPS = 1024;      // of a tensor at most: each leaves a row of partial sums of the weight's gradient

struct Tensor {
    const void *x, *g;                    // x by strides; g and y: [tokens, heads, columns]
    void *y;
    const float *w;
    float *parts;                         // [workgroups, columns] or null
    const void *positions;
    int64_t tokens, sb, st, sh, position_stride;
    int len, heads, chunks;               // chunks of HC heads
    int workgroups;
};

struct Args {
    Tensor t[2];
    const float *table;
    int table_rows, columns, rotary;
    bool wide;                            // positions of 64 bits
    float eps, inv_columns;
};

// What a lane holds of a row: vectors a and b (in units of 16 bytes), partners where the row is rotated by halves.
struct Slot {
    int a, b;
    bool has_a, has_b, turned;
};
template <typename R>
__device__ __forceinline__ Slot slot_of(int s, int columns, int rotary) {
    const int vectors = columns / R::N, turned = rotary / R::N, half = turned / 2, rest = 2 * (s - half);
    Slot o;
    o.a = s < half ? s : turned + rest;
    o.b = s < half ? s + half : turned + rest + 1;
    o.has_a = o.a < vectors;
    o.has_b = o.b < vectors;
    o.turned = s < half;
    return o;
}

// The angles of a lane's columns: by halves cos and sin of the N columns of vector a (and b); side by side of the N / 2 pairs of a, then of b.
template <typename R, bool INTERLEAVED>
__device__ __forceinline__ void load_angles(const Args &a, const Tensor &t, int64_t token, const Slot &s, float (&cos)[R::N], float (&sin)[R::N]) {
    const int half = a.rotary / 2;
    int64_t p = token % t.len;
    if (t.positions) {
        const int64_t at = token / t.len * t.position_stride + p;
        p = a.wide ? reinterpret_cast<const int64_t *>(t.positions)[at] : reinterpret_cast<const int32_t *>(t.positions)[at];
    }
    p = p < 0 ? 0 : p >= a.table_rows ? a.table_rows - 1 : p;
    const float *const row = a.table + p * a.rotary;
    auto read = [&](const float *from, int n, float *to) {
        for (int i = 0; i < n; i += (R::N == 8 || !INTERLEAVED) ? 4 : 2) {
            if (R::N == 8 || !INTERLEAVED) {
                const float4 v = *reinterpret_cast<const float4 *>(from + i);
                to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2 *>(from + i);
                to[i] = v.x, to[i + 1] = v.y;
            }
        }
    };
    if (INTERLEAVED) {
        constexpr int P = R::N / 2;
        read(row + s.a * P, P, cos), read(row + s.b * P, P, cos + P);
        read(row + half + s.a * P, P, sin), read(row + half + s.b * P, P, sin + P);
    } else {
        read(row + s.a * R::N, R::N, cos);
        read(row + half + s.a * R::N, R::N, sin);
    }
}

// (a, b) turned by the angles; back: by their opposites
template <int N, bool INTERLEAVED>
__device__ __forceinline__ void turn(float (&a)[N], float (&b)[N], const float (&cos)[N], const float (&sin)[N], float sign) {
    if (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float s0 = sign * sin[i], s1 = sign * sin[N / 2 + i];
            const float u = a[2 * i], v = a[2 * i + 1], x = b[2 * i], y = b[2 * i + 1];
            a[2 * i] = u * cos[i] - v * s0, a[2 * i + 1] = v * cos[i] + u * s0;
            b[2 * i] = x * cos[N / 2 + i] - y * s1, b[2 * i + 1] = y * cos[N / 2 + i] + x * s1;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float s = sign * sin[i], u = a[i], v = b[i];
            a[i] = u * cos[i] - v * s, b[i] = v * cos[i] + u * s;
        }
    }
}

template <int N>
__device__ __forceinline__ void load_weight(const float *w, int vector, bool has, float (&to)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 v = w && has ? *reinterpret_cast<const float4 *>(w + vector * N + i) : make_float4(1.f, 1.f, 1.f, 1.f);
        to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
    }
}

// LPR lanes a row, HC heads a lane group.
template <typename R, int LPR, int HC, bool INTERLEAVED, bool BACKWARD>
__global__ __launch_bounds__(WG) void norm_rotary_kernel(Args a) {
    constexpr int N = R::N, GROUPS = WG / LPR;
    const bool second = (int)blockIdx.x >= a.t[0].workgroups;
    const Tensor &t = a.t[second];
    const int wg = blockIdx.x - (second ? a.t[0].workgroups : 0), lane = threadIdx.x % LPR;
    const Slot s = slot_of<R>(lane, a.columns, a.rotary);
    const bool turned = s.turned;
    float wa[N], wb[N], ga[N] = {}, gb[N] = {};
    load_weight<N>(t.w, s.a, s.has_a, wa);
    load_weight<N>(t.w, s.b, s.has_b, wb);
    const int64_t units = t.tokens * t.chunks;
    for (int64_t unit = int64_t(wg) * GROUPS + threadIdx.x / LPR; unit < units; unit += int64_t(t.workgroups) * GROUPS) {
        const int64_t token = unit / t.chunks;
        const int first = int(unit - token * t.chunks) * HC;
        const char *const x = reinterpret_cast<const char *>(t.x) + (token / t.len * t.sb + token % t.len * t.st) * R::BYTES;
        const int64_t out = (token * t.heads + first) * a.columns * R::BYTES;
        uint4 xa[HC], xb[HC], da[HC], db[HC];
#pragma unroll
        for (int h = 0; h < HC; ++h) {
            const bool live = first + h < t.heads;
            const char *const row = x + (first + h) * t.sh * R::BYTES;
            xa[h] = xb[h] = da[h] = db[h] = make_uint4(0, 0, 0, 0);
            if (live && s.has_a) xa[h] = reinterpret_cast<const uint4 *>(row)[s.a];
            if (live && s.has_b) xb[h] = reinterpret_cast<const uint4 *>(row)[s.b];
            if (BACKWARD) {
                const uint4 *const g = reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(t.g) + out + h * a.columns * R::BYTES);
                if (live && s.has_a) da[h] = g[s.a];
                if (live && s.has_b) db[h] = g[s.b];
            }
        }
        float cos[N], sin[N];
        if (turned) load_angles<R, INTERLEAVED>(a, t, token, s, cos, sin);
#pragma unroll
        for (int h = 0; h < HC; ++h) {
            const bool live = first + h < t.heads;
            float u[N], v[N], squares = 0.f;
            R::unpack(xa[h], u);
            R::unpack(xb[h], v);
#pragma unroll
            for (int i = 0; i < N; ++i) squares = fmaf(u[i], u[i], fmaf(v[i], v[i], squares));
            const float r = 1.f / sqrtf(fmaf(lane_group_sum<LPR>(squares), a.inv_columns, a.eps));
            if (BACKWARD) {
                float hu[N], hv[N], dot = 0.f;
                R::unpack(da[h], hu);
                R::unpack(db[h], hv);
                if (turned) turn<N, INTERLEAVED>(hu, hv, cos, sin, -1.f);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    u[i] *= r, v[i] *= r;
                    if (live) ga[i] = fmaf(hu[i], u[i], ga[i]), gb[i] = fmaf(hv[i], v[i], gb[i]);
                    hu[i] *= wa[i], hv[i] *= wb[i];
                    dot = fmaf(hu[i], u[i], fmaf(hv[i], v[i], dot));
                }
                const float mean = lane_group_sum<LPR>(dot) * a.inv_columns;
#pragma unroll
                for (int i = 0; i < N; ++i) u[i] = r * fmaf(-mean, u[i], hu[i]), v[i] = r * fmaf(-mean, v[i], hv[i]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) u[i] *= r * wa[i], v[i] *= r * wb[i];
                if (turned) turn<N, INTERLEAVED>(u, v, cos, sin, 1.f);
            }
            uint4 *const y = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(t.y) + out + h * a.columns * R::BYTES);
            if (live && s.has_a) y[s.a] = R::pack(u);
            if (live && s.has_b) y[s.b] = R::pack(v);
        }
    }
    if (BACKWARD && t.parts) {
        // the workgroup's sum of its lane groups', in a fixed order
        __shared__ float4 red[WG / 64][LPR][2 * N / 4];
        auto over_groups = [](float v) {
            if constexpr (LPR <= 1) v += lane_xor<1>(v);
            if constexpr (LPR <= 2) v += lane_xor<2>(v);
            if constexpr (LPR <= 4) v += lane_xor<4>(v);
            if constexpr (LPR <= 8) v += lane_xor<8>(v);
            if constexpr (LPR <= 16) v += lane_xor<16>(v);
            if constexpr (LPR <= 32) v += lane_xor<32>(v);
            return v;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) ga[i] = over_groups(ga[i]), gb[i] = over_groups(gb[i]);
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 < LPR) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                red[wave][lane][i] = make_float4(ga[4 * i], ga[4 * i + 1], ga[4 * i + 2], ga[4 * i + 3]);
                red[wave][lane][N / 4 + i] = make_float4(gb[4 * i], gb[4 * i + 1], gb[4 * i + 2], gb[4 * i + 3]);
            }
        }
        __syncthreads();
        for (int n = threadIdx.x; n < LPR * (2 * N / 4); n += WG) {
            const int of = n / (2 * N / 4), i = n % (2 * N / 4);
            const Slot o = slot_of<R>(of, a.columns, a.rotary);
            const bool in_b = i >= N / 4;
            float4 sum = red[0][of][i];
#pragma unroll
            for (int w = 1; w < WG / 64; ++w) {
                const float4 v = red[w][of][i];
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            if (in_b ? o.has_b : o.has_a)
                *reinterpret_cast<float4 *>(t.parts + int64_t(wg) * a.columns + (in_b ? o.b : o.a) * N + 4 * (i % (N / 4))) = sum;
        }
    }
}

int lanes_of(const lffn_qk_norm_rotary &a) {
    const int n = a.format == LFFN_ROWS_F32 ? 4 : 8, vectors = int(a.columns) / n, half = int(a.rotary) / n / 2;
    const int slots = half + (vectors - 2 * half + 1) / 2;
    return 1 << lffn_log2(slots);
}

// Heads a lane group takes one after the other, their loads in flight together: as many as leave wavefronts enough.
int heads_of(const lffn_qk_norm_rotary &a, int lpr) {
    const int64_t rows = a.B * (a.q_len * a.q_heads + (a.k ? a.k_len * a.k_heads : 0)), waves = rows * lpr / 64;
    return waves >= 4 * 8192 ? 4 : waves >= 2 * 4096 ? 2 : 1;
}

int check(const lffn_qk_norm_rotary *a) {
    LFFN_REQUIRE(a, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->B >= 0 && a->q_len >= 0 && a->k_len >= 0 && a->q_heads >= 0 && a->k_heads >= 0 && a->columns >= 1 && a->rotary >= 0,
                 LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->format >= 0 && a->format <= 2, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->columns % 8 == 0 && a->columns <= 256 && a->rotary % 16 == 0, LFFN_ERR_UNSUPPORTED);
    LFFN_REQUIRE(a->rotary <= a->columns, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->eps >= 0.f, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->rotary == 0 || (a->table && lffn_aligned16(a->table) && a->table_rows >= 1), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->table_rows <= INT32_MAX, LFFN_ERR_UNSUPPORTED);
    const int64_t most = int64_t(1) << 31;
    LFFN_REQUIRE(a->q_len < most && a->k_len < most && a->q_heads <= 65536 && a->k_heads <= 65536 && a->B < most, LFFN_ERR_UNSUPPORTED);
    const int64_t size = a->format == LFFN_ROWS_F32 ? 4 : 2;
    for (int i = 0; i < 2; ++i) {
        const void *x = i ? a->k : a->q;
        const int64_t len = i ? a->k_len : a->q_len, heads = i ? a->k_heads : a->q_heads;
        const int64_t *s = i ? a->k_strides : a->q_strides;
        if (i && !x) continue;
        const bool empty = a->B == 0 || len == 0 || heads == 0;
        LFFN_REQUIRE(x || empty, LFFN_ERR_BAD_ARG);
        LFFN_REQUIRE(lffn_aligned16(x) && lffn_aligned16(i ? a->k_weight : a->q_weight), LFFN_ERR_BAD_ARG);
        for (int d = 0; d < 3; ++d) LFFN_REQUIRE(s[d] >= 0 && s[d] * size % 16 == 0, LFFN_ERR_BAD_ARG);
        LFFN_REQUIRE(empty || a->B <= (int64_t(1) << 40) / len / heads, LFFN_ERR_UNSUPPORTED);
    }
    return LFFN_OK;
}

// Fills the arguments in; the number of workgroups, or -1.
int64_t plan(const lffn_qk_norm_rotary &c, Args &a, int lpr, int hc, bool backward) {
    a.table = c.table;
    a.table_rows = (int)c.table_rows;
    a.columns = (int)c.columns;
    a.rotary = (int)c.rotary;
    a.wide = c.positions_64 != 0;
    a.eps = c.eps;
    a.inv_columns = 1.f / (float)c.columns;
    int64_t total = 0;
    for (int i = 0; i < 2; ++i) {
        Tensor &t = a.t[i];
        const int64_t *const s = i ? c.k_strides : c.q_strides;
        t.x = i ? c.k : c.q;
        t.w = i ? c.k_weight : c.q_weight;
        t.positions = i ? c.k_positions : c.q_positions;
        t.position_stride = i ? c.k_positions_stride : c.q_positions_stride;
        t.len = int(i ? c.k_len : c.q_len);
        t.heads = int(i ? c.k_heads : c.q_heads);
        t.tokens = t.x ? c.B * t.len : 0;
        t.sb = s[0], t.st = s[1], t.sh = s[2];
        t.chunks = (t.heads + hc - 1) / hc;
        const int64_t groups = WG / lpr, want = (t.tokens * t.chunks + groups - 1) / groups;
        if (!backward && total + want > UINT32_MAX / WG) return -1;           // (threads of a launch)
        t.workgroups = int(backward && want > BWD_WORKGROUPS ? BWD_WORKGROUPS : want);
        total += t.workgroups;
    }
    return total;
}

template <typename R, int LPR, bool INTERLEAVED, bool BACKWARD>
void launch(const Args &a, int hc, int64_t workgroups, hipStream_t stream) {
    const dim3 grid((unsigned)workgroups), block(WG);
    if (hc == 4) norm_rotary_kernel<R, LPR, 4, INTERLEAVED, BACKWARD><<<grid, block, 0, stream>>>(a);
    else if (hc == 2) norm_rotary_kernel<R, LPR, 2, INTERLEAVED, BACKWARD><<<grid, block, 0, stream>>>(a);
    else norm_rotary_kernel<R, LPR, 1, INTERLEAVED, BACKWARD><<<grid, block, 0, stream>>>(a);
}

template <typename R, bool BACKWARD>
void launch(const Args &a, int lpr, int hc, bool interleaved, int64_t workgroups, hipStream_t stream) {
    auto by_lanes = [&](auto pairs) {
        constexpr bool I = decltype(pairs)::value;
        switch (lpr) {
            case 1: return launch<R, 1, I, BACKWARD>(a, hc, workgroups, stream);
            case 2: return launch<R, 2, I, BACKWARD>(a, hc, workgroups, stream);
            case 4: return launch<R, 4, I, BACKWARD>(a, hc, workgroups, stream);
            case 8: return launch<R, 8, I, BACKWARD>(a, hc, workgroups, stream);
            case 16: return launch<R, 16, I, BACKWARD>(a, hc, workgroups, stream);
            default: return launch<R, 32, I, BACKWARD>(a, hc, workgroups, stream);
        }
    };
    if (interleaved) by_lanes(std::true_type{});
    else by_lanes(std::false_type{});
}

template <bool BACKWARD>
int launch_rows(const lffn_qk_norm_rotary &c, const Args &a, int lpr, int hc, int64_t workgroups, void *stream) {
    if (workgroups == 0) return LFFN_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool interleaved = c.interleaved != 0;
    if (c.format == LFFN_ROWS_F32) launch<F32Row, BACKWARD>(a, lpr, hc, interleaved, workgroups, s);
    else if (c.format == LFFN_ROWS_BF16) launch<BF16Row, BACKWARD>(a, lpr, hc, interleaved, workgroups, s);
    else launch<F16Row, BACKWARD>(a, lpr, hc, interleaved, workgroups, s);
    return lffn_launch_status();
}

}  // namespace

extern "C" int lffn_qk_norm_rotary_fwd(const lffn_qk_norm_rotary *c, void *q_out, void *k_out, void *stream) {
    if (const int rc = check(c)) return rc;
    Args a{};
    const int lpr = lanes_of(*c), hc = heads_of(*c, lpr);
    const int64_t workgroups = plan(*c, a, lpr, hc, false);
    LFFN_REQUIRE(workgroups >= 0, LFFN_ERR_UNSUPPORTED);
    a.t[0].y = q_out, a.t[1].y = k_out;
    for (const Tensor &t : a.t) LFFN_REQUIRE(t.workgroups == 0 || (t.y && lffn_aligned16(t.y)), LFFN_ERR_BAD_ARG);
    return launch_rows<false>(*c, a, lpr, hc, workgroups, stream);
}

extern "C" int lffn_qk_norm_rotary_bwd_workspace_bytes(const lffn_qk_norm_rotary *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    if (const int rc = check(c)) return rc;
    Args a{};
    const int lpr = lanes_of(*c);
    *bytes = plan(*c, a, lpr, heads_of(*c, lpr), true) * c->columns * 4;
    return LFFN_OK;
}

extern "C" int lffn_qk_norm_rotary_bwd(const lffn_qk_norm_rotary *c, const void *g_q, const void *g_k, void *grad_q, void *grad_k,
                                       float *grad_q_weight, float *grad_k_weight, void *workspace, int64_t workspace_bytes, void *stream) {
    if (const int rc = check(c)) return rc;
    Args a{};
    const int lpr = lanes_of(*c), hc = heads_of(*c, lpr);
    const int64_t workgroups = plan(*c, a, lpr, hc, true);
    float *const grads[2] = {grad_q_weight, grad_k_weight};
    LFFN_REQUIRE(workgroups == 0 || (!grad_q_weight && !grad_k_weight) ||
                     (workspace && lffn_aligned16(workspace) && workspace_bytes >= workgroups * c->columns * 4), LFFN_ERR_BAD_ARG);
    a.t[0].g = g_q, a.t[0].y = grad_q, a.t[1].g = g_k, a.t[1].y = grad_k;
    lffn_sum sums[2] = {};
    int count = 0;
    float *parts = static_cast<float *>(workspace);
    for (int i = 0; i < 2; ++i) {
        Tensor &t = a.t[i];
        LFFN_REQUIRE(lffn_aligned16(grads[i]), LFFN_ERR_BAD_ARG);
        if (grads[i]) {
            if (t.workgroups == 0) {          // a sum of nothing: one row of zeros would have to be cleared, so it is refused
                LFFN_REQUIRE(false, LFFN_ERR_BAD_ARG);
            }
            t.parts = parts;
            sums[count++] = {parts, grads[i], c->columns, t.workgroups};
            parts += int64_t(t.workgroups) * c->columns;
        }
        LFFN_REQUIRE(t.workgroups == 0 || (t.g && t.y && lffn_aligned16(t.g) && lffn_aligned16(t.y)), LFFN_ERR_BAD_ARG);
    }
    const int rc = launch_rows<true>(*c, a, lpr, hc, workgroups, stream);
    return rc != LFFN_OK || count == 0 ? rc : lffn_sum_many_f32(sums, count, stream);
}
