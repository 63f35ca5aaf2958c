// Layer norm over rows of any width, in fp32, bfloat16 or half, and its backward:
//
//   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps),  z = (x - m) r,  y = z w + b
//   g_x = r (g w - mean(g w) - z mean(g w z)),   g_w = sum over the rows of g z,   g_b = sum of g
//
// Bound by memory: a row is read once and held in the registers of T threads (16 or 64 lanes, or a workgroup), V 16-byte vectors each, mean and squares in two passes over
// registers; wider rows are read again, from cache.  Widths or addresses that 16 bytes do not divide are taken number by number.  The backward's threads keep their
// columns' sums over the rows they take; workgroups' sums are added by a second launch in a fixed order.
#include "rows16.h"

namespace {

constexpr int WG = 256;
constexpr int PARTS = 1024;              // workgroups of a backward, at most: each leaves two rows of sums
constexpr int64_t PARTS_NUMBERS = int64_t(1) << 22;      // columns times parts, at most
constexpr int WIDE_COLUMNS = 1024;       // columns of a workgroup that adds up a wide backward's columns

struct Args {
    const void *x, *w, *b, *g;
    void *y, *gx;
    float2 *stats;                       // mean, 1 / sigma
    float *parts;                        // [workgroups][2][columns]
    int64_t rows, stride;
    int columns, w32;                    // w32: w and b are fp32
    float eps, inv_columns;
};

template <typename R>
__device__ __forceinline__ void load(const void *p, int64_t at, float (&v)[R::N]) {
    R::unpack(*reinterpret_cast<const typename R::raw_t *>(static_cast<const char *>(p) + at * R::BYTES), v);
}
template <typename R>
__device__ __forceinline__ void store(void *p, int64_t at, const float (&v)[R::N]) {
    *reinterpret_cast<typename R::raw_t *>(static_cast<char *>(p) + at * R::BYTES) = R::pack(v);
}
// of a weight: `otherwise` where there is none
template <typename R>
__device__ __forceinline__ void load_weight(const void *p, int w32, int at, float otherwise, float (&v)[R::N]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < R::N; ++i) v[i] = otherwise;
    } else if (w32) {
#pragma unroll
        for (int i = 0; i < R::N; ++i) v[i] = static_cast<const float *>(p)[at + i];
    } else
        load<R>(p, at, v);
}

// Sum over a row's T threads.
template <int T>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
    for (int m = (T < 64 ? T : 64) / 2; m > 0; m /= 2) v += __shfl_xor(v, m);
    if constexpr (T > 64) {
        __syncthreads();                 // (what was read last time)
        if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < T / 64; ++i) v += red[i];
    }
    return v;
}

template <typename R, int T, int V>
__global__ __launch_bounds__(WG) void forward_kernel(Args a) {
    __shared__ float red[WG / 64];
    constexpr int N = R::N;
    const int in = threadIdx.x % T;
    const int64_t row = int64_t(blockIdx.x) * (WG / T) + threadIdx.x / T;
    const bool live = row < a.rows;
    const int64_t at = min(row, a.rows - 1) * a.stride;
    float x[V][N], w[V][N], b[V][N];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = min((j * T + in) * N, a.columns - N);
        load<R>(a.x, at + c, x[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = min((j * T + in) * N, a.columns - N);
        load_weight<R>(a.w, a.w32, c, 1.f, w[j]);
        load_weight<R>(a.b, a.w32, c, 0.f, b[j]);
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) sum += (j * T + in) * N < a.columns ? x[j][i] : 0.f;
    const float mean = row_sum<T>(sum, red) * a.inv_columns;
    float squares = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[j][i] -= mean;
            squares += (j * T + in) * N < a.columns ? x[j][i] * x[j][i] : 0.f;
        }
    const float r = 1.f / sqrtf(row_sum<T>(squares, red) * a.inv_columns + a.eps);
    if (!live) return;
    if (a.stats && in == 0) a.stats[row] = make_float2(mean, r);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (j * T + in) * N;
        if (c >= a.columns) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) x[j][i] = fmaf(x[j][i] * r, w[j][i], b[j][i]);
        store<R>(a.y, row * a.columns + c, x[j]);
    }
}

// Rows too wide for the registers: a workgroup reads them three times.
template <typename R>
__global__ __launch_bounds__(WG) void wide_forward_kernel(Args a) {
    __shared__ float red[WG / 64];
    constexpr int N = R::N;
    const int64_t row = blockIdx.x, at = row * a.stride;
    float sum = 0.f, squares = 0.f, x[N], w[N], b[N];
    for (int c = threadIdx.x * N; c < a.columns; c += WG * N) {
        load<R>(a.x, at + c, x);
#pragma unroll
        for (int i = 0; i < N; ++i) sum += x[i];
    }
    const float mean = row_sum<WG>(sum, red) * a.inv_columns;
    for (int c = threadIdx.x * N; c < a.columns; c += WG * N) {
        load<R>(a.x, at + c, x);
#pragma unroll
        for (int i = 0; i < N; ++i) squares += (x[i] - mean) * (x[i] - mean);
    }
    const float r = 1.f / sqrtf(row_sum<WG>(squares, red) * a.inv_columns + a.eps);
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mean, r);
    for (int c = threadIdx.x * N; c < a.columns; c += WG * N) {
        load<R>(a.x, at + c, x);
        load_weight<R>(a.w, a.w32, c, 1.f, w);
        load_weight<R>(a.b, a.w32, c, 0.f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf((x[i] - mean) * r, w[i], b[i]);
        store<R>(a.y, row * a.columns + c, x);
    }
}

template <typename R, int T, int V>
__global__ __launch_bounds__(WG) void backward_kernel(Args a) {
    __shared__ float red[WG / 64];
    __shared__ float sums[T < WG ? 2 * WG / T * T * R::N : 1];       // one of a thread's vectors at a time
    constexpr int N = R::N, ROWS = WG / T;
    const int in = threadIdx.x % T;
    float w[V][N], gw[V][N], gb[V][N];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        load_weight<R>(a.w, a.w32, min((j * T + in) * N, a.columns - N), 1.f, w[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) gw[j][i] = gb[j][i] = 0.f;
    }
    const int64_t step = int64_t(gridDim.x) * ROWS;
    // (all threads of a workgroup go round as often: rows behind the last are read as the last)
    for (int64_t first = int64_t(blockIdx.x) * ROWS; first < a.rows; first += step) {
        const int64_t own = first + threadIdx.x / T, row = min(own, a.rows - 1);
        const bool live = own < a.rows;
        float x[V][N], g[V][N];
        const float2 of = a.stats[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = min((j * T + in) * N, a.columns - N);
            load<R>(a.x, row * a.stride + c, x[j]);
            load<R>(a.g, row * a.columns + c, g[j]);
        }
        float first_sum = 0.f, second_sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool there = live && (j * T + in) * N < a.columns;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[j][i] = (x[j][i] - of.x) * of.y;
                if (there) {
                    gw[j][i] += g[j][i] * x[j][i];
                    gb[j][i] += g[j][i];
                    g[j][i] *= w[j][i];
                    first_sum += g[j][i];
                    second_sum += g[j][i] * x[j][i];
                }
            }
        }
        const float s1 = row_sum<T>(first_sum, red) * a.inv_columns, s2 = row_sum<T>(second_sum, red) * a.inv_columns;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * T + in) * N;
            if (!live || c >= a.columns || !a.gx) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) x[j][i] = of.y * (g[j][i] - s1 - x[j][i] * s2);
            store<R>(a.gx, row * a.columns + c, x[j]);
        }
    }
    if (!a.parts) return;
    float *const out = a.parts + int64_t(blockIdx.x) * 2 * a.columns;
    if constexpr (T == WG) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * T + in) * N;
            if (c >= a.columns) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) out[c + i] = gw[j][i], out[a.columns + c + i] = gb[j][i];
        }
    } else {
        float *const second = sums + ROWS * T * N;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sums[threadIdx.x * N + i] = gw[j][i];
                second[threadIdx.x * N + i] = gb[j][i];
            }
            __syncthreads();
            for (int k = threadIdx.x; k < T * N; k += WG) {
                float sw = 0.f, sb = 0.f;
#pragma unroll
                for (int o = 0; o < ROWS; ++o) sw += sums[o * T * N + k], sb += second[o * T * N + k];
                const int c = j * T * N + k;
                if (c < a.columns) out[c] = sw, out[a.columns + c] = sb;
            }
        }
    }
}

// Wide rows: the gradient of x, a workgroup a row.
template <typename R>
__global__ __launch_bounds__(WG) void wide_backward_kernel(Args a) {
    __shared__ float red[WG / 64];
    constexpr int N = R::N;
    const int64_t row = blockIdx.x;
    const float2 of = a.stats[row];
    float s1 = 0.f, s2 = 0.f, x[N], g[N], w[N];
    for (int c = threadIdx.x * N; c < a.columns; c += WG * N) {
        load<R>(a.x, row * a.stride + c, x);
        load<R>(a.g, row * a.columns + c, g);
        load_weight<R>(a.w, a.w32, c, 1.f, w);
#pragma unroll
        for (int i = 0; i < N; ++i) s1 += g[i] * w[i], s2 += g[i] * w[i] * ((x[i] - of.x) * of.y);
    }
    s1 = row_sum<WG>(s1, red) * a.inv_columns;
    s2 = row_sum<WG>(s2, red) * a.inv_columns;
    for (int c = threadIdx.x * N; c < a.columns; c += WG * N) {
        load<R>(a.x, row * a.stride + c, x);
        load<R>(a.g, row * a.columns + c, g);
        load_weight<R>(a.w, a.w32, c, 1.f, w);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = of.y * (g[i] * w[i] - s1 - (x[i] - of.x) * of.y * s2);
        store<R>(a.gx, row * a.columns + c, x);
    }
}

// Wide rows: the sums of blockIdx.x's columns over every gridDim.y-th row.
template <typename R>
__global__ __launch_bounds__(WG) void wide_sums_kernel(Args a) {
    constexpr int N = R::N, PER = WIDE_COLUMNS / N / WG > 0 ? WIDE_COLUMNS / N / WG : 1;
    float gw[PER][N] = {}, gb[PER][N] = {}, x[N], g[N];
    const int c0 = blockIdx.x * PER * WG * N + threadIdx.x * N;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float2 of = a.stats[row];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int c = min(c0 + k * WG * N, a.columns - N);
            load<R>(a.x, row * a.stride + c, x);
            load<R>(a.g, row * a.columns + c, g);
#pragma unroll
            for (int i = 0; i < N; ++i) gw[k][i] += g[i] * ((x[i] - of.x) * of.y), gb[k][i] += g[i];
        }
    }
    float *const out = a.parts + int64_t(blockIdx.y) * 2 * a.columns;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int c = c0 + k * WG * N;
        if (c >= a.columns) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) out[c + i] = gw[k][i], out[a.columns + c + i] = gb[k][i];
    }
}

struct SumArgs {
    const float *parts;
    void *gw, *gb;
    int num, columns, format;            // of the results
};

// The workgroups' sums of 16 columns of both gradients, 16 threads each (blockIdx.y: weight, bias).
__global__ __launch_bounds__(WG) void sum_kernel(SumArgs a) {
    __shared__ float red[16][17];
    const int in = threadIdx.x % 16, slice = threadIdx.x / 16, c = blockIdx.x * 16 + in;
    void *const to = blockIdx.y ? a.gb : a.gw;
    if (!to) return;
    float sum = 0.f;
    if (c < a.columns) {
        const float *from = a.parts + blockIdx.y * a.columns + c;
#pragma unroll 8
        for (int p = slice; p < a.num; p += 16) sum += from[int64_t(p) * 2 * a.columns];
    }
    red[slice][in] = sum;
    __syncthreads();
    if (slice == 0 && c < a.columns) {
#pragma unroll
        for (int i = 1; i < 16; ++i) sum += red[i][in];
        if (a.format == LFFN_ROWS_F32) static_cast<float *>(to)[c] = sum;
        else if (a.format == LFFN_ROWS_BF16) static_cast<__bf16 *>(to)[c] = (__bf16)sum;
        else static_cast<_Float16 *>(to)[c] = (_Float16)sum;
    }
}

__global__ void clear_kernel(SumArgs a) {
    const int c = blockIdx.x * WG + threadIdx.x;
    if (c >= a.columns) return;
    for (void *to : {a.gw, a.gb}) {
        if (!to) continue;
        if (a.format == LFFN_ROWS_F32) static_cast<float *>(to)[c] = 0.f;
        else static_cast<uint16_t *>(to)[c] = 0;
    }
}

// Threads a row and vectors a thread; 0: a workgroup that reads the row again.
struct Plan {
    int T, V;
};
Plan plan(int64_t vectors) {
    if (vectors <= 16) return {16, 1};
    if (vectors <= 64) return {64, 1};
    if (vectors <= 128) return {64, 2};
    if (vectors <= 192) return {64, 3};
    if (vectors <= 256) return {64, 4};
    if (vectors <= 512) return {WG, 2};
    if (vectors <= 1024) return {WG, 4};
    return {0, 0};
}

template <typename R, bool BACKWARD>
void launch(const Args &a, int parts, hipStream_t st) {
    const Plan p = plan((a.columns + R::N - 1) / R::N);
    const int64_t rows = p.T ? WG / p.T : 1;
    const dim3 grid(unsigned(BACKWARD && p.T ? parts : (a.rows + rows - 1) / rows)), block(WG);
#define LFFN_ROWS_CASE(TT, VV)                                                         \
    if (p.T == TT && p.V == VV) {                                                      \
        if constexpr (BACKWARD) backward_kernel<R, TT, VV><<<grid, block, 0, st>>>(a); \
        else forward_kernel<R, TT, VV><<<grid, block, 0, st>>>(a);                     \
        return;                                                                        \
    }
    LFFN_ROWS_CASE(16, 1)
    LFFN_ROWS_CASE(64, 1)
    LFFN_ROWS_CASE(64, 2)
    LFFN_ROWS_CASE(64, 3)
    LFFN_ROWS_CASE(64, 4)
    LFFN_ROWS_CASE(WG, 2)
    LFFN_ROWS_CASE(WG, 4)
#undef LFFN_ROWS_CASE
    if constexpr (BACKWARD) {
        if (a.gx) wide_backward_kernel<R><<<grid, block, 0, st>>>(a);
        constexpr int per = (WIDE_COLUMNS / R::N / WG > 0 ? WIDE_COLUMNS / R::N / WG : 1) * WG * R::N;
        if (a.parts) wide_sums_kernel<R><<<dim3(unsigned((a.columns + per - 1) / per), unsigned(parts)), block, 0, st>>>(a);
    } else
        wide_forward_kernel<R><<<grid, block, 0, st>>>(a);
}

bool by_vectors(const lffn_layer_norm_rows &a, const void *one, const void *two) {
    const int64_t size = a.format == LFFN_ROWS_F32 ? 4 : 2;
    return a.columns * size % 16 == 0 && a.stride * size % 16 == 0 && lffn_aligned16(a.x) && lffn_aligned16(one) && lffn_aligned16(two) &&
           (a.weight_f32 || (lffn_aligned16(a.weight) && lffn_aligned16(a.bias)));
}

template <bool BACKWARD>
void launch(const lffn_layer_norm_rows &c, const Args &a, int parts, bool vectors, hipStream_t st) {
    if (vectors) {
        if (c.format == LFFN_ROWS_F32) launch<Vectors<F32Row>, BACKWARD>(a, parts, st);
        else if (c.format == LFFN_ROWS_BF16) launch<Vectors<BF16Row>, BACKWARD>(a, parts, st);
        else launch<Vectors<F16Row>, BACKWARD>(a, parts, st);
    } else {
        if (c.format == LFFN_ROWS_F32) launch<Single<float, 4>, BACKWARD>(a, parts, st);
        else if (c.format == LFFN_ROWS_BF16) launch<Single<__bf16, 2>, BACKWARD>(a, parts, st);
        else launch<Single<_Float16, 2>, BACKWARD>(a, parts, st);
    }
}

int check(const lffn_layer_norm_rows *a) {
    LFFN_REQUIRE(a, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->format >= 0 && a->format <= 2 && a->rows >= 0 && a->columns >= 1 && a->stride >= 0 && a->eps >= 0.f, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->rows == 0 || a->x, LFFN_ERR_BAD_ARG);
    // (threads of a launch, one workgroup a row at most)
    LFFN_REQUIRE(a->rows < (int64_t(1) << 24) && a->columns <= (1 << 24), LFFN_ERR_UNSUPPORTED);
    return LFFN_OK;
}

Args arguments(const lffn_layer_norm_rows &c) {
    Args a{};
    a.x = c.x, a.w = c.weight, a.b = c.bias;
    a.rows = c.rows, a.stride = c.stride, a.columns = (int)c.columns, a.w32 = c.weight_f32;
    a.eps = c.eps, a.inv_columns = 1.f / (float)c.columns;
    return a;
}

// Of very wide rows fewer: a part's sums are as long as a row, and the columns by themselves give workgroups enough.  (BF16 512 x 65536, backward: 313 us with 512 parts, 113 with 64)
int parts_of(const lffn_layer_norm_rows &a) {
    const int64_t fewer = PARTS_NUMBERS / a.columns, most = fewer > PARTS ? PARTS : fewer < 32 ? 32 : fewer;
    return int(a.rows < most ? a.rows : most);
}

}  // namespace

extern "C" int lffn_layer_norm_rows_fwd(const lffn_layer_norm_rows *c, void *out, float *stats, void *stream) {
    const int rc = check(c);
    if (rc != LFFN_OK || c->rows == 0) return rc;
    LFFN_REQUIRE(out, LFFN_ERR_BAD_ARG);
    Args a = arguments(*c);
    a.y = out, a.stats = reinterpret_cast<float2 *>(stats);
    launch<false>(*c, a, 0, by_vectors(*c, out, nullptr), static_cast<hipStream_t>(stream));
    return lffn_launch_status();
}

extern "C" int lffn_layer_norm_rows_bwd_workspace_bytes(const lffn_layer_norm_rows *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    const int rc = check(c);
    if (rc == LFFN_OK) *bytes = parts_of(*c) * 2 * c->columns * 4;
    return rc;
}

extern "C" int lffn_layer_norm_rows_bwd(const lffn_layer_norm_rows *c, const float *stats, const void *g, void *grad_x, void *grad_weight, void *grad_bias,
                                        void *workspace, int64_t workspace_bytes, void *stream) {
    const int rc = check(c);
    if (rc != LFFN_OK) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool sums = grad_weight || grad_bias;
    SumArgs s{static_cast<const float *>(workspace), grad_weight, grad_bias, parts_of(*c), (int)c->columns, c->weight_f32 ? LFFN_ROWS_F32 : c->format};
    if (c->rows == 0) {
        if (sums) clear_kernel<<<dim3(unsigned((c->columns + WG - 1) / WG)), dim3(WG), 0, st>>>(s);
        return lffn_launch_status();
    }
    LFFN_REQUIRE(stats && g && (!sums || (workspace && lffn_aligned16(workspace) && workspace_bytes >= parts_of(*c) * 2 * c->columns * 4)), LFFN_ERR_BAD_ARG);
    Args a = arguments(*c);
    a.g = g, a.gx = grad_x, a.stats = reinterpret_cast<float2 *>(const_cast<float *>(stats));
    a.parts = sums ? static_cast<float *>(workspace) : nullptr;
    launch<true>(*c, a, s.num, by_vectors(*c, g, grad_x), st);
    if (sums) sum_kernel<<<dim3(unsigned((c->columns + 15) / 16), 2), dim3(WG), 0, st>>>(s);
    return lffn_launch_status();
}
