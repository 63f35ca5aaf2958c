// Softmax cross entropy of a projection to a large vocabulary, and its gradients, without the logits of many tokens in memory:
//
//   l_nv = h_n . W_v + b_v,   lse_n = log sum_v exp l_nv,   loss_n = lse_n - l_n,label(n)
//   d_nv = (exp(l_nv - lse_n) - [v = label(n)]) g_n,   dh_n = sum_v d_nv W_v,   dW_v = sum_n d_nv h_n,   db_v = sum_n d_nv
//
// Tokens without a label take no part and cost nothing: the labelled ones' rows are first laid together (`rows`), and how many there are stays on the device, so that
// every launch behind is of a fixed size and its workgroups, one a compute unit, share out what there is.
//
// Forward: tiles of 256 vocabulary entries x 256 tokens (product_tiles.h); a tile's logits become, in its registers, each token's largest and sum of exponentials, 8
// bytes for 256 logits, and a second launch joins those of a token.
// Backward: the logits of a piece of the vocabulary are formed once more, d is written in 16 bits (a float's in two terms), and one launch forms from it both gradients' products:
// dW, its sum over the tokens whole or, where its tiles are few and the tokens many, in shares of them, and dh in shares of the vocabulary, added up in fp32 in memory.  What a
// share adds to is its own: no atomics on results, the same bits on every call.
//
// fp32 in the backward: a sum's numbers have one power of two in common, so rows are laid by the largest of their array, and a row that is far below that would have few bits left.  Where rows,
// or logits, or tokens' gradients, are too far apart (far_apart) the rows are laid one by one, as in the forward, d stays a float, and both products are of the floats themselves (far_hidden, far_weight).
#include "product_tiles.h"

namespace {

using namespace product_tiles;

constexpr int TILE = 256;                       // tokens and vocabulary entries of a tile
constexpr int THREADS = 512, WAVES_M = 2, WAVES_N = 4, MB = TILE / WAVES_M / 32, NB = TILE / WAVES_N / 32;
constexpr int COMPUTE_UNITS = 256, XCDS = 8;
constexpr int CHUNK = 64;                       // tokens whose places a workgroup finds
constexpr int COUNTED = 4096;                   // tokens of a workgroup that counts the labelled ones of its chunks; with fewer every chunk looks at all before it
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LIFT = 16384.f;                 // d times 2^14: half's normal numbers then reach down to 2^-28 of a row's largest
constexpr int64_t D_BYTES = int64_t(1) << 30;   // of a piece's d, at most (with many tokens 2048 entries at least)
constexpr int64_t PARTS_BYTES = int64_t(256) << 20, WEIGHT_PARTS_BYTES = int64_t(512) << 20;
constexpr int CUT_FROM = 2048;                  // tokens (of one plane) from which on dW's sums over them may be cut
constexpr int SHARES = 64;                      // of the vocabulary, for dh, and of the tokens, for dW, at most

__host__ __device__ constexpr int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// What the backward needs beside the inputs, and what the forward's launches share.
struct Kept {
    int32_t *head;      // [8]: labelled tokens; of two-term numbers the exponents of the largest of their rows and of the weights, and of the least ones (rows of zeros aside)
    int32_t *pos;       // [N]: where a token's row is among the labelled ones, or -1
    int32_t *label;     // [labelled]
    float2 *level;      // [labelled]: a token's largest logit times log2(e) (level_of), and one over the sum of the exponentials of what they are below it
                        // (the last two up to a whole tile: tiles are read whole)
    float *logits;      // [labelled, up(vocabulary, 32)], or null: of few tokens, where they are no more than the weights
};

struct Sizes {
    int N, V, K;               // tokens, vocabulary, columns
    int64_t Kp, Vp;            // columns of laid-together rows, entries of padded arrays
};

struct Operands {
    Sizes s;
    Kept kept;
    Source weight;             // as the products read it
    char *rows;                // [Np, Kp] the labelled tokens' rows, zeros behind the columns
    float *bias;               // [Vp] fp32, -infinity behind the vocabulary
    float *weight_scale;       // two-term numbers: [Vp], [Np], by which sums are multiplied
    float *row_scale;
    const float2 *range;       // the backward of losses by token: [RANGES] the largest and the least finite gradients of labelled tokens, zeros aside; else null
};

__device__ __forceinline__ float wave_most(float v) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

__device__ __forceinline__ float wave_least(float v) { return -wave_most(-v); }

// Whether two-term numbers cannot be laid by the largest of their arrays in the backward.  Rows whose largest is 2^-16 of the array's have 22 bits of it left, what a second term has at the
// least.  And the logits that are formed of them must be those whose levels the forward left: laid either way they are off from each other by 2^-38 of the largest number of a row, of an
// entry and the columns, which has to be no more than 2^-18.  (A row's largest is less than 2^14 times the power of two that it was divided by; kept logits are not formed again.)  d is scaled by
// the largest of the tokens' gradients and held to 2^-38 of it: a token's at 2^-8 of that to 2^-30 of its own.  Called by whole wavefronts.
constexpr int ROWS_APART = 16, LOGITS_LARGEST = 20, GRADIENTS_APART = 8, RANGES = 64;
__device__ __forceinline__ bool far_apart(const Operands &o) {
    const int32_t *h = o.kept.head;
    if (o.range) {
        const float2 r = o.range[threadIdx.x % RANGES];
        const float most = wave_most(r.x), least = wave_least(r.y);
        if (most > 0.f && ilogbf(most) - ilogbf(least) > GRADIENTS_APART) return true;
    }
    return max(h[1] - min(h[1], h[3]), h[2] - min(h[2], h[4])) > ROWS_APART || (!o.kept.logits && h[1] + h[2] + 28 + (32 - __clz(o.s.K - 1)) > LOGITS_LARGEST);
}

template <int PLANES>
__device__ __forceinline__ Source rows_of(const Operands &o, int labelled) {
    return {o.rows, o.s.Kp * 2 * PLANES, (int)up(labelled, TILE), (int)o.s.Kp};
}

// ---------------------------------------------------------------- the labelled tokens

struct RowsArgs {
    Operands o;
    const void *hidden, *labels, *bias;
    int64_t hidden_stride, ignore;
    int32_t labels_64, bias_format;            // of the gather's row formats; -1: none
    const int32_t *counts, *groups;            // labelled tokens of every chunk and of every COUNTED, or null
    int parts;                                 // workgroups that lay a chunk's rows
    int32_t *token;                            // [labelled], or null
    float *loss;                               // [N]: zeros for the others, or null
    const float *g_loss;                       // the backward of losses by token: [N]
    float *coefficient, *power;                // and what becomes of it (BackwardArgs), or null
};

__device__ __forceinline__ int label_of(const void *labels, int wide, int64_t i, int64_t ignore, int V) {
    const int64_t y = wide ? static_cast<const int64_t *>(labels)[i] : static_cast<const int32_t *>(labels)[i];
    return y == ignore || y < 0 || y >= V ? -1 : (int)y;
}

__global__ __launch_bounds__(1024) void count_kernel(const void *labels, int wide, int64_t ignore, int V, int N, int32_t *counts, int32_t *groups) {
    __shared__ int sums[16];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    int sum = 0;
#pragma unroll
    for (int i = 0; i < COUNTED / 1024; ++i) {
        const int n = blockIdx.x * COUNTED + i * 1024 + (int)threadIdx.x;
        const int live = __popcll(__ballot(n < N && label_of(labels, wide, n, ignore, V) >= 0));
        if (lane == 0 && n < N) counts[n / CHUNK] = live;
        sum += live;
    }
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) sum += sums[i];
        groups[blockIdx.x] = sum;
    }
}

// A row of `columns` numbers as the products read it, zeros up to `padded`, by one wavefront.  Two-term numbers: scaled by the row's largest, or to `exponent` where that is
// given; -> the power of two of the way back, 0 of a row of zeros (no sum of it is anything else) and of an infinite one (which is lost).
template <typename R, int PLANES>
__device__ __forceinline__ float lay_row(const char *from, char *to, int columns, int64_t padded, const int *exponent) {
    const int lane = threadIdx.x % 64;
    if constexpr (PLANES == 1) {
        for (int c = lane * 8; c < padded; c += 512)
            *reinterpret_cast<uint4 *>(to + c * 2) = c < columns ? *reinterpret_cast<const uint4 *>(from + c * 2) : make_uint4(0, 0, 0, 0);
        return 1.f;
    } else {
        float scale, back;
        if (exponent) {
            scale = __builtin_amdgcn_ldexpf(1.f, -*exponent), back = __builtin_amdgcn_ldexpf(1.f, *exponent);
        } else {
            float most = 0.f;
            for (int c = lane * 4; c < columns; c += 256) {
                const float4 v = *reinterpret_cast<const float4 *>(from + c * 4);
                most = fmaxf(fmaxf(fmaxf(most, fabsf(v.x)), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
            }
            most = wave_most(most);
            int e;
            scale = scale_to(most == INFINITY ? 0.f : most, 13, e);        // (the backward's exponents are the others')
            back = most == INFINITY || most == 0.f ? 0.f : __builtin_amdgcn_ldexpf(1.f, e);
        }
        for (int c = lane * 8; c < padded; c += 512) {
            uint32_t h[4] = {0, 0, 0, 0}, l[4] = {0, 0, 0, 0};
            if (c < columns) {
                const float4 a = *reinterpret_cast<const float4 *>(from + c * 4), b = *reinterpret_cast<const float4 *>(from + c * 4 + 16);
                const float v[8] = {a.x * scale, a.y * scale, a.z * scale, a.w * scale, b.x * scale, b.y * scale, b.z * scale, b.w * scale};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[i] = split_hi(v[2 * i], v[2 * i + 1], 1.f);
                    l[i] = split_rest(v[2 * i], v[2 * i + 1], h[i]);
                }
            }
            *reinterpret_cast<uint4 *>(to + byte_of<2>(c)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4 *>(to + byte_of<2>(c) + 64) = make_uint4(l[0], l[1], l[2], l[3]);
        }
        return back;
    }
}

__device__ __forceinline__ float bias_of(const void *bias, int format, int v) {
    if (format == LFFN_ROWS_F32) return static_cast<const float *>(bias)[v];
    if (format == LFFN_ROWS_BF16) return (float)static_cast<const __bf16 *>(bias)[v];
    return (float)static_cast<const _Float16 *>(bias)[v];
}

// The exponents of the largest and the least of n powers of two, zeros aside, to *most and *least, by a workgroup that others may be beside: an atomic for each.  red: 32 numbers.
__device__ __forceinline__ void find_exponents(int32_t *most, int32_t *least, const float *scales, int first, int n, int step, float *red) {
    float high = 0.f, low = INFINITY;
    for (int i = first; i < n; i += step) {
        const float v = scales[i];
        high = fmaxf(high, v), low = v > 0.f ? fminf(low, v) : low;
    }
    high = wave_most(high), low = wave_least(low);
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = high, red[16 + threadIdx.x / 64] = low;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (unsigned i = 1; i < blockDim.x / 64; ++i) high = fmaxf(high, red[i]), low = fminf(low, red[16 + i]);
        if (high > 0.f) atomicMax(most, ilogbf(high)), atomicMin(least, ilogbf(low));
    }
}

// (as low an exponent as any, and a higher one than any: the launch that joins raises and lowers them)
__device__ __forceinline__ void begin_head(const Kept &k, int labelled) { k.head[0] = labelled, k.head[1] = k.head[2] = -116, k.head[3] = k.head[4] = 1000; }

// Workgroups parts (tokens / CHUNK): the labelled tokens of a chunk take their places (in the forward; the backward reads where they are) and their rows are laid there; the last
// one fills the last tile's rows up with zeros.  The workgroups behind: the bias in fp32.
template <typename R, int PLANES, bool BACKWARD>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
    const Sizes &s = a.o.s;
    const Kept &k = a.o.kept;
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, chunks = (s.N + CHUNK - 1) / CHUNK, chunk = (int)blockIdx.x / a.parts, part = (int)blockIdx.x % a.parts;
    if (chunk >= chunks) {
        const int v = ((int)blockIdx.x - chunks * a.parts) * 256 + tid;
        if (v < s.Vp) a.o.bias[v] = v >= s.V ? -INFINITY : a.bias_format < 0 ? 0.f : bias_of(a.bias, a.bias_format, v);
        return;
    }
    __shared__ int place[CHUNK], before[4];
    const int t0 = chunk * CHUNK;
    const bool far = PLANES == 2 && BACKWARD && far_apart(a.o);
    int labelled = 0;              // up to and with this chunk
    if constexpr (!BACKWARD) {
        int n = 0;
        if (a.counts) {
            const int group = t0 / COUNTED, first = group * (COUNTED / CHUNK);
            for (int i = tid; i < group; i += 256) n += a.groups[i];
            if (first + tid < chunk) n += a.counts[first + tid];
        } else
            for (int i = tid; i < t0; i += 256) n += label_of(a.labels, a.labels_64, i, a.ignore, s.V) >= 0;
#pragma unroll
        for (int m = 32; m > 0; m /= 2) n += __shfl_xor(n, m);
        if (lane == 0) before[wave] = n;
        __syncthreads();
        const int first = before[0] + before[1] + before[2] + before[3], t = t0 + lane;
        const int y = t < s.N ? label_of(a.labels, a.labels_64, t, a.ignore, s.V) : -1;
        const uint64_t live = __ballot(y >= 0);
        labelled = first + __popcll(live);
        if (wave == 0) {
            const int at = y >= 0 ? first + __popcll(live & ((uint64_t(1) << lane) - 1)) : -1;
            place[lane] = at;
            if (t < s.N && part == 0) {
                k.pos[t] = at;
                if (y >= 0) k.label[at] = y, a.token[at] = t;
                else if (a.loss) a.loss[t] = 0.f;
            }
            if (chunk == chunks - 1 && part == 0 && lane == 0) begin_head(k, labelled);
        }
    } else {
        labelled = k.head[0];
        if (wave == 0) {
            const int at = t0 + lane < s.N ? k.pos[t0 + lane] : -1;
            place[lane] = at;
            if (a.token && part == 0 && at >= 0) a.token[at] = t0 + lane;
            if (a.coefficient && part == 0) {
                // Tokens' own gradients by the power of two of their largest; far apart as they are, but for very large ones (d is lifted)
                const float most = wave_most(a.o.range[lane].x);
                int e = most > 0x1p100f ? 28 : 0;
                const float scale = far ? __builtin_amdgcn_ldexpf(1.f, -e) : scale_to(most, 0, e);
                if (at >= 0) a.coefficient[at] = a.g_loss[t0 + lane] * scale;
                if (chunk == 0 && lane == 0) *a.power = __builtin_amdgcn_ldexpf(1.f / LIFT, e);
            }
        }
    }
    __syncthreads();
    const int64_t row_bytes = s.Kp * 2 * PLANES;
    const int *const exponent = BACKWARD && !far ? k.head + 1 : nullptr;
    for (int i = part * 4 + wave; i < CHUNK; i += 4 * a.parts) {
        const int at = place[i];
        if (at < 0) continue;
        const char *from = static_cast<const char *>(a.hidden) + (int64_t(t0) + i) * a.hidden_stride * R::BYTES;
        const float back = lay_row<R, PLANES>(from, a.o.rows + at * row_bytes, s.K, s.Kp, exponent);
        if (PLANES == 2 && lane == 0) a.o.row_scale[at] = back;
    }
    if (chunk == chunks - 1) {
        const int64_t from = labelled * row_bytes / 16, to = up(labelled, TILE) * row_bytes / 16;
        for (int64_t i = from + part * 256 + tid; i < to; i += 256 * a.parts) *reinterpret_cast<uint4 *>(a.o.rows + i * 16) = make_uint4(0, 0, 0, 0);
        if (PLANES == 2)
            for (int i = labelled + tid; i < up(labelled, TILE); i += 256) a.o.row_scale[i] = 1.f;
    }
}

// fp32 weights in two half-precision terms: each row by its largest, or, in the backward, all by the array's (far_apart).
template <bool BACKWARD>
__global__ __launch_bounds__(256) void weight_kernel(Operands o, const float *w, int64_t stride) {
    const int v = blockIdx.x * 4 + threadIdx.x / 64;
    if (v >= o.s.Vp) return;
    float back = 0.f;              // (of entries behind the vocabulary, and nothing to the largest and the least)
    if (v < o.s.V)
        back = lay_row<F32Row, 2>(reinterpret_cast<const char *>(w + v * stride), const_cast<char *>(o.weight.at) + v * o.weight.stride, o.s.K, o.weight.columns,
                                  BACKWARD && !far_apart(o) ? o.kept.head + 2 : nullptr);
    if (threadIdx.x % 64 == 0) o.weight_scale[v] = back;
}

// ---------------------------------------------------------------- logits

// A workgroup's tasks of `total`, in turn: those of an XCD follow each other, so that its compute units read the same ones.
struct Turns {
    int at, end, step;
    __device__ __forceinline__ explicit Turns(int total) {
        const int xcd = blockIdx.x % XCDS, share = (total + XCDS - 1) / XCDS;
        step = gridDim.x / XCDS;
        at = xcd * share + blockIdx.x / XCDS;
        end = min(total, (xcd + 1) * share);
    }
    __device__ __forceinline__ bool any() const { return at < end; }
};

// A tile of vt x nt: eight tiles of the vocabulary at a time against one tile of tokens after the other.
struct Place {
    int v, n;
    __device__ __forceinline__ Place(int id, int vt, int nt) {
        const int group = id / (8 * nt), in = id - group * 8 * nt, height = min(8, vt - group * 8);
        v = (group * 8 + in % height) * TILE;
        n = in / height * TILE;
    }
};

// How eight wavefronts share a tile of TILE entries, or columns, x TOKENS_ tokens: M x N of them along its entries and tokens.  Up to 64 labelled tokens take a tile of as many, here and in
// dh: a quarter of the products (58 of 385 tokens labelled, 50265 x 768 bfloat16: logits 18.6 us for 27.2, d 21.5 for 28.4, both gradients 46 for 56; 9 labelled, 50265 x 840 fp32: 55 for 70, 61 for 84, 99 for 121).
constexpr int NARROW = 64;
template <int TOKENS_, int M_, int N_>
struct OfLogits {
    static constexpr int TOKENS = TOKENS_, M = M_, N = N_, MB = TILE / M / 32, NB = TOKENS / N / 32;
};
typedef OfLogits<TILE, WAVES_M, WAVES_N> WideLogits;
typedef OfLogits<NARROW, 4, 2> NarrowLogits;

typedef Along<TILE, THREADS, 1> AlongOne;
constexpr uint32_t STREAM_LDS = Stream<F16, MB, NB, AlongOne, AlongOne>::LDS;      // (of any operands)

// What a tile's logits become takes numbers of its entries and its tokens: 1 KB of each, brought to LDS with the tile's first step, a wavefront a kilobyte, two tiles' places in turn.  Loads
// from memory would return behind the next tile's copies and be waited for as long.
enum Beside { BIAS, LABEL, WEIGHT_SCALE, ROW_SCALE, LEVEL, LEVEL_END = LEVEL + 2, COEFFICIENT = LEVEL_END, BESIDES };
constexpr uint32_t BESIDE_BYTES = BESIDES * 1024;
static_assert(TILE == 256 && BESIDES <= THREADS / 64, "a wavefront's copy is one array's share of a tile");

template <bool BACKWARD>
__device__ __forceinline__ void bring_beside(const Operands &o, const float *coefficient, int v0, int n0, uint32_t lds) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const void *from = nullptr;
    if (wave == BIAS) from = o.bias + v0;
    else if (wave == LABEL) from = o.kept.label + n0;
    else if (wave == WEIGHT_SCALE && o.weight_scale) from = o.weight_scale + v0;
    else if (wave == ROW_SCALE && o.row_scale) from = o.row_scale + n0;
    else if (BACKWARD && wave >= LEVEL && wave < LEVEL_END) from = o.kept.level + n0 + (wave - LEVEL) * 128;
    else if (BACKWARD && wave == COEFFICIENT && coefficient) from = coefficient + n0;
    if (from) copy_to_lds((const char *)uniform((uint64_t)from), threadIdx.x % 64 * 16, lds + wave * 1024);
}
template <typename T>
__device__ __forceinline__ T beside(uint32_t lds, Beside of, int at) {
    typedef uint32_t words_t __attribute__((ext_vector_type(sizeof(T) / 4)));
    return __builtin_bit_cast(T, *(const __attribute__((address_space(3))) words_t *)(uintptr_t)(lds + of * 1024 + at * sizeof(T)));
}

// The logits of one tile after the other: entries from v0 on, in all `width`, and the labelled tokens; each(sums, place, lds) has the sums of a tile's products, of one plane with the bias, and
// what came beside it, and calls landed() before it stores anything.
template <typename F, typename S, bool BACKWARD, typename Each>
__device__ __forceinline__ void for_logits(const Operands &o, const float *coefficient, int labelled, int v0, int width, uint32_t lds, Each &&each) {
    typedef Along<TILE, THREADS, F::PLANES> Side;
    typedef Along<S::TOKENS, THREADS, F::PLANES> Rows;
    const int wave = threadIdx.x / 64, half = threadIdx.x % 64 / 32, vt = (width + TILE - 1) / TILE, nt = (labelled + TILE - 1) / TILE;
    const int steps = max(2, (o.s.K + Side::K - 1) / Side::K);
    Turns turns(vt * nt);
    if (!turns.any()) return;
    const Source rows = rows_of<F::PLANES>(o, labelled);
    Place place(turns.at, vt, nt);
    Side a(o.weight, v0 + place.v);
    Rows b(rows, place.n);
    Stream<F, S::MB, S::NB, Side, Rows> stream(lds, wave / S::N * S::MB * 32, wave % S::N * S::NB * 32);
    uint32_t by = lds + STREAM_LDS, next_by = by + BESIDE_BYTES;
    bring_beside<BACKWARD>(o, coefficient, v0 + place.v, place.n, by);
    stream.prime(a, b, 0);
    for (;;) {
        const int next = turns.at + turns.step;
        const bool more = next < turns.end;
        const Place then(more ? next : turns.at, vt, nt);
        const Side next_a(o.weight, v0 + then.v);
        const Rows next_b(rows, then.n);
        Sums<S::MB, S::NB> sums;
        if constexpr (F::PLANES == 1) {
#pragma unroll
            for (int i = 0; i < S::MB; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 bias = beside<float4>(by, BIAS, (wave / S::N * S::MB + i) * 8 + 2 * g + half);
#pragma unroll
                    for (int j = 0; j < S::NB; ++j)
                        sums.v[i][j][4 * g] = bias.x, sums.v[i][j][4 * g + 1] = bias.y, sums.v[i][j][4 * g + 2] = bias.z, sums.v[i][j][4 * g + 3] = bias.w;
                }
        } else
            sums.clear();
        stream.multiply(sums, a, b, 0, steps, next_a, next_b, 0, [](int, const uint4 &) {},
                        [&] { bring_beside<BACKWARD>(o, coefficient, v0 + then.v, then.n, next_by); });
        each(sums, place, by);
        if (!more) break;
        turns.at = next, place = then;
        const uint32_t swap = by;
        by = next_by;
        next_by = swap;
    }
    stream.done();
}

// The logits of block i's 16 entries, `row` of the tile's first of them, for a token: l[e] of entry mfma_row(e, half).
template <typename F>
__device__ __forceinline__ void logits_of(float (&l)[16], const f32x16_t &sum, uint32_t lds, int row, float row_scale) {
    const int half = threadIdx.x % 64 / 32;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        if constexpr (F::PLANES == 1) {
#pragma unroll
            for (int e = 4 * g; e < 4 * g + 4; ++e) l[e] = sum[e];
        } else {
            const float4 b = beside<float4>(lds, BIAS, row / 4 + 2 * g + half), w = beside<float4>(lds, WEIGHT_SCALE, row / 4 + 2 * g + half);
            l[4 * g] = fmaf(sum[4 * g] * w.x, row_scale, b.x), l[4 * g + 1] = fmaf(sum[4 * g + 1] * w.y, row_scale, b.y);
            l[4 * g + 2] = fmaf(sum[4 * g + 2] * w.z, row_scale, b.z), l[4 * g + 3] = fmaf(sum[4 * g + 3] * w.w, row_scale, b.w);
        }
    }
}

struct ForwardArgs {
    Operands o;
    float2 *parts;         // [tiles of the vocabulary, Np]: largest, sum of exponentials of what they are below it
    float *at_label;       // [labelled]
    int64_t Np;
};

__device__ __forceinline__ float2 joined(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), from = m == -INFINITY ? 0.f : m;
    return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - from) + b.y * __builtin_amdgcn_exp2f(b.x - from));
}

// Levels are logits times log2(e): an exponential is one product with a sum, rounded once, and the power of two of that; what the level's own rounding is off by, all of a token's have, and
// it falls out.  From 2^30 on it would be more than an exponential's range, and logits are 64 apart or equal: there a level is twice the logit, exactly, and the others' powers are none.
constexpr float LARGE = 1073741824.f;
__device__ __forceinline__ float level_of(float logit) { return fabsf(logit) >= LARGE ? logit + logit : logit * LOG2E; }
// what logits are multiplied with to be compared with a level
__device__ __forceinline__ float scale_of(float level) { return fabsf(level) >= 2.f * LARGE ? 2.f : LOG2E; }

// Adds 16 logits of a token to its largest and sum so far.
__device__ __forceinline__ float2 with_logits(float2 of, const float (&l)[16]) {
    float most = l[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) most = fmaxf(most, l[e]);
    most = fmaxf(of.x, level_of(most));
    const float from = most == -INFINITY ? 0.f : most, scale = scale_of(from);
    float sum = of.y * __builtin_amdgcn_exp2f(of.x - from);
#pragma unroll
    for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(fmaf(l[e], scale, -from));
    return make_float2(most, sum);
}

template <typename F, typename S>
__device__ __forceinline__ void forward_tiles(const ForwardArgs &a, uint32_t lds, float2 *parts) {
    const Operands &o = a.o;
    const int labelled = o.kept.head[0], tid = threadIdx.x, wave = tid / 64, lane = tid % 64, half = lane / 32;
    const int wm = wave / S::N, wn = wave % S::N;
    for_logits<F, S, false>(o, nullptr, labelled, 0, o.s.V, lds, [&](const Sums<S::MB, S::NB> &sums, const Place &p, uint32_t by) {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            const int column = wn * S::NB * 32 + j * 32 + lane % 32, n = p.n + column;
            const float row_scale = F::PLANES == 2 ? beside<float>(by, ROW_SCALE, column) : 1.f;
            const int at = n < labelled ? beside<int>(by, LABEL, column) - p.v - wm * S::MB * 32 : -1;
            float2 of = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < S::MB; ++i) {
                float l[16];
                logits_of<F>(l, sums.v[i][j], by, (wm * S::MB + i) * 32, row_scale);
                of = with_logits(of, l);
                const int r = at - 32 * i;
                if (r >= 0 && r < 32 && r / 4 % 2 == half) {
                    float found = l[0];
#pragma unroll
                    for (int e = 1; e < 16; ++e) found = mfma_row(e, half) == r ? l[e] : found;
                    arrived();
                    a.at_label[n] = found;
                }
            }
            const float2 other = make_float2(__shfl_xor(of.x, 32), __shfl_xor(of.y, 32));
            if (half == 0) parts[wm * S::TOKENS + column] = joined(of, other);
        }
        arrived();
        __syncthreads();
        if (tid < S::TOKENS) {
            float2 of = parts[tid];
#pragma unroll
            for (int m = 1; m < S::M; ++m) of = joined(of, parts[m * S::TOKENS + tid]);
            a.parts[p.v / TILE * a.Np + p.n + tid] = of;
        }
        // (the next tile's products have barriers before the parts are written again)
    });
}

template <typename F>
__global__ __launch_bounds__(THREADS, 2) void forward_kernel(ForwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint4 lds_words[];
    const uint32_t lds = lds_byte_of(lds_words);
    float2 *const parts = reinterpret_cast<float2 *>(reinterpret_cast<char *>(lds_words) + STREAM_LDS + 2 * BESIDE_BYTES);     // of a tile's tokens, by wavefronts along the entries
    if (a.o.kept.head[0] <= NARROW) forward_tiles<F, NarrowLogits>(a, lds, parts);
    else forward_tiles<F, WideLogits>(a, lds, parts);
}
static_assert(NarrowLogits::M * NarrowLogits::TOKENS <= WAVES_M * TILE, "the parts' room");


// ---------------------------------------------------------------- few tokens

// Up to 64 tokens whose rows fit LDS, and whose logits are no more bytes than the weights: reading the weights is all there is.  The labelled tokens' rows lie in every workgroup's LDS as a
// whole; a wavefront takes 32 entries of the vocabulary at a time, whose rows go from memory straight to its registers as operands, 64 bytes a lane, half a line, six such in flight.  Nothing is
// laid together before: a launch less.  (64 x 50265 x 768 bfloat16 22.7 us, 3.4 TB/s: 50265 entries are 1571 blocks for 2048 wavefronts, of which a quarter have none, and the others' single blocks
// begin and end together.)
// fp32 is multiplied as it is (v_mfma_f32_32x32x2_f32): 32 x 50265 x 840 64 us, where the weights' bytes are 33 and the products 17, but each wavefront's loads and products follow one another
// (splitting the weights to memory took 71 and the tiles' products 71).  The exponents that the backward's two-term numbers have in common, and the least ones, are found on the way.
constexpr int FEW = 64, LINE = 128;                                                            // bytes of a row that a step has
constexpr int few_stride(int64_t row_bytes) { return int(up(row_bytes, LINE)) / 16 | 1; }      // 16-byte pieces of a row in LDS: odd, so that 16 rows meet every bank once
constexpr int64_t few_lds(int64_t tokens, int64_t row_bytes) {
    return (tokens <= 32 ? 32 : 64) * int64_t(few_stride(row_bytes)) * 16 + 8 * FEW * 8 + FEW * 4;
}
int64_t row_bytes(const lffn_linear_cross_entropy &a) { return a.columns * (a.format == LFFN_ROWS_F32 ? 4 : 2); }
// The backward of few tokens takes their logits from the forward, which are no more bytes than the weights, that it would read for them once more (both directions, 19 tokens, 50265 x 768 fp32:
// 291 us with them formed again, 246 with these).  Formed again they would be sums in another order, and a softmax has to see both directions' logits alike; so tokens that are more than a
// row's columns in floats take the tiles, as many tokens do, in both.
constexpr int64_t logits_stride(int64_t vocabulary) { return up(vocabulary, 32); }
bool few_tokens(const lffn_linear_cross_entropy &a) { return a.tokens <= FEW && a.tokens * 4 <= row_bytes(a) && few_lds(a.tokens, row_bytes(a)) <= 160 * 1024; }
constexpr int64_t HEAD_BYTES = 32;
int64_t kept_bytes(const lffn_linear_cross_entropy &a, bool logits) {
    return HEAD_BYTES + up(a.tokens * 4, 16) + up(a.tokens, TILE) * 12 + (logits ? a.tokens * logits_stride(a.vocabulary) * 4 : 0);
}
Kept kept_at(const lffn_linear_cross_entropy &a, void *at) {
    char *p = static_cast<char *>(at);
    const int64_t n = up(a.tokens * 4, 16), tiles = up(a.tokens, TILE);
    int32_t *const head = reinterpret_cast<int32_t *>(p);
    p += HEAD_BYTES;
    return {head, reinterpret_cast<int32_t *>(p), reinterpret_cast<int32_t *>(p + n), reinterpret_cast<float2 *>(p + n + tiles * 4),
            few_tokens(a) ? reinterpret_cast<float *>(p + n + tiles * 12) : nullptr};
}

int few_workgroups(const lffn_linear_cross_entropy &a) { return (int)min((a.vocabulary + 31) / 32, int64_t(COMPUTE_UNITS)); }

struct FewArgs {
    RowsArgs r;
    float2 *parts;
    float *at_label, *logits;      // the last: null without a backward
    int64_t Np;
};

// Adds the products of 16 bytes of both operands.
template <typename F>
struct Few {
    static constexpr int BYTES = 2, SUMS = 1;
    static __device__ __forceinline__ void add(f32x16_t (&sums)[SUMS], const uint4 &w, const uint4 &x) { sums[0] = F::mma(w, x, sums[0]); }
};
template <>
struct Few<F32Row> {
    static constexpr int BYTES = 4, SUMS = 2;                  // (two sums: half as many roundings each, of half the size)
    static __device__ __forceinline__ void add(f32x16_t (&sums)[SUMS], const uint4 &w, const uint4 &x) {
        const float4 a = __builtin_bit_cast(float4, w), b = __builtin_bit_cast(float4, x);
        sums[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, b.x, sums[0], 0, 0, 0);
        sums[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, b.y, sums[1], 0, 0, 0);
        sums[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, b.z, sums[0], 0, 0, 0);
        sums[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, b.w, sums[1], 0, 0, 0);
    }
};
__device__ __forceinline__ float most_of(const uint4 &u, float most) {
    const float4 v = __builtin_bit_cast(float4, u);
    return fmaxf(fmaxf(fmaxf(most, fabsf(v.x)), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
}
// The largest and the least of rows' largest magnitudes, zeros and infinite ones aside.
struct Range {
    float most = 0.f, least = INFINITY;
    __device__ __forceinline__ void add(float of_row) {
        if (of_row > 0.f && of_row < INFINITY) most = fmaxf(most, of_row), least = fminf(least, of_row);
    }
};
// The powers of two that two-term numbers of a workgroup's are divided by, to scales[0] and [1], zeros of none.
__device__ __forceinline__ void put_scales(float *scales, Range r, float *red) {
    r.most = wave_most(r.most), r.least = wave_least(r.least);
    __syncthreads();
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = r.most, red[16 + threadIdx.x / 64] = r.least;
    __syncthreads();
    if (threadIdx.x < 2) {
        for (unsigned i = 0; i < blockDim.x / 64; ++i) r.most = fmaxf(r.most, red[i]), r.least = fminf(r.least, red[16 + i]);
        int e;
        scale_to(threadIdx.x == 0 ? r.most : r.least, 13, e);
        scales[threadIdx.x] = r.most > 0.f ? __builtin_amdgcn_ldexpf(1.f, e) : 0.f;
    }
}

template <typename F, int TOKENS>
__global__ __launch_bounds__(THREADS, 2) void few_kernel(FewArgs a) {
    typedef Few<F> Of;
    constexpr int JB = TOKENS / 32, WAVES = THREADS / 64, BYTES = Of::BYTES;
    constexpr bool WHOLE = BYTES == 4;
    constexpr int AHEAD = WHOLE && TOKENS == 64 ? 4 : 6;       // steps in flight (what the registers have room for)
    extern __shared__ __attribute__((aligned(16))) uint4 lds_words[];
    const Operands &o = a.r.o;
    const int V = o.s.V, K = o.s.K, tid = threadIdx.x, wave = tid / 64, lane = tid % 64, half = lane / 32;
    const int bytes = K * BYTES, stride = few_stride(bytes), pieces = int(up(bytes, LINE)) / 16, steps = pieces / 8;
    float2 *const waves = reinterpret_cast<float2 *>(lds_words + TOKENS * stride);       // [WAVES][TOKENS]
    int *const tokens = reinterpret_cast<int *>(waves + WAVES * TOKENS);                 // [TOKENS]
    // the labelled tokens: every wavefront sees them all
    const int y = lane < o.s.N ? label_of(a.r.labels, a.r.labels_64, lane, a.r.ignore, V) : -1;
    const uint64_t live = __ballot(y >= 0);
    const int labelled = __popcll(live), place = __popcll(live & ((uint64_t(1) << lane) - 1));
    if (wave == 0 && y >= 0) tokens[place] = lane;
    if (blockIdx.x == 0 && wave == 0) {
        if (lane == 0) begin_head(o.kept, labelled);
        if (lane < o.s.N) {
            o.kept.pos[lane] = y >= 0 ? place : -1;
            if (y >= 0) o.kept.label[place] = y, a.r.token[place] = lane;
            else if (a.r.loss) a.r.loss[lane] = 0.f;
        }
    }
    if (labelled == 0) return;
    const int blocks = (V + 31) / 32, all = gridDim.x * WAVES;
    int block = wave * gridDim.x + blockIdx.x;
    uint4 w[AHEAD][4];
    Range of_weights, of_rows;
    float most = 0.f;                              // of the lane's numbers of an entry
    const char *row = nullptr;
    auto begin_block = [&] { row = o.weight.at + int64_t(min(block * 32 + lane % 32, V - 1)) * o.weight.stride; };
    auto load = [&](int s, uint4 (&to)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) to[c] = *reinterpret_cast<const uint4 *>(row + min(s * LINE + half * 64 + c * 16, bytes - 16));
    };
    if (block < blocks) {
        begin_block();
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) load(s, w[s]);
    }
    __syncthreads();
    // (six pieces a thread in flight: 22.0 us for 64 x 50265 x 768 instead of 24.2 one after the other)
    constexpr int BATCH = 6;
    for (int i0 = tid; i0 < TOKENS * pieces; i0 += BATCH * THREADS) {
        uint4 v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + k * THREADS, r = i / pieces, p = i - r * pieces;
            v[k] = make_uint4(0, 0, 0, 0);
            if (r < labelled && p * 16 < bytes) v[k] = *reinterpret_cast<const uint4 *>(static_cast<const char *>(a.r.hidden) + tokens[r] * a.r.hidden_stride * BYTES + p * 16);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + k * THREADS, r = i / pieces, p = i - r * pieces;
            if (r < TOKENS) lds_words[r * stride + p] = v[k];
        }
    }
    __syncthreads();
    const uint32_t lds = lds_byte_of(lds_words) + (lane % 32 * stride + half * 4) * 16;
    int label[JB];
    float2 of[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) {
        const int n = 32 * j + lane % 32;
        label[j] = n < labelled ? label_of(a.r.labels, a.r.labels_64, tokens[n], a.r.ignore, V) : -1;
        of[j] = make_float2(-INFINITY, 0.f);
    }
    for (; block < blocks; block += all) {
        f32x16_t sums[JB][Of::SUMS];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int v = block * 32 + mfma_row(e, half);
            const float b = v >= V ? -INFINITY : a.r.bias_format < 0 ? 0.f : bias_of(a.r.bias, a.r.bias_format, v);
#pragma unroll
            for (int j = 0; j < JB; ++j) {
                sums[j][0][e] = b;
                if constexpr (WHOLE) sums[j][1][e] = 0.f;
            }
        }
        for (int s0 = 0; s0 < steps; s0 += AHEAD) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int s = s0 + k;
                if (s < steps) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int j = 0; j < JB; ++j)
                            Of::add(sums[j], w[k][c], __builtin_bit_cast(uint4, *(const lds_word_t *)(uintptr_t)(lds + (j * 32 * stride + s * 8 + c) * 16)));
                        if constexpr (WHOLE) most = most_of(w[k][c], most);
                    }
                    if (s + AHEAD < steps) load(s + AHEAD, w[k]);
                }
            }
        }
        const int v0 = block * 32;
        if constexpr (WHOLE) {
            of_weights.add(fmaxf(most, __shfl_xor(most, 32)));
            most = 0.f;
        }
        if (block + all < blocks) {                 // the next block's first steps
            block += all;
            begin_block();
            block -= all;
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) load(s, w[s]);
        }
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            float l[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) l[e] = WHOLE ? sums[j][0][e] + sums[j][Of::SUMS - 1][e] : sums[j][0][e];
            of[j] = with_logits(of[j], l);
            if (a.logits && label[j] >= 0) {
                float *const to = a.logits + (32 * j + lane % 32) * logits_stride(V) + v0 + 4 * half;
#pragma unroll
                for (int g = 0; g < 4; ++g) *reinterpret_cast<float4 *>(to + 8 * g) = make_float4(l[4 * g], l[4 * g + 1], l[4 * g + 2], l[4 * g + 3]);
            }
            const int r = label[j] - v0;
            if (label[j] >= 0 && r >= 0 && r < 32 && r / 4 % 2 == half) {
                float found = l[0];
#pragma unroll
                for (int e = 1; e < 16; ++e) found = mfma_row(e, half) == r ? l[e] : found;
                a.at_label[32 * j + lane % 32] = found;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
        const float2 other = make_float2(__shfl_xor(of[j].x, 32), __shfl_xor(of[j].y, 32));
        if (half == 0) waves[wave * TOKENS + 32 * j + lane] = joined(of[j], other);
    }
    __syncthreads();
    if (tid < TOKENS) {
        float2 sum = waves[tid];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) sum = joined(sum, waves[i * TOKENS + tid]);
        a.parts[blockIdx.x * a.Np + tid] = sum;
    }
    if constexpr (WHOLE) {
        put_scales(o.weight_scale + 2 * blockIdx.x, of_weights, reinterpret_cast<float *>(waves));
        // (the last workgroup has no more blocks than any)
        if (blockIdx.x == gridDim.x - 1) {
            for (int r = wave; r < labelled; r += WAVES) {
                float of_row = 0.f;
                for (int p = lane; p < pieces; p += 64) of_row = most_of(lds_words[r * stride + p], of_row);
                of_rows.add(wave_most(of_row));
            }
            put_scales(o.row_scale, of_rows, reinterpret_cast<float *>(waves));
        }
    }
}

struct JoinArgs {
    Kept kept;
    const float2 *parts;
    const float *at_label;
    const int32_t *token;
    int64_t Np;
    int tiles;
    float *loss;           // by token
    double *sums;          // of a workgroup's
    const float *weight_scale, *row_scale;       // two-term numbers: of `entries`, and of the labelled tokens; of few, every workgroup's largest and least and all tokens'
    int entries, few, joining;                   // the last: workgroups that join; those behind look for the largest and the least of the scales
};

constexpr int LOOKING = 16;

// A token's parts: 16 threads.
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
    __shared__ float2 shares[16][17];
    const int labelled = a.kept.head[0], in = threadIdx.x % 16, slice = threadIdx.x / 16, n = blockIdx.x * 16 + in;
    if ((int)blockIdx.x >= a.joining) {
        const int i = blockIdx.x - a.joining;
        if (labelled == 0) return;                   // (no numbers are multiplied)
        int32_t *const head = a.kept.head;
        if (i < LOOKING) find_exponents(head + 2, head + 4, a.weight_scale, i * 256 + threadIdx.x, a.entries, LOOKING * 256, &shares[0][0].x);
        else find_exponents(head + 1, head + 3, a.row_scale, (i - LOOKING) * 256 + threadIdx.x, a.few ? 2 : labelled, LOOKING * 256, &shares[0][0].x);
        return;
    }
    if ((int)blockIdx.x * 16 >= labelled) return;
    float2 of = make_float2(-INFINITY, 0.f);
#pragma unroll 4
    for (int t = slice; t < a.tiles; t += 16) of = joined(of, a.parts[t * a.Np + n]);
    shares[slice][in] = of;
    __syncthreads();
    if (slice != 0) return;
    double sum = 0;
    if (n < labelled) {
#pragma unroll
        for (int i = 1; i < 16; ++i) of = joined(of, shares[i][in]);
        // (log2(e), rounded alike in both, falls out)
        const float scale = scale_of(of.x), loss = (fmaf(-a.at_label[n], scale, of.x) + __builtin_amdgcn_logf(of.y)) * (scale == LOG2E ? 1.f / LOG2E : 0.5f);
        a.kept.level[n] = make_float2(of.x, 1.f / of.y);
        if (a.loss) a.loss[a.token[n]] = loss;
        sum = loss;
    }
    if (!a.sums) return;
#pragma unroll
    for (int m = 8; m > 0; m /= 2) sum += __shfl_xor(sum, m);
    if (in == 0) a.sums[blockIdx.x] = sum;
}

// The tokens' sum, or mean (0 of none), in 64 bits.
__global__ __launch_bounds__(1024) void sum_kernel(const int32_t *head, const double *parts, float *loss, int mean) {
    __shared__ double sums[16];
    const int labelled = head ? head[0] : 0;
    double sum = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < (labelled + 15) / 16; i += 1024) sum += parts[i];
#pragma unroll
    for (int m = 32; m > 0; m /= 2) sum += __shfl_xor(sum, m);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) sum += sums[i];
        *loss = (float)(mean ? sum / (labelled > 0 ? labelled : 1) : sum);
    }
}

// ---------------------------------------------------------------- gradients

struct BackwardArgs {
    Operands o;
    char *d;                   // [Np, ld]: a piece's
    int64_t d_bytes;           // how large it may be
    float *parts;              // [shares, labelled, K]
    int64_t parts_bytes;
    const float *g_loss;       // [1] or [N]
    float *coefficient;        // [labelled] or null: what d is multiplied with beside `factor`
    float *power;              // [1]: of both gradients, where there are coefficients
    float *weight_parts;       // [shares, vocabulary, K] and [shares, vocabulary] of the bias, where dW's sums may be cut
    float *bias_parts;
    int32_t *shares;           // [3]: of the vocabulary, for dh; pieces that there are; of the tokens, for dW (all from the first piece's launch)
    const float *hidden, *whole_weight;        // numbers that are far apart: the arrays as they were given, the labelled tokens
    int64_t hidden_stride, weight_stride;
    const int32_t *token;
    void *grad_hidden, *grad_weight, *grad_bias;
    int32_t bias_format, reduction, pieces, weight_shares;         // the last: at most
};

// Entries of a piece, whole tiles, that fit so many bytes.  d's rows are some more apart: rows at a distance of a power of two would share few of the cache's channels.
constexpr int APART = 64;
__host__ __device__ constexpr int64_t widest(int64_t bytes, int64_t rows, int planes) { return (bytes / (rows * 2 * planes) - APART) / TILE * TILE; }

// How a piece is laid out, from the number of labelled tokens, alike in every launch.
struct Piece {
    int v0, width, ld, nt;     // entries; numbers from row to row of d; tiles of tokens
    int steps;                 // of dh's sum over the entries of a whole piece
    int pieces;
};
template <typename F>
__device__ __forceinline__ Piece piece_of(const BackwardArgs &a, int labelled, int piece) {
    constexpr int K = STEP / F::PLANES;
    Piece p;
    p.nt = (labelled + TILE - 1) / TILE;
    const int64_t rows = max(p.nt, 1) * int64_t(TILE);
    const int tiles = int(a.o.s.Vp / TILE), most = (int)min(int64_t(tiles), widest(a.d_bytes, rows, F::PLANES) / TILE);
    p.pieces = (tiles + most - 1) / most;                  // as few as fit, and all alike
    const int whole = (tiles + p.pieces - 1) / p.pieces * TILE;
    p.ld = whole + APART;
    p.v0 = (int)min(int64_t(piece) * whole, int64_t(a.o.s.V));
    p.width = min(whole, a.o.s.V - p.v0);
    p.steps = (min(whole, a.o.s.V) + K - 1) / K;
    return p;
}

// A piece's tasks on the compute units: tiles of dW, steps_w steps each, go round, and the `more` first compute units have one more than the others; dh's tiles, whose sums over the
// entries can be cut anywhere, fill up: all compute units take `all` of its tasks, steps_h steps each, and those with a tile less of dW go on to `some`.
struct Balance {
    int more, all, some;
    int length, shorter, longer;               // steps of the units that take longer and of the others, whole rounds of dW aside; how many take longer
    __device__ __forceinline__ Balance(int weight_tasks, int steps_w, int hidden_tasks, int steps_h) {
        more = weight_tasks % COMPUTE_UNITS;
        length = INT32_MAX;
        for (int less = steps_w / steps_h, last = less + 1; less <= last; ++less) {       // tasks that a tile of dW is worth
            int s = (hidden_tasks + more * less + COMPUTE_UNITS - 1) / COMPUTE_UNITS, a = s - less;
            if (a < 0) a = 0, s = (hidden_tasks + COMPUTE_UNITS - more - 1) / (COMPUTE_UNITS - more);
            const int l1 = s * steps_h, l2 = a * steps_h + (more ? steps_w : 0), l = max(l1, l2);
            if (l < length) length = l, shorter = more ? min(l1, l2) : l1, longer = l2 == l ? more : COMPUTE_UNITS - more, all = a, some = s;
        }
    }
    // In steps of all compute units: those take 2.1 us, of power, and steps of a few units 1.3.
    __device__ __forceinline__ float cost() const {
        return shorter + (length - shorter) * (0.6f + 0.4f / COMPUTE_UNITS * longer);
    }
};

// How dW's sums over the tokens are cut: whole, or in shares of an even number of steps.
struct TokenShares {
    int steps, length, shares;
    // (rows and d have zeros behind the last token, up to a whole tile)
    template <typename F>
    static __device__ __forceinline__ TokenShares of(int labelled, int wanted) {
        constexpr int K = STEP / F::PLANES;
        const int steps = labelled ? max(2, (labelled + K - 1) / K) : 0;
        if (wanted <= 1 || steps == 0) return {steps, steps, 1};
        const int even = (steps + 1) / 2 * 2, length = (even + 2 * wanted - 1) / (2 * wanted) * 2;
        return {even, length, (even + length - 1) / length};
    }
};

// Into how many shares of the vocabulary dh's sums are cut, by how long a piece's launch takes and what the shares cost in memory; lane i looks at i + 1.  A step of all compute units takes
// 2.1 us, memory moves 5.1 TB/s.  (4915 labelled tokens, 50265 x 512: 9 shares are 253 steps, 10 in whole rounds were 314.)
// And into how many of the tokens dW's: the next power of two while that is 4 % better, the units that take longer priced as Balance's cost and memory as it was found beside products,
// 1.75 times as much.  (BF16: 32768 tokens, 1000 x 64, forward and backward 676 us whole and 129 cut; both gradients' sums of 65536 tokens, 50265 x 512, 12450 and 7170, of 32768 tokens 3630,
// and 4450 if cut.)
struct Shares {
    int vocabulary, tokens;
};
template <typename F>
__device__ __forceinline__ Shares shares_of(const BackwardArgs &a, int labelled) {
    const Piece p = piece_of<F>(a, labelled, 0);
    const int ht = (a.o.s.K + TILE - 1) / TILE, vt = (p.width + TILE - 1) / TILE, fit = (int)min(int64_t(SHARES), a.parts_bytes / (max(labelled, 1) * int64_t(a.o.s.K) * 4));
    const int n = threadIdx.x % 64 + 1, share = (p.steps + 2 * n - 1) / (2 * n) * 2, shares = (p.steps + share - 1) / share;
    Shares best{1, 1};
    float least = INFINITY;
    for (int w = 1; w <= a.weight_shares; w *= 2) {
        const TokenShares t = TokenShares::of<F>(labelled, w);
        const Balance b(vt * ht * t.shares, t.length, shares * p.nt * ht, share);      // (whether or not dW is wanted: the same bits)
        const float in_memory = (shares * (float)labelled + (t.shares > 1 ? t.shares * (float)p.width : 0.f)) * a.o.s.K * 7.5e-7f;
        const float cost = n > max(1, fit) ? INFINITY : b.length + in_memory;
        const int of = __ffsll((unsigned long long)__ballot(cost == wave_least(cost))) - 1;
        const float all = __shfl(vt * ht * t.shares / COMPUTE_UNITS * t.length + b.cost() + 1.75f * in_memory, of);
        if (all < 0.96f * least) least = all, best = {of + 1, w};
    }
    return best;
}

template <typename F>
__device__ __forceinline__ void put_shares(const BackwardArgs &a, int labelled, const Piece &p) {
    const Shares shares = shares_of<F>(a, labelled);
    if (threadIdx.x % 64 == 0) a.shares[0] = shares.vocabulary, a.shares[1] = p.pieces, a.shares[2] = shares.tokens;
}

// What both gradients' sums are multiplied with: of a sum or mean what all tokens' d are, nothing without any (whatever the loss's gradient is), else the power of two that their
// coefficients were divided by.
__device__ __forceinline__ float factor_of(const BackwardArgs &a, int labelled) {
    if (labelled == 0) return 0.f;
    if (a.coefficient) return *a.power;
    return *a.g_loss / (a.reduction == 1 ? (float)labelled : 1.f) * (1.f / LIFT);
}

// The range of the tokens' own gradients, RANGES workgroups' shares of the tokens.
__global__ __launch_bounds__(1024) void range_kernel(const int32_t *pos, const float *g_loss, int N, float2 *range) {
    __shared__ float high[16], low[16];
    const int tid = threadIdx.x;
    float most = 0.f, least = INFINITY;
#pragma unroll 4
    for (int n = blockIdx.x * 1024 + tid; n < N; n += RANGES * 1024) {
        const float g = pos[n] >= 0 ? fabsf(g_loss[n]) : 0.f;
        if (g > 0.f && g < INFINITY) most = fmaxf(most, g), least = fminf(least, g);
    }
    most = wave_most(most), least = wave_least(least);
    if (tid % 64 == 0) high[tid / 64] = most, low[tid / 64] = least;
    __syncthreads();
    if (tid > 0) return;
    for (int i = 1; i < 16; ++i) most = fmaxf(most, high[i]), least = fminf(least, low[i]);
    range[blockIdx.x] = make_float2(most, least);
}

// A block's 32 numbers of each column, 16 a lane (mfma_row), packed: w[k] has 16 bytes of column 16 k + lane % 16, the piece_of_lane-th of its four.  Lanes 32 apart and then lanes 16 apart
// exchange halves, so that what four lanes store of a row is 64 bytes together (32 bytes at a time took the cache twice as many writes).
__device__ __forceinline__ int piece_of_lane(int lane) { return lane / 16 % 2 * 2 + lane / 32; }
template <typename F>
__device__ __forceinline__ void pieces_of(const float (&l)[16], uint4 (&w)[2]) {
    uint32_t p[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const auto s = __builtin_amdgcn_permlane32_swap(F::pack2(l[8 * h + 2 * e], l[8 * h + 2 * e + 1]), F::pack2(l[8 * h + 4 + 2 * e], l[8 * h + 5 + 2 * e]), false, false);
            p[h][e] = s[0], p[h][2 + e] = s[1];
        }
    uint32_t q[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const auto s = __builtin_amdgcn_permlane16_swap(p[0][e], p[1][e], false, false);
        q[0][e] = s[0], q[1][e] = s[1];
    }
    w[0] = make_uint4(q[0][0], q[0][1], q[0][2], q[0][3]);
    w[1] = make_uint4(q[1][0], q[1][1], q[1][2], q[1][3]);
}

constexpr int FEW_ROWS = 2 * STEP;              // tokens that dW's sums over few have, at least
static_assert(FEW_ROWS >= FEW && FEW_ROWS <= TILE && FEW_ROWS == 2 * NARROW, "two steps; twice a narrow tile");

// d is rounded to the type of what it is multiplied with, as the matrix cores take operands of one type: two terms of it would be twice the products of both gradients.  What that costs is a
// rounding of each summand, 2^-9 or 2^-12 of it and of either sign (32768 x 512 half, the largest error of hidden's gradient 3.6e-4 of its largest number; with d in fp32 and the result
// rounded 2.4e-4).
template <typename F, typename S>
__device__ __forceinline__ void d_tiles(const BackwardArgs &a, const Piece &p, int labelled, uint32_t lds) {
    const Operands &o = a.o;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, half = lane / 32, wm = wave / S::N, wn = wave % S::N;
    const bool far = F::PLANES == 2 && far_apart(o);
    for_logits<F, S, true>(o, a.coefficient, labelled, p.v0, p.width, lds, [&](const Sums<S::MB, S::NB> &sums, const Place &tile, uint32_t beside_) {
        const int in = tile.v + wm * S::MB * 32;
        bool stored = false;
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            const int column = wn * S::NB * 32 + j * 32 + lane % 32, n = tile.n + column;
            const bool live = n < labelled;
            // (a token behind the last: exponentials of minus infinity, times zero)
            const float2 level = live ? beside<float2>(beside_, LEVEL, column) : make_float2(INFINITY, 0.f);
            const float by = LIFT * (a.coefficient ? beside<float>(beside_, COEFFICIENT, column) : 1.f), p_by = live ? level.y * by : 0.f, to_level = scale_of(level.x);
            const int at = live ? beside<int>(beside_, LABEL, column) - p.v0 - in : -1;
            const float row_scale = F::PLANES == 2 ? beside<float>(beside_, ROW_SCALE, column) : 1.f;
            char *const row = a.d + (int64_t(n - lane % 32 + lane % 16) * p.ld + in) * 2 * F::PLANES + 16 * piece_of_lane(lane);       // (of the block's first 16 tokens)
#pragma unroll
            for (int i = 0; i < S::MB; ++i) {
                float l[16];
                logits_of<F>(l, sums.v[i][j], beside_, (wm * S::MB + i) * 32, row_scale);
#pragma unroll
                for (int e = 0; e < 16; ++e) l[e] = __builtin_amdgcn_exp2f(fmaf(l[e], to_level, -level.x)) * p_by;
                const int r = at - 32 * i;
                if (r >= 0 && r < 32 && r / 4 % 2 == half) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) l[e] -= mfma_row(e, half) == r ? by : 0.f;
                }
                if (!stored) {
                    arrived();
                    stored = true;
                }
                if (far) {
                    float *const to = reinterpret_cast<float *>(a.d) + int64_t(n) * p.ld + in + 32 * i + 4 * half;
#pragma unroll
                    for (int g = 0; g < 4; ++g) *reinterpret_cast<float4 *>(to + 8 * g) = make_float4(l[4 * g], l[4 * g + 1], l[4 * g + 2], l[4 * g + 3]);
                    continue;
                }
                auto put = [&](char *to) {
                    uint4 w[2];
                    pieces_of<F>(l, w);
                    *reinterpret_cast<uint4 *>(to + 64 * F::PLANES * i) = w[0];
                    *reinterpret_cast<uint4 *>(to + 64 * F::PLANES * i + 32 * F::PLANES * int64_t(p.ld)) = w[1];
                };
                put(row);
                if constexpr (S::TOKENS < FEW_ROWS && F::PLANES == 1) {              // (dW's sums are two steps at least)
                    char *const behind = row + S::TOKENS * int64_t(p.ld) * 2 + 64 * i;
                    *reinterpret_cast<uint4 *>(behind) = *reinterpret_cast<uint4 *>(behind + 32 * int64_t(p.ld)) = make_uint4(0, 0, 0, 0);
                }
                if constexpr (F::PLANES == 2) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) l[e] -= (float)(_Float16)l[e];
                    put(row + 64);
                }
            }
        }
    });
}

template <typename F>
__global__ __launch_bounds__(THREADS, 2) void d_kernel(BackwardArgs a, int piece) {
    if (piece > 0 && piece >= a.shares[1]) return;
    extern __shared__ __attribute__((aligned(16))) uint4 lds_words[];
    const uint32_t lds = lds_byte_of(lds_words);
    const int labelled = a.o.kept.head[0];
    const Piece p = piece_of<F>(a, labelled, piece);
    if (labelled <= NARROW) d_tiles<F, NarrowLogits>(a, p, labelled, lds);
    else d_tiles<F, WideLogits>(a, p, labelled, lds);
    // (one of the workgroups that have the fewest tiles)
    if (piece == 0 && blockIdx.x == gridDim.x - 1 && threadIdx.x / 64 == 0) {
        put_shares<F>(a, labelled, p);
    }
}

// Eight numbers in the results' format.
template <typename R>
__device__ __forceinline__ void store8(char *to, const float (&v)[8]) {
    if constexpr (R::BYTES == 4) {
        *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4 *>(to + 16) = make_float4(v[4], v[5], v[6], v[7]);
    } else
        *reinterpret_cast<uint4 *>(to) = R::pack(v);
}

// d of few tokens from their logits: eight entries of a token a thread, zeros for the tokens behind (as far as dW's sums go; what dh's tile reads behind those is not stored).
template <typename F>
__global__ __launch_bounds__(256) void few_d_kernel(BackwardArgs a, int piece) {
    const int labelled = a.o.kept.head[0], n = blockIdx.y, V = a.o.s.V;
    const Piece p = piece_of<F>(a, labelled, piece);
    const bool far = F::PLANES == 2 && far_apart(a.o);
    if (piece == 0 && n == FEW_ROWS - 1 && blockIdx.x == 0 && threadIdx.x < 64) put_shares<F>(a, labelled, p);
    const int in = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 8;
    if (in >= p.ld - APART || p.width <= 0) return;
    float l[8] = {};
    if (n < labelled) {
        const float2 level = a.o.kept.level[n];
        const float by = LIFT * (a.coefficient ? a.coefficient[n] : 1.f), p_by = level.y * by, to_level = scale_of(level.x);
        const float *from = a.o.kept.logits + n * logits_stride(V) + p.v0 + in;
        const int at = a.o.kept.label[n] - p.v0 - in;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (in + 4 * g >= p.width) continue;               // (the last ones may be behind the vocabulary: within the row)
            const float4 v = *reinterpret_cast<const float4 *>(from + 4 * g);
            const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                l[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(w[e], to_level, -level.x)) * p_by - (at == 4 * g + e ? by : 0.f);
                if (in + 4 * g + e >= p.width) l[4 * g + e] = 0.f;
            }
        }
    }
    if (far) {
        store8<F32Row>(a.d + (int64_t(n) * p.ld + in) * 4, l);
        return;
    }
    char *const to = a.d + int64_t(n) * p.ld * 2 * F::PLANES + byte_of<F::PLANES>(in);
    auto put = [&](char *at) {
        *reinterpret_cast<uint4 *>(at) = make_uint4(F::pack2(l[0], l[1]), F::pack2(l[2], l[3]), F::pack2(l[4], l[5]), F::pack2(l[6], l[7]));
    };
    put(to);
    if constexpr (F::PLANES == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) l[e] -= (float)(_Float16)l[e];
        put(to + 64);
    }
}

__device__ __forceinline__ float dot_ones(BF16, uint4 u, float sum) {
    typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
    const pair_t one = {(__bf16)1.f, (__bf16)1.f};
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair_t, w[i]), one, sum, false);
    return sum;
}
__device__ __forceinline__ float dot_ones(F16, uint4 u, float sum) {
    typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
    const pair_t one = {(_Float16)1.f, (_Float16)1.f};
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair_t, w[i]), one, sum, false);
    return sum;
}

// dh: shares of the piece's entries x tiles of tokens x tiles of columns, one after the other; each adds to its own part.
template <typename F, int TOKENS>
__device__ __forceinline__ void hidden_tasks(const BackwardArgs &a, const Piece &p, int labelled, int piece, int unit, uint32_t lds) {
    typedef Along<TOKENS, THREADS, F::PLANES> Left;
    constexpr int MB = TOKENS / WAVES_M / 32;
    typedef Across<TILE, THREADS, F::PLANES> Right;
    const Operands &o = a.o;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, half = lane / 32, ht = (o.s.K + TILE - 1) / TILE;
    const Source d{a.d, int64_t(p.ld) * 2 * F::PLANES, p.nt * TILE, p.ld};
    Source w = o.weight;
    w.at += p.v0 * w.stride;
    w.rows = p.width;
    struct Task {
        int share, n, h, first, end;
        // (d has zeros behind the piece's last entry, up to a whole tile: an odd number of steps is followed by one of them)
        __device__ __forceinline__ Task(int id, const Piece &p, int ht, int length, int steps)
            : share(id / ht / p.nt), n(id / ht % p.nt * TILE), h(id % ht * TILE), first(share * length), end(min((steps + 1) / 2 * 2, first + length)) {}
    };
    // shares of an even number of steps, alike in all pieces; the last piece may have fewer
    const int wanted = *a.shares, length = (p.steps + 2 * wanted - 1) / (2 * wanted) * 2, steps = (p.width + Left::K - 1) / Left::K;
    const int tasks = (steps + length - 1) / length * p.nt * ht;
    const TokenShares of_weight = TokenShares::of<F>(labelled, a.shares[2]);
    const Balance balance(a.grad_weight ? (p.width + TILE - 1) / TILE * ht * of_weight.shares : 0, of_weight.length, tasks, length);
    const int rounds = unit < balance.more ? balance.all : balance.some;
    // a compute unit's round-th task: neighbours take neighbouring ones
    auto id_of = [&](int round) {
        return round < balance.all ? round * COMPUTE_UNITS + unit
                                   : balance.all * COMPUTE_UNITS + (round - balance.all) * (COMPUTE_UNITS - balance.more) + unit - balance.more;
    };
    if (rounds == 0 || id_of(0) >= tasks) return;
    int round = 0;
    Task task(id_of(0), p, ht, length, steps);
    Left left(d, task.n);
    Right right(w, task.h);
    Stream<F, MB, NB, Left, Right> stream(lds, wave / WAVES_N * MB * 32, wave % WAVES_N * NB * 32);
    stream.prime(left, right, task.first);
    for (;;) {
        const int next = id_of(round + 1);
        const bool more = round + 1 < rounds && next < tasks;
        const Task then(more ? next : id_of(round), p, ht, length, steps);
        const Left next_left(d, then.n);
        const Right next_right(w, then.h);
        Sums<MB, NB> sums;
        sums.clear();
        stream.multiply(sums, left, right, task.first, task.end, next_left, next_right, then.first, [](int, const uint4 &) {}, [] {});
        stream.landed();
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int h = task.h + (wave % WAVES_N * NB + j) * 32 + lane % 32;
            if (h >= o.s.K) continue;
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int n = task.n + (wave / WAVES_N * MB + i) * 32;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = n + mfma_row(e, half);
                    float *const at = a.parts + (int64_t(task.share) * labelled + row) * o.s.K + h;
                    if (row < labelled) *at = piece == 0 ? sums.v[i][j][e] : *at + sums.v[i][j][e];
                }
            }
        }
        if (!more) break;
        ++round, task = then;
    }
    stream.done();
}

__device__ __forceinline__ void put_bias(const BackwardArgs &a, int v, float sum) {
    if (a.bias_format == LFFN_ROWS_F32) static_cast<float *>(a.grad_bias)[v] = sum;
    else if (a.bias_format == LFFN_ROWS_BF16) static_cast<__bf16 *>(a.grad_bias)[v] = (__bf16)sum;
    else static_cast<_Float16 *>(a.grad_bias)[v] = (_Float16)sum;
}

// dW: shares of the tokens x tiles of the piece's entries x tiles of columns, and, with the first columns, db.
template <typename F, typename R>
__device__ __forceinline__ void weight_tasks(const BackwardArgs &a, const Piece &p, int labelled, int unit, uint32_t lds) {
    typedef Across<TILE, THREADS, F::PLANES> Side;
    const Operands &o = a.o;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, half = lane / 32, wm = wave / WAVES_N, wn = wave % WAVES_N, ht = (o.s.K + TILE - 1) / TILE;
    const Source rows = rows_of<F::PLANES>(o, labelled), d{a.d, int64_t(p.ld) * 2 * F::PLANES, p.nt * TILE, p.ld};
    const TokenShares shares = TokenShares::of<F>(labelled, a.shares[2]);
    const bool whole = shares.shares == 1;
    const float factor = factor_of(a, labelled), by = F::PLANES == 2 ? factor * __builtin_amdgcn_ldexpf(1.f, o.kept.head[1]) : factor;
    struct Task {
        int share, v, h, first, end;
        __device__ __forceinline__ Task(int id, int vt, int ht, const TokenShares &s)
            : share(id / ht / vt), v(id / ht % vt * TILE), h(id % ht * TILE), first(share * s.length), end(min(s.steps, first + s.length)) {}
    };
    const int vt = (p.width + TILE - 1) / TILE, tasks = shares.shares * vt * ht;
    int id = unit;
    if (id >= tasks) return;
    Task task(id, vt, ht, shares);
    Side left(rows, task.h), right(d, task.v);
    Stream<F, MB, NB, Side, Side> stream(lds, wm * MB * 32, wn * NB * 32);
    if (shares.steps) stream.prime(left, right, task.first);
    for (;;) {
        const bool more = id + COMPUTE_UNITS < tasks;
        const int v0 = task.v, h0 = task.h;
        if (more) id += COMPUTE_UNITS;
        const Task then(id, vt, ht, shares);
        const Side next_left(rows, then.h), next_right(d, then.v);
        Sums<MB, NB> sums;
        sums.clear();
        float bias[NB] = {};
        const bool of_bias = h0 == 0 && wm == 0 && a.grad_bias;
        if (shares.steps)
            stream.multiply(sums, left, right, task.first, task.end, next_left, next_right, then.first, [&](int j, const uint4 &u) {
                if (of_bias) bias[j] = dot_ones(F(), u, bias[j]);
            }, [] {});
        stream.landed();
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int in = v0 + (wn * NB + j) * 32 + lane % 32, v = p.v0 + in;
            const bool live = in < p.width;
            if (of_bias) {
                const float sum = (bias[j] + __shfl_xor(bias[j], 32)) * factor;
                if (half == 0 && live) {
                    if (!whole) a.bias_parts[int64_t(task.share) * o.s.V + v] = sum;
                    else put_bias(a, v, sum);
                }
            }
            if (R::BYTES == 2 && whole) {
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    float l[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) l[e] = sums.v[i][j][e] * by;
                    uint4 w[2];
                    pieces_of<F>(l, w);
                    const int h = h0 + (wm * MB + i) * 32 + 8 * piece_of_lane(lane), first = in - lane % 32 + lane % 16;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (first + 16 * k < p.width && h < o.s.K)
                            *reinterpret_cast<uint4 *>(static_cast<char *>(a.grad_weight) + (int64_t(p.v0 + first + 16 * k) * o.s.K + h) * 2) = w[k];
                }
                continue;
            }
            float *const row = whole ? static_cast<float *>(a.grad_weight) + int64_t(v) * o.s.K : a.weight_parts + (int64_t(task.share) * o.s.V + v) * o.s.K;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int g = 0; g < 4; g += 2) {
                    float t[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(sums.v[i][j][4 * g + e] * by), __float_as_uint(sums.v[i][j][4 * g + 4 + e] * by),
                                                                        false, false);
                        t[e] = __uint_as_float(s[0]), t[4 + e] = __uint_as_float(s[1]);
                    }
                    const int h = h0 + (wm * MB + i) * 32 + 8 * (g + half);
                    if (live && h < o.s.K) store8<F32Row>(reinterpret_cast<char *>(row + h), t);
                }
        }
        if (!more) break;
        task = then;
    }
    stream.done();
}

// ---------------------------------------------------------------- numbers that are far apart

// Products of floats as they are (v_mfma_f32_32x32x2_f32), 64 x 64 results a wavefront, operands from memory straight to its registers: 16 products, 1024 clocks, to 16 loads.  An instruction's two
// summed indices are four apart, so that four in a row are 16 bytes of d.  (Both directions with one token of 10^9 and without: 4096 x 50265 x 768 12.5 ms and 3.2, 385 x 32003 x 520 687 us and
// 300, 32768 x 1000 x 64 603 and 188.)  load(k, a, b): index k + 4 (lane / 32) + q of 32 i + lane % 32, zeros of b or a behind the last; of a share at least one.
template <typename Load, typename Seen>
__device__ __forceinline__ void far_products(f32x16_t (&sums)[2][2], int first, int end, Load &&load, Seen &&seen) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) sums[i][j][e] = 0.f;
    float a[2][2][4], b[2][2][4];
    auto form = [&](int at) {
        seen(b[at]);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) sums[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[at][i][q], b[at][j][q], sums[i][j], 0, 0, 0);
    };
    load(first, a[0], b[0]);
    for (int k = first; k < end; k += 16) {
        load(k + 8, a[1], b[1]);
        form(0);
        load(k + 16, a[0], b[0]);
        form(1);
    }
}

constexpr int FAR = 64, FAR_WAVES = COMPUTE_UNITS * THREADS / 64;

// dh in the shares of hidden_tasks.
template <typename F>
__device__ __forceinline__ void far_hidden(const BackwardArgs &a, const Piece &p, int labelled, int piece, int unit) {
    constexpr int STEPS_OF = STEP / F::PLANES;
    const Sizes &s = a.o.s;
    const int lane = threadIdx.x % 64, half = lane / 32, nt = (labelled + FAR - 1) / FAR, ht = (s.K + FAR - 1) / FAR;
    const int wanted = *a.shares, length = (p.steps + 2 * wanted - 1) / (2 * wanted) * 2, steps = (p.width + STEPS_OF - 1) / STEPS_OF, tasks = (steps + length - 1) / length * nt * ht;
    const float *const d = reinterpret_cast<const float *>(a.d);
    for (int id = unit * (THREADS / 64) + threadIdx.x / 64; id < tasks; id += FAR_WAVES) {
        const int share = id / ht / nt, n0 = id / ht % nt * FAR, h0 = id % ht * FAR, first = share * length * STEPS_OF, end = min(p.width, first + length * STEPS_OF);
        f32x16_t sums[2][2];
        far_products(sums, first, end, [&](int k, float (&x)[2][4], float (&w)[2][4]) {
            const int v = k + 4 * half;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // (behind the piece's last entry d has zeros up to a whole tile)
                float4 of = make_float4(0.f, 0.f, 0.f, 0.f);
                if (v < end) of = *reinterpret_cast<const float4 *>(d + int64_t(min(n0 + 32 * i + lane % 32, labelled - 1)) * p.ld + v);
                x[i][0] = of.x, x[i][1] = of.y, x[i][2] = of.z, x[i][3] = of.w;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float *const row = a.whole_weight + (p.v0 + min(v + q, p.width - 1)) * a.weight_stride;
#pragma unroll
                for (int j = 0; j < 2; ++j) w[j][q] = row[min(h0 + 32 * j + lane % 32, s.K - 1)];
            }
        }, [](const float (&)[2][4]) {});
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = h0 + 32 * j + lane % 32;
            if (h >= s.K) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = n0 + 32 * i + mfma_row(e, half);
                    float *const at = a.parts + (int64_t(share) * labelled + row) * s.K + h;
                    if (row < labelled) *at = piece == 0 ? sums[i][j][e] : *at + sums[i][j][e];
                }
        }
    }
}

// dW in the shares of weight_tasks, and, with the first columns, db.
template <typename F>
__device__ __forceinline__ void far_weight(const BackwardArgs &a, const Piece &p, int labelled, int unit) {
    constexpr int STEPS_OF = STEP / F::PLANES;
    const Sizes &s = a.o.s;
    const int lane = threadIdx.x % 64, half = lane / 32, vt = (p.width + FAR - 1) / FAR, ht = (s.K + FAR - 1) / FAR;
    const TokenShares shares = TokenShares::of<F>(labelled, a.shares[2]);
    const bool whole = shares.shares == 1;
    const float factor = factor_of(a, labelled);
    const float *const d = reinterpret_cast<const float *>(a.d);
    for (int id = unit * (THREADS / 64) + threadIdx.x / 64; id < shares.shares * vt * ht; id += FAR_WAVES) {
        const int share = id / ht / vt, v0 = id / ht % vt * FAR, h0 = id % ht * FAR, first = share * shares.length * STEPS_OF, end = min(labelled, first + shares.length * STEPS_OF);
        const bool of_bias = h0 == 0 && a.grad_bias;
        float bias[2] = {};
        f32x16_t sums[2][2];
        far_products(sums, first, end, [&](int k, float (&x)[2][4], float (&w)[2][4]) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = k + 4 * half + q, in = min(n, end - 1);
                const float *const row = a.hidden + a.token[in] * a.hidden_stride, *const of = d + int64_t(in) * p.ld + v0 + lane % 32;
#pragma unroll
                for (int i = 0; i < 2; ++i) x[i][q] = row[min(h0 + 32 * i + lane % 32, s.K - 1)];
#pragma unroll
                for (int j = 0; j < 2; ++j) w[j][q] = n < end ? of[32 * j] : 0.f;
            }
        }, [&](const float (&w)[2][4]) {
#pragma unroll
            for (int j = 0; j < 2; ++j) bias[j] += (w[j][0] + w[j][1]) + (w[j][2] + w[j][3]);
        });
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int in = v0 + 32 * j + lane % 32, v = p.v0 + in;
            const float sum = (bias[j] + __shfl_xor(bias[j], 32)) * factor;
            if (in >= p.width) continue;
            if (of_bias && half == 0) {
                if (!whole) a.bias_parts[int64_t(share) * s.V + v] = sum;
                else put_bias(a, v, sum);
            }
            float *const row = whole ? static_cast<float *>(a.grad_weight) + int64_t(v) * s.K : a.weight_parts + (int64_t(share) * s.V + v) * s.K;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int h = h0 + 32 * i + 8 * g + 4 * half;
                    if (h < s.K)
                        *reinterpret_cast<float4 *>(row + h) =
                            make_float4(sums[i][j][4 * g] * factor, sums[i][j][4 * g + 1] * factor, sums[i][j][4 * g + 2] * factor, sums[i][j][4 * g + 3] * factor);
                }
        }
    }
}

// Both gradients of a piece.
template <typename F, typename R>
__global__ __launch_bounds__(THREADS, 2) void gradients_kernel(BackwardArgs a, int piece) {
    if (piece > 0 && piece >= a.shares[1]) return;
    extern __shared__ __attribute__((aligned(16))) uint4 lds_words[];
    const uint32_t lds = lds_byte_of(lds_words);
    const int labelled = a.o.kept.head[0];
    const Piece p = piece_of<F>(a, labelled, piece);
    if (p.width <= 0) return;
    // (COMPUTE_UNITS workgroups; the units of an XCD have neighbouring numbers)
    const int unit = blockIdx.x % XCDS * (COMPUTE_UNITS / XCDS) + blockIdx.x / XCDS;
    if constexpr (F::PLANES == 2) {
        if (far_apart(a.o)) {
            if (a.grad_hidden) far_hidden<F>(a, p, labelled, piece, unit);
            if (a.grad_weight) far_weight<F>(a, p, labelled, unit);
            return;
        }
    }
    if (a.grad_hidden && labelled > NARROW) hidden_tasks<F, TILE>(a, p, labelled, piece, unit, lds);
    else if (a.grad_hidden && labelled) hidden_tasks<F, NARROW>(a, p, labelled, piece, unit, lds);
    if (a.grad_weight) weight_tasks<F, R>(a, p, labelled, unit, lds);
}

// dh: a labelled token's shares added up, zeros for the others; EACH threads for eight columns.
template <typename F, typename R, int EACH>
__global__ __launch_bounds__(256) void hidden_kernel(BackwardArgs a) {
    constexpr int PLACES = 256 / EACH;
    __shared__ float4 sums[EACH][EACH > 1 ? PLACES : 1][2];
    const Sizes &s = a.o.s;
    const int in = threadIdx.x % PLACES, part = threadIdx.x / PLACES, pieces = s.K / 8;
    const int64_t i = int64_t(blockIdx.x) * PLACES + in, t = i / pieces, c = i % pieces * 8;
    const int at = t < s.N ? a.o.kept.pos[t] : -1, labelled = a.o.kept.head[0];
    const bool far = F::PLANES == 2 && far_apart(a.o);
    float v[8] = {};
    auto add = [&](const float4 &x, const float4 &y) { v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w; };
    if (at >= 0) {
        const int steps = piece_of<F>(a, labelled, 0).steps, wanted = *a.shares, length = (steps + 2 * wanted - 1) / (2 * wanted) * 2, shares = (steps + length - 1) / length;
#pragma unroll 4
        for (int p = part; p < shares; p += EACH) {
            const float *from = a.parts + (int64_t(p) * labelled + at) * s.K + c;
            add(*reinterpret_cast<const float4 *>(from), *reinterpret_cast<const float4 *>(from + 4));
        }
    }
    if constexpr (EACH > 1) {
        sums[part][in][0] = make_float4(v[0], v[1], v[2], v[3]), sums[part][in][1] = make_float4(v[4], v[5], v[6], v[7]);
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int p = 1; p < EACH; ++p) add(sums[p][in][0], sums[p][in][1]);
    }
    if (t >= s.N) return;
    if (at >= 0) {
        const float by = factor_of(a, labelled) * (F::PLANES == 2 && !far ? __builtin_amdgcn_ldexpf(1.f, a.o.kept.head[2]) : 1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= by;
    }
    store8<R>(static_cast<char *>(a.grad_hidden) + (t * s.K + c) * R::BYTES, v);
}

// dW and db: shares added up, where there are any; a thread has eight columns or, in the workgroups behind, an entry's bias.
template <typename F, typename R>
__global__ __launch_bounds__(256) void weight_sum_kernel(BackwardArgs a) {
    const Sizes &s = a.o.s;
    const int shares = TokenShares::of<F>(a.o.kept.head[0], a.shares[2]).shares;
    if (shares == 1) return;
    const int64_t all = int64_t(s.V) * s.K, of_weight = (all / 8 + 255) / 256;
    if (blockIdx.x >= of_weight) {
        const int64_t v = (blockIdx.x - of_weight) * 256 + threadIdx.x;
        if (v >= s.V) return;
        float sum = 0.f;
#pragma unroll 8
        for (int i = 0; i < shares; ++i) sum += a.bias_parts[int64_t(i) * s.V + v];
        put_bias(a, (int)v, sum);
        return;
    }
    const int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 8;
    if (at >= all) return;
    float v[8] = {};
#pragma unroll 8
    for (int i = 0; i < shares; ++i) {
        const float4 x = *reinterpret_cast<const float4 *>(a.weight_parts + i * all + at), y = *reinterpret_cast<const float4 *>(a.weight_parts + i * all + at + 4);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    store8<R>(static_cast<char *>(a.grad_weight) + at * R::BYTES, v);
}

}  // namespace

// ---------------------------------------------------------------- C entries

namespace {

int planes_of(const lffn_linear_cross_entropy &a) { return a.format == LFFN_ROWS_F32 ? 2 : 1; }

int check(const lffn_linear_cross_entropy *a) {
    LFFN_REQUIRE(a, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->format >= 0 && a->format <= 2 && a->bias_format >= 0 && a->bias_format <= 2 && a->reduction >= 0 && a->reduction <= 2, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->tokens >= 0 && a->vocabulary >= 1 && a->columns >= 8, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->columns % 8 == 0 && a->columns <= 65536 && a->tokens <= (1 << 24) && a->vocabulary <= (1 << 22) && a->tokens * a->columns <= int64_t(1) << 32,
                 LFFN_ERR_UNSUPPORTED);
    const int64_t size = a->format == LFFN_ROWS_F32 ? 4 : 2, most = int64_t(1) << 22;
    LFFN_REQUIRE(a->weight && lffn_aligned16(a->weight) && a->weight_stride >= a->columns && a->weight_stride * size % 16 == 0, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->tokens == 0 || (a->hidden && a->labels), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(lffn_aligned16(a->hidden) && a->hidden_stride >= 0 && a->hidden_stride * size % 16 == 0, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->weight_stride <= most, LFFN_ERR_UNSUPPORTED);
    return LFFN_OK;
}

// Takes pieces of a workspace one after the other; with base null it only counts.
struct Carver {
    char *base;
    int64_t used = 0;
    template <typename T>
    T *take(int64_t n) {
        T *const p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += up(n * (int64_t)sizeof(T), 256);
        return p;
    }
};

Operands operands(const lffn_linear_cross_entropy &a, Carver &c, bool split) {
    Operands o{};
    const int64_t Np = up(a.tokens, TILE);
    o.s = {(int)a.tokens, (int)a.vocabulary, (int)a.columns, up(a.columns, 2 * STEP), up(a.vocabulary, TILE)};
    const int planes = planes_of(a);
    o.rows = c.take<char>(Np * o.s.Kp * 2 * planes);
    o.bias = c.take<float>(o.s.Vp);
    o.weight = {static_cast<const char *>(a.weight), a.weight_stride * (planes == 2 ? 4 : 2), o.s.V, o.s.K};
    if (planes == 2) {
        o.weight_scale = c.take<float>(o.s.Vp);          // (of few tokens: two a workgroup, and two of the tokens)
        o.row_scale = c.take<float>(Np);
    }
    if (split) {
        const int64_t columns = up(a.columns, STEP / 2);
        o.weight = {c.take<char>(a.vocabulary * columns * 4), columns * 4, o.s.V, (int)columns};
    }
    return o;
}

struct Forward {
    ForwardArgs f;
    RowsArgs r;
    JoinArgs j;
    void *kept;
    float *logits;
    int32_t *counts, *groups;
};
int64_t carve(const lffn_linear_cross_entropy &a, char *base, bool with_kept, Forward &f) {
    Carver c{base};
    const int64_t Np = up(a.tokens, TILE);
    f = {};
    f.f.o = operands(a, c, a.format == LFFN_ROWS_F32 && !few_tokens(a));
    f.f.Np = f.j.Np = Np;
    f.j.tiles = int((a.vocabulary + TILE - 1) / TILE);
    f.j.parts = f.f.parts = c.take<float2>((few_tokens(a) ? few_workgroups(a) : f.j.tiles) * Np);
    f.j.at_label = f.f.at_label = c.take<float>(Np);
    f.j.sums = c.take<double>(Np / 16);
    f.j.token = f.r.token = c.take<int32_t>(Np);
    f.counts = c.take<int32_t>(a.tokens / CHUNK + 1);
    f.groups = c.take<int32_t>(a.tokens / COUNTED + 1);
    f.kept = with_kept ? c.take<char>(kept_bytes(a, false)) : nullptr;
    return c.used;
}

struct Backward {
    BackwardArgs b;
    RowsArgs r;
};
int64_t carve(const lffn_linear_cross_entropy &a, char *base, Backward &w) {
    Carver c{base};
    w = {};
    const int64_t Np = up(a.tokens, TILE), planes = planes_of(a), K = a.columns;
    BackwardArgs &b = w.b;
    b.o = operands(a, c, planes == 2);
    const int64_t Vp = b.o.s.Vp, least = Np * ((Vp < 2048 ? Vp : 2048) + APART) * 2 * planes, whole = Np * (Vp + APART) * 2 * planes;
    b.d_bytes = least > D_BYTES ? least : whole < D_BYTES ? whole : D_BYTES;
    b.d = c.take<char>(b.d_bytes);
    const int64_t one = a.tokens * K * 4;
    b.parts_bytes = one > PARTS_BYTES ? one : one * SHARES < PARTS_BYTES ? one * SHARES : PARTS_BYTES;
    b.parts = c.take<float>(b.parts_bytes / 4);
    b.coefficient = c.take<float>(a.reduction == 0 ? Np : 0);
    float2 *const range = c.take<float2>(a.reduction == 0 ? RANGES : 0);
    b.power = c.take<float>(1);
    b.shares = c.take<int32_t>(3);
    if (planes == 2) b.token = w.r.token = c.take<int32_t>(Np);
    if (a.reduction == 0) b.o.range = range, w.r.coefficient = b.coefficient, w.r.power = b.power;
    else b.coefficient = nullptr;
    // as many launches as pieces if all tokens are labelled; with fewer the last ones find nothing
    const int64_t entries = a.tokens == 0 ? 0 : widest(b.d_bytes, Np, (int)planes);
    b.pieces = a.tokens == 0 ? 0 : int((a.vocabulary + entries - 1) / entries);
    // dW's sums may be cut into as many shares as a piece's tiles leave compute units without one, if a sum is long enough to be worth a launch
    const int64_t each = b.pieces == 0 ? 0 : (Vp / TILE + b.pieces - 1) / b.pieces * ((K + TILE - 1) / TILE), rows = a.vocabulary * (K + 1) * 4;
    const bool cut = b.pieces > 0 && a.tokens * planes >= CUT_FROM && each * 2 <= COMPUTE_UNITS;
    const int64_t most = cut ? min(min(int64_t(SHARES), COMPUTE_UNITS / each), WEIGHT_PARTS_BYTES / rows) : 1;
    b.weight_shares = 1;
    while (b.weight_shares * 2 <= most) b.weight_shares *= 2;
    if (b.weight_shares > 1) {
        b.weight_parts = c.take<float>(b.weight_shares * a.vocabulary * K);
        b.bias_parts = c.take<float>(b.weight_shares * a.vocabulary);
    }
    return c.used;
}

void fill(RowsArgs &r, const lffn_linear_cross_entropy &a, const Operands &o) {
    r.o = o;
    r.hidden = a.hidden, r.labels = a.labels, r.bias = a.bias;
    r.hidden_stride = a.hidden_stride, r.ignore = a.ignore_index;
    r.labels_64 = a.labels_64, r.bias_format = a.bias ? a.bias_format : -1;
    r.parts = a.tokens > COUNTED ? 4 : 16;         // (few tokens: a row a wavefront; 385 x 520 fp32 6.5 us, by four 12.8)
}

template <bool BACKWARD>
void launch_rows(const lffn_linear_cross_entropy &a, const RowsArgs &r, hipStream_t st) {
    const dim3 grid(unsigned((a.tokens + CHUNK - 1) / CHUNK * r.parts + (r.o.s.Vp + 255) / 256));
    if (a.format == LFFN_ROWS_F32) {
        weight_kernel<BACKWARD><<<dim3(unsigned(r.o.s.Vp / 4)), dim3(256), 0, st>>>(r.o, static_cast<const float *>(a.weight), a.weight_stride);
        rows_kernel<F32Row, 2, BACKWARD><<<grid, dim3(256), 0, st>>>(r);
    } else
        rows_kernel<F16Row, 1, BACKWARD><<<grid, dim3(256), 0, st>>>(r);
}

unsigned workgroups(int64_t tiles) { return unsigned(tiles >= COMPUTE_UNITS ? COMPUTE_UNITS : up(tiles, XCDS)); }

constexpr size_t LDS_BYTES = STREAM_LDS + 2 * BESIDE_BYTES + WAVES_M * TILE * sizeof(float2);

template <typename F, int TOKENS>
int few(const lffn_linear_cross_entropy &a, Forward &f, hipStream_t st) {
    static LdsGrant granted;
    const int64_t lds = few_lds(a.tokens, row_bytes(a));
    if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&few_kernel<F, TOKENS>), lds, granted)) return LFFN_ERR_LAUNCH;
    f.j.tiles = few_workgroups(a);
    few_kernel<F, TOKENS><<<dim3(f.j.tiles), dim3(THREADS), lds, st>>>({f.r, f.f.parts, f.f.at_label, f.logits, f.f.Np});
    return LFFN_OK;
}
template <typename F>
int few(const lffn_linear_cross_entropy &a, Forward &f, hipStream_t st) {
    return a.tokens <= 32 ? few<F, 32>(a, f, st) : few<F, 64>(a, f, st);
}

template <typename F>
int forward(const Forward &f, hipStream_t st) {
    static LdsGrant granted;
    if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&forward_kernel<F>), LDS_BYTES, granted)) return LFFN_ERR_LAUNCH;
    forward_kernel<F><<<dim3(workgroups(f.j.tiles * (f.f.Np / TILE))), dim3(THREADS), LDS_BYTES, st>>>(f.f);
    return LFFN_OK;
}

template <typename F, typename R>
int backward(const BackwardArgs &b, hipStream_t st) {
    static LdsGrant granted_d, granted_g;
    if (!lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&d_kernel<F>), LDS_BYTES, granted_d) ||
        !lffn_grant_dynamic_lds(reinterpret_cast<const void *>(&gradients_kernel<F, R>), STREAM_LDS, granted_g))
        return LFFN_ERR_LAUNCH;
    for (int p = 0; p < b.pieces; ++p) {
        if (b.o.kept.logits) {
            const int64_t widest_piece = up((b.o.s.Vp / TILE + b.pieces - 1) / b.pieces * TILE, 2048);
            few_d_kernel<F><<<dim3(unsigned(widest_piece / 2048), FEW_ROWS), dim3(256), 0, st>>>(b, p);
        } else
            d_kernel<F><<<dim3(COMPUTE_UNITS), dim3(THREADS), LDS_BYTES, st>>>(b, p);
        gradients_kernel<F, R><<<dim3(COMPUTE_UNITS), dim3(THREADS), STREAM_LDS, st>>>(b, p);
    }
    if (b.grad_hidden) {
        const int64_t n = int64_t(b.o.s.N) * (b.o.s.K / 8);
        // four threads where one each would leave the chip without enough in flight (385 x 520 fp32 16.4 us with one, 11.4 with four; 32768 x 512, 4915 labelled, half 27 and 36)
        if (n < COMPUTE_UNITS * 256) hidden_kernel<F, R, 4><<<dim3(unsigned((n + 63) / 64)), dim3(256), 0, st>>>(b);
        else hidden_kernel<F, R, 1><<<dim3(unsigned((n + 255) / 256)), dim3(256), 0, st>>>(b);
    }
    if (b.grad_weight && b.weight_shares > 1) {
        const int64_t n = int64_t(b.o.s.V) * (b.o.s.K / 8), of_bias = b.grad_bias ? (b.o.s.V + 255) / 256 : 0;
        weight_sum_kernel<F, R><<<dim3(unsigned((n + 255) / 256 + of_bias)), dim3(256), 0, st>>>(b);
    }
    return LFFN_OK;
}

}  // namespace

extern "C" int lffn_linear_cross_entropy_kept_bytes(const lffn_linear_cross_entropy *a, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    const int rc = check(a);
    if (rc == LFFN_OK) *bytes = kept_bytes(*a, few_tokens(*a));
    return rc;
}

extern "C" int lffn_linear_cross_entropy_workspace_bytes(const lffn_linear_cross_entropy *a, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    const int rc = check(a);
    Forward f;
    if (rc == LFFN_OK) *bytes = carve(*a, nullptr, true, f);
    return rc;
}

extern "C" int lffn_linear_cross_entropy_fwd(const lffn_linear_cross_entropy *a, float *loss, void *kept, void *workspace, int64_t workspace_bytes, void *stream) {
    const int rc = check(a);
    if (rc != LFFN_OK) return rc;
    LFFN_REQUIRE(loss || (a->reduction == 0 && a->tokens == 0), LFFN_ERR_BAD_ARG);
    Forward f;
    LFFN_REQUIRE(workspace && lffn_aligned16(workspace) && workspace_bytes >= carve(*a, static_cast<char *>(workspace), true, f), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(lffn_aligned16(kept), LFFN_ERR_BAD_ARG);
    if (a->reduction == 0 && a->tokens == 0) return LFFN_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    f.f.o.kept = f.j.kept = kept_at(*a, kept ? kept : f.kept);
    f.logits = kept ? f.f.o.kept.logits : nullptr;
    fill(f.r, *a, f.f.o);
    if (a->reduction == 0) f.j.loss = f.r.loss = loss, f.j.sums = nullptr;
    // (workgroups that look for the largest and the least scales behind those that join)
    const int looking = a->format == LFFN_ROWS_F32 ? 2 * LOOKING : 0;
    f.j.weight_scale = f.f.o.weight_scale, f.j.row_scale = f.f.o.row_scale;
    if (a->tokens > 0 && few_tokens(*a)) {
        const int done = a->format == LFFN_ROWS_F32 ? few<F32Row>(*a, f, st) : a->format == LFFN_ROWS_BF16 ? few<BF16>(*a, f, st) : few<F16>(*a, f, st);
        if (done != LFFN_OK) return done;
        f.j.joining = int((a->tokens + 15) / 16), f.j.entries = 2 * f.j.tiles, f.j.few = 1;
        join_kernel<<<dim3(f.j.joining + looking), dim3(256), 0, st>>>(f.j);
    } else if (a->tokens > 0) {
        if (a->tokens > COUNTED) {
            count_kernel<<<dim3(unsigned((a->tokens + COUNTED - 1) / COUNTED)), dim3(1024), 0, st>>>(a->labels, a->labels_64, a->ignore_index, f.f.o.s.V, f.f.o.s.N, f.counts, f.groups);
            f.r.counts = f.counts, f.r.groups = f.groups;
        }
        launch_rows<false>(*a, f.r, st);
        const int done = a->format == LFFN_ROWS_F32 ? forward<F32Two>(f, st) : a->format == LFFN_ROWS_BF16 ? forward<BF16>(f, st) : forward<F16>(f, st);
        if (done != LFFN_OK) return done;
        f.j.joining = int(f.f.Np / 16), f.j.entries = (int)a->vocabulary;
        join_kernel<<<dim3(f.j.joining + looking), dim3(256), 0, st>>>(f.j);
    }
    if (a->reduction != 0) sum_kernel<<<dim3(1), dim3(1024), 0, st>>>(a->tokens > 0 ? f.f.o.kept.head : nullptr, f.j.sums, loss, a->reduction == 1);
    return lffn_launch_status();
}

extern "C" int lffn_linear_cross_entropy_bwd_workspace_bytes(const lffn_linear_cross_entropy *a, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    const int rc = check(a);
    Backward w;
    if (rc == LFFN_OK) *bytes = carve(*a, nullptr, w);
    return rc;
}

extern "C" int lffn_linear_cross_entropy_bwd(const lffn_linear_cross_entropy *a, const void *kept, const float *g_loss, void *grad_hidden, void *grad_weight,
                                             void *grad_bias, void *workspace, int64_t workspace_bytes, void *stream) {
    const int rc = check(a);
    if (rc != LFFN_OK) return rc;
    LFFN_REQUIRE(a->tokens >= 1, LFFN_ERR_UNSUPPORTED);
    LFFN_REQUIRE(kept && g_loss && lffn_aligned16(kept) && lffn_aligned16(grad_hidden) && lffn_aligned16(grad_weight), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(grad_weight || !grad_bias, LFFN_ERR_BAD_ARG);
    Backward w;
    LFFN_REQUIRE(workspace && lffn_aligned16(workspace) && workspace_bytes >= carve(*a, static_cast<char *>(workspace), w), LFFN_ERR_BAD_ARG);
    hipStream_t st = static_cast<hipStream_t>(stream);
    BackwardArgs &b = w.b;
    b.o.kept = kept_at(*a, const_cast<void *>(kept));
    b.g_loss = g_loss;
    b.grad_hidden = grad_hidden, b.grad_weight = grad_weight, b.grad_bias = grad_bias;
    b.bias_format = a->bias_format, b.reduction = a->reduction;
    b.hidden = static_cast<const float *>(a->hidden), b.whole_weight = static_cast<const float *>(a->weight);
    b.hidden_stride = a->hidden_stride, b.weight_stride = a->weight_stride;
    fill(w.r, *a, b.o);
    w.r.g_loss = g_loss;
    if (a->reduction == 0) range_kernel<<<dim3(RANGES), dim3(1024), 0, st>>>(b.o.kept.pos, g_loss, (int)a->tokens, const_cast<float2 *>(b.o.range));
    launch_rows<true>(*a, w.r, st);
    const int done = a->format == LFFN_ROWS_F32    ? backward<F32Two, F32Row>(b, st)
                     : a->format == LFFN_ROWS_BF16 ? backward<BF16, BF16Row>(b, st)
                                                   : backward<F16, F16Row>(b, st);
    return done != LFFN_OK ? done : lffn_launch_status();
}
