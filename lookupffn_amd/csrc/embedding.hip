// Rows of an embedding table by token number, and the table's gradient:
//
//   out[n] = s W[id_n],   dW[r] = s sum of g[n] over the tokens n with id_n = r
//
// Both are bound by memory.  Backward: the tokens are sorted by their numbers (stable, 9 bits a pass: a launch that counts and one that sorts; up to 2048 tokens one launch for all), their list is cut into pieces of equal
// length, whatever the numbers' frequencies, and a wavefront adds up a piece's runs of equal numbers, 16 bytes of a row a lane.  A run inside a piece is a row of the result; of one that
// passes a piece's end each piece leaves its part, and a last launch adds those.  While the tokens are sorted, on a few compute units, the others clear the table's gradient.
#include "rows16.h"

namespace {

constexpr int WG = 256;
constexpr int BITS = 9, DIGITS = 1 << BITS;
constexpr int SORT_WG = 1024, CHUNK = SORT_WG;      // tokens that a workgroup sorts, a thread each (two: 14.3 us for two passes over 32768 tokens instead of 13.1)
constexpr int ONE_MOST = 2;                  // tokens a thread has, at most, where one workgroup sorts all (2048 tokens 17.7 us with their sums; 4096 tokens would be 23.2 instead of 22.1)
constexpr int FILL_BYTES = 64 * 1024;        // of a workgroup that clears
constexpr int JOIN_WG = 512;

struct Args {
    const void *ids, *weight;
    void *out;
    int64_t stride;
    uint32_t tokens, rows, columns, pieces;      // pieces: of R::N columns
    int32_t ids_64;
    float scale;
};

// A token's row, or `rows`.
__device__ __forceinline__ uint32_t row_of(const void *ids, int wide, int64_t n, uint32_t rows) {
    const int64_t id = wide ? static_cast<const int64_t *>(ids)[n] : static_cast<const int32_t *>(ids)[n];
    return id >= 0 && id < int64_t(rows) ? (uint32_t)id : rows;
}

// LANES threads take a row, AHEAD of their 16 bytes (or numbers) at a time.
template <typename R, int LANES>
__global__ __launch_bounds__(WG) void forward_kernel(Args a) {
    constexpr int AHEAD = 4;
    const uint32_t n = blockIdx.x * (WG / LANES) + threadIdx.x / LANES, in = threadIdx.x % LANES;
    if (n >= a.tokens) return;
    const uint32_t row = row_of(a.ids, a.ids_64, n, a.rows);
    const bool there = row < a.rows;
    const char *from = static_cast<const char *>(a.weight) + (there ? row * a.stride : 0) * R::BYTES;
    char *to = static_cast<char *>(a.out) + int64_t(n) * a.columns * R::BYTES;
    constexpr int SIZE = R::N * R::BYTES;
    for (uint32_t p0 = in; p0 < a.pieces; p0 += AHEAD * LANES) {
        typename R::raw_t raw[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (p0 + k * LANES < a.pieces && there) raw[k] = *reinterpret_cast<const typename R::raw_t *>(from + int64_t(p0 + k * LANES) * SIZE);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (p0 + k * LANES >= a.pieces) continue;
            float v[R::N] = {};
            if (there) {
                R::unpack(raw[k], v);
#pragma unroll
                for (int i = 0; i < R::N; ++i) v[i] *= a.scale;
            }
            *reinterpret_cast<typename R::raw_t *>(to + int64_t(p0 + k * LANES) * SIZE) = R::pack(v);
        }
    }
}

// ---------------------------------------------------------------- sorting

struct Fill {
    char *at;                  // this launch's share: 16-byte pieces, and what is left of fewer bytes
    int64_t bytes;
};

struct SortArgs {
    const void *ids;
    int64_t padding;
    const uint2 *from;         // (row, token), or null: the tokens themselves
    uint2 *to;
    int32_t *counts;           // [chunks][DIGITS]: this pass's
    uint32_t tokens, rows;
    int chunks, shift, ids_64;
    int scanned;               // counts are those of the chunks before, and behind the last chunk's all
    Fill fill;
};

__device__ __forceinline__ uint2 entry(const SortArgs &a, uint32_t i) {
    if (a.from) return a.from[i];
    const uint32_t row = row_of(a.ids, a.ids_64, i, a.rows);
    return make_uint2(int64_t(row) == a.padding ? a.rows : row, i);
}

// A workgroup behind the sorting ones: 64 KB of zeros.
__device__ __forceinline__ void clear(const Fill &f, int64_t workgroup) {
    const int64_t first = workgroup * FILL_BYTES, end = min(first + FILL_BYTES, f.bytes);
    for (int64_t i = first + threadIdx.x * 16; i + 16 <= end; i += SORT_WG * 16) *reinterpret_cast<uint4 *>(f.at + i) = make_uint4(0, 0, 0, 0);
    if (end == f.bytes && threadIdx.x < f.bytes % 16 / 2) reinterpret_cast<uint16_t *>(f.at + f.bytes / 16 * 16)[threadIdx.x] = 0;
}

// How often a chunk has each of a pass's digits.
__global__ __launch_bounds__(SORT_WG) void count_kernel(SortArgs a) {
    if ((int)blockIdx.x >= a.chunks) return clear(a.fill, blockIdx.x - a.chunks);
    __shared__ int32_t count[DIGITS];
    if (threadIdx.x < DIGITS) count[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t i = blockIdx.x * uint32_t(CHUNK) + threadIdx.x;
    if (i < a.tokens) atomicAdd(&count[entry(a, i).x >> a.shift & (DIGITS - 1)], 1);
    __syncthreads();
    if (threadIdx.x < DIGITS) a.counts[int64_t(blockIdx.x) * DIGITS + threadIdx.x] = count[threadIdx.x];
}

// Many chunks (each reading all counts would be as much as the square of them): counts become those of the chunks before, and of all behind the last one.  16 digits a workgroup, 64 threads each.
constexpr int SCANNED_FROM = 128;            // (a backward of 131072 tokens x 64 57 us without and with, 262144 93 and 80, 1048576 293 and 127)
__global__ __launch_bounds__(SORT_WG) void scan_kernel(int32_t *counts, int chunks) {
    __shared__ int32_t sums[SORT_WG / 16][17];
    const int in = threadIdx.x % 16, slice = threadIdx.x / 16, share = (chunks + SORT_WG / 16 - 1) / (SORT_WG / 16), first = min(slice * share, chunks), end = min(first + share, chunks);
    int32_t *const at = counts + blockIdx.x * 16 + in;
    int sum = 0;
#pragma unroll 8
    for (int c = first; c < end; ++c) sum += at[int64_t(c) * DIGITS];
    sums[slice][in] = sum;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < slice; ++i) before += sums[i][in];
    for (int c = first; c < end; ++c) {
        const int n = at[int64_t(c) * DIGITS];
        at[int64_t(c) * DIGITS] = before;
        before += n;
    }
    if (slice == SORT_WG / 16 - 1) at[int64_t(chunks) * DIGITS] = before;
}

// What a workgroup needs to put a chunk's entries in the order of a digit.
struct Sorter {
    int32_t place[DIGITS];                     // where a digit's entries of this chunk begin
    int32_t had[SORT_WG / 64][DIGITS];         // how many of a digit a wavefront has had
    int32_t total[DIGITS / 64];
};

// A thread's entries are numbers (wave * EACH + k) * 64 + lane of the chunk: -> which of its digit's an entry is within its wavefront.
template <int EACH>
__device__ __forceinline__ void rank_entries(Sorter &s, const uint2 (&e)[EACH], const bool (&live)[EACH], int shift, int (&rank)[EACH]) {
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    for (int d = lane; d < DIGITS; d += 64) s.had[wave][d] = 0;
    __builtin_amdgcn_wave_barrier();           // (a wavefront's LDS accesses keep their order)
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const uint32_t digit = e[k].x >> shift & (DIGITS - 1);
        // the lanes of the same digit
        uint64_t same = __ballot(live[k]);
#pragma unroll
        for (int b = 0; b < BITS; ++b) {
            const uint64_t set = __ballot(digit >> b & 1);
            same &= digit >> b & 1 ? set : ~set;
        }
        const int earlier = __popcll(same & ((uint64_t(1) << lane) - 1));
        rank[k] = live[k] ? s.had[wave][digit] + earlier : 0;
        __builtin_amdgcn_wave_barrier();
        if (live[k] && earlier == 0) s.had[wave][digit] = rank[k] + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// A digit's entries in all chunks (thread d's) -> where they begin.  Barriers inside.
__device__ __forceinline__ int begin_of_digit(Sorter &s, int all) {
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    int upto = all;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const int v = __shfl_up(upto, m);
        if (lane >= m) upto += v;
    }
    if (threadIdx.x < DIGITS && lane == 63) s.total[wave] = upto;
    __syncthreads();
    if (threadIdx.x < DIGITS)
        for (int w = 0; w < wave; ++w) upto += s.total[w];
    return upto - all;
}

__device__ __forceinline__ int place_of(const Sorter &s, uint32_t digit, int rank) {
    int at = s.place[digit] + rank;
    for (int w = 0; w < (int)threadIdx.x / 64; ++w) at += s.had[w][digit];
    return at;
}

// One pass: a chunk's entries go to their places, those of a digit in the order they had.
__global__ __launch_bounds__(SORT_WG) void sort_kernel(SortArgs a) {
    if ((int)blockIdx.x >= a.chunks) return clear(a.fill, blockIdx.x - a.chunks);
    __shared__ Sorter s;
    const int tid = threadIdx.x;
    uint2 e[1];
    bool live[1];
    int rank[1];
    const uint32_t i = blockIdx.x * uint32_t(CHUNK) + tid;
    live[0] = i < a.tokens;
    e[0] = live[0] ? entry(a, i) : make_uint2(0, 0);
    // a digit's entries in the chunks before this one and in all
    int before = 0, all = 0;
    if (tid < DIGITS && a.scanned) {
        before = a.counts[int64_t(blockIdx.x) * DIGITS + tid];
        all = a.counts[int64_t(a.chunks) * DIGITS + tid];
    } else if (tid < DIGITS) {
#pragma unroll 8
        for (int c = 0; c < a.chunks; ++c) {
            const int n = a.counts[int64_t(c) * DIGITS + tid];
            if (c < (int)blockIdx.x) before += n;
            all += n;
        }
    }
    const int begin = begin_of_digit(s, all);
    if (tid < DIGITS) s.place[tid] = begin + before;
    rank_entries(s, e, live, a.shift, rank);
    __syncthreads();
    if (live[0]) a.to[place_of(s, e[0].x >> a.shift & (DIGITS - 1), rank[0])] = e[0];
}

// All passes of EACH * SORT_WG tokens, by one workgroup in LDS.
template <int EACH>
__global__ __launch_bounds__(SORT_WG) void sort_one_kernel(SortArgs a, int passes) {
    if (blockIdx.x >= 1) return clear(a.fill, blockIdx.x - 1);
    __shared__ Sorter s;
    __shared__ uint2 list[EACH * SORT_WG];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    uint2 e[EACH];
    bool live[EACH];
    int rank[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const uint32_t i = (wave * EACH + k) * 64 + lane;
        live[k] = i < a.tokens;
        e[k] = live[k] ? entry(a, i) : make_uint2(0, 0);
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * BITS;
        rank_entries(s, e, live, shift, rank);
        __syncthreads();
        int all = 0;
        if (tid < DIGITS)
#pragma unroll
            for (int w = 0; w < SORT_WG / 64; ++w) all += s.had[w][tid];
        const int begin = begin_of_digit(s, all);
        if (tid < DIGITS) s.place[tid] = begin;
        __syncthreads();
        uint2 *const to = p + 1 < passes ? list : a.to;
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if (live[k]) to[place_of(s, e[k].x >> shift & (DIGITS - 1), rank[k])] = e[k];
        __syncthreads();
        if (p + 1 < passes) {
#pragma unroll
            for (int k = 0; k < EACH; ++k)
                if (live[k]) e[k] = list[(wave * EACH + k) * 64 + lane];
        }
    }
}

// ---------------------------------------------------------------- sums

struct SumArgs {
    const uint2 *list;
    const void *g;
    void *grad;
    float *parts;              // [pieces][2][columns]: of the run that came in, of the one that goes out
    uint32_t tokens, rows, columns, vectors;
    int length;                // of a piece
    int64_t pieces;
    float scale;
};

template <typename R>
__device__ __forceinline__ void put_row(const SumArgs &a, uint32_t row, uint32_t vector, float (&sum)[R::N]) {
#pragma unroll
    for (int i = 0; i < R::N; ++i) sum[i] *= a.scale;
    *reinterpret_cast<typename R::raw_t *>(static_cast<char *>(a.grad) + (int64_t(row) * a.columns + int64_t(vector) * R::N) * R::BYTES) = R::pack(sum);
}

// A wavefront a piece and 64 vectors of its rows.
template <typename R>
__global__ __launch_bounds__(WG) void sum_kernel(SumArgs a) {
    constexpr int N = R::N, AHEAD = 8;
    const int64_t piece = int64_t(blockIdx.x) * (WG / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (piece >= a.pieces) return;
    const uint32_t lane = threadIdx.x % 64, vector = blockIdx.y * 64 + lane, at = min(vector, a.vectors - 1);
    const uint32_t first = uint32_t(piece) * a.length, end = min(first + uint32_t(a.length), a.tokens);
    const uint32_t came = first > 0 ? a.list[first - 1].x : a.rows, goes = end < a.tokens ? a.list[end].x : a.rows;
    const bool live = vector < a.vectors;
    float sum[N] = {};
    uint32_t now = a.list[first].x;
    bool from_before = now == came && now < a.rows;
    auto flush = [&](bool goes_on) {
        if (!live || now >= a.rows) return;
        if (from_before || goes_on) {
            float *to = a.parts + (piece * 2 + (from_before ? 0 : 1)) * a.columns + int64_t(vector) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) to[i] = sum[i];
        } else
            put_row<R>(a, now, vector, sum);
    };
    for (uint32_t i = first; i < end; i += AHEAD) {
        uint2 e[AHEAD];
        typename R::raw_t raw[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) e[k] = a.list[min(i + k, end - 1)];
        if (e[0].x >= a.rows) break;                   // sorted behind all rows: nothing more
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            raw[k] = *reinterpret_cast<const typename R::raw_t *>(static_cast<const char *>(a.g) + (int64_t(e[k].y) * a.columns + int64_t(at) * N) * R::BYTES);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (i + k >= end) break;
            const uint32_t row = __builtin_amdgcn_readfirstlane(e[k].x);
            if (row != now) {
                flush(false);
                now = row;
                from_before = false;
#pragma unroll
                for (int c = 0; c < N; ++c) sum[c] = 0.f;
            }
            float v[N];
            R::unpack(raw[k], v);
#pragma unroll
            for (int c = 0; c < N; ++c) sum[c] += v[c];
        }
    }
    flush(now == goes);
}

// The run that goes out of piece blockIdx.x, if one does: its part there and those of the pieces that it came into.
template <typename R>
__global__ __launch_bounds__(JOIN_WG) void join_kernel(SumArgs a) {
    constexpr int N = R::N, WAVES = JOIN_WG / 64;
    __shared__ float red[WAVES][64 * N];
    const int64_t piece = blockIdx.x;
    const uint32_t end = uint32_t(piece + 1) * a.length;             // (less than the tokens: there is a piece behind)
    const uint32_t row = a.list[end - 1].x;
    if (row >= a.rows || a.list[end].x != row) return;
    const uint32_t first = uint32_t(piece) * a.length;
    if (first > 0 && a.list[first - 1].x == row) return;             // it came in: an earlier piece's
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    // pieces that it came into
    int64_t more = 0;
    for (;;) {
        const int64_t next = piece + 1 + more + lane;
        const uint64_t in = __ballot(next < a.pieces && a.list[next * a.length].x == row);
        const int run = in == ~uint64_t(0) ? 64 : __ffsll((unsigned long long)~in) - 1;
        more += run;
        if (run < 64) break;
    }
    const uint32_t vector = blockIdx.y * 64 + lane, at = min(vector, a.vectors - 1);
    float sum[N] = {};
    const float *from = a.parts + int64_t(at) * N;
    // the parts one after the other, a wavefront's together
    const int64_t all = more + 1, share = (all + WAVES - 1) / WAVES, last = min(all, (wave + 1) * share);
#pragma unroll 4
    for (int64_t k = wave * share; k < last; ++k) {
        const float *p = from + ((piece + k) * 2 + (k == 0 ? 1 : 0)) * a.columns;
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += p[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) red[wave][lane * N + i] = sum[i];
    __syncthreads();
    if (wave == 0 && vector < a.vectors) {
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += red[w][lane * N + i];
        put_row<R>(a, row, vector, sum);
    }
}

int check(const lffn_embedding *a) {
    LFFN_REQUIRE(a, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->format >= 0 && a->format <= 2 && a->tokens >= 0 && a->rows >= 0 && a->columns >= 1 && a->stride >= 0, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->tokens == 0 || a->ids, LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(a->tokens < (int64_t(1) << 31) && a->rows < (int64_t(1) << 31) - 1 && a->columns <= (1 << 20), LFFN_ERR_UNSUPPORTED);
    return LFFN_OK;
}

int passes_of(int64_t rows) {
    int passes = 1;
    while (rows >> (passes * BITS)) ++passes;          // (the numbers are 0 .. rows)
    return passes;
}

// Tokens of a piece: enough pieces to fill the chip, and few enough that a run through all of them is soon added up.
int length_of(int64_t tokens) {
    int length = 16;
    while (length < 256 && tokens / length > 1024) length *= 2;
    return length;
}

struct Space {
    int64_t chunks, pieces, counts, lists, parts, bytes;
    int passes, length;
};
Space space_of(const lffn_embedding &a) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    Space s{};
    s.chunks = (a.tokens + CHUNK - 1) / CHUNK;
    s.passes = passes_of(a.rows);
    s.length = length_of(a.tokens);
    s.pieces = (a.tokens + s.length - 1) / s.length;
    s.counts = up((s.chunks + 1) * DIGITS * 4);
    s.lists = up(a.tokens * 8);
    s.parts = s.pieces * 2 * a.columns * 4;
    s.bytes = s.counts + 2 * s.lists + s.parts;
    return s;
}

template <typename R>
void sums(const SumArgs &a, hipStream_t st) {
    const unsigned blocks = (a.vectors + 63) / 64;
    sum_kernel<R><<<dim3(unsigned((a.pieces + WG / 64 - 1) / (WG / 64)), blocks), dim3(WG), 0, st>>>(a);
    if (a.pieces > 1) join_kernel<R><<<dim3(unsigned(a.pieces - 1), blocks), dim3(JOIN_WG), 0, st>>>(a);
}

template <typename R>
int forward(Args a, hipStream_t st) {
    a.pieces = a.columns / R::N;
    const int lanes = a.pieces <= 4 ? 4 : a.pieces <= 16 ? 16 : a.pieces <= 64 || a.pieces % 64 == 0 ? 64 : a.pieces % 32 == 0 ? 32 : 64;
    const int64_t groups = WG / lanes, grid = (a.tokens + groups - 1) / groups;
    if (grid >= (int64_t(1) << 32) / WG) return LFFN_ERR_UNSUPPORTED;
    const dim3 g((unsigned)grid), b(WG);
    if (lanes == 4) forward_kernel<R, 4><<<g, b, 0, st>>>(a);
    else if (lanes == 16) forward_kernel<R, 16><<<g, b, 0, st>>>(a);
    else if (lanes == 32) forward_kernel<R, 32><<<g, b, 0, st>>>(a);
    else forward_kernel<R, 64><<<g, b, 0, st>>>(a);
    return LFFN_OK;
}

}  // namespace

extern "C" int lffn_embedding_fwd(const lffn_embedding *c, void *out, void *stream) {
    const int rc = check(c);
    if (rc != LFFN_OK || c->tokens == 0) return rc;
    LFFN_REQUIRE(out && (c->weight || c->rows == 0), LFFN_ERR_BAD_ARG);
    Args a{c->ids, c->weight, out, c->stride, (uint32_t)c->tokens, (uint32_t)c->rows, (uint32_t)c->columns, 0, c->ids_64, c->scale};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t size = c->format == LFFN_ROWS_F32 ? 4 : 2;
    const bool vectors = c->columns * size % 16 == 0 && c->stride * size % 16 == 0 && lffn_aligned16(c->weight) && lffn_aligned16(out);
    int done;
    if (vectors)
        done = c->format == LFFN_ROWS_F32    ? forward<Vectors<F32Row>>(a, st)
               : c->format == LFFN_ROWS_BF16 ? forward<Vectors<BF16Row>>(a, st)
                                             : forward<Vectors<F16Row>>(a, st);
    else
        done = c->format == LFFN_ROWS_F32    ? forward<Single<float, 4>>(a, st)
               : c->format == LFFN_ROWS_BF16 ? forward<Single<__bf16, 2>>(a, st)
                                             : forward<Single<_Float16, 2>>(a, st);
    return done != LFFN_OK ? done : lffn_launch_status();
}

extern "C" int lffn_embedding_bwd_workspace_bytes(const lffn_embedding *c, int64_t *bytes) {
    LFFN_REQUIRE(bytes, LFFN_ERR_BAD_ARG);
    const int rc = check(c);
    if (rc == LFFN_OK) *bytes = space_of(*c).bytes;
    return rc;
}

extern "C" int lffn_embedding_bwd(const lffn_embedding *c, const void *g, void *grad, void *workspace, int64_t workspace_bytes, void *stream) {
    const int rc = check(c);
    if (rc != LFFN_OK || c->rows == 0) return rc;
    const Space s = space_of(*c);
    LFFN_REQUIRE(grad && lffn_aligned16(grad), LFFN_ERR_BAD_ARG);
    LFFN_REQUIRE(c->tokens == 0 || (g && workspace && lffn_aligned16(workspace) && workspace_bytes >= s.bytes), LFFN_ERR_BAD_ARG);
    hipStream_t st = static_cast<hipStream_t>(stream);
    char *const ws = static_cast<char *>(workspace);
    int32_t *const counts = reinterpret_cast<int32_t *>(ws);
    uint2 *const lists[2] = {reinterpret_cast<uint2 *>(ws + s.counts), reinterpret_cast<uint2 *>(ws + s.counts + s.lists)};
    const int64_t size = c->format == LFFN_ROWS_F32 ? 4 : 2, bytes = c->rows * c->columns * size;
    // every launch that sorts clears an equal share
    const bool one = c->tokens > 0 && c->tokens <= ONE_MOST * SORT_WG;
    const int launches = c->tokens == 0 || one ? 1 : 2 * s.passes;
    const int64_t share = (bytes / launches + 1023) / 1024 * 1024;
    const bool vectors = c->columns * size % 16 == 0 && lffn_aligned16(g);
    const int64_t width = vectors ? c->columns * size / 16 : c->columns;
    LFFN_REQUIRE(share / FILL_BYTES + 1 + s.chunks < (int64_t(1) << 32) / SORT_WG && s.pieces * ((width + 63) / 64) < (int64_t(1) << 32) / JOIN_WG, LFFN_ERR_UNSUPPORTED);
    SortArgs a{};
    a.ids = c->ids, a.padding = c->padding, a.ids_64 = c->ids_64;
    a.tokens = (uint32_t)c->tokens, a.rows = (uint32_t)c->rows, a.chunks = (int)s.chunks;
    a.counts = counts, a.to = lists[0];
    a.scanned = a.chunks > SCANNED_FROM;
    for (int i = 0; i < launches; ++i) {
        const int64_t first = i * share < bytes ? i * share : bytes, end = i + 1 == launches || (i + 1) * share > bytes ? bytes : (i + 1) * share;
        a.fill = {static_cast<char *>(grad) + first, end - first};
        const dim3 grid(unsigned((one ? 1 : s.chunks) + (a.fill.bytes + FILL_BYTES - 1) / FILL_BYTES)), block(SORT_WG);
        if (one && c->tokens <= SORT_WG) sort_one_kernel<1><<<grid, block, 0, st>>>(a, s.passes);
        else if (one) sort_one_kernel<ONE_MOST><<<grid, block, 0, st>>>(a, s.passes);
        else if (i % 2 == 0) {
            if (i > 0) a.from = a.to, a.to = lists[i / 2 % 2];
            a.shift = i / 2 * BITS;
            count_kernel<<<grid, block, 0, st>>>(a);
            if (a.scanned) scan_kernel<<<dim3(DIGITS / 16), block, 0, st>>>(counts, a.chunks);
        } else
            sort_kernel<<<grid, block, 0, st>>>(a);
    }
    if (c->tokens > 0) {
        const SumArgs m{a.to,     g, grad, reinterpret_cast<float *>(ws + s.counts + 2 * s.lists), a.tokens, a.rows, (uint32_t)c->columns, (uint32_t)width,
                        s.length, s.pieces, c->scale};
        if (vectors) {
            if (c->format == LFFN_ROWS_F32) sums<Vectors<F32Row>>(m, st);
            else if (c->format == LFFN_ROWS_BF16) sums<Vectors<BF16Row>>(m, st);
            else sums<Vectors<F16Row>>(m, st);
        } else {
            if (c->format == LFFN_ROWS_F32) sums<Single<float, 4>>(m, st);
            else if (c->format == LFFN_ROWS_BF16) sums<Single<__bf16, 2>>(m, st);
            else sums<Single<_Float16, 2>>(m, st);
        }
    }
    return lffn_launch_status();
}
