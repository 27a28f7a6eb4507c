// Kernels of the matrix operators: momentum pass, normalisation, the Newton-Schulz products.
// Included by matrix.hip only.
//
// The iteration.  For U (rows x cols) let X be U / max(|U|_F, eps), turned so that its short side s comes first
// (s x l, s <= l).  One step with coefficients (a, b, c) is
//     A = X X^T,    B = b A + c A A,    X <- a X + B X,
// which maps every singular value x of X to a x + b x^3 + c x^5 and leaves the singular vectors.  A and B are
// symmetric: only the tiles on and under their diagonal are computed, each is stored at its mirror place too.
//
// How numbers are held.  Frobenius norm 1 bounds the singular values of X0 by 1; the host follows that bound through
// the polynomial (step_bounds in matrix.hip), and no entry of a matrix is larger than its largest singular value.  So
// X, A and B are kept as halves times a power of two that the bound allows: 11 bits each and no overflow, which
// bfloat16 (8 bits) would pay for a range that is not needed.  A second half holds what the first leaves over (22 bits):
//   * X always has it, for the term a X: a > 3 there multiplies the rounding of X at every step, and for directions
//     of small singular values nothing takes it back (rounding X to 11 bits: error 4e-2 after five steps on a matrix
//     of rank 8 plus 1 % noise; with the second half 4e-4, simulated against 64 bits);
//   * with PLANES == 2 the products use it as well: hi hi + hi lo + lo hi in one fp32 accumulator, three matrix
//     instructions in place of one, and errors like those of fp32 products (the dropped lo lo is 2^-22 of the sum).
// Sums are held in fp32 (matrix instructions), norms in fp64.
//
// Storage in the workspace, all sizes padded to 64 with zeros (zero rows and columns stay zero through the iteration,
// so no product needs a mask): X is s64 x l64, A and B are s64 x s64, the planes one behind the other.  A matrix lies in blocks of
// column_block() columns (what a panel of a product is deep: 64 halves, 32 with two planes), each block's rows one behind the other: a
// panel's rows, wherever it is cut, are then one contiguous span, every load of a wave 1 KiB of it.  Row-major, a wave's load
// of 64-byte pieces fills half lines only and gets through at half the rate (62 against 115 GB/s for a compute unit).
#pragma once

#include <cstdint>
#include <type_traits>

#include "fsadam_common.h"  // store_through

namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float float4_t __attribute__((ext_vector_type(4)));

#define FM_LDS __attribute__((address_space(3)))
#define FM_GLOBAL __attribute__((address_space(1)))

enum { kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 2 };

// Which of a row's tile counts a launch goes by.
enum {
    kTilesSym64, kTilesFull64, kTilesGram64, kTilesSym128, kTilesFull128, kTilesGram128, kTilesSym256, kTilesFull256, kTilesGram256,
    kTilesPart, kTilesAllParts, kTilesJoin, kTilesPrep, kTilesChunk, kTileKinds
};

// One row of a call's table: `batch` matrices of one shape, equally spaced.
struct alignas(16) MatrixRow {
    const void* src;   // orthogonalize: the matrices.  step: the gradients
    float* buf;        // step: the momentum
    void* dst;         // orthogonalize: the results.  step: the parameters (fp32 masters in mixed precision)
    void* copy;        // step, mixed precision: the 16-bit parameters
    int64_t src_ld, src_stride, dst_ld, dst_stride;  // elements from row to row, from matrix to matrix
    int64_t x_off[2];  // workspace: X and its successor (halves from the workspace's start)
    int64_t sq_off[3]; // workspace: square matrices (A and B; a pair of steps uses all three)
    int32_t batch, rows, cols;
    int32_t s, l, s64, l64;
    int32_t tall;      // rows > cols: X is the transpose
    int32_t first_matrix;           // index of the row's first matrix in the chunk
    int32_t chunks;                 // partial sums per matrix
    int32_t parts;                  // of the Gram matrix's inner products; 1: not split
    float step_ratio;               // step: lr * ratio of this shape
    int32_t first[kTileKinds];      // tiles of the rows before this one
    int32_t n[kTileKinds];          // tiles of one matrix
};

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int type) {
    if (type == kTypeF32) return static_cast<const float*>(p)[i];
    if (type == kTypeF16) return (float)static_cast<const _Float16*>(p)[i];
    return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}
// Round to nearest even; NaN stays NaN (one instruction for two values on this part).
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, bf16x2_t)); }
__device__ __forceinline__ uint16_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ void store_from_float(void* p, int64_t i, int type, float v) {
    if (type == kTypeF32) static_cast<float*>(p)[i] = v;
    else if (type == kTypeF16) static_cast<_Float16*>(p)[i] = (_Float16)v;
    else static_cast<uint16_t*>(p)[i] = bf16_bits(v);
}
// What a stored value of this type reads back as.
__device__ __forceinline__ float round_to(float v, int type) {
    if (type == kTypeF32) return v;
    if (type == kTypeF16) return (float)(_Float16)v;
    return __builtin_bit_cast(float, (uint32_t)bf16_bits(v) << 16);
}

// Eight neighbours p[i .. i + 7], of which the first `left` are there: 16-byte accesses where all are and the address allows it.
typedef uint32_t words4_t __attribute__((ext_vector_type(4)));
typedef uint32_t words2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float high_half(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ float low_half(uint32_t w) { return __builtin_bit_cast(float, w << 16); }

__device__ __forceinline__ void load_eight(const void* p, int64_t i, int type, int left, float (&v)[8]) {
    const char* at = static_cast<const char*>(p) + i * (type == kTypeF32 ? 4 : 2);
    if (left >= 8 && ((uintptr_t)at & 15) == 0) {
        if (type == kTypeF32) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = reinterpret_cast<const float4_t*>(at)[q >> 2][q & 3];
        } else if (type == kTypeF16) {
            const half8_t h = *reinterpret_cast<const half8_t*>(at);
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (float)h[q];
        } else {
            const words4_t w = *reinterpret_cast<const words4_t*>(at);
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = q & 1 ? high_half(w[q >> 1]) : low_half(w[q >> 1]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < left ? load_as_float(p, i + q, type) : 0.0f;
    }
}
__device__ __forceinline__ void store_eight(void* p, int64_t i, int type, int left, const float (&v)[8]) {
    char* at = static_cast<char*>(p) + i * (type == kTypeF32 ? 4 : 2);
    if (left >= 8 && ((uintptr_t)at & 15) == 0) {
        if (type == kTypeF32) {
            reinterpret_cast<float4_t*>(at)[0] = float4_t{v[0], v[1], v[2], v[3]};
            reinterpret_cast<float4_t*>(at)[1] = float4_t{v[4], v[5], v[6], v[7]};
        } else if (type == kTypeF16) {
            half8_t h;
#pragma unroll
            for (int q = 0; q < 8; ++q) h[q] = (_Float16)v[q];
            *reinterpret_cast<half8_t*>(at) = h;
        } else {
            *reinterpret_cast<words4_t*>(at) = words4_t{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < left) store_from_float(p, i + q, type, v[q]);
    }
}

// Four neighbours for passes that stream: the lanes of a wave lie side by side (16 bytes each in fp32, 8 in 16 bits), so that an
// instruction covers one span; loads do not stay in the caches and stores are written through to memory (store_through).
// `whole`: all four are there and the addresses allow it.
template <int TYPE>
__device__ __forceinline__ void load_four(const void* p, int64_t i, bool whole, int left, float (&v)[4]) {
    const uintptr_t at = (uintptr_t)p + i * (TYPE == kTypeF32 ? 4 : 2);
    if (whole) {
        if constexpr (TYPE == kTypeF32) {
            const float4_t w = __builtin_nontemporal_load((gptr<const float4_t>)at);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = w[q];
        } else if constexpr (TYPE == kTypeF16) {
            const half4_t w = __builtin_nontemporal_load((gptr<const half4_t>)at);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = (float)w[q];
        } else {
            const words2_t w = __builtin_nontemporal_load((gptr<const words2_t>)at);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = q & 1 ? high_half(w[q >> 1]) : low_half(w[q >> 1]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = q < left ? load_as_float(p, i + q, TYPE) : 0.0f;
    }
}
template <int TYPE>
__device__ __forceinline__ void store_four(void* p, int64_t i, bool whole, int left, const float (&v)[4]) {
    const uintptr_t at = (uintptr_t)p + i * (TYPE == kTypeF32 ? 4 : 2);
    if (whole) {
        if constexpr (TYPE == kTypeF32) {
            store_through((gptr<void>)at, float4_t{v[0], v[1], v[2], v[3]});
        } else if constexpr (TYPE == kTypeF16) {
            store_through((gptr<void>)at, half4_t{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]});
        } else {
            store_through((gptr<void>)at, words2_t{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])});
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < left) store_from_float(p, i + q, TYPE, v[q]);
    }
}

__device__ __forceinline__ void split_halves(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// Eight values as one or two planes of halves.
template <int PLANES>
__device__ __forceinline__ void store_planes(_Float16* at, int64_t plane, const float (&v)[8]) {
    half8_t hi, lo;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        _Float16 h, o;
        split_halves(v[q], h, o);
        hi[q] = h;
        lo[q] = o;
    }
    *reinterpret_cast<half8_t*>(at) = hi;
    if constexpr (PLANES == 2) *reinterpret_cast<half8_t*>(at + plane) = lo;
}
template <int PLANES>
__device__ __forceinline__ void load_planes(const _Float16* at, int64_t plane, float (&v)[8]) {
    const half8_t hi = *reinterpret_cast<const half8_t*>(at);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = (float)hi[q];
    if constexpr (PLANES == 2) {
        const half8_t lo = *reinterpret_cast<const half8_t*>(at + plane);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] += (float)lo[q];
    }
}

constexpr int column_block(int planes) { return planes == 2 ? 32 : 64; }
// Where element (i, j) of a matrix of `rows` rows lies.
__device__ __forceinline__ int64_t in_blocks(int i, int j, int rows, int log_block) {
    return (((int64_t)(j >> log_block) * rows + i) << log_block) + (j & ((1 << log_block) - 1));
}

// Workgroups are handed to the 8 XCDs in turn, each with an L2 of its own: give every XCD a contiguous range of tiles.
__device__ __forceinline__ uint32_t xcd_contiguous(uint32_t block, uint32_t n) {
    const uint32_t per = n / 8, extra = n % 8, xcd = block % 8, at = block / 8;
    return xcd * per + (xcd < extra ? xcd : extra) + at;
}

// The last of n rows whose first(row) is not past t; first(0) is not.  A wave looks at 64 rows at a time: one trip to memory for a
// list of up to 64, where halving takes one behind the other (12 rows: four, before a workgroup knows what to do; products of 768 deep
// in one round of tiles 30 -> 28 us).
template <typename First>
__device__ __forceinline__ int find_row(int n, int64_t t, First&& first) {
    if (n == 1) return 0;
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (;;) {
        const int step = (n + 63) / 64;
        const bool before = lane * step < n && (int64_t)first(base + lane * step) <= t;
        const int at = (__builtin_popcountll(__ballot(before)) - 1) * step;
        base += at;
        if (step == 1) return __builtin_amdgcn_readfirstlane(base);
        n = n - at < step ? n - at : step;
    }
}

// The row, the matrix in it and the tile in that of the launch's tile `t`.
__device__ __forceinline__ const MatrixRow& find_tile(const MatrixRow* table, int n_rows, int kind, uint32_t t, int& matrix, uint32_t& tile) {
    const MatrixRow& row = table[find_row(n_rows, t, [&](int r) { return table[r].first[kind]; })];
    const uint32_t at = t - (uint32_t)row.first[kind], per = (uint32_t)row.n[kind];
    matrix = (int)(at / per);
    tile = at - (uint32_t)matrix * per;
    return row;
}

// ---- momentum -----------------------------------------------------------------------------------------------------

struct MomentumArgs {
    const float* scale_dev;  // when not NULL the gradients are divided by this instead of `scale`
    float scale;
    float momentum, one_minus;
    int nesterov;
};

// The divisor of the gradients.  A power of two with a normal reciprocal is multiplied by that: the same bits, and a
// division takes ten instructions that a pass over 16-bit gradients has no time for.
struct Divisor {
    float scale, inverse;
    bool exact;
    __device__ __forceinline__ explicit Divisor(const MomentumArgs& k) {
        scale = k.scale_dev ? *k.scale_dev : k.scale;
        inverse = 1.0f / scale;
        exact = (__builtin_bit_cast(uint32_t, scale) & 0x7fffffu) == 0 && __builtin_isnormal(scale) && __builtin_isnormal(inverse);
    }
    __device__ __forceinline__ float operator()(float g) const { return exact ? g * inverse : g / scale; }
};

//     r = g / scale;   m <- m + (1 - mu) (r - m);   u = nesterov ? r + mu (m - r) : m
__device__ __forceinline__ float momentum_update(float r, float& m, const MomentumArgs& k) {
    m = m + (r - m) * k.one_minus;
    return k.nesterov ? r + (m - r) * k.momentum : m;
}
__device__ __forceinline__ float update_again(float r, float m, const MomentumArgs& k) {  // from the stored m
    return k.nesterov ? r + (m - r) * k.momentum : m;
}

constexpr int kChunkThreads = 256;
constexpr int kChunkElems = 8192;  // elements of one partial sum
constexpr int kMomentumElems = 1024;  // likewise, of the momentum pass: four to a thread (8 and 16 are 4 and 12 % slower)

// Sum over a workgroup in a fixed order; the result is valid in thread 0.
template <int THREADS = kChunkThreads>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 64];
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int n = 0; n < THREADS / 64; ++n) v += part[n];
    return v;
}

// A thread's share of the sum of p[0 .. n - 1], eight loads at a time in flight.
template <int THREADS = kChunkThreads>
__device__ __forceinline__ double sum_of(const double* p, int64_t n) {
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 8 * THREADS) {
        double v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = i + q * THREADS < n ? p[i + q * THREADS] : 0.0;
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += v[q];
    }
    return sum;
}

// One row of the momentum pass's table: a tensor as a line of elements.
struct alignas(16) MomentumRow {
    const void* g;
    float* m;
    void* u;
    int64_t numel;
    int64_t first;    // chunks of the rows before this one
};
// Short tables travel in the arguments of the launches that use them, longer ones in those of launches that write them to
// memory first: nothing is copied from the host, and a captured graph holds all of it.
constexpr int kMomentumRowsPerLaunch = 64;
struct MomentumRows {
    MomentumRow row[kMomentumRowsPerLaunch];
};
// What a kernel takes: the address of a table, or the table.
struct InMemory {
    const MomentumRow* row;
    int n;
};
struct InArguments {
    MomentumRows rows;
    int n;
};
__device__ __forceinline__ const MomentumRow* rows_of(const InMemory& t) { return t.row; }
__device__ __forceinline__ const MomentumRow* rows_of(const InArguments& t) { return t.rows.row; }

// Elements `begin` to `end` of a line, eight to a thread: calls each(first element, how many) for every piece.  With whole eights
// all pieces of a thread are independent, so that their loads are all in flight before the first is used.
template <typename Each>
__device__ __forceinline__ void for_eights(int64_t begin, int64_t end, Each&& each) {
    if (end - begin == kChunkElems) {
#pragma unroll
        for (int n = 0; n < kChunkElems / 8 / kChunkThreads; ++n) each(begin + (n * kChunkThreads + threadIdx.x) * 8, 8);
    } else {
        for (int64_t i = begin + threadIdx.x * 8; i < end; i += kChunkThreads * 8) each(i, end - i < 8 ? (int)(end - i) : 8);
    }
}

// Bound by HBM: 2 + 4 bytes read and 2 + 4 written per element with 16-bit gradients and updates.  The matrices of a layer of 4096
// with an FFN of 11008 (202 million elements): 374 us, 6.5 TB/s (382 us the call), where a plain copy of a tensor reaches 4.8 and this library's
// parameter pass 6.7.  Short workgroups of one piece a thread, all loads before the first store, and stores that write through
// the L2 (store_through) as in the parameter pass; the L2 would hold the lines until they are in the way of the reads.
template <int GT, int UT, typename Table>
__global__ __launch_bounds__(kChunkThreads) void fsadam_momentum_chunks(Table tables, MomentumArgs k, double* partials, float* cleared) {
    if (cleared && blockIdx.x == 0 && threadIdx.x == 0) *cleared = 0.0f;
    const MomentumRow* table = rows_of(tables);
    const int n_rows = tables.n;
    // by halving: workgroups this short find the table in the scalar cache (a layer's list 382 us; with find_row 404)
    int low = 0, high = n_rows - 1;
    const int64_t t = blockIdx.x;
    while (low < high) {
        const int mid = (low + high + 1) >> 1;
        if (table[mid].first <= t) low = mid;
        else high = mid - 1;
    }
    const MomentumRow& row = table[low];
    const int64_t begin = (t - row.first) * kMomentumElems;
    const int64_t end = begin + kMomentumElems < row.numel ? begin + kMomentumElems : row.numel;
    const Divisor by(k);
    double sum = 0.0;
    constexpr int kPieces = kMomentumElems / 4 / kChunkThreads;
    float g[kPieces][4], m[kPieces][4], u[kPieces][4];
    const uintptr_t any = (uintptr_t)row.g * (GT == kTypeF32 ? 1 : 2) | (uintptr_t)row.m | (uintptr_t)row.u * (UT == kTypeF32 ? 1 : 2);
    const bool whole = end - begin == kMomentumElems && (any & 15) == 0;
    const int64_t i0 = begin + threadIdx.x * 4;
    constexpr int kStep = kChunkThreads * 4;
    auto left = [&](int n) { const int64_t here = end - (i0 + n * kStep); return here < 4 ? (int)here : 4; };
    auto load = [&](bool whole) {
#pragma unroll
        for (int n = 0; n < kPieces; ++n) {
            load_four<GT>(row.g, i0 + n * kStep, whole, left(n), g[n]);
            load_four<kTypeF32>(row.m, i0 + n * kStep, whole, left(n), m[n]);
        }
    };
    if (whole) load(true);
    else load(false);
    if (by.exact) {
#pragma unroll
        for (int n = 0; n < kPieces; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) g[n][q] *= by.inverse;
    } else {
#pragma unroll
        for (int n = 0; n < kPieces; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) g[n][q] /= by.scale;
    }
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) u[n][q] = momentum_update(g[n][q], m[n][q], k);
    auto store = [&](bool whole) {
#pragma unroll
        for (int n = 0; n < kPieces; ++n) {
            store_four<kTypeF32>(row.m, i0 + n * kStep, whole, left(n), m[n]);
            store_four<UT>(row.u, i0 + n * kStep, whole, left(n), u[n]);
        }
    };
    if (whole) store(true);
    else store(false);
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // elements past the end are zeros: g and m were loaded as such
            const double r = (double)round_to(u[n][q], UT);
            sum = __builtin_fma(r, r, sum);
        }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partials[t] = sum;
}

// norms[row] = sqrt of the row's sum of squares; found_inf is raised where that is not finite (a double holds the sum of
// squares of any floats, so it is not finite exactly where an update is not).
constexpr int kNormThreads = 1024;  // a tensor of 45 million elements has 44000 partial sums
template <typename Table>
__global__ __launch_bounds__(kNormThreads) void fsadam_momentum_norms(Table tables, const double* partials, float* norms, float* found_inf) {
    const MomentumRow& row = rows_of(tables)[blockIdx.x];
    const int64_t n = (row.numel + kMomentumElems - 1) / kMomentumElems;
    const double sum = block_sum<kNormThreads>(sum_of<kNormThreads>(partials + row.first, n));
    if (threadIdx.x == 0) {
        if (norms) norms[blockIdx.x] = (float)sqrt(sum);
        if (found_inf && !__builtin_isfinite(sum)) *found_inf = 1.0f;
    }
}

// ---- norms and normalisation of the matrices ----------------------------------------------------------------------

// STEP: the source is the gradient, the momentum is updated and what is summed is the update, which is not stored: the next pass
// makes it again from the gradient and the new momentum, 6 bytes read in place of 4 written and 4 read.  Bound by HBM: 16-bit
// gradients, 202 million elements: 342 us, 5.9 TB/s.  Where X is read alone (4096 x 4096 bf16, 34 MB): 8.8 us, 3.8 TB/s.
template <int ST, bool STEP>
__global__ __launch_bounds__(kChunkThreads) void fsadam_matrix_chunks(const MatrixRow* table, int n_rows, MomentumArgs k, double* partials) {
    int matrix;
    uint32_t chunk;
    const MatrixRow& row = find_tile(table, n_rows, kTilesChunk, blockIdx.x, matrix, chunk);
    const int64_t numel = (int64_t)row.rows * row.cols;
    const int64_t begin = (int64_t)chunk * kChunkElems;
    const int64_t end = begin + kChunkElems < numel ? begin + kChunkElems : numel;
    double sum = 0.0;
    if constexpr (STEP) {
        const Divisor by(k);
        const int64_t base = (int64_t)matrix * numel;
        for_eights(begin, end, [&](int64_t i, int n) {
            float g[8], m[8];
            load_eight(row.src, base + i, ST, n, g);
            load_eight(row.buf, base + i, kTypeF32, n, m);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const double u = q < n ? (double)momentum_update(by(g[q]), m[q], k) : 0.0;
                sum = __builtin_fma(u, u, sum);
            }
            store_eight(row.buf, base + i, kTypeF32, n, m);
        });
    } else if (row.src_ld == row.cols) {
        const int64_t base = (int64_t)matrix * row.src_stride;
        for_eights(begin, end, [&](int64_t i, int n) {
            float v[8];
            load_eight(row.src, base + i, ST, n, v);
#pragma unroll
            for (int q = 0; q < 8; ++q) sum = __builtin_fma((double)v[q], (double)v[q], sum);  // what is not there was loaded as 0
        });
    } else {
        const int64_t base = (int64_t)matrix * row.src_stride;
        for (int64_t i = begin + threadIdx.x; i < end; i += kChunkThreads) {
            const int64_t r = i / row.cols;
            const double u = (double)load_as_float(row.src, base + r * row.src_ld + (i - r * row.cols), ST);
            sum += u * u;
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// One workgroup per matrix: inverse[matrix] = 1 / max(norm, eps), NaN where the norm is not finite (every entry of the
// result is then NaN, which is what one product of the iteration would make of it).
__global__ __launch_bounds__(kChunkThreads) void fsadam_matrix_norms(const MatrixRow* table, int n_rows, double eps, const double* partials, double* inverse) {
    const MatrixRow& row = table[find_row(n_rows, blockIdx.x, [&](int r) { return table[r].first_matrix; })];
    const double* p = partials + row.first[kTilesChunk] + (int64_t)((int)blockIdx.x - row.first_matrix) * row.chunks;
    const double sum = block_sum(sum_of(p, row.chunks));
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum);
        inverse[blockIdx.x] = __builtin_isfinite(sum) ? 1.0 / (norm > eps ? norm : eps) : __builtin_nan("");
    }
}

// X0 * 2^k as two halves, 64 x 64 elements a workgroup, turned (through LDS) where the matrix is tall; the padding is written as
// zeros.  Bound by HBM: 16-bit gradients and momentum in, 10 bytes an element in all: 8 x 1024 x 2816 and turned 83 us, 5.5 TB/s.
template <int ST, bool STEP>
__global__ __launch_bounds__(256) void fsadam_matrix_normalise(const MatrixRow* table, int n_rows, MomentumArgs k, const double* inverse, double power, int log_block,
                                                                _Float16* work) {
    __shared__ float tile[64][65];
    int matrix;
    uint32_t t;
    const MatrixRow& row = find_tile(table, n_rows, kTilesPrep, blockIdx.x, matrix, t);
    const uint32_t across = (uint32_t)row.l64 / 64;
    const int i0 = (int)(t / across) * 64, j0 = (int)(t % across) * 64;  // in X
    const int r0 = row.tall ? j0 : i0, c0 = row.tall ? i0 : j0;         // in the source
    const double factor = inverse[row.first_matrix + matrix] * power;
    const Divisor by(k);
    const int64_t plane = (int64_t)row.s64 * row.l64;
    _Float16* x = work + row.x_off[0] + (int64_t)matrix * 2 * plane;
    auto put = [&](int i, int j, const float (&v)[8]) { store_planes<2>(x + in_blocks(i0 + i, j0 + j, row.s64, log_block), plane, v); };
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int e = threadIdx.x + part * 256, r = e >> 3, c = (e & 7) * 8;  // eight neighbours in the source
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = 0.0f;
        const int left = r0 + r < row.rows ? row.cols - (c0 + c) : 0;
        if (left > 0) {
            if constexpr (STEP) {
                const int64_t at = (int64_t)matrix * row.rows * row.cols + (int64_t)(r0 + r) * row.cols + c0 + c;
                float m[8];
                load_eight(row.src, at, ST, left, v);
                load_eight(row.buf, at, kTypeF32, left, m);
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = q < left ? update_again(by(v[q]), m[q], k) : 0.0f;
            } else {
                load_eight(row.src, (int64_t)matrix * row.src_stride + (int64_t)(r0 + r) * row.src_ld + c0 + c, ST, left, v);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (float)((double)v[q] * factor);
        }
        if (!row.tall) {
            put(r, c, v);
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) tile[r][c + q] = v[q];
        }
    }
    if (!row.tall) return;
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int e = threadIdx.x + part * 256, i = e >> 3, j = (e & 7) * 8;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = tile[j + q][i];
        put(i, j, v);
    }
}

// ---- the products -------------------------------------------------------------------------------------------------

enum { kStageJoin, kStageGram, kStageSquare, kStageUpdate, kStageOut, kStageStep };

// Depth of a part of a Gram matrix's inner products, where they are split.
constexpr int kPartDepth = 512;

struct StageArgs {
    int from, to;       // which of the two X buffers is read and written
    int p, q, add, into;  // square matrices: operands, what is added (< 0: nothing), result.  Update: p is the left operand
    float linear, product;  // result = linear * (what is added) + product * (accumulator), powers of two included
    float diagonal;     // square matrices: added on the diagonal
    float keep;         // step: 1 - lr * weight_decay
    int kind;           // Gram matrix in tiles of 64: which tile counts the launch goes by
    int dst_type, copy_type;  // out, step: kType*; copy_type < 0: no copies
};

// A tile's operand panel in LDS, K contiguous ("NT"): `rows` x BK halves, 16-byte chunks of a row exchanged (xor) so that
// the 16 rows a fragment reads spread over the banks.
template <int BK>
__device__ __forceinline__ int swizzle_nt(int row) {
    return BK == 64 ? (row & 7) : ((row >> 1) & 3);
}
// K x columns ("NN", read with the transposing LDS loads): blocks of BK columns as in memory, pairs of chunks (32 bytes, 16
// columns) of a row exchanged so that the rows one load touches (8g + 0..3 for the four groups g of 16 lanes) spread over the banks.
template <int BK>
__device__ __forceinline__ int swizzle_nn(int row) {
    return BK == 32 ? (row >> 3) & 1 : ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
}

// An address that all lanes hold, in scalar registers.
__device__ __forceinline__ const _Float16* uniform(const _Float16* p) {
    const uint64_t a = (uint64_t)p;
    return (const _Float16*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)a));
}

// 1 KiB straight from memory into LDS: 16 bytes from src + `bytes` of every lane land at dst + 16 * lane.
// From assembly because of the wait: behind the builtin the compiler places a wait for ALL loads before the next read
// of LDS (it cannot tell the buffer being filled from the one being read), which takes away the overlap the two
// buffers are there for.  The statement has no output register; what it writes is LDS, and nothing reads that before
// loads_arrived() and the barrier behind it.  m0 is a reserved register: the compiler writes it right before each use of
// its own and keeps nothing in it.  The s_nop: a write of m0 needs one wait state before the load that uses
// it, a vector instruction's write of the scalar address (readfirstlane) five, and the compiler does not look into the statement.
__device__ __forceinline__ void load_to_lds(const _Float16* src, uint32_t bytes, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(bytes), "s"(src) : "memory");
}
template <int LEFT>
__device__ __forceinline__ void loads_arrived() {  // all but the last LEFT loads of this wave
    static_assert(LEFT < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(FM_LDS const void*)p; }

// What bounds it.  With two planes every 32 of depth take three matrix instructions for each pair of fragments, and the matrix cores
// are busy 72 % of the time at the 1.9 GHz that the power limit leaves: update of 5120 x 13824 in 1.73 ms, 419 TFLOP/s, which is
// 1.26 PFLOP/s of matrix instructions; a plain 16-bit matrix product of the library runs at 1.26 to 1.32 PFLOP/s on this card.
// With one plane the panels' way from the L2 to LDS is the longer part (64 KiB per 64 of depth of a 256 x 256 tile, at 100 to
// 135 GB/s a compute unit): update of 4096 x 4096 in 141 us, 975 TFLOP/s.
// Fragments: lane (g, c) of 16 x 4 holds row c, eight deep from 8 g on; NN operands lie deep-major and are turned by the
// transposing LDS loads, four deep of 16 columns each.
//
// C tile (TM x TN) = P Q^T (NT) or P Q (NN) over K, by WM x WN waves; the caller's epilogue takes acc.  DEPTH panels are in LDS:
// one is multiplied while the others are on their way.
template <int TM, int TN, int WM, int WN, int BK, int DEPTH, int PLANES, bool NN>
struct Product {
    static constexpr int kThreads = 64 * WM * WN, kWaves = WM * WN;
    static constexpr int MI = TM / WM / 16, NJ = TN / WN / 16;
    static constexpr int kPanelP = TM * BK, kPanelQ = TN * BK;             // halves of one plane
    static constexpr int kStageHalves = PLANES * (kPanelP + kPanelQ);
    static constexpr int kLdsHalves = DEPTH * kStageHalves;
    static constexpr int kLoadsP = kPanelP / 512 / kWaves, kLoadsQ = kPanelQ / 512 / kWaves;  // 1 KiB loads of a wave, one plane
    // registers for a second slice of operands beside the accumulators and the first: 256 per lane with two waves to a SIMD
    static constexpr bool kAhead = MI * NJ * 4 + 2 * PLANES * (MI + NJ) * 4 <= 228;
    static_assert(BK == 32 || BK == 64, "one or two slices of 32");
    static_assert(kLoadsP * 512 * kWaves == kPanelP && kLoadsQ * 512 * kWaves == kPanelQ, "panels divide among the waves");

    float4_t acc[MI][NJ];

    // p: element (first row, first depth) of a matrix of `rows` rows, in blocks of BK columns; rows_p: how many rows there are from it
    // on (further ones are read as the last).  q: NT as p; NN element (first depth, first column), blocks_q blocks of columns from it on.
    __device__ __forceinline__ void run(const _Float16* p, int rows, int64_t plane_p, int rows_p, const _Float16* q, int64_t plane_q, int rows_q, int blocks_q,
                                        int k_total, _Float16* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / WN, wn = wave % WN;
        constexpr int kRowsPerLoad = 512 / BK, kChunks = BK / 8;  // of 1 KiB; 16-byte chunks of a row
        uint32_t off_p[kLoadsP], off_q[kLoadsQ];                  // bytes
#pragma unroll
        for (int n = 0; n < kLoadsP; ++n) {
            int r = (wave * kLoadsP + n) * kRowsPerLoad + lane / kChunks;
            const int chunk = (lane % kChunks) ^ swizzle_nt<BK>(r);
            r = r < rows_p ? r : rows_p - 1;
            off_p[n] = (uint32_t)(r * BK + chunk * 8) * 2;
        }
#pragma unroll
        for (int n = 0; n < kLoadsQ; ++n) {
            const int at = (wave * kLoadsQ + n) * kRowsPerLoad + lane / kChunks, slot = lane % kChunks;
            if constexpr (NN) {
                const int r = at % BK;
                int block = at / BK;
                block = block < blocks_q ? block : blocks_q - 1;
                const int chunk = (((slot >> 1) ^ swizzle_nn<BK>(r)) << 1) | (slot & 1);
                off_q[n] = (uint32_t)((block * rows + r) * BK + chunk * 8) * 2;
            } else {
                const int r = at < rows_q ? at : rows_q - 1;
                off_q[n] = (uint32_t)(r * BK + (slot ^ swizzle_nt<BK>(at)) * 8) * 2;
            }
        }
        const int64_t next_p = (int64_t)__builtin_amdgcn_readfirstlane(rows) * BK, next_q = NN ? BK * BK : next_p;
        p = uniform(p), q = uniform(q);
        const _Float16 *low_p = uniform(p + plane_p), *low_q = uniform(q + plane_q);
        const uint32_t lds_at = __builtin_amdgcn_readfirstlane((int)lds_address(lds));
        auto fetch = [&](uint32_t stage) {
#pragma unroll
            for (int plane = 0; plane < PLANES; ++plane) {
                const _Float16 *gp = plane ? low_p : p, *gq = plane ? low_q : q;
                const uint32_t lp = stage + 2 * (plane * kPanelP + wave * kLoadsP * 512);
                const uint32_t lq = stage + 2 * (PLANES * kPanelP + plane * kPanelQ + wave * kLoadsQ * 512);
#pragma unroll
                for (int n = 0; n < kLoadsP; ++n) load_to_lds(gp, off_p[n], lp + n * 1024);
#pragma unroll
                for (int n = 0; n < kLoadsQ; ++n) load_to_lds(gq, off_q[n], lq + n * 1024);
            }
            p += next_p, low_p += next_p;
            q += next_q, low_q += next_q;
        };
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

        const int g = lane >> 4, c = lane & 15;
        const int row_p = wm * (TM / WM) + c, row_q = wn * (TN / WN) + c;
        const int turn_p = swizzle_nt<BK>(row_p), turn_q = swizzle_nt<BK>(row_q);
        int nn_at[NJ];
        if constexpr (NN) {
            const int r = 8 * g + (c >> 2);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int column = wn * (TN / WN) + j * 16;
                nn_at[j] = column / BK * (BK * BK) + r * BK + ((column % BK / 16) ^ swizzle_nn<BK>(r)) * 16 + (c & 3) * 4;
            }
        }

        constexpr int kLoads = PLANES * (kLoadsP + kLoadsQ);  // of a wave for one panel pair
        constexpr int kSlices = BK / 32;                      // of a panel, 32 deep: what one matrix instruction takes
        const int n_k = k_total / BK;
        int fetched = 0, into = 0;
        for (; fetched < DEPTH - 1 && fetched < n_k; ++fetched) fetch(lds_at + fetched * kStageHalves * 2);
        into = fetched % DEPTH;
        int waited = 0;  // panels that are there
        // Panel `waited` is there for this wave, behind the barrier for all; and behind it every wave has read all of the
        // panel before, whose place the next fetch takes.
        auto next_panel = [&] {
            if (fetched - waited == DEPTH - 1) loads_arrived<kLoads*(DEPTH - 2)>();
            else loads_arrived<0>();
            __syncthreads();
            ++waited;
            if (fetched < n_k) {
                fetch(lds_at + into * kStageHalves * 2);
                ++fetched;
                into = into + 1 == DEPTH ? 0 : into + 1;
            }
        };
        struct Slice {
            half8_t p[PLANES][MI], q[PLANES][NJ];
        };
        auto read = [&](Slice& f, const _Float16* now, int kk) {
#pragma unroll
            for (int plane = 0; plane < PLANES; ++plane) {
                const _Float16* lp = now + plane * kPanelP + row_p * BK + ((kk * 4 + g) ^ turn_p) * 8;
                const _Float16* lq = now + PLANES * kPanelP + plane * kPanelQ;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    if constexpr (NN) {
                        const short4_t low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FM_LDS short4_t*)(lq + nn_at[j] + kk * 32 * BK));
                        const short4_t high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FM_LDS short4_t*)(lq + nn_at[j] + (kk * 32 + 4) * BK));
                        const half4_t l4 = __builtin_bit_cast(half4_t, low), h4 = __builtin_bit_cast(half4_t, high);
                        f.q[plane][j] = __builtin_shufflevector(l4, h4, 0, 1, 2, 3, 4, 5, 6, 7);
                    } else {
                        f.q[plane][j] = *reinterpret_cast<const half8_t*>(lq + row_q * BK + ((kk * 4 + g) ^ turn_q) * 8 + j * 16 * BK);
                    }
                }
#pragma unroll
                for (int i = 0; i < MI; ++i) f.p[plane][i] = *reinterpret_cast<const half8_t*>(lp + i * 16 * BK);
            }
        };
        auto multiply = [&](const Slice& f) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    if constexpr (PLANES == 2) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.p[1][i], f.q[0][j], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.p[0][i], f.q[1][j], acc[i][j], 0, 0, 0);
                    }
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.p[0][i], f.q[0][j], acc[i][j], 0, 0, 0);
                }
        };
        const _Float16* now = lds;
        if constexpr (kWaves == 8 && PLANES == 2) {
            // (22 bits: 1.86 -> 1.79 ms on the update of 5120 x 13824.  With 11 bits the loads are the longer part, and two waves of a SIMD
            // in step, each a slice ahead of itself, are faster: 1.69 against 1.83 ms on a layer of the 7B list.)
            // Two groups of four waves, one of each on every SIMD, half a slice apart: while one multiplies, the other reads its
            // operands and sends for the next panel, so that the matrix cores always have a wave that has nothing else to do.
            // Time goes in ticks between barriers.  Group 0 reads slice j in tick 2j and multiplies it in 2j + 1, group 1 a tick
            // later.  A panel of S slices is read for the last time (by group 1) in the tick before group 0 reads the first slice of the
            // next: from that tick on its buffer may be filled again, and both groups send for the panel after next in it, group 0 as
            // it reads, group 1 as it multiplies.  Before group 0 reads a panel, every wave has waited for its own loads of it and passed a barrier:
            // group 0 after multiplying the last slice of the panel before, group 1 after reading it.
            static_assert(DEPTH == 2, "two buffers");
            const bool late = wave >= 4;
            auto tick = [] {
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            };
            loads_arrived<0>();
            tick();
            if (late) {
                if (n_k > 1) fetch(lds_at + kStageHalves * 2);
                tick();
            }
            for (int panel = 0; panel < n_k; ++panel) {
                const _Float16* here = lds + (panel & 1) * kStageHalves;
#pragma unroll
                for (int kk = 0; kk < kSlices; ++kk) {
                    Slice f;
                    read(f, here, kk);
                    if (kk == 0 && !late && panel + 1 < n_k) fetch(lds_at + ((panel + 1) & 1) * kStageHalves * 2);
                    if (kk == kSlices - 1 && late) loads_arrived<0>();
                    tick();
                    if (kk == kSlices - 1 && late && panel + 2 < n_k) fetch(lds_at + (panel & 1) * kStageHalves * 2);
                    __builtin_amdgcn_s_setprio(1);
                    multiply(f);
                    __builtin_amdgcn_s_setprio(0);
                    if (kk == kSlices - 1 && !late) loads_arrived<0>();
                    tick();
                }
            }
            if (!late) tick();
        } else if constexpr (kAhead) {
            // the next slice is read while this one is multiplied, across the barrier between panels too
            constexpr int kReads = PLANES * (MI + NJ * (NN ? 2 : 1)), kProducts = MI * NJ * (PLANES == 2 ? 3 : 1);
            Slice f[2];
            next_panel();
            read(f[0], now, 0);
            for (int step = 0; step < n_k; step += 2 / kSlices) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {  // two slices: f[0], f[1]
                    const int panel = step + n / kSlices, kk = n % kSlices;
                    if (kSlices == 1 && panel >= n_k) break;
                    if (kk + 1 < kSlices) {
                        read(f[1 - n], now, kk + 1);
                    } else if (panel + 1 < n_k) {
                        next_panel();
                        now = (panel + 1) % DEPTH == 0 ? lds : now + kStageHalves;
                        read(f[1 - n], now, 0);
                    }
                    multiply(f[n]);
                    // a few matrix instructions behind every read: in the order of the text the matrix cores would wait
                    // until a wave has got all its reads into the queue
#pragma unroll
                    for (int r = 0; r < kReads; ++r) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, kProducts / kReads, 0);
                    }
                }
            }
        } else {
            for (int step = 0; step < n_k; ++step) {
                next_panel();
#pragma unroll
                for (int kk = 0; kk < kSlices; ++kk) {
                    Slice f;
                    read(f, now, kk);
                    multiply(f);
                }
                now = step % DEPTH == DEPTH - 1 ? lds : now + kStageHalves;
            }
        }
        __syncthreads();  // the epilogue writes over the panels
    }
};

// One stage of the iteration over every matrix of the chunk.  The tile is chosen on the host (choose_tiles), a product's result stays
// in registers until its epilogue: the polynomial, the mirror image of a symmetric result, the split into halves, or the
// update of the parameters.  Accumulators pass through LDS, 64 rows at a time, so that every store and every load of what is
// added is 16 bytes of a line that its neighbours fill.
template <int STAGE, int TM, int TN, int WM, int WN, int BK, int DEPTH, int PLANES>
__global__ __launch_bounds__(64 * WM * WN) void fsadam_matrix_stage(const MatrixRow* table, int n_rows, StageArgs k, _Float16* work) {
    constexpr bool kSym = STAGE <= kStageSquare;
    constexpr bool kNN = !kSym;
    using Prod = Product<TM, TN, WM, WN, BK, DEPTH, PLANES, kNN>;
    constexpr int kSlab = 64, kStride = TN + 4;  // the accumulators pass through LDS 64 rows at a time
    constexpr int kLdsBytes = Prod::kLdsHalves * 2 > kSlab * kStride * 4 ? Prod::kLdsHalves * 2 : kSlab * kStride * 4;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kLdsBytes];

    const int kind = STAGE == kStageGram && TM == 64 ? k.kind : STAGE == kStageJoin ? kTilesJoin
                         : (TM == 64 ? kTilesSym64 : TM == 128 ? kTilesSym128 : kTilesSym256) + (STAGE == kStageGram ? 2 : kSym ? 0 : 1);
    static_assert(kTilesFull64 == kTilesSym64 + 1 && kTilesGram64 == kTilesSym64 + 2 && kTilesGram128 == kTilesSym128 + 2 && kTilesGram256 == kTilesSym256 + 2);
    int matrix;
    uint32_t tile;
    const MatrixRow& row = find_tile(table, n_rows, kind, xcd_contiguous(blockIdx.x, gridDim.x), matrix, tile);
    const int s64 = row.s64, l64 = row.l64;
    constexpr int kLog = PLANES == 2 ? 5 : 6;
    static_assert(BK == column_block(PLANES) && BK == 1 << kLog, "a panel is as deep as a block");
    auto place = [&](int i, int j) { return in_blocks(i, j, s64, kLog); };
    uint32_t part_of = 0;  // which part of a split inner product
    if constexpr (STAGE == kStageGram && TM == 64) {
        part_of = tile % (uint32_t)row.parts;
        tile /= (uint32_t)row.parts;
    }
    int ti, tj;
    if constexpr (kSym) {  // row by row under the diagonal
        ti = (int)((__builtin_sqrtf(8.0f * (float)tile + 1.0f) - 1.0f) * 0.5f);
        while ((uint32_t)((ti + 1) * (ti + 2) / 2) <= tile) ++ti;
        while ((uint32_t)(ti * (ti + 1) / 2) > tile) --ti;
        tj = (int)tile - ti * (ti + 1) / 2;
    } else {
        const int down = (s64 + TM - 1) / TM;
        ti = (int)(tile % (uint32_t)down);
        tj = (int)(tile / (uint32_t)down);
    }
    const int64_t plane_x = (int64_t)s64 * l64, plane_a = (int64_t)s64 * s64;
    const _Float16* x = work + row.x_off[k.from] + (int64_t)matrix * 2 * plane_x;
    auto square = [&](int which) { return work + row.sq_off[which] + (int64_t)matrix * PLANES * plane_a; };
    const int i0 = ti * TM, j0 = tj * TN;

    Prod prod;
    // The partial sums of a split product, in the X buffer that the next update writes: tile by tile, part by part, every lane's
    // accumulators side by side.
    constexpr int kTile = TM * TN / 4;  // float4
    auto partial = [&](int part) {
        return reinterpret_cast<float4_t*>(work + row.x_off[k.to] + (int64_t)matrix * 2 * plane_x) + ((int64_t)tile * row.parts + part) * kTile + threadIdx.x;
    };
    if constexpr (STAGE == kStageGram && TM == 64) {
        const int from = (int)part_of * kPartDepth, left = l64 - from;
        const int depth = row.parts > 1 && left > kPartDepth ? kPartDepth : left;
        prod.run(x + place(i0, from), s64, plane_x, s64 - i0, x + place(j0, from), plane_x, s64 - j0, 0, depth, reinterpret_cast<_Float16*>(lds));
        if (row.parts > 1) {
            float4_t* to = partial((int)part_of);
#pragma unroll
            for (int i = 0; i < Prod::MI; ++i)
#pragma unroll
                for (int j = 0; j < Prod::NJ; ++j) to[(i * Prod::NJ + j) * Prod::kThreads] = prod.acc[i][j];
            return;
        }
    } else if constexpr (STAGE == kStageJoin) {
#pragma unroll
        for (int i = 0; i < Prod::MI; ++i)
#pragma unroll
            for (int j = 0; j < Prod::NJ; ++j) prod.acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int n = 0; n < row.parts; ++n)  // in their order
#pragma unroll
            for (int i = 0; i < Prod::MI; ++i)
#pragma unroll
                for (int j = 0; j < Prod::NJ; ++j) prod.acc[i][j] += partial(n)[(i * Prod::NJ + j) * Prod::kThreads];
    } else if constexpr (STAGE == kStageGram)
        prod.run(x + place(i0, 0), s64, plane_x, s64 - i0, x + place(j0, 0), plane_x, s64 - j0, 0, l64, reinterpret_cast<_Float16*>(lds));
    else if constexpr (STAGE == kStageSquare)
        prod.run(square(k.p) + place(i0, 0), s64, plane_a, s64 - i0, square(k.q) + place(j0, 0), plane_a, s64 - j0, 0, s64,
                 reinterpret_cast<_Float16*>(lds));
    else
        prod.run(square(k.p) + place(i0, 0), s64, plane_a, s64 - i0, x + place(0, j0), plane_x, 0, (l64 - j0) / BK, s64, reinterpret_cast<_Float16*>(lds));

    float* slab = reinterpret_cast<float*>(lds);
    // element (i, j) of the slab; columns are exchanged in blocks of 8 by the rows' block of 8, so that reading eight
    // rows of a column at a time (mirror images, tall matrices) spreads over the banks as well
    auto at_slab = [&](int i, int j) { return slab + i * kStride + (j ^ (((i >> 3) & 7) << 3)); };
    auto along_row = [&](int i, int j, float (&v)[8]) {  // (i, j .. j + 7)
        const float4_t* from = reinterpret_cast<const float4_t*>(at_slab(i, j));
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = from[q >> 2][q & 3];
    };
    auto along_column = [&](int i, int j, float (&v)[8]) {  // (i .. i + 7, j)
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = at_slab(i, j)[q * kStride];
    };
    // eight neighbours of a square result, at `at` of its storage; element `on_diagonal` of them is on the diagonal
    auto finish = [&](float (&v)[8], int64_t at, int on_diagonal) {
        float w[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] *= k.product;
        if constexpr (STAGE == kStageSquare) {
            if (k.add >= 0) {
                load_planes<PLANES>(square(k.add) + at, plane_a, w);
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] += k.linear * w[q];
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q == on_diagonal) v[q] += k.diagonal;
        }
        store_planes<PLANES>(square(k.into) + at, plane_a, v);
    };
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    constexpr int kWaveRows = TM / WM, kPieces = kSlab * TN / 8;  // pieces of eight elements
    constexpr int kPer = (kSlab < kWaveRows ? kSlab : kWaveRows) / 16;  // blocks of 16 rows a wave has in a slab
    constexpr int kMine = kPieces / Prod::kThreads;  // pieces of a thread
    // The n-th piece of this thread.  Where results lie in blocks, lanes go through a block's rows (contiguous); where they lie in rows of
    // their own, along those.
    auto piece = [&](int n, int& i, int& j) {
        const int e = threadIdx.x + n * Prod::kThreads;
        if constexpr (STAGE > kStageUpdate) {
            i = e / (TN / 8);
            j = e % (TN / 8) * 8;
        } else {
            i = e / (BK / 8) % kSlab;
            j = e / (BK / 8 * kSlab) * BK + e % (BK / 8) * 8;
        }
    };
    static_assert(kMine * Prod::kThreads == kPieces, "slabs divide among the threads");
    constexpr bool kAddsX = STAGE >= kStageUpdate;
#pragma unroll
    for (int part = 0; part < TM / kSlab; ++part) {
        // What is added to the slab's product is on its way while the slab is written.
        half8_t add_hi[kMine], add_lo[kMine];
        if constexpr (kAddsX) {
#pragma unroll
            for (int n = 0; n < kMine; ++n) {
                int i, j;
                piece(n, i, j);
                if (i0 + part * kSlab < s64 && j0 + j < l64) {
                    const _Float16* from = x + place(i0 + part * kSlab + i, j0 + j);
                    add_hi[n] = *reinterpret_cast<const half8_t*>(from);
                    add_lo[n] = *reinterpret_cast<const half8_t*>(from + plane_x);
                }
            }
        }
        if (kWaveRows > kSlab ? wm == part * kSlab / kWaveRows : wm * kWaveRows / kSlab == part) {
            const int first = (part * kSlab % kWaveRows) / 16;  // of the wave's blocks
            const int down = kWaveRows < kSlab ? wm * kWaveRows % kSlab : 0;  // its rows in the slab
#pragma unroll
            for (int i = 0; i < kPer; ++i)
#pragma unroll
                for (int j = 0; j < Prod::NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        *at_slab(down + i * 16 + (lane >> 4) * 4 + r, wn * (TN / WN) + j * 16 + (lane & 15)) = prod.acc[first + i][j][r];
        }
        __syncthreads();
        const int r0 = i0 + part * kSlab;  // the slab's first row in the result
        if (r0 < s64) {  // sizes are multiples of 64: all rows of the slab are there, or none
            if constexpr (STAGE <= kStageUpdate) {
                const int width = kSym ? s64 : l64;
#pragma unroll
                for (int n = 0; n < kMine; ++n) {
                    int i, j;
                    piece(n, i, j);
                    if (j0 + j >= width) continue;
                    // Every element of a symmetric result is its lower triangle's, also in a tile on the diagonal: what a matrix
                    // gives does not depend on the tiles, and so not on the rest of the list.
                    if (kSym && j0 + j > r0 + i) continue;
                    const int64_t at = place(r0 + i, j0 + j);
                    float v[8];
                    along_row(i, j, v);
                    if constexpr (kSym) {
                        if (j0 + j + 7 > r0 + i) {  // the diagonal runs through these eight
                            const int down = j0 + j - r0;  // the first one's column as a row of the slab
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (j0 + j + q > r0 + i) v[q] = *at_slab(down + q, r0 + i - j0);
                        }
                        finish(v, at, r0 + i - (j0 + j));
                    } else {
#pragma unroll
                        for (int q = 0; q < 8; ++q) v[q] = k.linear * ((float)add_hi[n][q] + (float)add_lo[n][q]) + k.product * v[q];
                        store_planes<2>(work + row.x_off[k.to] + (int64_t)matrix * 2 * plane_x + at, plane_x, v);
                    }
                }
                if constexpr (kSym) {
                    {  // the mirror image
                        for (int e = threadIdx.x; e < kPieces; e += Prod::kThreads) {
                            // rows j of the result: lanes through the rows of a block of its columns
                            const int j = e / (BK / 8) % TN, i = e / (BK / 8 * TN) * BK + e % (BK / 8) * 8;
                            if (j0 + j >= s64 || (j0 + j) / 8 >= (r0 + i) / 8) continue;
                            const int64_t at = place(j0 + j, r0 + i);
                            float v[8];
                            along_column(i, j, v);
                            finish(v, at, -8);
                        }
                    }
                }
            } else {
                // the last product: into the results or the parameters, in their own orientation, eight elements along
                // their rows at a time
                const int64_t numel = (int64_t)row.rows * row.cols;
                const float ratio = row.step_ratio;
                if (row.tall) {  // a X + B X along the rows of X first, in the slab: its columns are what is written
#pragma unroll
                    for (int n = 0; n < kMine; ++n) {
                        int i, j;
                        piece(n, i, j);
                        if (j0 + j >= l64) continue;
                        float o[8];
                        along_row(i, j, o);
#pragma unroll
                        for (int q = 0; q < 8; ++q) o[q] = k.linear * ((float)add_hi[n][q] + (float)add_lo[n][q]) + k.product * o[q];
                        float4_t* to = reinterpret_cast<float4_t*>(at_slab(i, j));
                        to[0] = float4_t{o[0], o[1], o[2], o[3]};
                        to[1] = float4_t{o[4], o[5], o[6], o[7]};
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int n = 0; n < kMine; ++n) {
                    int i, j;
                    float o[8], w[8];
                    if (row.tall) {
                        const int e = threadIdx.x + n * Prod::kThreads;
                        j = e / (kSlab / 8);
                        i = (e % (kSlab / 8)) * 8;
                        if (r0 + i >= row.s || j0 + j >= row.l) continue;
                        along_column(i, j, o);
                    } else {
                        piece(n, i, j);
                        if (r0 + i >= row.s || j0 + j >= row.l) continue;
                        along_row(i, j, o);
#pragma unroll
                        for (int q = 0; q < 8; ++q) o[q] = k.linear * ((float)add_hi[n][q] + (float)add_lo[n][q]) + k.product * o[q];
                    }
                    const int64_t r = row.tall ? j0 + j : r0 + i, c = row.tall ? r0 + i : j0 + j;
                    const int left = row.cols - (int)c;  // elements of the row from here on
                    if constexpr (STAGE == kStageOut) {
                        store_eight(row.dst, (int64_t)matrix * row.dst_stride + r * row.dst_ld + c, k.dst_type, left, o);
                    } else {
                        const int64_t to = (int64_t)matrix * numel + r * row.cols + c;
                        load_eight(row.dst, to, k.dst_type, left, w);
#pragma unroll
                        for (int q = 0; q < 8; ++q) o[q] = w[q] * k.keep - ratio * o[q];
                        store_eight(row.dst, to, k.dst_type, left, o);
                        if (k.copy_type >= 0) store_eight(row.copy, to, k.copy_type, left, o);
                    }
                }
            }
        }
        __syncthreads();
    }
}

// ---- matrices that fit a compute unit's LDS -----------------------------------------------------------------------

// One workgroup takes a matrix from the source to the result: X (two planes) and one square matrix stay in LDS, products
// go through registers, nothing is written to memory in between.  Bound by latency: a compute unit reads its operands from LDS at
// 128 bytes a clock, and between the products all its waves wait for each other.  Five steps of 16 x 16 16 us, 64 x 256 36 us, 128 x 128 73 us, where the launches of the
// stages take 100 us for any matrix this small.  All the launches and the trips to the L2 and back
// that the stages above are made of are what such a matrix would wait for.
struct alignas(16) ResidentRow {
    const void* src;
    float* buf;
    void* dst;
    void* copy;
    int64_t src_ld, src_stride, dst_ld, dst_stride;
    int32_t rows, cols;
    int32_t first_matrix;
    float step_ratio;
};
constexpr int kResidentRowsPerLaunch = 24;
struct ResidentRows {
    ResidentRow row[kResidentRowsPerLaunch];
};
struct ResidentInMemory {
    const ResidentRow* row;
    int n;
};
struct ResidentInArguments {
    ResidentRows rows;
    int n;
};
__device__ __forceinline__ const ResidentRow* rows_of(const ResidentInMemory& t) { return t.row; }
__device__ __forceinline__ const ResidentRow* rows_of(const ResidentInArguments& t) { return t.rows.row; }
constexpr int kMaxSteps = 32;
enum { kFactorGram, kFactorLinearB, kFactorProductB, kFactorLinearX, kFactorProductX };
struct ResidentArgs {
    int steps, src_type, dst_type, copy_type;
    float keep;
    double eps, power;  // of the norm; 2^x of X0
    float factors[5][kMaxSteps];  // [kFactor...][step]
};

// Storage in LDS: sides padded to 32 (the depth of a matrix instruction), rows 8 halves longer than that, which spreads the 16
// rows a fragment is read from over the banks.
constexpr int kResidentThreads = 1024, kResidentWaves = kResidentThreads / 64;
constexpr int kResidentElems = 38912;  // of X and the square matrix, rows' ends included: 4 bytes each in 152 of the 160 KiB
constexpr int kResidentSide = 128;
constexpr int kResidentBatch = 16;        // elements of a thread in registers
__host__ __device__ constexpr int resident_pitch(int side) { return (side + 31) / 32 * 32 + 8; }
__host__ __device__ constexpr bool resident_fits(int64_t s, int64_t l) {
    return s <= kResidentSide && l <= kResidentElems && (s + 31) / 32 * 32 * (resident_pitch((int)l) + resident_pitch((int)s)) <= kResidentElems;
}

// SIDE: the short side in tiles of 16, padded to 32: 2, 4, 6 or 8.  A constant, so that the addresses of the square matrix's tiles
// are one register and offsets in the instructions.
template <int SIDE, bool STEP>
__device__ __forceinline__ void resident_matrix(const ResidentRow& row, const ResidentArgs& k, const MomentumArgs& mk, unsigned char* lds, double* part,
                                                const float (*factors)[kMaxSteps]) {
    const int steps = k.steps, src_type = k.src_type, dst_type = k.dst_type, copy_type = k.copy_type;
    const float keep = k.keep;
    const int64_t matrix = (int)blockIdx.x - row.first_matrix;
    const int rows = row.rows, cols = row.cols;
    const bool tall = rows > cols;
    const int s = tall ? cols : rows, l = tall ? rows : cols;
    constexpr int sp = SIDE * 16, pitch_a = sp + 8, plane_a = sp * pitch_a;  // halves
    const int lp = (l + 31) / 32 * 32, pitch_x = lp + 8, plane_x = sp * pitch_x;
    _Float16* a = reinterpret_cast<_Float16*>(lds);
    _Float16* x = a + 2 * plane_a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;

    // the padding is zero and stays zero
    for (int e = tid; e < 2 * plane_x / 8; e += kResidentThreads) *reinterpret_cast<half8_t*>(x + e * 8) = half8_t{};
    __syncthreads();
    // element e of the matrix, row-major as in the source
    const int numel = rows * cols;
    const float per_row = 1.0f / (float)cols;
    auto place = [&](int e, int& r, int& q) {  // e < 2^17, so half a column is far more than the rounding of the product
        r = (int)(((float)e + 0.5f) * per_row);
        q = e - r * cols;
    };
    const Divisor by(mk);
    const int64_t base = matrix * row.src_stride, flat = matrix * numel;
    double sum = 0.0;
    float u[kResidentBatch];
    // elements e0, e0 + 1024, ... : all loads first
    auto fetch = [&](int e0, bool first) {
        int64_t at[kResidentBatch];
#pragma unroll
        for (int n = 0; n < kResidentBatch; ++n) {
            const int e = e0 + n * kResidentThreads;
            int r, q;
            place(e, r, q);
            at[n] = e >= numel ? -1 : STEP ? flat + e : base + r * row.src_ld + q;
        }
        if (src_type == kTypeF32) {
#pragma unroll
            for (int n = 0; n < kResidentBatch; ++n) u[n] = at[n] >= 0 ? static_cast<const float*>(row.src)[at[n]] : 0.0f;
        } else {
            uint16_t raw[kResidentBatch];
#pragma unroll
            for (int n = 0; n < kResidentBatch; ++n) raw[n] = at[n] >= 0 ? static_cast<const uint16_t*>(row.src)[at[n]] : (uint16_t)0;
#pragma unroll
            for (int n = 0; n < kResidentBatch; ++n) u[n] = src_type == kTypeF16 ? (float)__builtin_bit_cast(_Float16, raw[n]) : low_half(raw[n]);
        }
        if constexpr (STEP) {
            float m[kResidentBatch];
#pragma unroll
            for (int n = 0; n < kResidentBatch; ++n) m[n] = at[n] >= 0 ? row.buf[at[n]] : 0.0f;
#pragma unroll
            for (int n = 0; n < kResidentBatch; ++n) {
                if (first) {
                    u[n] = momentum_update(by(u[n]), m[n], mk);
                    if (at[n] >= 0) row.buf[at[n]] = m[n];
                } else {
                    u[n] = update_again(by(u[n]), m[n], mk);
                }
            }
        }
    };
    auto spread = [&](int e0, double factor) {
#pragma unroll
        for (int n = 0; n < kResidentBatch; ++n) {
            const int e = e0 + n * kResidentThreads;
            if (e >= numel) continue;
            int r, q;
            place(e, r, q);
            const int at = tall ? q * pitch_x + r : r * pitch_x + q;
            split_halves((float)((double)u[n] * factor), x[at], x[plane_x + at]);
        }
    };
    constexpr int kTurn = kResidentThreads * kResidentBatch;  // elements of one turn; a matrix of no more is read once
    for (int e0 = tid; e0 < numel; e0 += kTurn) {
        fetch(e0, true);
#pragma unroll
        for (int n = 0; n < kResidentBatch; ++n) sum = __builtin_fma((double)u[n], (double)u[n], sum);
    }
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_down(sum, d);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int n = 0; n < kResidentWaves; ++n) sum += part[n];
    const double norm = sqrt(sum);
    const double factor = __builtin_isfinite(sum) ? k.power / (norm > k.eps ? norm : k.eps) : __builtin_nan("");
    if (numel <= kTurn) {
        spread(tid, factor);
    } else {
        for (int e0 = tid; e0 < numel; e0 += kTurn) {
            fetch(e0, false);
            spread(e0, factor);
        }
    }
    __syncthreads();

    auto read8 = [](const _Float16* p) { return *reinterpret_cast<const half8_t*>(p); };
    auto turned = [](const _Float16* at, int pitch) {  // rows at, at + pitch, ... + 7 pitch of 16 columns: eight deep for every column
        const short4_t first = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FM_LDS short4_t*)at);
        const short4_t second = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FM_LDS short4_t*)(at + 4 * pitch));
        return __builtin_shufflevector(__builtin_bit_cast(half4_t, first), __builtin_bit_cast(half4_t, second), 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto mfma = [](const half8_t& p, const half8_t& q, const float4_t& v) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, v, 0, 0, 0); };
    // lane (g, c): operands hold row c, eight deep from 8 g on; a product holds rows 4 g .. 4 g + 3 of column c
    const _Float16* const row_a = a + c * pitch_a + g * 8;
    const _Float16* const row_x = x + c * pitch_x + g * 8;
    constexpr int kSquare = SIDE * (SIDE + 1) / 2, kRounds = (kSquare + kResidentWaves - 1) / kResidentWaves;
    auto triangle = [&](int t, int& ti, int& tj) {  // row by row under the diagonal
        ti = 0;
#pragma unroll
        for (int n = 1; n < SIDE; ++n) ti += t >= n * (n + 1) / 2;
        tj = t - ti * (ti + 1) / 2;
    };
    auto put_square = [&](int ti, int tj, const float4_t& v) {  // the lower triangle and its mirror image
        half4_t hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            _Float16 h, o;
            split_halves(v[r], h, o);
            hi[r] = h;
            lo[r] = o;
        }
        _Float16* const here = a + (ti * 16 + 4 * g) * pitch_a + tj * 16 + c;
        _Float16* const there = a + (tj * 16 + c) * pitch_a + ti * 16 + 4 * g;
        if (ti != tj) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                here[r * pitch_a] = hi[r];
                here[plane_a + r * pitch_a] = lo[r];
            }
            *reinterpret_cast<half4_t*>(there) = hi;
            *reinterpret_cast<half4_t*>(there + plane_a) = lo;
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (c > 4 * g + r) continue;
                here[r * pitch_a] = there[r] = hi[r];
                here[plane_a + r * pitch_a] = there[plane_a + r] = lo[r];
            }
        }
    };
    // A wave takes whole columns of tiles of X: what it overwrites, it alone has read.
    constexpr int kAtOnce = SIDE % 4 == 0 ? 4 : 2;
    const int along = lp / 16;
    auto columns = [&](int step, auto&& done) {
        const float linear = factors[kFactorLinearX][step], scale = factors[kFactorProductX][step];
        for (int tj = wave; tj < along; tj += kResidentWaves) {
            float4_t next[SIDE];
#pragma unroll
            for (int ti = 0; ti < SIDE; ++ti) next[ti] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            const _Float16* column = x + (8 * g + (c >> 2)) * pitch_x + (c & 3) * 4 + tj * 16;
#pragma unroll 1
            for (int d = 0; d < SIDE / 2; ++d, column += 32 * pitch_x) {
                const half8_t q0 = turned(column, pitch_x), q1 = turned(column + plane_x, pitch_x);
#pragma unroll
                for (int t0 = 0; t0 < SIDE; t0 += kAtOnce) {
                    half8_t p0[kAtOnce], p1[kAtOnce];
#pragma unroll
                    for (int t = 0; t < kAtOnce; ++t) {
                        p0[t] = read8(row_a + d * 32 + (t0 + t) * 16 * pitch_a);
                        p1[t] = read8(row_a + d * 32 + plane_a + (t0 + t) * 16 * pitch_a);
                    }
#pragma unroll
                    for (int t = 0; t < kAtOnce; ++t) next[t0 + t] = mfma(p1[t], q0, next[t0 + t]);
#pragma unroll
                    for (int t = 0; t < kAtOnce; ++t) next[t0 + t] = mfma(p0[t], q1, next[t0 + t]);
#pragma unroll
                    for (int t = 0; t < kAtOnce; ++t) next[t0 + t] = mfma(p0[t], q0, next[t0 + t]);
                }
            }
            _Float16* at = x + 4 * g * pitch_x + tj * 16 + c;
#pragma unroll
            for (int ti = 0; ti < SIDE; ++ti, at += 16 * pitch_x) {
                float o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = linear * ((float)at[r * pitch_x] + (float)at[plane_x + r * pitch_x]) + scale * next[ti][r];
                done(at, ti * 16 + 4 * g, tj * 16 + c, o);
            }
        }
    };
    for (int step = 0; step < steps; ++step) {
#pragma unroll
        for (int n = 0; n < kRounds; ++n) {
            const int t = wave + n * kResidentWaves;
            if (t >= kSquare) break;
            int ti, tj;
            triangle(t, ti, tj);
            const _Float16 *p = row_x + ti * 16 * pitch_x, *q = row_x + tj * 16 * pitch_x;
            float4_t high = {0.0f, 0.0f, 0.0f, 0.0f}, cross = high, cross2 = high;
            for (int d = 0; d < lp; d += 32) {
                const half8_t p0 = read8(p + d), p1 = read8(p + plane_x + d), q0 = read8(q + d), q1 = read8(q + plane_x + d);
                cross = mfma(p1, q0, cross);
                cross2 = mfma(p0, q1, cross2);
                high = mfma(p0, q0, high);
            }
            put_square(ti, tj, (high + (cross + cross2)) * factors[kFactorGram][step]);
        }
        __syncthreads();
        float4_t b[kRounds];
#pragma unroll
        for (int n = 0; n < kRounds; ++n) {
            const int t = wave + n * kResidentWaves;
            if (t >= kSquare) break;
            int ti, tj;
            triangle(t, ti, tj);
            const _Float16 *p = row_a + ti * 16 * pitch_a, *q = row_a + tj * 16 * pitch_a;
            float4_t high = {0.0f, 0.0f, 0.0f, 0.0f}, cross = high, cross2 = high;
#pragma unroll
            for (int d = 0; d < sp; d += 32) {
                const half8_t p0 = read8(p + d), p1 = read8(p + plane_a + d), q0 = read8(q + d), q1 = read8(q + plane_a + d);
                cross = mfma(p1, q0, cross);
                cross2 = mfma(p0, q1, cross2);
                high = mfma(p0, q0, high);
            }
            const _Float16* here = a + (ti * 16 + 4 * g) * pitch_a + tj * 16 + c;
            const float linear = factors[kFactorLinearB][step], scale = factors[kFactorProductB][step];
            b[n] = (high + (cross + cross2)) * scale;
#pragma unroll
            for (int r = 0; r < 4; ++r) b[n][r] += linear * ((float)here[r * pitch_a] + (float)here[plane_a + r * pitch_a]);
        }
        __syncthreads();  // A has been read: B takes its place
#pragma unroll
        for (int n = 0; n < kRounds; ++n) {
            const int t = wave + n * kResidentWaves;
            if (t >= kSquare) break;
            int ti, tj;
            triangle(t, ti, tj);
            put_square(ti, tj, b[n]);
        }
        __syncthreads();
        if (step + 1 < steps) {
            columns(step, [&](_Float16* at, int, int, const float (&o)[4]) {
#pragma unroll
                for (int r = 0; r < 4; ++r) split_halves(o[r], at[r * pitch_x], at[plane_x + r * pitch_x]);
            });
            __syncthreads();
        } else {
            columns(step, [&](_Float16*, int i, int j, const float (&o)[4]) {
                const int64_t step_i = tall ? 1 : STEP ? cols : row.dst_ld, step_j = tall ? (STEP ? cols : row.dst_ld) : 1;
                const int64_t to = (STEP ? flat : matrix * row.dst_stride) + i * step_i + j * step_j;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (i + r >= s || j >= l) continue;
                    if constexpr (STEP) {
                        const float p = load_as_float(row.dst, to + r * step_i, dst_type) * keep - row.step_ratio * o[r];
                        store_from_float(row.dst, to + r * step_i, dst_type, p);
                        if (copy_type >= 0) store_from_float(row.copy, to + r * step_i, copy_type, p);
                    } else {
                        store_from_float(row.dst, to + r * step_i, dst_type, o[r]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // one tile's addresses at a time: the registers do not hold those of eight
            });
        }
    }
}

template <bool STEP, typename Table>
__global__ __launch_bounds__(kResidentThreads) void fsadam_matrix_resident(Table tables, ResidentArgs k, MomentumArgs mk) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ double part[kResidentWaves];
    const ResidentRow* table = rows_of(tables);
    const ResidentRow row = table[find_row(tables.n, blockIdx.x, [&](int r) { return table[r].first_matrix; })];
    // The arguments of a launch are not in the GPU's memory: the factors of all steps are fetched together, once.
    __shared__ float factors[5][kMaxSteps];
    if (threadIdx.x < 5 * kMaxSteps) (&factors[0][0])[threadIdx.x] = (&k.factors[0][0])[threadIdx.x];
    switch (((row.rows < row.cols ? row.rows : row.cols) + 31) / 32) {
        case 1: resident_matrix<2, STEP>(row, k, mk, lds, part, factors); break;
        case 2: resident_matrix<4, STEP>(row, k, mk, lds, part, factors); break;
        case 3: resident_matrix<6, STEP>(row, k, mk, lds, part, factors); break;
        default: resident_matrix<8, STEP>(row, k, mk, lds, part, factors); break;
    }
}

// Rows of a call's table, in the arguments of the launch: nothing is allocated or copied, and a captured graph holds them.
constexpr int kRowsPerPut = 14;
struct MatrixRows {
    MatrixRow row[kRowsPerPut];
};
__global__ void fsadam_put_matrix_rows(MatrixRow* table, int n, MatrixRows rows) {
    constexpr int kWords = sizeof(MatrixRow) / 16;
    typedef uint32_t word_t __attribute__((ext_vector_type(4)));
    for (int e = threadIdx.x; e < n * kWords; e += blockDim.x) reinterpret_cast<word_t*>(table)[e] = reinterpret_cast<const word_t*>(rows.row)[e];
}
__global__ void fsadam_put_resident_rows(ResidentRow* table, int n, ResidentRows rows) {
    constexpr int kWords = sizeof(ResidentRow) / 16;
    for (int e = threadIdx.x; e < n * kWords; e += blockDim.x) reinterpret_cast<words4_t*>(table)[e] = reinterpret_cast<const words4_t*>(rows.row)[e];
}
__global__ void fsadam_clear_flag(float* flag) { *flag = 0.0f; }
__global__ void fsadam_put_momentum_rows(MomentumRow* table, int n, MomentumRows rows) {
    constexpr int kWords = sizeof(MomentumRow) / 16;
    typedef uint32_t word_t __attribute__((ext_vector_type(4)));
    for (int e = threadIdx.x; e < n * kWords; e += blockDim.x) reinterpret_cast<word_t*>(table)[e] = reinterpret_cast<const word_t*>(rows.row)[e];
}

}  // namespace
