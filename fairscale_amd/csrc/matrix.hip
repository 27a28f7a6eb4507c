// Matrix operators of libfsadam for MI355X (gfx950): momentum pass, orthogonalisation by Newton-Schulz products, and the
// optimizer step made of both.  Host code and C ABI (include/fsadam.h); the kernels are in matrix_kernels.h.
//
// A call covers a list of matrices of any shapes.  Its work is cut into chunks whose intermediate matrices fit the
// workspace; a chunk is a table of rows (one per list entry) and a fixed sequence of launches, each over the tiles of every
// matrix in it, so that the number of launches does not grow with the list and small matrices share the machine:
//     table | sums of squares per 8192 elements (the step: momentum update too) | norms | normalise and split |
//     steps x (Gram, polynomial, update) -- the last update writes the results or the parameters.
// Nothing outlives a call: tables travel in kernel arguments, everything else is in the caller's workspace.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>
#include <string>
#include <type_traits>
#include <vector>

#include "fsadam.h"

#include "matrix_kernels.h"

__attribute__((visibility("hidden"))) int fsadam_fail(int code, const char* msg) noexcept;  // fsadam.hip: the message of this thread

namespace {

int fail(int code, const std::string& msg) { return fsadam_fail(code, msg.c_str()); }
int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FSADAM_OK : fail(FSADAM_EHIP, std::string("kernel launch: ") + hipGetErrorString(e));
}

// No exception crosses the C boundary.
template <typename F>
int guarded(F&& body) noexcept {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fsadam_fail(FSADAM_ENOMEM, "out of host memory");
    } catch (const std::exception& e) {
        return fsadam_fail(FSADAM_EINVAL, e.what());
    } catch (...) {
        return fsadam_fail(FSADAM_EINVAL, "unknown exception");
    }
}

bool valid_type(int t) { return t == FSADAM_TYPE_F32 || t == FSADAM_TYPE_F16 || t == FSADAM_TYPE_BF16; }
int size_of(int t) { return t == FSADAM_TYPE_F32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

constexpr int64_t kMaxSide = 1 << 20;
// A launch takes fewer than 2^32 threads.
constexpr int64_t most_workgroups(int64_t threads) { return UINT32_MAX / threads; }
constexpr int64_t kMaxTiles = most_workgroups(512);  // of a chunk, of any kind: no launch over them has larger workgroups
// Intermediate matrices of one chunk.  Enough for eight 4096 x 11008 matrices, whose products then have thousands of
// tiles for the 256 compute units; a matrix that needs more gets what it needs.
constexpr int64_t kChunkBytes = int64_t(4) << 30;

// ---- numbers of the iteration -------------------------------------------------------------------------------------

// Where u + v t + w t^2 vanishes: up to two values of t, NaN where there are fewer.
void roots(double u, double v, double w, double (&t)[2]) {
    t[0] = t[1] = std::nan("");
    if (w == 0.0) {
        if (v != 0.0) t[0] = -u / v;
        return;
    }
    const double d = v * v - 4.0 * u * w;
    if (d < 0.0) return;
    const double h = -0.5 * (v + std::copysign(std::sqrt(d), v));  // no cancellation: the other root is u / h
    t[0] = h / w;
    t[1] = h != 0.0 ? u / h : 0.0;
}
// Largest |f(t)| on [0, top]: at the ends, or at `at` (where its derivative vanishes).
template <typename F>
double largest(const F& f, double top, const double (&at)[2]) {
    double most = std::max(std::fabs(f(0.0)), std::fabs(f(top)));
    for (double t : at)
        if (t > 0.0 && t < top) most = std::max(most, std::fabs(f(t)));
    return most;
}

// The powers of two that a step's matrices are held with.  With t the square of a singular value (a: step's polynomial
// q(t) = a + b t + c t^2, so that X <- q(A) X):  A: t,  B: b t + c t^2,  R: q(t),  T: t q(t).
struct StepNumbers {
    int x, a, b, r, t;
    double q_bound;  // of |q|
};
int exponent_for(double bound) {  // the largest k with bound * 2^k <= 60000 (halves end at 65504), at most 15
    if (!(bound > 0x1p-15)) return 15;
    return std::min(15, (int)std::floor(std::log2(60000.0 / bound)));
}

// How large the eigenvalues of those matrices can be at every step, when the singular values of X0 are in [0, 1].  2 % a step stands
// for what its rounding adds: with 11-bit products (local_error below) at most 1.76 % of the largest value that an odd polynomial of
// fifth degree takes on the interval, reached by Chebyshev's 5 x - 20 x^3 + 16 x^5.  Errors of earlier steps need no room: the bound is
// that of every value in the interval, and so of the one that was moved.
int step_bounds(const FsOrthOptions& o, std::vector<StepNumbers>& numbers) {
    const double a = o.a, b = o.b, c = o.c;
    const auto q = [&](double t) { return a + t * (b + t * c); };
    double q_flat[2], t_flat[2], p_flat[2];
    roots(b, 2.0 * c, 0.0, q_flat);          // of q and of b t + c t^2
    roots(a, 2.0 * b, 3.0 * c, t_flat);      // of t q(t)
    roots(a, 3.0 * b, 5.0 * c, p_flat);      // of t q(t)^2, but for the zeros of q
    numbers.clear();
    double m = 1.0;
    for (int k = 0; k < o.steps; ++k) {
        m *= 1.02;
        StepNumbers n;
        const double top = m * m, most_q = largest(q, top, q_flat);
        const double most_b = largest([&](double t) { return t * (b + t * c); }, top, q_flat);
        const double most_t = largest([&](double t) { return t * q(t); }, top, t_flat);
        m = std::sqrt(largest([&](double t) { return t * q(t) * q(t); }, top, p_flat));
        if (!(m <= 1024.0))
            return fail(FSADAM_EINVAL, "the coefficients let singular values in [0, 1] grow past 1024 by step " + std::to_string(k + 1));
        n.x = exponent_for(std::sqrt(top));
        n.a = exponent_for(top);
        n.b = exponent_for(most_b);
        n.r = exponent_for(most_q);
        n.t = exponent_for(most_t);
        n.q_bound = most_q;
        numbers.push_back(n);
    }
    return FSADAM_OK;
}

// What 11-bit products can do to a singular value.  With each of them off by at most u = 2^-11 of itself -- X's first half (d), A (e)
// and B (f) -- a step is off, to first order, by
//     x ((b x^2 + 2 c x^4) (2 d + e) + (b x^2 + c x^4) (f + d)),
// and multiplies what was off before by its slope a + 3 b x^2 + 5 c x^4.  That is what happens to a matrix of one entry in a row and
// column, or of rank one with entries of one size, where all roundings of a kind are alike; in others they average.  The usual
// coefficients and five steps: 0.057 (the worst of 4e5 singular values with these roundings made: 0.024, and 2.9 % of what a value is sent to;
// Gaussian matrices 2e-3 of the norm).  Slopes over 1 multiply it: 0.094 for six steps, 0.62 for five steps of (4.0848, -6.8946, 2.9270).  Above 1/16 the products
// take 22 bits, whatever was asked for.  256 values tell it to 4 % there.
constexpr double kMostHalfError = 1.0 / 16;
int products_of(const FsOrthOptions& o) {
    if (o.products == FSADAM_PRODUCTS_SPLIT) return FSADAM_PRODUCTS_SPLIT;
    const double a = o.a, b = o.b, c = o.c, u = 0x1p-11;
    constexpr int kValues = 256;
    double x[kValues], error[kValues];
    for (int k = 0; k < kValues; ++k) x[k] = (k + 1.0) / kValues, error[k] = 0.0;
    for (int s = 0; s < o.steps; ++s) {
        int over = 0;
        for (int k = 0; k < kValues; ++k) {
            const double t = x[k] * x[k], in_a = t * (b + 2.0 * c * t), in_b = t * (b + c * t);
            const double local_error = u * std::fabs(x[k]) * (std::fabs(2.0 * in_a + in_b) + std::fabs(in_a) + std::fabs(in_b));
            error[k] = error[k] * std::fabs(a + t * (3.0 * b + 5.0 * c * t)) + local_error;
            x[k] *= a + in_b;
            over |= !(error[k] <= kMostHalfError);
        }
        if (over) return FSADAM_PRODUCTS_SPLIT;
    }
    return FSADAM_PRODUCTS_HALF;
}

int check_options(const FsOrthOptions* o) {
    if (!o) return fail(FSADAM_EINVAL, "options is NULL");
    if (o->steps < 1 || o->steps > kMaxSteps) return fail(FSADAM_EINVAL, "steps must be in [1, 32], got " + std::to_string(o->steps));
    if (!std::isfinite(o->a) || !std::isfinite(o->b) || !std::isfinite(o->c)) return fail(FSADAM_EINVAL, "the coefficients must be finite");
    if (!(o->eps > 0.0f) || !std::isfinite(o->eps)) return fail(FSADAM_EINVAL, "eps must be positive and finite");
    if (o->products != FSADAM_PRODUCTS_HALF && o->products != FSADAM_PRODUCTS_SPLIT) return fail(FSADAM_EINVAL, "unknown products " + std::to_string(o->products));
    std::vector<StepNumbers> numbers;
    return step_bounds(*o, numbers);
}

// ---- chunks -------------------------------------------------------------------------------------------------------

struct Chunk {
    std::vector<MatrixRow> rows;
    int64_t matrices = 0;
    int64_t tiles[kTileKinds] = {};
    int64_t halves = 0;  // of the intermediate matrices
    int products = 0;    // FSADAM_PRODUCTS_* of its launches
    bool pairs() const { return products == FSADAM_PRODUCTS_SPLIT; }  // steps are taken two at a time (run_chunk)
    int64_t head_bytes() const { return up((int64_t)rows.size() * sizeof(MatrixRow), 256) + up(matrices * 8, 256) + up(tiles[kTilesChunk] * 8, 256); }
    int64_t bytes() const { return head_bytes() + halves * 2; }
    int64_t mean_depth() const {  // of the updates' products, over their tiles
        int64_t tiles = 0, deep = 0;
        for (const MatrixRow& row : rows) {
            const int64_t n = (int64_t)row.batch * row.n[kTilesFull64];
            tiles += n;
            deep += n * row.s64;
        }
        return std::max<int64_t>(64, deep / std::max<int64_t>(1, tiles));
    }
};

int64_t symmetric_tiles(int64_t s, int64_t t) { const int64_t n = (s + t - 1) / t; return n * (n + 1) / 2; }
int64_t full_tiles(int64_t s, int64_t l, int64_t t) { return ((s + t - 1) / t) * ((l + t - 1) / t); }

// Adds up to `batch` matrices of a row to the chunk; returns how many fit.  A chunk takes at least one.
int64_t add_to_chunk(Chunk& chunk, const MatrixRow& proto, int64_t batch) {
    const int64_t products = chunk.products;
    const int64_t x = 2 * (int64_t)proto.s64 * proto.l64, a = products * (int64_t)proto.s64 * proto.s64;  // halves of one matrix, one buffer
    const int squares = chunk.pairs() ? 3 : 2;
    const int64_t per = 2 * x + squares * a, room = kChunkBytes / 2 - chunk.halves;
    int64_t n = std::min(batch, room / per);
    int64_t most = kMaxTiles;
    for (int k = 0; k < kTileKinds; ++k)
        if (proto.n[k]) most = std::min(most, (kMaxTiles - chunk.tiles[k]) / proto.n[k]);
    n = std::min(n, most);
    if (n < 1) {
        if (!chunk.rows.empty()) return 0;
        n = 1;
    }
    MatrixRow row = proto;
    row.batch = (int32_t)n;
    row.first_matrix = (int32_t)chunk.matrices;
    for (int k = 0; k < kTileKinds; ++k) {
        row.first[k] = (int32_t)chunk.tiles[k];
        chunk.tiles[k] += n * proto.n[k];
    }
    row.x_off[0] = chunk.halves;
    row.x_off[1] = row.x_off[0] + n * x;
    chunk.halves = row.x_off[1] + n * x;
    for (int k = 0; k < squares; ++k) {
        row.sq_off[k] = chunk.halves;
        chunk.halves += n * a;
    }
    chunk.matrices += n;
    chunk.rows.push_back(row);
    return n;
}

struct Source {  // what a list entry's row starts from
    const void* src; float* buf; void* dst; void* copy;
    int64_t batch, rows, cols, src_ld, src_stride, dst_ld, dst_stride;
    float step_ratio;
    int src_size, dst_size, copy_size;
};

// Matrices of a short side up to this are always multiplied to 22 bits: their products are too small to be what a call waits for,
// and few singular values are where the error of 11 bits averages least (products_of; larger matrices can have few as well, so this is
// no promise about the error).
constexpr int64_t kAlwaysSplit = 128;

// A Gram matrix of few tiles and long inner products keeps a few compute units busy for long: parts of kPartDepth are summed by
// workgroups of their own and joined in order by a second launch.  By the matrix alone, so that its bits do not depend on the
// list.  32 matrices of 128 x 4096: 39 -> 23 us, both launches.
int gram_parts(int64_t s64, int64_t l64) {
    if (s64 > 384 || l64 < 2 * kPartDepth) return 1;
    return (int)((l64 + kPartDepth - 1) / kPartDepth);
}

bool resident(const Source& in) { return resident_fits(std::min(in.rows, in.cols), std::max(in.rows, in.cols)); }

void make_chunks(const std::vector<Source>& all, const FsOrthOptions& options, std::vector<Chunk>& chunks) {
  const bool large = std::any_of(all.begin(), all.end(), [](const Source& in) { return std::min(in.rows, in.cols) > kAlwaysSplit; });
  const int asked = large ? products_of(options) : options.products;
  for (int products : {FSADAM_PRODUCTS_HALF, FSADAM_PRODUCTS_SPLIT}) {
    bool fresh = true;  // a chunk is of one kind
    for (const Source& in : all) {
        if (resident(in) || (std::min(in.rows, in.cols) <= kAlwaysSplit ? FSADAM_PRODUCTS_SPLIT : asked) != products) continue;
        MatrixRow row{};
        row.rows = (int32_t)in.rows;
        row.cols = (int32_t)in.cols;
        row.tall = in.rows > in.cols;
        row.s = row.tall ? row.cols : row.rows;
        row.l = row.tall ? row.rows : row.cols;
        row.s64 = (int32_t)up(row.s, 64);
        row.l64 = (int32_t)up(row.l, 64);
        row.src_ld = in.src_ld; row.src_stride = in.src_stride;
        row.dst_ld = in.dst_ld; row.dst_stride = in.dst_stride;
        row.step_ratio = in.step_ratio;
        row.chunks = (int32_t)(up(in.rows * in.cols, kChunkElems) / kChunkElems);
        row.parts = gram_parts(row.s64, row.l64);
        for (int t = 64, k = kTilesSym64; t <= 256; t *= 2, k += 3) {
            row.n[k] = (int32_t)symmetric_tiles(row.s64, t);
            row.n[k + 1] = (int32_t)full_tiles(row.s64, row.l64, t);
            row.n[k + 2] = row.parts > 1 ? 0 : row.n[k];  // the Gram matrix
        }
        row.n[kTilesJoin] = row.parts > 1 ? row.n[kTilesSym64] : 0;
        row.n[kTilesPart] = row.n[kTilesJoin] * row.parts;
        row.n[kTilesAllParts] = row.n[kTilesSym64] * row.parts;
        row.n[kTilesPrep] = (int32_t)full_tiles(row.s64, row.l64, 64);
        row.n[kTilesChunk] = row.chunks;
        int64_t done = 0;
        while (done < in.batch) {
            row.src = static_cast<const char*>(in.src) + done * in.src_stride * in.src_size;
            row.buf = in.buf ? in.buf + done * in.rows * in.cols : nullptr;
            row.dst = static_cast<char*>(in.dst) + done * in.dst_stride * in.dst_size;
            row.copy = in.copy ? static_cast<char*>(in.copy) + done * in.rows * in.cols * in.copy_size : nullptr;
            if (fresh) {
                chunks.emplace_back();
                chunks.back().products = products;
            }
            const int64_t n = add_to_chunk(chunks.back(), row, in.batch - done);
            fresh = n == 0;
            done += n;
        }
    }
  }
}

// The rows of the list that fit LDS.
struct Residents {
    std::vector<ResidentRow> rows;
    int64_t matrices = 0;
    int lds_bytes = 0;  // of the largest
    int check() const {
        return matrices <= most_workgroups(kResidentThreads) ? FSADAM_OK : fail(FSADAM_EINVAL, "the list has too many matrices of a short side up to 128 for one call (2^22 or more)");
    }
    int64_t bytes() const { return rows.size() > kResidentRowsPerLaunch ? up((int64_t)(rows.size() * sizeof(ResidentRow)), 256) : 0; }
};

struct Plan {
    Residents residents;
    std::vector<Chunk> chunks;
    Plan(const std::vector<Source>& list, const FsOrthOptions& options) {
        for (const Source& in : list) {
            if (!resident(in)) continue;
            const int s = (int)std::min(in.rows, in.cols), l = (int)std::max(in.rows, in.cols);
            ResidentRow row{};
            row.src = in.src; row.buf = in.buf; row.dst = in.dst; row.copy = in.copy;
            row.src_ld = in.src_ld; row.src_stride = in.src_stride; row.dst_ld = in.dst_ld; row.dst_stride = in.dst_stride;
            row.rows = (int32_t)in.rows; row.cols = (int32_t)in.cols;
            row.first_matrix = (int32_t)residents.matrices;
            row.step_ratio = in.step_ratio;
            residents.rows.push_back(row);
            residents.matrices += in.batch;
            residents.lds_bytes = std::max(residents.lds_bytes, (int)up(s, 32) * (resident_pitch(s) + resident_pitch(l)) * 4);
        }
        make_chunks(list, options, chunks);
    }
    int64_t workspace() const {
        int64_t bytes = residents.bytes();  // their table is done with when the chunks begin
        for (const Chunk& c : chunks) bytes = std::max(bytes, c.bytes());
        return bytes;
    }
};

int check_shape(int64_t t, int64_t batch, int64_t rows, int64_t cols) {
    if (batch < 0 || rows < 0 || cols < 0) return fail(FSADAM_EINVAL, "matrix " + std::to_string(t) + ": negative size");
    if (rows > kMaxSide || cols > kMaxSide || batch > kMaxSide)
        return fail(FSADAM_EINVAL, "matrix " + std::to_string(t) + ": sides and batches over 2^20 are not supported");
    if (rows * cols > (int64_t(1) << 34)) return fail(FSADAM_EINVAL, "matrix " + std::to_string(t) + ": more than 2^34 elements");
    return FSADAM_OK;
}

// ---- launches -----------------------------------------------------------------------------------------------------

// The tile of a launch: 64, 128 or 256 square, by what the busiest compute unit is given to do.  A unit of 64 x 64 is 13, what
// takes 0.65 us per 64 of depth with 22-bit products; 128 takes 1.5 us and 256 takes 4.6 us, so that the larger tiles do 1.7 and
// 2.2 times the work in the same time -- where there are enough of them for 256 compute units.  (11-bit products: about half
// the times in the same proportion.)  With 64 / 128 / 256, 22 bits, six matrices of 768 x 2304 and six of 768 x 768: update
// 101 / 73 / 73 us, square products 34 / 29 / 61.  11 bits, 4096 x 4096: update 268 / 178 / 145 us, square products 155 / 117 / 137.
// `last`: what a round of 256 takes longer when the parameters are updated in it.  Their traffic comes in one burst behind the
// products, with nothing on the compute unit to do meanwhile; two workgroups of 128 share one and take turns.  Per 64 of depth it
// weighs the less the deeper the products are.  With 128 / 256: the matrices above (768 deep) 95 / 112 us, a layer's (4096 deep) 2.18 / 1.88 ms.
struct Tiles {
    int size;
    int64_t count;
};
Tiles choose_tiles(int64_t t64, int64_t t128, int64_t t256, int64_t last) {
    const auto cost = [](int64_t tiles, int64_t unit) { return (tiles + 255) / 256 * unit; };
    const int64_t c64 = cost(t64, 13), c128 = cost(t128, 30), c256 = cost(t256, 92 + last);
    if (c256 < c128 && c256 < c64) return {256, t256};
    if (c128 < c64) return {128, t128};
    return {64, t64};
}

template <int STAGE, int TILE, int PLANES, int DEPTH>
void launch_tile(int64_t count, int n_rows, const MatrixRow* table, const StageArgs& k, _Float16* work, hipStream_t stream) {
    constexpr int WM = 2, WN = TILE == 64 ? 2 : 4, BK = column_block(PLANES);
    if (count) hipLaunchKernelGGL((fsadam_matrix_stage<STAGE, TILE, TILE, WM, WN, BK, DEPTH, PLANES>), dim3((uint32_t)count), dim3(64 * WM * WN), 0, stream, table, n_rows, k, work);
}

// Panels in LDS.  Tiles of 64 are taken where there are few of them, one workgroup to a compute unit: what hides the loads' latency is
// then its own panels alone (11 bits, 2 / 3 / 4 panels: 512 x 2048 184 / 165 / 164 us, four of 512 x 1024 155 / 149 / 150; 22 bits, half as
// deep, 3 / 4 / 6: 231 / 225 / 226, 214 / 207 / 228).  Tiles of 128 take four panels while no compute unit has two of them (11 bits, 2 / 4
// panels: 1600 x 1600 287 / 262 us, 2048 x 2048 417 / 377; with 22 bits, where the two groups of waves wait for something else, 816 /
// 801 and no difference elsewhere: left at two).  256 has no room for a third.
template <int STAGE, int TILE, int PLANES>
void launch_tiles(int64_t count, int n_rows, const MatrixRow* table, const StageArgs& k, _Float16* work, hipStream_t stream) {
    if constexpr (TILE == 128)
        PLANES == 1 && count <= 256 ? launch_tile<STAGE, TILE, PLANES, PLANES == 1 ? 4 : 2>(count, n_rows, table, k, work, stream) : launch_tile<STAGE, TILE, PLANES, 2>(count, n_rows, table, k, work, stream);
    else launch_tile<STAGE, TILE, PLANES, TILE == 256 ? 2 : PLANES == 2 ? 4 : 3>(count, n_rows, table, k, work, stream);
}

template <int STAGE, int PLANES>
int launch_stage(const Chunk& c, const MatrixRow* table, StageArgs k, _Float16* work, hipStream_t stream) {
    constexpr int kind = STAGE == kStageGram ? 2 : STAGE == kStageSquare ? 0 : 1;
    const int n = (int)c.rows.size();
    const int64_t last = STAGE == kStageStep ? 550 * 64 / c.mean_depth() : 0;
    const Tiles t = choose_tiles(c.tiles[kTilesSym64 + kind], c.tiles[kTilesSym128 + kind], c.tiles[kTilesSym256 + kind], last);
    if (t.size == 256) launch_tiles<STAGE, 256, PLANES>(t.count, n, table, k, work, stream);
    else if (t.size == 128) launch_tiles<STAGE, 128, PLANES>(t.count, n, table, k, work, stream);
    else if (STAGE != kStageGram) launch_tiles<STAGE, 64, PLANES>(t.count, n, table, k, work, stream);
    if constexpr (STAGE == kStageGram) {  // split products are in tiles of 64; the others join their launch where they are too
        k.kind = t.size == 64 ? kTilesAllParts : kTilesPart;
        launch_tiles<kStageGram, 64, PLANES>(c.tiles[k.kind], n, table, k, work, stream);
        launch_tiles<kStageJoin, 64, PLANES>(c.tiles[kTilesJoin], n, table, k, work, stream);
    }
    return launched();
}

struct Call {
    bool step;
    int src_type, dst_type, copy_type;
    FsOrthOptions options;
    std::vector<StepNumbers> numbers;
    MomentumArgs momentum;
    float keep;
};

template <bool STEP>
void launch_prepare(const Chunk& c, const Call& call, const MatrixRow* table, double* inverse, double* partials, _Float16* work, hipStream_t stream) {
    const int n = (int)c.rows.size();
    const dim3 chunks((uint32_t)c.tiles[kTilesChunk]), matrices((uint32_t)c.matrices), tiles((uint32_t)c.tiles[kTilesPrep]), block(256);
    const double power = std::ldexp(1.0, call.numbers[0].x);
#define FM_TYPE(T, EACH) \
    if (call.src_type == T) { EACH(T); }
#define FM_CHUNKS(T) hipLaunchKernelGGL((fsadam_matrix_chunks<T, STEP>), chunks, block, 0, stream, table, n, call.momentum, partials)
#define FM_NORMALISE(T) hipLaunchKernelGGL((fsadam_matrix_normalise<T, STEP>), tiles, block, 0, stream, table, n, call.momentum, (const double*)inverse, power, c.products == FSADAM_PRODUCTS_SPLIT ? 5 : 6, work)
    FM_TYPE(kTypeF32, FM_CHUNKS) FM_TYPE(kTypeF16, FM_CHUNKS) FM_TYPE(kTypeBF16, FM_CHUNKS)
    hipLaunchKernelGGL(fsadam_matrix_norms, matrices, block, 0, stream, table, n, (double)call.options.eps, (const double*)partials, inverse);
    FM_TYPE(kTypeF32, FM_NORMALISE) FM_TYPE(kTypeF16, FM_NORMALISE) FM_TYPE(kTypeBF16, FM_NORMALISE)
#undef FM_TYPE
#undef FM_CHUNKS
#undef FM_NORMALISE
}

int run_chunk(const Chunk& c, const Call& call, void* workspace, hipStream_t stream) {
    char* at = static_cast<char*>(workspace);
    MatrixRow* table = reinterpret_cast<MatrixRow*>(at);
    at += up((int64_t)c.rows.size() * sizeof(MatrixRow), 256);
    double* inverse = reinterpret_cast<double*>(at);
    at += up(c.matrices * 8, 256);
    double* partials = reinterpret_cast<double*>(at);
    at += up(c.tiles[kTilesChunk] * 8, 256);
    _Float16* work = reinterpret_cast<_Float16*>(at);

    for (size_t first = 0; first < c.rows.size(); first += kRowsPerPut) {
        MatrixRows rows;
        const size_t n = std::min<size_t>(kRowsPerPut, c.rows.size() - first);
        std::memcpy(rows.row, c.rows.data() + first, n * sizeof(MatrixRow));
        hipLaunchKernelGGL(fsadam_put_matrix_rows, dim3(1), dim3(256), 0, stream, table + first, (int)n, rows);
    }
    if (call.step) launch_prepare<true>(c, call, table, inverse, partials, work, stream);
    else launch_prepare<false>(c, call, table, inverse, partials, work, stream);
    int rc = launched();
    if (rc) return rc;

    const FsOrthOptions& o = call.options;
    const std::vector<StepNumbers>& n = call.numbers;
    StageArgs k{};
    k.dst_type = call.dst_type;
    k.copy_type = call.copy_type;
    k.keep = call.keep;
    auto stage = [&](auto which) {
        constexpr int kStage = decltype(which)::value;
        return c.products == FSADAM_PRODUCTS_SPLIT ? launch_stage<kStage, 2>(c, table, k, work, stream) : launch_stage<kStage, 1>(c, table, k, work, stream);
    };
    constexpr std::integral_constant<int, kStageGram> gram{};
    constexpr std::integral_constant<int, kStageSquare> square_stage{};
    constexpr std::integral_constant<int, kStageUpdate> update{};
    constexpr std::integral_constant<int, kStageOut> out{};
    constexpr std::integral_constant<int, kStageStep> step{};
    auto square = [&](int p, int q, int add, double linear, int linear_exp, double product, int product_exp, double diagonal, int into) {
        k.p = p; k.q = q; k.add = add; k.into = into;
        k.linear = (float)std::ldexp(linear, linear_exp);
        k.product = (float)std::ldexp(product, product_exp);
        k.diagonal = (float)diagonal;
        return stage(square_stage);
    };
    int s = 0, from = 0;
    while (s < o.steps) {
        const bool pair = c.pairs() && s + 2 <= o.steps;
        const StepNumbers& n0 = n[s];
        const int after = s + (pair ? 2 : 1), next_x = after < o.steps ? n[after].x : 0;
        k.from = from;
        k.to = from ^ 1;
        k.into = 0;
        k.product = (float)std::ldexp(1.0, n0.a - 2 * n0.x);
        if ((rc = stage(gram))) return rc;  // 0: A
        if (pair) {
            const StepNumbers& n1 = n[s + 1];
            const int q = exponent_for(n0.q_bound * n1.q_bound);
            if ((rc = square(0, 0, 0, o.b, n0.r - n0.a, o.c, n0.r - 2 * n0.a, std::ldexp((double)o.a, n0.r), 1))) return rc;  // 1: R
            if ((rc = square(1, 0, -1, 0.0, 0, 1.0, n0.t - n0.r - n0.a, 0.0, 2))) return rc;                                  // 2: R A
            if ((rc = square(2, 1, -1, 0.0, 0, 1.0, n1.a - n0.t - n0.r, 0.0, 0))) return rc;                                  // 0: R A R, the next A
            if ((rc = square(0, 0, 0, o.b, n1.r - n1.a, o.c, n1.r - 2 * n1.a, std::ldexp((double)o.a, n1.r), 2))) return rc;  // 2: the next R
            if ((rc = square(2, 1, -1, 0.0, 0, 1.0, q - n1.r - n0.r, 0.0, 0))) return rc;                                     // 0: their product
            k.p = 0;
            k.linear = 0.0f;
            k.product = (float)std::ldexp(1.0, next_x - q - n0.x);
        } else {
            if ((rc = square(0, 0, 0, o.b, n0.b - n0.a, o.c, n0.b - 2 * n0.a, 0.0, 1))) return rc;  // 1: B
            k.p = 1;
            k.linear = (float)std::ldexp((double)o.a, next_x - n0.x);
            k.product = (float)std::ldexp(1.0, next_x - n0.b - n0.x);
        }
        if ((rc = after < o.steps ? stage(update) : call.step ? stage(step) : stage(out))) return rc;
        from ^= 1;
        s = after;
    }
    return FSADAM_OK;
}

int run_residents(const Residents& r, const Call& call, void* workspace, hipStream_t stream) {
    if (r.rows.empty()) return FSADAM_OK;
    const FsOrthOptions& o = call.options;
    ResidentArgs k{};
    k.steps = o.steps;
    k.src_type = call.src_type; k.dst_type = call.dst_type; k.copy_type = call.copy_type;
    k.keep = call.keep;
    k.eps = o.eps;
    k.power = std::ldexp(1.0, call.numbers[0].x);
    for (int s = 0; s < o.steps; ++s) {
        const StepNumbers& n = call.numbers[s];
        const int next_x = s + 1 < o.steps ? call.numbers[s + 1].x : 0;
        k.factors[kFactorGram][s] = (float)std::ldexp(1.0, n.a - 2 * n.x);
        k.factors[kFactorLinearB][s] = (float)std::ldexp((double)o.b, n.b - n.a);
        k.factors[kFactorProductB][s] = (float)std::ldexp((double)o.c, n.b - 2 * n.a);
        k.factors[kFactorLinearX][s] = (float)std::ldexp((double)o.a, next_x - n.x);
        k.factors[kFactorProductX][s] = (float)std::ldexp(1.0, next_x - n.b - n.x);
    }
    auto launch = [&](const auto& table) {
        using Table = std::decay_t<decltype(table)>;
        const dim3 grid((uint32_t)r.matrices), block(kResidentThreads);
        if (call.step) hipLaunchKernelGGL((fsadam_matrix_resident<true, Table>), grid, block, r.lds_bytes, stream, table, k, call.momentum);
        else hipLaunchKernelGGL((fsadam_matrix_resident<false, Table>), grid, block, r.lds_bytes, stream, table, k, call.momentum);
        return launched();
    };
    if (r.rows.size() <= kResidentRowsPerLaunch) {
        ResidentInArguments table{};
        table.n = (int)r.rows.size();
        std::memcpy(table.rows.row, r.rows.data(), r.rows.size() * sizeof(ResidentRow));
        return launch(table);
    }
    ResidentRow* memory = static_cast<ResidentRow*>(workspace);
    for (size_t first = 0; first < r.rows.size(); first += kResidentRowsPerLaunch) {
        ResidentRows rows;
        const size_t n = std::min<size_t>(kResidentRowsPerLaunch, r.rows.size() - first);
        std::memcpy(rows.row, r.rows.data() + first, n * sizeof(ResidentRow));
        hipLaunchKernelGGL(fsadam_put_resident_rows, dim3(1), dim3(256), 0, stream, memory + first, (int)n, rows);
    }
    return launch(ResidentInMemory{memory, (int)r.rows.size()});
}

int run_call(const Plan& plan, Call& call, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    int rc = step_bounds(call.options, call.numbers);
    if (rc || (rc = plan.residents.check())) return rc;
    const std::vector<Chunk>& chunks = plan.chunks;
    const int64_t need = plan.workspace();
    if (need && (!workspace || !aligned(workspace, 256))) return fail(FSADAM_EINVAL, "the workspace must be a device pointer aligned to 256 bytes");
    if (workspace_bytes < need)
        return fail(FSADAM_EINVAL, "the workspace holds " + std::to_string(workspace_bytes) + " bytes, this list needs " + std::to_string(need));
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    if ((rc = run_residents(plan.residents, call, workspace, stream))) return rc;
    for (const Chunk& c : chunks) {
        rc = run_chunk(c, call, workspace, stream);
        if (rc) return rc;
    }
    return FSADAM_OK;
}

int sources_of(const FsMatrix* m, int64_t n, int size, std::vector<Source>& list) {
    if (n < 0 || (n > 0 && !m)) return fail(FSADAM_EINVAL, "matrices is NULL, or their number negative");
    for (int64_t t = 0; t < n; ++t) {
        const FsMatrix& r = m[t];
        int rc = check_shape(t, r.batch, r.rows, r.cols);
        if (rc) return rc;
        if (r.batch == 0 || r.rows == 0 || r.cols == 0) continue;
        const std::string name = "matrix " + std::to_string(t);
        if (!r.src || !r.dst) return fail(FSADAM_EINVAL, name + ": NULL pointer");
        if (!aligned(r.src, size) || !aligned(r.dst, size)) return fail(FSADAM_EINVAL, name + ": pointer not aligned to its element size");
        for (int64_t ld : {r.src_ld, r.dst_ld})
            if (ld < r.cols || ld > (int64_t(1) << 40)) return fail(FSADAM_EINVAL, name + ": rows overlap (ld < cols), or lie too far apart");
        const int64_t dst_end = (r.rows - 1) * r.dst_ld + r.cols;
        if (r.batch > 1 && (r.src_stride < 0 || r.dst_stride < dst_end || r.src_stride > (int64_t(1) << 40) || r.dst_stride > (int64_t(1) << 40)))
            return fail(FSADAM_EINVAL, name + ": matrices of the batch overlap, or lie too far apart");
        if (r.src == r.dst && (r.src_ld != r.dst_ld || (r.batch > 1 && r.src_stride != r.dst_stride)))
            return fail(FSADAM_EINVAL, name + ": results over the matrices need the same strides");
        list.push_back({r.src, nullptr, r.dst, nullptr, r.batch, r.rows, r.cols, r.src_ld, r.src_stride, r.dst_ld, r.dst_stride, 0.0f, size, size, 0});
    }
    return FSADAM_OK;
}

int sources_of(const FsMuonTensor* m, int64_t n, int p_size, int g_size, int c_size, double lr, std::vector<Source>& list) {
    if (n < 0 || (n > 0 && !m)) return fail(FSADAM_EINVAL, "tensors is NULL, or their number negative");
    for (int64_t t = 0; t < n; ++t) {
        const FsMuonTensor& r = m[t];
        int rc = check_shape(t, r.batch, r.rows, r.cols);
        if (rc) return rc;
        if (r.batch == 0 || r.rows == 0 || r.cols == 0) continue;
        const std::string name = "tensor " + std::to_string(t);
        if (!r.p || !r.g || !r.m) return fail(FSADAM_EINVAL, name + ": NULL p/g/m pointer");
        if (c_size && !r.p_copy) return fail(FSADAM_EINVAL, name + ": this combination of types needs p_copy");
        if (!aligned(r.p, p_size) || !aligned(r.g, g_size) || !aligned(r.m, 4) || (c_size && !aligned(r.p_copy, c_size)))
            return fail(FSADAM_EINVAL, name + ": pointer not aligned to its element size");
        if (!std::isfinite(r.ratio)) return fail(FSADAM_EINVAL, name + ": ratio must be finite");
        const int64_t numel = r.rows * r.cols;
        list.push_back({r.g, r.m, r.p, c_size ? r.p_copy : nullptr, r.batch, r.rows, r.cols, r.cols, numel, r.cols, numel, (float)(lr * r.ratio), g_size, p_size, c_size});
    }
    return FSADAM_OK;
}

int check_momentum(double momentum, float scale, const float* scale_dev) {
    if (!(momentum >= 0.0 && momentum < 1.0)) return fail(FSADAM_EINVAL, "momentum must be in [0, 1)");
    if (!scale_dev && !(std::isfinite(scale) && scale != 0.0f)) return fail(FSADAM_EINVAL, "scale must be finite and not 0");
    return FSADAM_OK;
}
MomentumArgs momentum_args(double momentum, int nesterov, float scale, const float* scale_dev) {
    return {scale_dev, scale, (float)momentum, (float)(1.0 - momentum), nesterov != 0};
}

// The momentum pass's table: rows that hold something; returns how many chunks they have.
int momentum_rows(const FsMomentumTensor* t, int64_t n, std::vector<MomentumRow>& rows, int64_t& chunks) {
    if (n < 0 || (n > 0 && !t)) return fail(FSADAM_EINVAL, "tensors is NULL, or their number negative");
    chunks = 0;
    for (int64_t k = 0; k < n; ++k) {
        if (t[k].numel < 0 || t[k].numel > (int64_t(1) << 42)) return fail(FSADAM_EINVAL, "tensor " + std::to_string(k) + ": numel out of range");
        rows.push_back({t[k].g, t[k].m, t[k].u, t[k].numel, chunks});
        chunks += up(t[k].numel, kMomentumElems) / kMomentumElems;
    }
    if (chunks > most_workgroups(kChunkThreads)) return fail(FSADAM_EINVAL, "the list has too many elements for one call (about 2^34 or more)");
    if (n > most_workgroups(kNormThreads)) return fail(FSADAM_EINVAL, "the list has too many tensors for one call (2^22 or more)");
    return FSADAM_OK;
}
// The arguments of a launch are slow to read (they are not in the GPU's memory): worth it for a few workgroups only.
bool table_in_arguments(int64_t rows, int64_t chunks) { return rows <= kMomentumRowsPerLaunch && chunks <= 2048; }
int64_t momentum_table_bytes(int64_t rows) { return up(rows * (int64_t)sizeof(MomentumRow), 256); }
int64_t momentum_bytes(int64_t rows, int64_t chunks) { return momentum_table_bytes(rows) + up(chunks * 8, 256); }

}  // namespace

extern "C" {

int fsadam_momentum_workspace(const FsMomentumTensor* tensors, int64_t n_tensors, int64_t* bytes) {
    return guarded([&] {
        if (!bytes) return fail(FSADAM_EINVAL, "bytes is NULL");
        std::vector<MomentumRow> rows;
        int64_t chunks;
        const int rc = momentum_rows(tensors, n_tensors, rows, chunks);
        if (rc) return rc;
        *bytes = momentum_bytes(n_tensors, chunks);
        return FSADAM_OK;
    });
}

int fsadam_momentum_pass(const FsMomentumTensor* tensors, int64_t n_tensors, int grad_type, int update_type, double momentum, int nesterov,
                         float scale, const float* scale_dev, float* norms_dev, float* found_inf_dev, int clear_found_inf, void* workspace,
                         int64_t workspace_bytes, void* hip_stream) {
    return guarded([&] {
        if (!valid_type(grad_type) || !valid_type(update_type)) return fail(FSADAM_EINVAL, "unknown type");
        int rc = check_momentum(momentum, scale, scale_dev);
        if (rc) return rc;
        std::vector<MomentumRow> rows;
        int64_t chunks;
        if ((rc = momentum_rows(tensors, n_tensors, rows, chunks))) return rc;
        for (int64_t t = 0; t < n_tensors; ++t) {
            if (tensors[t].numel == 0) continue;
            if (!tensors[t].g || !tensors[t].m || !tensors[t].u) return fail(FSADAM_EINVAL, "tensor " + std::to_string(t) + ": NULL g/m/u pointer");
            if (!aligned(tensors[t].g, size_of(grad_type)) || !aligned(tensors[t].m, 4) || !aligned(tensors[t].u, size_of(update_type)))
                return fail(FSADAM_EINVAL, "tensor " + std::to_string(t) + ": pointer not aligned to its element size");
            if (tensors[t].u == tensors[t].g && size_of(grad_type) != size_of(update_type))
                return fail(FSADAM_EINVAL, "tensor " + std::to_string(t) + ": updates over the gradients need elements of the same size");
        }
        if (n_tensors == 0) return FSADAM_OK;
        if (!workspace || !aligned(workspace, 256)) return fail(FSADAM_EINVAL, "the workspace must be a device pointer aligned to 256 bytes");
        if (workspace_bytes < momentum_bytes(n_tensors, chunks))
            return fail(FSADAM_EINVAL, "the workspace holds " + std::to_string(workspace_bytes) + " bytes, this list needs " + std::to_string(momentum_bytes(n_tensors, chunks)));
        hipStream_t stream = static_cast<hipStream_t>(hip_stream);
        double* partials = reinterpret_cast<double*>(static_cast<char*>(workspace) + momentum_table_bytes(n_tensors));
        const MomentumArgs k = momentum_args(momentum, nesterov, scale, scale_dev);
        float* cleared = clear_found_inf ? found_inf_dev : nullptr;
        if (cleared && !chunks) hipLaunchKernelGGL(fsadam_clear_flag, dim3(1), dim3(1), 0, stream, cleared);
        auto launch = [&](const auto& table) {
            using Table = std::decay_t<decltype(table)>;
            const dim3 grid((uint32_t)chunks), block(kChunkThreads);
#define FM_PASS(G, U) \
    if (grad_type == G && update_type == U) hipLaunchKernelGGL((fsadam_momentum_chunks<G, U, Table>), grid, block, 0, stream, table, k, partials, cleared)
            if (chunks) {
                FM_PASS(kTypeF32, kTypeF32); FM_PASS(kTypeF32, kTypeF16); FM_PASS(kTypeF32, kTypeBF16);
                FM_PASS(kTypeF16, kTypeF32); FM_PASS(kTypeF16, kTypeF16); FM_PASS(kTypeF16, kTypeBF16);
                FM_PASS(kTypeBF16, kTypeF32); FM_PASS(kTypeBF16, kTypeF16); FM_PASS(kTypeBF16, kTypeBF16);
            }
#undef FM_PASS
            if (norms_dev || found_inf_dev)
                hipLaunchKernelGGL((fsadam_momentum_norms<Table>), dim3((uint32_t)n_tensors), dim3(kNormThreads), 0, stream, table, (const double*)partials, norms_dev, found_inf_dev);
            return launched();
        };
        if (table_in_arguments(n_tensors, chunks)) {
            InArguments table{};
            table.n = (int)n_tensors;
            std::memcpy(table.rows.row, rows.data(), (size_t)n_tensors * sizeof(MomentumRow));
            return launch(table);
        }
        MomentumRow* memory = static_cast<MomentumRow*>(workspace);
        for (int64_t first = 0; first < n_tensors; first += kMomentumRowsPerLaunch) {
            MomentumRows put;
            const int64_t n = std::min<int64_t>(kMomentumRowsPerLaunch, n_tensors - first);
            std::memcpy(put.row, rows.data() + first, (size_t)n * sizeof(MomentumRow));
            hipLaunchKernelGGL(fsadam_put_momentum_rows, dim3(1), dim3(256), 0, stream, memory + first, (int)n, put);
        }
        return launch(InMemory{memory, (int)n_tensors});
    });
}

int fsadam_orth_workspace(const FsMatrix* matrices, int64_t n, const FsOrthOptions* options, int64_t* bytes) {
    return guarded([&] {
        if (!bytes) return fail(FSADAM_EINVAL, "bytes is NULL");
        int rc = check_options(options);
        if (rc) return rc;
        std::vector<Source> list;
        if ((rc = sources_of(matrices, n, 1, list))) return rc;
        const Plan plan(list, *options);
        if ((rc = plan.residents.check())) return rc;
        *bytes = plan.workspace();
        return FSADAM_OK;
    });
}

int fsadam_orthogonalize(const FsMatrix* matrices, int64_t n, int type, const FsOrthOptions* options, void* workspace, int64_t workspace_bytes,
                         void* hip_stream) {
    return guarded([&] {
        if (!valid_type(type)) return fail(FSADAM_EINVAL, "unknown type");
        int rc = check_options(options);
        if (rc) return rc;
        std::vector<Source> list;
        if ((rc = sources_of(matrices, n, size_of(type), list))) return rc;
        const Plan plan(list, *options);
        Call call{};
        call.src_type = call.dst_type = type;
        call.copy_type = -1;
        call.options = *options;
        return run_call(plan, call, workspace, workspace_bytes, hip_stream);
    });
}

int fsadam_muon_workspace(const FsMuonTensor* tensors, int64_t n, const FsOrthOptions* options, int64_t* bytes) {
    return guarded([&] {
        if (!bytes) return fail(FSADAM_EINVAL, "bytes is NULL");
        int rc = check_options(options);
        if (rc) return rc;
        std::vector<Source> list;
        if ((rc = sources_of(tensors, n, 1, 1, 0, 0.0, list))) return rc;
        const Plan plan(list, *options);
        if ((rc = plan.residents.check())) return rc;
        *bytes = plan.workspace();
        return FSADAM_OK;
    });
}

int fsadam_muon_step(const FsMuonTensor* tensors, int64_t n, int param_type, int grad_type, int copy_type, const FsOrthOptions* options,
                     double lr, double momentum, int nesterov, double weight_decay, float scale, const float* scale_dev, void* workspace,
                     int64_t workspace_bytes, void* hip_stream) {
    return guarded([&] {
        const bool plain = copy_type == -1 && param_type == grad_type && valid_type(param_type);
        const bool mixed = param_type == FSADAM_TYPE_F32 && copy_type == grad_type && (grad_type == FSADAM_TYPE_F16 || grad_type == FSADAM_TYPE_BF16);
        if (!plain && !mixed) return fail(FSADAM_EINVAL, "unsupported combination of parameter, gradient and copy types");
        if (!std::isfinite(lr) || !std::isfinite(weight_decay)) return fail(FSADAM_EINVAL, "lr and weight_decay must be finite");
        int rc = check_options(options);
        if (rc) return rc;
        if ((rc = check_momentum(momentum, scale, scale_dev))) return rc;
        std::vector<Source> list;
        if ((rc = sources_of(tensors, n, size_of(param_type), size_of(grad_type), mixed ? 2 : 0, lr, list))) return rc;
        const Plan plan(list, *options);
        Call call{};
        call.step = true;
        call.src_type = grad_type;
        call.dst_type = param_type;
        call.copy_type = copy_type;
        call.options = *options;
        call.momentum = momentum_args(momentum, nesterov, scale, scale_dev);
        call.keep = (float)(1.0 - lr * weight_decay);
        return run_call(plan, call, workspace, workspace_bytes, hip_stream);
    });
}

}  // extern "C"
