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
constexpr int kMaxSteps = 32;
constexpr int64_t kMaxTiles = INT32_MAX / 2;  // of one launch
// Intermediate matrices of one chunk.  Enough for eight 4096 x 11008 matrices, whose products then have thousands of
// tiles for the 256 compute units; a matrix that needs more gets what it needs.
constexpr int64_t kChunkBytes = int64_t(4) << 30;

// ---- numbers of the iteration -------------------------------------------------------------------------------------

// Exponents of the powers of two that X, A and B are held with at every step.
struct StepNumbers {
    int x[kMaxSteps + 1], a[kMaxSteps], b[kMaxSteps];
};

int exponent_for(double bound) {  // the largest k with bound * 2^k <= 60000 (halves end at 65504), at most 15
    if (!(bound > 0x1p-15)) return 15;
    return std::min(15, (int)std::floor(std::log2(60000.0 / bound)));
}

// How large singular values of X, A and B can be at every step, when those of X0 are in [0, 1].  The polynomial's extremes on
// [0, m] are at the ends and where its derivative (quadratic in x^2) vanishes.  2 % a step stands for what rounding adds.
int step_bounds(const FsOrthOptions& o, StepNumbers& n) {
    const double a = o.a, b = o.b, c = o.c;
    double m = 1.0;
    for (int k = 0; k < o.steps; ++k) {
        m *= 1.02;
        n.x[k] = exponent_for(m);
        n.a[k] = exponent_for(m * m);
        const double top = m * m;
        double most_b = std::fabs(b * top + c * top * top);
        if (c != 0.0) {
            const double at = -b / (2.0 * c);
            if (at > 0.0 && at < top) most_b = std::max(most_b, std::fabs(b * at + c * at * at));
        }
        n.b[k] = exponent_for(most_b);
        auto p = [&](double t) { return std::fabs(std::sqrt(t) * (a + b * t + c * t * t)); };  // t = x^2
        double next = p(top);
        const double d = 9.0 * b * b - 20.0 * a * c;
        if (c != 0.0 && d >= 0.0) {
            for (double sign : {-1.0, 1.0}) {
                const double t = (-3.0 * b + sign * std::sqrt(d)) / (10.0 * c);
                if (t > 0.0 && t < top) next = std::max(next, p(t));
            }
        } else if (c == 0.0 && b != 0.0) {
            const double t = -a / (3.0 * b);
            if (t > 0.0 && t < top) next = std::max(next, p(t));
        }
        m = next;
        if (!(m <= 1024.0) || !(most_b <= 1024.0))
            return fail(FSADAM_EINVAL, "the coefficients let singular values in [0, 1] grow past 1024 by step " + std::to_string(k + 1));
    }
    n.x[o.steps] = 0;
    return FSADAM_OK;
}

int check_options(const FsOrthOptions* o) {
    if (!o) return fail(FSADAM_EINVAL, "options is NULL");
    if (o->steps < 1 || o->steps > kMaxSteps) return fail(FSADAM_EINVAL, "steps must be in [1, 32], got " + std::to_string(o->steps));
    if (!std::isfinite(o->a) || !std::isfinite(o->b) || !std::isfinite(o->c)) return fail(FSADAM_EINVAL, "the coefficients must be finite");
    if (!(o->eps > 0.0f) || !std::isfinite(o->eps)) return fail(FSADAM_EINVAL, "eps must be positive and finite");
    if (o->products != FSADAM_PRODUCTS_HALF && o->products != FSADAM_PRODUCTS_SPLIT) return fail(FSADAM_EINVAL, "unknown products " + std::to_string(o->products));
    StepNumbers numbers;
    return step_bounds(*o, numbers);
}

// ---- chunks -------------------------------------------------------------------------------------------------------

struct Chunk {
    std::vector<MatrixRow> rows;
    int64_t matrices = 0;
    int64_t tiles[kTileKinds] = {};
    int64_t halves = 0;  // of the intermediate matrices
    int products = 0;    // FSADAM_PRODUCTS_* of its launches
    int64_t head_bytes() const { return up((int64_t)rows.size() * sizeof(MatrixRow), 256) + up(matrices * 8, 256) + up(tiles[kTilesChunk] * 8, 256); }
    int64_t bytes() const { return head_bytes() + halves * 2; }
};

int64_t symmetric_tiles(int64_t s, int64_t t) { const int64_t n = (s + t - 1) / t; return n * (n + 1) / 2; }
int64_t full_tiles(int64_t s, int64_t l, int64_t t) { return ((s + t - 1) / t) * ((l + t - 1) / t); }

// Adds up to `batch` matrices of a row to the chunk; returns how many fit.  A chunk takes at least one.
int64_t add_to_chunk(Chunk& chunk, const MatrixRow& proto, int64_t batch) {
    const int64_t products = chunk.products;
    const int64_t x = 2 * (int64_t)proto.s64 * proto.l64, a = products * (int64_t)proto.s64 * proto.s64;  // halves of one matrix, one buffer
    const int64_t per = 2 * (x + a), room = kChunkBytes / 2 - chunk.halves;
    int64_t n = std::min(batch, room / per);
    int64_t most = kMaxTiles;
    for (int k = 0; k < kTileKinds; ++k) most = std::min(most, (kMaxTiles - chunk.tiles[k]) / proto.n[k]);
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
    row.a_off = row.x_off[1] + n * x;
    row.b_off = row.a_off + n * a;
    chunk.halves = row.b_off + n * a;
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

// Matrices of a short side up to this are always multiplied to 22 bits.  The error of 11-bit products is about 2e-3 of the
// result where it averages over many singular values, but a matrix that has few of them can be off by 2 % (rounding A, B
// and X by 2^-11 each moves b x^3 + c x^5 by up to 32 * 2^-11 at x = 1); and their products are too small to be what a
// call waits for.
constexpr int64_t kAlwaysSplit = 128;

void make_chunks(const std::vector<Source>& all, int asked, std::vector<Chunk>& chunks) {
  for (int products : {FSADAM_PRODUCTS_HALF, FSADAM_PRODUCTS_SPLIT}) {
    bool fresh = true;  // a chunk is of one kind
    for (const Source& in : all) {
        if ((std::min(in.rows, in.cols) <= kAlwaysSplit ? FSADAM_PRODUCTS_SPLIT : asked) != products) continue;
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
        row.n[kTilesSym128] = (int32_t)symmetric_tiles(row.s64, 128);
        row.n[kTilesFull128] = (int32_t)full_tiles(row.s64, row.l64, 128);
        row.n[kTilesSym256] = (int32_t)symmetric_tiles(row.s64, 256);
        row.n[kTilesFull256] = (int32_t)full_tiles(row.s64, row.l64, 256);
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

int64_t workspace_of(const std::vector<Chunk>& chunks) {
    int64_t bytes = 0;
    for (const Chunk& c : chunks) bytes = std::max(bytes, c.bytes());
    return bytes;
}

int check_shape(int64_t t, int64_t batch, int64_t rows, int64_t cols) {
    if (batch < 0 || rows < 0 || cols < 0) return fail(FSADAM_EINVAL, "matrix " + std::to_string(t) + ": negative size");
    if (rows > kMaxSide || cols > kMaxSide || batch > kMaxSide)
        return fail(FSADAM_EINVAL, "matrix " + std::to_string(t) + ": sides and batches over 2^20 are not supported");
    if (rows * cols > (int64_t(1) << 34)) return fail(FSADAM_EINVAL, "matrix " + std::to_string(t) + ": more than 2^34 elements");
    return FSADAM_OK;
}

// ---- launches -----------------------------------------------------------------------------------------------------

template <int PLANES>
int launch_stage(int stage, const Chunk& c, const MatrixRow* table, const StageArgs& k, _Float16* work, hipStream_t stream) {
    const int n = (int)c.rows.size();
    constexpr int BK = PLANES == 2 ? 32 : 64;
    const bool sym = stage == kStageGram || stage == kStagePoly;
    const dim3 grid((uint32_t)c.tiles[sym ? kTilesSym128 : kTilesFull128]), block(256);
#define FM_STAGE(S) \
    case S: hipLaunchKernelGGL((fsadam_matrix_stage<S, 128, 128, 2, 2, BK, 2, PLANES>), grid, block, 0, stream, table, n, k, work); break
    switch (stage) {
        FM_STAGE(kStageGram);
        FM_STAGE(kStagePoly);
        FM_STAGE(kStageUpdate);
        FM_STAGE(kStageOut);
        FM_STAGE(kStageStep);
    }
#undef FM_STAGE
    return launched();
}

struct Call {
    bool step;
    int src_type, dst_type, copy_type;
    FsOrthOptions options;
    StepNumbers numbers;
    MomentumArgs momentum;
    float keep;
};

template <bool STEP>
void launch_prepare(const Chunk& c, const Call& call, const MatrixRow* table, double* inverse, double* partials, _Float16* work, hipStream_t stream) {
    const int n = (int)c.rows.size();
    const dim3 chunks((uint32_t)c.tiles[kTilesChunk]), matrices((uint32_t)c.matrices), tiles((uint32_t)c.tiles[kTilesPrep]), block(256);
    const double power = std::ldexp(1.0, call.numbers.x[0]);
#define FM_TYPE(T, EACH) \
    if (call.src_type == T) { EACH(T); }
#define FM_CHUNKS(T) hipLaunchKernelGGL((fsadam_matrix_chunks<T, STEP>), chunks, block, 0, stream, table, n, call.momentum, partials)
#define FM_NORMALISE(T) hipLaunchKernelGGL((fsadam_matrix_normalise<T, STEP>), tiles, block, 0, stream, table, n, call.momentum, (const double*)inverse, power, work)
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
    const StepNumbers& n = call.numbers;
    for (int s = 0; s < o.steps; ++s) {
        StageArgs k{};
        k.from = s & 1;
        k.to = k.from ^ 1;
        k.dst_type = call.dst_type;
        k.copy_type = call.copy_type;
        k.keep = call.keep;
        auto stage = [&](int which, double linear, int linear_exp, double product, int product_exp) {
            k.linear = (float)std::ldexp(linear, linear_exp);
            k.product = (float)std::ldexp(product, product_exp);
            return c.products == FSADAM_PRODUCTS_SPLIT ? launch_stage<2>(which, c, table, k, work, stream) : launch_stage<1>(which, c, table, k, work, stream);
        };
        if ((rc = stage(kStageGram, 0.0, 0, 1.0, n.a[s] - 2 * n.x[s]))) return rc;
        if ((rc = stage(kStagePoly, o.b, n.b[s] - n.a[s], o.c, n.b[s] - 2 * n.a[s]))) return rc;
        const int which = s + 1 < o.steps ? kStageUpdate : call.step ? kStageStep : kStageOut;
        if ((rc = stage(which, o.a, n.x[s + 1] - n.x[s], 1.0, n.x[s + 1] - n.b[s] - n.x[s]))) return rc;
    }
    return FSADAM_OK;
}

int run_call(const std::vector<Chunk>& chunks, Call& call, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    int rc = step_bounds(call.options, call.numbers);
    if (rc || chunks.empty()) return rc;
    if (!workspace || !aligned(workspace, 256)) return fail(FSADAM_EINVAL, "the workspace must be a device pointer aligned to 256 bytes");
    if (workspace_bytes < workspace_of(chunks))
        return fail(FSADAM_EINVAL, "the workspace holds " + std::to_string(workspace_bytes) + " bytes, this list needs " + std::to_string(workspace_of(chunks)));
    for (const Chunk& c : chunks) {
        rc = run_chunk(c, call, workspace, static_cast<hipStream_t>(hip_stream));
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
        const int64_t src_end = (r.rows - 1) * r.src_ld + r.cols, dst_end = (r.rows - 1) * r.dst_ld + r.cols;
        if (r.batch > 1 && (r.src_stride < 0 || r.dst_stride < dst_end || r.src_stride > (int64_t(1) << 40) || r.dst_stride > (int64_t(1) << 40)))
            return fail(FSADAM_EINVAL, name + ": matrices of the batch overlap, or lie too far apart");
        if (r.src == r.dst && (r.src_ld != r.dst_ld || (r.batch > 1 && r.src_stride != r.dst_stride)))
            return fail(FSADAM_EINVAL, name + ": results over the matrices need the same strides");
        (void)src_end;
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
        chunks += up(t[k].numel, kChunkElems) / kChunkElems;
    }
    if (chunks > kMaxTiles || n > kMaxTiles) return fail(FSADAM_EINVAL, "the list has too many elements for one call");
    return FSADAM_OK;
}
int64_t momentum_bytes(int64_t rows, int64_t chunks) { return up(rows * (int64_t)sizeof(MomentumRow), 256) + up(chunks * 8, 256); }

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
                         float scale, const float* scale_dev, float* norms_dev, float* found_inf_dev, void* workspace,
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
        MomentumRow* table = static_cast<MomentumRow*>(workspace);
        double* partials = reinterpret_cast<double*>(static_cast<char*>(workspace) + up(n_tensors * (int64_t)sizeof(MomentumRow), 256));
        for (int64_t first = 0; first < n_tensors; first += kMomentumRowsPerPut) {
            MomentumRows put;
            const int64_t n = std::min<int64_t>(kMomentumRowsPerPut, n_tensors - first);
            std::memcpy(put.row, rows.data() + first, (size_t)n * sizeof(MomentumRow));
            hipLaunchKernelGGL(fsadam_put_momentum_rows, dim3(1), dim3(256), 0, stream, table + first, (int)n, put);
        }
        const MomentumArgs k = momentum_args(momentum, nesterov, scale, scale_dev);
        if (chunks) {
            const dim3 grid((uint32_t)chunks), block(kChunkThreads);
#define FM_PASS(G, U) \
    if (grad_type == G && update_type == U) hipLaunchKernelGGL((fsadam_momentum_chunks<G, U>), grid, block, 0, stream, table, (int)n_tensors, k, partials)
            FM_PASS(kTypeF32, kTypeF32); FM_PASS(kTypeF32, kTypeF16); FM_PASS(kTypeF32, kTypeBF16);
            FM_PASS(kTypeF16, kTypeF32); FM_PASS(kTypeF16, kTypeF16); FM_PASS(kTypeF16, kTypeBF16);
            FM_PASS(kTypeBF16, kTypeF32); FM_PASS(kTypeBF16, kTypeF16); FM_PASS(kTypeBF16, kTypeBF16);
#undef FM_PASS
        }
        if (norms_dev || found_inf_dev)
            hipLaunchKernelGGL(fsadam_momentum_norms, dim3((uint32_t)n_tensors), dim3(kChunkThreads), 0, stream, table, (const double*)partials, norms_dev, found_inf_dev);
        return launched();
    });
}

int fsadam_orth_workspace(const FsMatrix* matrices, int64_t n, const FsOrthOptions* options, int64_t* bytes) {
    return guarded([&] {
        if (!bytes) return fail(FSADAM_EINVAL, "bytes is NULL");
        int rc = check_options(options);
        if (rc) return rc;
        std::vector<Source> list;
        if ((rc = sources_of(matrices, n, 1, list))) return rc;
        std::vector<Chunk> chunks;
        make_chunks(list, options->products, chunks);
        *bytes = workspace_of(chunks);
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
        std::vector<Chunk> chunks;
        make_chunks(list, options->products, chunks);
        Call call{};
        call.src_type = call.dst_type = type;
        call.copy_type = -1;
        call.options = *options;
        return run_call(chunks, call, workspace, workspace_bytes, hip_stream);
    });
}

int fsadam_muon_workspace(const FsMuonTensor* tensors, int64_t n, const FsOrthOptions* options, int64_t* bytes) {
    return guarded([&] {
        if (!bytes) return fail(FSADAM_EINVAL, "bytes is NULL");
        int rc = check_options(options);
        if (rc) return rc;
        std::vector<Source> list;
        if ((rc = sources_of(tensors, n, 1, 1, 0, 0.0, list))) return rc;
        std::vector<Chunk> chunks;
        make_chunks(list, options->products, chunks);
        *bytes = workspace_of(chunks);
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
        std::vector<Chunk> chunks;
        make_chunks(list, options->products, chunks);
        Call call{};
        call.step = true;
        call.src_type = grad_type;
        call.dst_type = param_type;
        call.copy_type = copy_type;
        call.options = *options;
        call.momentum = momentum_args(momentum, nesterov, scale, scale_dev);
        call.keep = (float)(1.0 - lr * weight_decay);
        return run_call(chunks, call, workspace, workspace_bytes, hip_stream);
    });
}

}  // extern "C"
