// gated_linear.hip — the gated pair of Linear layers of a feed-forward block, forward and backward (gfx950).
//
//   g = x . Wg + bg,  u = x . Wu + bu,  h = act(g) * u                          act: silu, gelu (erf), relu, sigmoid
//   dg = dh * u * act'(g),  du = dh * act(g),  dx = dg . Wg^T + du . Wu^T,  dW = x^T . d{g,u},  db = column sums of d{g,u}
// No counterpart in the reference; it stands beside nn::Linear (nn/linear.cpp:42-50) followed by an activation.
//
// Bound: the matrix cores for many rows (4 and 8 rows x inner x hidden flop), HBM (the weights) for a few.
#include "gated.h"

#include <initializer_list>

namespace ttamd {
namespace {

template <typename T>
struct VecOf;
template <>
struct VecOf<float> {
    static constexpr int W = 4;
    typedef float type __attribute__((ext_vector_type(4)));
};
template <>
struct VecOf<double> {
    static constexpr int W = 2;
    typedef double type __attribute__((ext_vector_type(2)));
};

// h = act(g) * u over n elements.  VEC: whole vectors at aligned addresses; the elements behind the last one go one by one.
// `out` may be `gate`: an element is read before it is written.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256) gated_product_kernel(const T *gate, const T *up, T *out, int64_t n) {
    using V = typename VecOf<T>::type;
    constexpr int W = VEC ? VecOf<T>::W : 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, whole = n / W;
    for (int64_t i = first; i < whole; i += step) {
        if constexpr (VEC) {
            const V g = reinterpret_cast<const V *>(gate)[i], u = reinterpret_cast<const V *>(up)[i];
            V h;
#pragma unroll
            for (int k = 0; k < W; ++k) h[k] = activate<T, ACT>(g[k]) * u[k];
            reinterpret_cast<V *>(out)[i] = h;
        } else {
            out[i] = activate<T, ACT>(gate[i]) * up[i];
        }
    }
    if (VEC && first < n - whole * W) out[whole * W + first] = activate<T, ACT>(gate[whole * W + first]) * up[whole * W + first];
}

// What a pass needs before its products, in one launch: the gradients of the two products' results, and copies of operands
// whose rows are no whole aligned vectors.
//   dg = dh * u * act'(g), du = dh * act(g): dense dh, g, u [rows, hidden] in, rows of d_row elements out (a multiple of the
//   vector; zeros behind the columns).  A workgroup has 64 vectors of columns and slope_rows rows, a wave every fourth of
//   them; with `sums` it also leaves its rows' column sums, the bias gradients' parts: sums[row block][2][d_row].
//   slope_rows: kSlopeRows with sums (their parts are read again), else kFewSlopeRows: more waves with fewer loads one after
//   the other (1024 x 784 x 1024 f32 forward and backward 107 -> 103 us; 4 or 16 rows 104).
//   A copy: element (r, c) of any view to dst[r * dst_row + c], zeros from (rows, cols) to (dst_rows, dst_row).
constexpr int kSlopeRows = 32, kFewSlopeRows = 8, kCopies = 3;
template <typename T>
struct CopyJob {
    const T *src;
    int64_t s0, s1, rows, cols, dst_rows, dst_row;
    T *dst;
    int blocks;  // tiles of dst, copy_rows() x 64: little more than 2^30 for the 2^40 elements that check_gated allows; 0: nothing to copy
};
template <typename T>
struct PrepareArgs {
    const T *dh, *gate, *up;
    T *dg, *du, *sums;
    int64_t rows, d_row;
    int hidden;
    int slope_rows, slope_blocks, slope_blocks_n;  // rows a workgroup; workgroups of the gradients; of them side by side
    CopyJob<T> copy[kCopies];
    unsigned first;  // number of the launch's first workgroup (launch_prepare)
};

// Rows of a tile: rows in order go by vectors, one to three a lane; others are turned in LDS.
template <typename T>
__host__ __device__ constexpr int copy_rows(const CopyJob<T> &j) { return j.s1 == 1 ? 16 : 64; }

template <typename T>
__device__ __forceinline__ void copy_tile(const CopyJob<T> &j, int block, T (*tile)[65]) {
    using V = typename VecOf<T>::type;
    typedef T near_t __attribute__((ext_vector_type(VecOf<T>::W), aligned(sizeof(T))));
    constexpr int W = VecOf<T>::W, kVecs = 64 / W;
    const int tiles_n = static_cast<int>((j.dst_row + 63) / 64);
    const int64_t r0 = static_cast<int64_t>(block / tiles_n) * copy_rows(j), c0 = static_cast<int64_t>(block % tiles_n) * 64;
    if (j.s1 == 1) {  // rows in order: vectors, wherever the source's begin (dst_row is whole vectors)
#pragma unroll
        for (int i = threadIdx.x; i < 16 * kVecs; i += 256) {
            const int64_t r = r0 + i / kVecs, c = c0 + i % kVecs * W;
            if (r >= j.dst_rows || c >= j.dst_row) continue;
            const T *src = j.src + r * j.s0 + c;
            V v = {};
            if (r < j.rows && c + W <= j.cols) {
                v = *reinterpret_cast<const near_t *>(src);
            } else if (r < j.rows) {
#pragma unroll
                for (int k = 0; k < W; ++k) v[k] = c + k < j.cols ? src[k] : T(0);
            }
            *reinterpret_cast<V *>(j.dst + r * j.dst_row + c) = v;
        }
        return;
    }
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const bool by_rows = j.s0 < j.s1;  // lanes run along the rows (a transposed view) and the tile is turned in LDS
#pragma unroll 4
    for (int i = wave; i < 64; i += 4) {
        const int64_t r = r0 + (by_rows ? lane : i), c = c0 + (by_rows ? i : lane);
        const T v = r < j.rows && c < j.cols ? j.src[r * j.s0 + c * j.s1] : T(0);
        if (by_rows) tile[i][lane] = v;
        else if (r < j.dst_rows && c < j.dst_row) j.dst[r * j.dst_row + c] = v;
    }
    if (!by_rows) return;  // (the same for the whole workgroup)
    __syncthreads();
#pragma unroll 4
    for (int i = wave; i < 64; i += 4)
        if (r0 + i < j.dst_rows && c0 + lane < j.dst_row) j.dst[(r0 + i) * j.dst_row + c0 + lane] = tile[lane][i];
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_prepare_kernel(PrepareArgs<T> a) {
    using V = typename VecOf<T>::type;
    typedef T near_t __attribute__((ext_vector_type(VecOf<T>::W), aligned(sizeof(T))));
    constexpr int W = VecOf<T>::W;
    __shared__ T lds[64][65];
    unsigned job = a.first + blockIdx.x;
    if (job >= static_cast<unsigned>(a.slope_blocks)) {
        job -= a.slope_blocks;
#pragma unroll
        for (int k = 0; k < kCopies; ++k) {
            if (job < static_cast<unsigned>(a.copy[k].blocks)) {
                copy_tile(a.copy[k], static_cast<int>(job), lds);
                return;
            }
            job -= a.copy[k].blocks;
        }
        return;
    }
    const int block = static_cast<int>(job);
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int row_block = block / a.slope_blocks_n, col_block = block - row_block * a.slope_blocks_n;
    const int64_t c = (static_cast<int64_t>(col_block) * 64 + lane) * W;
    const int64_t r0 = static_cast<int64_t>(row_block) * a.slope_rows;
    T sg[W], su[W];
#pragma unroll
    for (int k = 0; k < W; ++k) sg[k] = su[k] = T(0);
    if (c < a.d_row) {
        const bool whole = c + W <= a.hidden;
#pragma unroll 2
        for (int i = wave; i < a.slope_rows; i += 4) {
            if (r0 + i >= a.rows) break;
            const int64_t at = (r0 + i) * a.hidden + c;
            T d[W], g[W], u[W];
            if (whole) {
                const near_t x = *reinterpret_cast<const near_t *>(a.dh + at), y = *reinterpret_cast<const near_t *>(a.gate + at),
                             z = *reinterpret_cast<const near_t *>(a.up + at);
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    d[k] = x[k];
                    g[k] = y[k];
                    u[k] = z[k];
                }
            } else {
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    const bool in = c + k < a.hidden;
                    d[k] = in ? a.dh[at + k] : T(0);
                    g[k] = in ? a.gate[at + k] : T(0);
                    u[k] = in ? a.up[at + k] : T(0);
                }
            }
            V x, y;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                T value, slope;
                activate<T, ACT>(g[k], value, slope);
                x[k] = d[k] * u[k] * slope;
                y[k] = d[k] * value;
                sg[k] += x[k];
                su[k] += y[k];
            }
            *reinterpret_cast<V *>(a.dg + (r0 + i) * a.d_row + c) = x;
            *reinterpret_cast<V *>(a.du + (r0 + i) * a.d_row + c) = y;
        }
    }
    if (!a.sums) return;
    T *const part = &lds[0][0];  // [wave][2][W][64]
#pragma unroll
    for (int k = 0; k < W; ++k) {
        part[((wave * 2 + 0) * W + k) * 64 + lane] = sg[k];
        part[((wave * 2 + 1) * W + k) * 64 + lane] = su[k];
    }
    __syncthreads();
    if (wave < 2 && c < a.d_row) {  // wave 0 adds up dg's columns, wave 1 du's
#pragma unroll
        for (int k = 0; k < W; ++k) {
            T v = T(0);
#pragma unroll
            for (int w = 0; w < 4; ++w) v += part[((w * 2 + wave) * W + k) * 64 + lane];
            a.sums[(static_cast<int64_t>(row_block) * 2 + wave) * a.d_row + c + k] = v;
        }
    }
}

// Bias gradients from the parts: dbg[c] = sum over b of sums[b][0][c], dbu of sums[b][1][c].  A wave adds every fourth row
// block, the waves' sums are added in order.
template <typename T>
__global__ void __launch_bounds__(256) gated_bias_kernel(const T *sums, int64_t blocks, int64_t d_row, int hidden, T *dbg, T *dbu) {
    __shared__ T part[4][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    T *const out = blockIdx.y == 0 ? dbg : dbu;
    if (!out) return;
    T v = T(0);
    if (c < hidden) {
#pragma unroll 8
        for (int64_t b = wave; b < blocks; b += 4) v += sums[(b * 2 + blockIdx.y) * d_row + c];
    }
    part[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < hidden) out[c] = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
}

// A few rows (a token or a handful while generating): bound by the weights, which are read once.  A workgroup owns 8 vectors of
// columns of both weights and the whole reduction: lane group g of 128 takes every 128th row of the weights, so that its loads
// are 128 neighbouring bytes and each feeds R rows of x out of LDS; the groups' sums are added by shuffles, then wave by
// wave in order through LDS, and the same workgroup applies biases and activation: one launch.  Weights' rows may begin
// anywhere; the last vector of a row is moved back to end with it (its first columns come out twice, the same).
constexpr int kRowThreads = 1024, kRowLanes = 8, kRowGroups = kRowThreads / kRowLanes, kRowWaves = kRowThreads / 64;
constexpr int kRowChunk = 1024;  // of the reduction whose x is in LDS at a time
template <typename T>
struct RowArgs {
    const T *x, *wg, *wu, *bg, *bu;
    int64_t x0, x1, wg_row, wu_row;
    T *out, *gate, *up;
    int rows, inner, hidden;  // rows: up to R
};
template <typename T, int R, int ACT>
__global__ void __launch_bounds__(kRowThreads) gated_rows_kernel(RowArgs<T> a) {
    constexpr int W = VecOf<T>::W;
    typedef T near_t __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    constexpr int kCols = kRowLanes * W;
    __shared__ T xs[kRowChunk][R];
    __shared__ T part[kRowWaves][2][R][kCols];
    const int tid = threadIdx.x, lane = tid % kRowLanes, group = tid / kRowLanes;
    const int c0 = blockIdx.x * kCols;
    const int at = c0 + lane * W;
    const int c = at + W <= a.hidden ? at : a.hidden - W;  // (lanes beyond the row repeat its last columns)
    T g[R][W], u[R][W];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < W; ++k) g[r][k] = u[r][k] = T(0);
    for (int k0 = 0; k0 < a.inner; k0 += kRowChunk) {
        const int n = a.inner - k0 < kRowChunk ? a.inner - k0 : kRowChunk;
        if (k0) __syncthreads();
        for (int i = tid; i < n * R; i += kRowThreads) {
            const int r = i / n, k = i - r * n;
            xs[k][r] = r < a.rows ? a.x[r * a.x0 + (k0 + k) * a.x1] : T(0);
        }
        __syncthreads();
        const T *wg = a.wg + static_cast<int64_t>(k0) * a.wg_row + c, *wu = a.wu + static_cast<int64_t>(k0) * a.wu_row + c;
#pragma unroll 4
        for (int k = group; k < n; k += kRowGroups) {
            const near_t p = *reinterpret_cast<const near_t *>(wg + k * a.wg_row), q = *reinterpret_cast<const near_t *>(wu + k * a.wu_row);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const T v = xs[k][r];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    g[r][j] += v * p[j];
                    u[r][j] += v * q[j];
                }
            }
        }
    }
    const int wave = tid / 64;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < W; ++j) {
#pragma unroll
            for (int d = kRowLanes; d < 64; d *= 2) {
                g[r][j] += __shfl_xor(g[r][j], d, 64);
                u[r][j] += __shfl_xor(u[r][j], d, 64);
            }
            if (tid % 64 < kRowLanes) {
                part[wave][0][r][lane * W + j] = g[r][j];
                part[wave][1][r][lane * W + j] = u[r][j];
            }
        }
    __syncthreads();
    for (int i = tid; i < a.rows * kCols; i += kRowThreads) {
        const int r = i / kCols, k = i - r * kCols;
        const int from = c0 + k / W * W;
        const int col = (from + W <= a.hidden ? from : a.hidden - W) + k % W;  // the column that this place holds
        T gv = T(0), uv = T(0);
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) {
            gv += part[w][0][r][k];
            uv += part[w][1][r][k];
        }
        if (a.bg) gv += a.bg[col];
        if (a.bu) uv += a.bu[col];
        const int64_t to = static_cast<int64_t>(r) * a.hidden + col;
        if (a.gate) {
            a.gate[to] = gv;
            a.up[to] = uv;
        }
        a.out[to] = activate<T, ACT>(gv) * uv;
    }
}

template <typename F>
void for_activation(int act, F f) {
    switch (act) {
    case kSilu: f.template operator()<kSilu>(); break;
    case kGelu: f.template operator()<kGelu>(); break;
    case kRelu: f.template operator()<kRelu>(); break;
    default: f.template operator()<kSigmoid>(); break;
    }
}

unsigned stream_blocks(int64_t vectors) {
    const int64_t b = (vectors + 255) / 256;
    return static_cast<unsigned>(b < 1 ? 1 : b > (1 << 22) ? (1 << 22) : b);
}
bool aligned16(std::initializer_list<const void *> ptrs) {
    for (const void *p : ptrs)
        if (misaligned(p, 16)) return false;
    return true;
}

template <typename T>
ttamd_status launch_product(int act, const void *gate, const void *up, void *out, int64_t n, hipStream_t st) {
    if (n == 0) return TTAMD_OK;
    const bool vec = aligned16({gate, up, out});
    const unsigned blocks = stream_blocks(vec ? n / VecOf<T>::W : n);
    for_activation(act, [&]<int ACT>() {
        const auto *g = static_cast<const T *>(gate), *u = static_cast<const T *>(up);
        if (vec) gated_product_kernel<T, ACT, true><<<blocks, 256, 0, st>>>(g, u, static_cast<T *>(out), n);
        else gated_product_kernel<T, ACT, false><<<blocks, 256, 0, st>>>(g, u, static_cast<T *>(out), n);
    });
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

// Sizes of a pass: padded row lengths and the workspace's layout (bytes).  What a call needs of it depends on its views;
// the space covers every case.
struct GatedSizes {
    size_t item;
    int64_t vec;                   // elements of 16 bytes
    int64_t inner_row, hidden_row; // inner and hidden rounded up to whole vectors
    size_t first, second;          // forward: g and u; backward: dg and du, rows of hidden_row elements
    size_t sums;                   // backward: the bias gradients' parts
    size_t x, wg, wu;              // copies of operands
    size_t parts;                  // backward: parts of reductions that the tile kernel cuts
    GatedSplit split;
    size_t scratch, scratch_bytes; // lent to separate products: partial tiles of split reductions
    size_t bytes;
};

GatedSizes sizes_of(ttamd_dtype dtype, int64_t rows, int64_t inner, int64_t hidden, bool backward) {
    GatedSizes z{};
    z.item = dtype_size(dtype);
    z.vec = 16 / static_cast<int64_t>(z.item);
    z.inner_row = (inner + z.vec - 1) / z.vec * z.vec;
    z.hidden_row = (hidden + z.vec - 1) / z.vec * z.vec;
    size_t at = 0;
    const auto take = [&](int64_t elements) {
        const size_t here = at;
        at += (static_cast<size_t>(elements) * z.item + 255) / 256 * 256;
        return here;
    };
    z.first = take(rows * z.hidden_row);
    z.second = take(rows * z.hidden_row);
    z.sums = take(backward ? (rows + kSlopeRows - 1) / kSlopeRows * 2 * z.hidden_row : 0);
    z.x = take(rows * z.inner_row);
    z.wg = take(z.inner_row * z.hidden_row);
    z.wu = take(z.inner_row * z.hidden_row);
    // (the last stretch serves the tile kernel or the separate products)
    z.parts = z.scratch = at;
    size_t parts = 0;
    if (backward && rows > 0) {
        z.split = plan_gated_split(z.item, rows, inner, hidden, z.hidden_row);
        parts = static_cast<size_t>(z.split.x_parts + z.split.w_parts + z.split.b_parts) * z.item;
    }
    // A product of fewer than 128 tiles of 64 x 64 may be split into up to 64 reductions, 32 MiB of partial tiles at most.
    const auto split = [&](int64_t m, int64_t n) {
        if ((m + 63) / 64 * ((n + 63) / 64) >= 128) return size_t(0);
        const size_t b = static_cast<size_t>(64 * m * n) * z.item;
        return b < (size_t(32) << 20) ? b : size_t(32) << 20;
    };
    const size_t a = backward ? split(rows, inner) : split(rows, hidden), b = backward ? split(inner, hidden) : 0;
    z.scratch_bytes = a > b ? a : b;
    z.bytes = at + (z.scratch_bytes > parts ? z.scratch_bytes : parts);
    return z;
}

ttamd_status check_gated(const char *what, ttamd_dtype dtype, int64_t rows, int64_t inner, int64_t hidden) {
    if (dtype != TTAMD_F32 && dtype != TTAMD_F64) {
        set_error("%s: floating point dtypes only", what);
        return TTAMD_ERR_UNSUPPORTED_DTYPE;
    }
    // Every size in bytes fits 64 bits, and a launch fewer than 2^32 lanes: launch_prepare goes in runs, launch_rows is left to
    // narrower layers, and the operands, results and workspace of a call that 288 GB hold keep a grid of tiles (64 x 64 results and 256
    // lanes at least) below 2^24 workgroups.
    constexpr int64_t most_lines = int64_t(1) << 26, most = int64_t(1) << 40;
    if (rows < 0 || inner < 1 || hidden < 1 || rows > most_lines || inner > most_lines || hidden > most_lines || rows * inner > most ||
        rows * hidden > most || inner * hidden > most) {
        set_error("%s: rows %lld, inner %lld, hidden %lld: rows from 0, the others from 1, up to 2^26 each and 2^40 elements a matrix", what,
                  static_cast<long long>(rows), static_cast<long long>(inner), static_cast<long long>(hidden));
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    return TTAMD_OK;
}

ttamd_status check_activation(const char *what, int act) {
    if (act >= kSilu && act <= kSigmoid) return TTAMD_OK;
    set_error("%s: unknown activation %d", what, act);
    return TTAMD_ERR_INVALID_ARGUMENT;
}

ttamd_status check_view(const char *what, const char *name, const ttamd_view2 *v, size_t item, bool need_data) {
    if (!v || (need_data && !v->data)) {
        set_error("%s: NULL view or data of %s", what, name);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    constexpr int64_t most = int64_t(1) << 32;  // (reaches are computed in 64 bits)
    if (v->offset < 0 || v->stride[0] < 0 || v->stride[1] < 0 || v->stride[0] > most || v->stride[1] > most || misaligned(v->data, item)) {
        set_error("%s: %s: a negative offset, a stride outside 0 to 2^32, or a pointer off the element size", what, name);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    return TTAMD_OK;
}

// A matrix as the kernels take it: the caller's own, or its copy in the workspace.
template <typename T>
struct Operand {
    const T *data;
    int64_t s0, s1;
};

template <typename T>
Operand<T> operand_of(const ttamd_view2 &v) {
    return {static_cast<const T *>(v.data) + v.offset, v.stride[0], v.stride[1]};
}
// Rows of whole 16-byte vectors at aligned addresses, in order.
template <typename T>
bool row_vectors(const Operand<T> &m, int64_t cols) {
    constexpr int64_t W = VecOf<T>::W;
    return m.s1 == 1 && m.s0 % W == 0 && cols % W == 0 && !misaligned(m.data, 16);
}
template <typename T>
CopyJob<T> copy_job(Operand<T> &m, int64_t rows, int64_t cols, int64_t dst_rows, int64_t dst_row, void *dst) {
    CopyJob<T> j{m.data, m.s0, m.s1, rows, cols, dst_rows, dst_row, static_cast<T *>(dst), 0};
    j.blocks = static_cast<int>((dst_rows + copy_rows(j) - 1) / copy_rows(j) * ((dst_row + 63) / 64));
    m = {static_cast<const T *>(dst), dst_row, 1};
    return j;
}
template <typename T>
ttamd_view3 view_of(const Operand<T> &m, bool transposed = false) {
    return {m.data, 0, {0, transposed ? m.s1 : m.s0, transposed ? m.s0 : m.s1}};
}

template <typename T>
ttamd_status launch_prepare(int act, const PrepareArgs<T> &a, hipStream_t st) {
    int64_t blocks = a.slope_blocks;
    for (const CopyJob<T> &j : a.copy) blocks += j.blocks;
    // A launch holds fewer than 2^32 lanes; copies of more than 2^32 elements have more (2^26 rows of 257 f32: 2^22 x 5 workgroups).
    constexpr int64_t kRun = int64_t(1) << 23;
    PrepareArgs<T> run = a;
    for (int64_t at = 0; at < blocks; at += kRun) {
        run.first = static_cast<unsigned>(at);
        const unsigned n = static_cast<unsigned>(blocks - at < kRun ? blocks - at : kRun);
        for_activation(act, [&]<int ACT>() { gated_prepare_kernel<T, ACT><<<n, 256, 0, st>>>(run); });
        TTAMD_HIP_CHECK(hipGetLastError());
    }
    return TTAMD_OK;
}

// Offsets inside a tile's operand or result are 32-bit: `lines` rows of `row` elements must lie within 2^31 bytes.
bool within_reach(size_t item, int64_t lines, int64_t row) { return (lines + 64) * row < 0x7fffffffLL / static_cast<int64_t>(item); }
constexpr int64_t kTileLines = 256;  // of the largest tile

struct Pass {
    int device, act;
    ttamd_dtype dtype;
    int64_t rows, inner, hidden;
    ttamd_view2 x, wg, wu;
    char *ws;
    void *stream;
};

// Up to 4 rows (f32; 2 f64) in one launch: 1 x 2048 x 2048 f32 13.2 us against 18.6 on the matrix cores (gated_few_kernel),
// 4 x 4000 x 512 27 against 33, f64 2 x 2048 x 2048 16.7 against 23.2.  f32 of more than 4096 columns only 1 row: 4 x 2048 x 8192 28.7
// against 21.8, while 1 row gains up to a fifth (1 x 2048 x 8200 36.5 against 44.6, 4096 x 12000 69 against 84) and loses up to
// an eighth (2048 x 8192 22.4 against 21.5, 2048 x 16384 55 against 48).
template <typename T>
ttamd_status launch_rows(int act, const RowArgs<T> &a, int64_t rows, hipStream_t st) {
    constexpr int kCols = kRowLanes * VecOf<T>::W;
    const unsigned blocks = static_cast<unsigned>((a.hidden + kCols - 1) / kCols);
    for_activation(act, [&]<int ACT>() {
        if (rows > 2) {
            if constexpr (sizeof(T) == 4) gated_rows_kernel<T, 4, ACT><<<blocks, kRowThreads, 0, st>>>(a);
        } else if (rows > 1) {
            gated_rows_kernel<T, 2, ACT><<<blocks, kRowThreads, 0, st>>>(a);
        } else {
            gated_rows_kernel<T, 1, ACT><<<blocks, kRowThreads, 0, st>>>(a);
        }
    });
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

// How the forward pass goes: the row kernel, blocks of rows, one grid of tiles, or two products and a launch behind them.
enum class Way { rows, few, tiles, products };
template <typename T>
Way forward_way(const GatedSizes &z, int64_t rows, int64_t inner, int64_t hidden, const Operand<T> &x, const Operand<T> &wg, const Operand<T> &wu) {
    const bool f32 = z.item == 4;
    const bool in_order = x.s1 == 1 && wg.s1 == 1 && wu.s1 == 1;
    const int64_t handful = f32 ? (hidden <= 4096 ? 4 : 1) : 2;
    // (a launch of 2^32 lanes, f64 from 2^26 - 15 columns on, is one too many)
    const bool in_a_launch = (hidden + kRowLanes * z.vec - 1) / (kRowLanes * z.vec) * kRowThreads < int64_t(1) << 32;
    if (rows <= handful && wg.s1 == 1 && wu.s1 == 1 && hidden >= z.vec && in_a_launch) return Way::rows;
    // One grid of both products (gated_tiles.hip), unless it would be few tiles of a long reduction, which the separate
    // products cut (f32, 64 x 128 tiles: 128 x 1024 x 2048, 64 tiles, 38 us against 28 in three launches; 256 x 1024 x 4096,
    // 256 tiles, 38 against 49; f64, 64 x 64 tiles: 200 x 2001 x 1003, 128 tiles, 98 against 77; 256 x 1024 x 4096, 512
    // tiles, 65 against 79), or the weights are beyond its reach.
    const int64_t tiles = (rows + 63) / 64 * ((hidden + (f32 ? 63 : 31)) / (f32 ? 64 : 32));
    const bool cut = inner > 256 && (rows <= 32 || tiles < (f32 ? 96 : 144));
    const bool tiled = !cut && within_reach(z.item, z.inner_row, z.hidden_row) && within_reach(z.item, kTileLines, z.inner_row) &&
                       within_reach(z.item, kTileLines, z.hidden_row);
    if (rows <= 256 && in_order && hidden >= 2) {
        // What the others take, in us: a round of tiles (0.034 a k) and a copy launch where an operand needs one, or two
        // products and the launch behind them.
        const bool copies = !row_vectors(x, inner) || !row_vectors(wg, hidden) || !row_vectors(wu, hidden);
        const double others = tiled ? static_cast<double>((tiles + 255) / 256 * inner) * 0.034 + (copies ? 11 : 3)
                                    : 17 + 0.0035 * static_cast<double>(inner) + 4e-6 * static_cast<double>(rows * inner) * static_cast<double>(hidden) / (f32 ? 153 : 73);
        if (few_rows_estimate(z.item, rows, inner, hidden) < others) return Way::few;
    }
    return tiled ? Way::tiles : Way::products;
}

template <typename T>
ttamd_status forward(const Pass &p, const void *gate_bias, const void *up_bias, void *out, void *gate, void *up) {
    hipStream_t st = static_cast<hipStream_t>(p.stream);
    const int64_t rows = p.rows, inner = p.inner, hidden = p.hidden;
    const GatedSizes z = sizes_of(p.dtype, rows, inner, hidden, false);
    Operand<T> x = operand_of<T>(p.x), wg = operand_of<T>(p.wg), wu = operand_of<T>(p.wu);
    const Way way = forward_way(z, rows, inner, hidden, x, wg, wu);
    if (way == Way::rows) {
        const RowArgs<T> a{x.data, wg.data, wu.data, static_cast<const T *>(gate_bias), static_cast<const T *>(up_bias), x.s0, x.s1, wg.s0, wu.s0,
                           static_cast<T *>(out), static_cast<T *>(gate), static_cast<T *>(up), static_cast<int>(rows), static_cast<int>(inner), static_cast<int>(hidden)};
        return launch_rows<T>(p.act, a, rows, st);
    }
    if (way == Way::few) {
        const GatedForward<T> a{x.data, wg.data, wu.data, x.s0, wg.s0, wu.s0, static_cast<int>(rows), static_cast<int>(inner), static_cast<int>(hidden),
                                static_cast<int>(hidden), p.act, static_cast<const T *>(gate_bias), static_cast<const T *>(up_bias),
                                static_cast<T *>(out), static_cast<T *>(gate), static_cast<T *>(up)};
        return launch_gated_few_rows<T>(a, p.device, st);
    }
    if (way == Way::tiles) {
        PrepareArgs<T> prep{};
        const bool own = inner % z.vec == 0;  // (x's padding meets rows of zeros in the weights' copies)
        const auto far = [&](const Operand<T> &w) { return !own || !row_vectors(w, hidden) || !within_reach(z.item, inner, w.s0); };
        if (!row_vectors(x, inner) || !within_reach(z.item, kTileLines, x.s0)) prep.copy[0] = copy_job(x, rows, inner, rows, z.inner_row, p.ws + z.x);
        if (far(wg)) prep.copy[1] = copy_job(wg, inner, hidden, z.inner_row, z.hidden_row, p.ws + z.wg);
        if (far(wu)) prep.copy[2] = copy_job(wu, inner, hidden, z.inner_row, z.hidden_row, p.ws + z.wu);
        if (ttamd_status s = launch_prepare(p.act, prep, st)) return s;
        const GatedForward<T> a{x.data, wg.data, wu.data, x.s0, wg.s0, wu.s0, static_cast<int>(rows), static_cast<int>(z.inner_row),
                                static_cast<int>(z.hidden_row), static_cast<int>(hidden), p.act, static_cast<const T *>(gate_bias),
                                static_cast<const T *>(up_bias), static_cast<T *>(out), static_cast<T *>(gate), static_cast<T *>(up)};
        return launch_gated_forward_tiles<T>(a, p.device, st);
    }
    const ScratchLoan loan(p.ws + z.scratch, z.scratch_bytes);
    void *g = gate ? gate : p.ws + z.first, *u = gate ? up : p.ws + z.second;
    const int R = static_cast<int>(rows), K = static_cast<int>(inner), H = static_cast<int>(hidden);
    const ttamd_view3 xv = view_of(x), gv = view_of(wg), uv = view_of(wu);
    ttamd_epilogue eg{}, eu{};
    eg.bias = gate_bias;
    eg.bias_mode = gate_bias ? 1 : 0;
    eu.bias = up_bias;
    eu.bias_mode = up_bias ? 1 : 0;
    if (ttamd_status s = ttamd_batched_matmul(p.device, p.dtype, 1, R, K, H, &xv, &gv, g, &eg, p.stream)) return s;
    if (ttamd_status s = ttamd_batched_matmul(p.device, p.dtype, 1, R, K, H, &xv, &uv, u, &eu, p.stream)) return s;
    return launch_product<T>(p.act, g, u, out, rows * hidden, st);
}

// One grid of all three products (gated_tiles.hip) unless rows or weights are beyond its reach.
bool backward_in_a_grid(const GatedSizes &z, int64_t rows) {
    const int64_t piece = z.split.w_splits ? z.split.w_chunk : rows;  // rows under a tile of a weight's gradient
    return rows > 0 && within_reach(z.item, piece, z.hidden_row) && within_reach(z.item, piece, z.inner_row) &&
           within_reach(z.item, kTileLines, z.hidden_row) && within_reach(z.item, kTileLines, z.inner_row);
}

template <typename T>
ttamd_status backward(const Pass &p, const void *grad_out, const void *gate, const void *up, void *dx, void *dwg, void *dwu, void *dbg, void *dbu) {
    hipStream_t st = static_cast<hipStream_t>(p.stream);
    const int64_t rows = p.rows, inner = p.inner, hidden = p.hidden;
    const GatedSizes z = sizes_of(p.dtype, rows, inner, hidden, true);
    Operand<T> x = operand_of<T>(p.x), wg = operand_of<T>(p.wg), wu = operand_of<T>(p.wu);
    PrepareArgs<T> prep{};
    T *const dg = reinterpret_cast<T *>(p.ws + z.first), *const du = reinterpret_cast<T *>(p.ws + z.second);
    if (rows > 0) {
        prep.dh = static_cast<const T *>(grad_out);
        prep.gate = static_cast<const T *>(gate);
        prep.up = static_cast<const T *>(up);
        prep.dg = dg;
        prep.du = du;
        prep.rows = rows;
        prep.d_row = z.hidden_row;
        prep.hidden = static_cast<int>(hidden);
        prep.slope_blocks_n = static_cast<int>((z.hidden_row / z.vec + 63) / 64);
        prep.slope_rows = kFewSlopeRows;
        prep.slope_blocks = static_cast<int>((rows + kFewSlopeRows - 1) / kFewSlopeRows) * prep.slope_blocks_n;
    }
    if (backward_in_a_grid(z, rows)) {
        const int64_t piece = z.split.w_splits ? z.split.w_chunk : rows;
        const auto far = [&](const Operand<T> &w) { return !row_vectors(w, hidden) || !within_reach(z.item, kTileLines, w.s0); };
        if (!row_vectors(x, inner) || !within_reach(z.item, piece, x.s0)) prep.copy[0] = copy_job(x, rows, inner, rows, z.inner_row, p.ws + z.x);
        if (far(wg)) prep.copy[1] = copy_job(wg, inner, hidden, inner, z.hidden_row, p.ws + z.wg);
        if (far(wu)) prep.copy[2] = copy_job(wu, inner, hidden, inner, z.hidden_row, p.ws + z.wu);
        if (ttamd_status s = launch_prepare(p.act, prep, st)) return s;
        const GatedBackward<T> a{x.data, wg.data, wu.data, x.s0, wg.s0, wu.s0, dg, du, z.hidden_row, static_cast<int>(rows), static_cast<int>(inner),
                                 static_cast<int>(z.inner_row), static_cast<int>(hidden), static_cast<int>(z.hidden_row), static_cast<T *>(dx),
                                 static_cast<T *>(dwg), static_cast<T *>(dwu), static_cast<T *>(dbg), static_cast<T *>(dbu),
                                 z.split, reinterpret_cast<T *>(p.ws + z.parts), reinterpret_cast<T *>(p.ws + z.parts) + z.split.x_parts,
                                 reinterpret_cast<T *>(p.ws + z.parts) + z.split.x_parts + z.split.w_parts};
        return launch_gated_backward_tiles<T>(a, p.device, st);
    }
    T *const sums = reinterpret_cast<T *>(p.ws + z.sums);
    if (dbg || dbu) {
        prep.sums = sums;
        prep.slope_rows = kSlopeRows;
        prep.slope_blocks = static_cast<int>((rows + kSlopeRows - 1) / kSlopeRows) * prep.slope_blocks_n;
    }
    if (ttamd_status s = launch_prepare(p.act, prep, st)) return s;
    if (dbg || dbu) {
        gated_bias_kernel<T><<<dim3(static_cast<unsigned>((hidden + 63) / 64), 2), 256, 0, st>>>(
            sums, (rows + kSlopeRows - 1) / kSlopeRows, z.hidden_row, static_cast<int>(hidden), static_cast<T *>(dbg), static_cast<T *>(dbu));
        TTAMD_HIP_CHECK(hipGetLastError());
    }
    const ScratchLoan loan(p.ws + z.scratch, z.scratch_bytes);
    const int R = static_cast<int>(rows), K = static_cast<int>(inner), H = static_cast<int>(hidden);
    const ttamd_view3 gv{dg, 0, {0, z.hidden_row, 1}}, uv{du, 0, {0, z.hidden_row, 1}};
    const ttamd_view3 xt = view_of(x, true), wgt = view_of(wg, true), wut = view_of(wu, true);
    ttamd_epilogue add{};
    add.accumulate = 1;
    if (rows > 0) {
        if (ttamd_status s = ttamd_batched_matmul(p.device, p.dtype, 1, R, H, K, &gv, &wgt, dx, nullptr, p.stream)) return s;
        if (ttamd_status s = ttamd_batched_matmul(p.device, p.dtype, 1, R, H, K, &uv, &wut, dx, &add, p.stream)) return s;
    }
    // the weights' gradients in runs of rows whose offsets fit the products' 32 bits
    const int64_t longest = z.hidden_row > x.s0 + x.s1 * inner ? z.hidden_row : x.s0 + x.s1 * inner;
    int64_t run = 0x3fffffffLL / static_cast<int64_t>(z.item) / longest;
    if (run < 64) run = 64;
    for (int64_t r = 0; r == 0 || r < rows; r += run) {
        const int n = static_cast<int>(rows - r < run ? rows - r : run);
        ttamd_view3 xr = xt, gr = gv, ur = uv;
        xr.offset += r * x.s0;
        gr.offset += r * z.hidden_row;
        ur.offset += r * z.hidden_row;
        const ttamd_epilogue *ep = r ? &add : nullptr;
        if (ttamd_status s = ttamd_batched_matmul(p.device, p.dtype, 1, K, n, H, &xr, &gr, dwg, ep, p.stream)) return s;
        if (ttamd_status s = ttamd_batched_matmul(p.device, p.dtype, 1, K, n, H, &xr, &ur, dwu, ep, p.stream)) return s;
    }
    return TTAMD_OK;
}

Extent extent_of(const char *name, const ttamd_view2 &v, int64_t rows, int64_t cols, size_t item) {
    return {name, v.data ? static_cast<const char *>(v.data) + v.offset * static_cast<int64_t>(item) : nullptr, rows, cols, v.stride[0], v.stride[1], item};
}

ttamd_status check_workspace(const char *what, const void *workspace, size_t given, size_t needed) {
    if (workspace && !misaligned(workspace, 16) && given >= needed) return TTAMD_OK;
    set_error("%s: workspace %p of %zu bytes: %zu are needed, aligned to 16", what, workspace, given, needed);
    return TTAMD_ERR_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" {

ttamd_status ttamd_gated_linear_workspace(ttamd_dtype dtype, int64_t rows, int64_t inner, int64_t hidden, int backward, size_t *bytes) {
    if (ttamd_status s = check_gated("gated_linear", dtype, rows, inner, hidden)) return s;
    if (!bytes) {
        set_error("gated_linear: bytes is NULL");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    *bytes = rows > 0 ? sizes_of(dtype, rows, inner, hidden, backward != 0).bytes : 0;
    return TTAMD_OK;
}

const char *ttamd_gated_linear_variant(ttamd_dtype dtype, int64_t rows, int64_t inner, int64_t hidden, const ttamd_view2 *input,
                                       const ttamd_view2 *gate_weight, const ttamd_view2 *up_weight, int backward) {
    const char *const what = "gated_linear_variant";
    if (check_gated(what, dtype, rows, inner, hidden)) return "invalid";
    const size_t item = dtype_size(dtype);
    if (check_view(what, "input", input, item, false) || check_view(what, "gate weight", gate_weight, item, false) ||
        check_view(what, "up weight", up_weight, item, false))
        return "invalid";
    if (rows == 0) return "empty";
    const GatedSizes z = sizes_of(dtype, rows, inner, hidden, backward != 0);
    static thread_local char name[64];
    const char *const type = item == 4 ? "f32" : "f64";
    if (backward) {
        if (!backward_in_a_grid(z, rows)) return item == 4 ? "gated_backward_f32_products" : "gated_backward_f64_products";
        char x[16] = "", w[16] = "";
        if (z.split.x_splits) snprintf(x, sizeof(x), "_x%d", z.split.x_splits);
        if (z.split.w_splits) snprintf(w, sizeof(w), "_w%d", z.split.w_splits);
        snprintf(name, sizeof(name), "gated_backward_%s_%dx%d%s%s", type, z.split.tile, z.split.tile, x, w);
        return name;
    }
    const auto way_of = [&]<typename T>() { return forward_way<T>(z, rows, inner, hidden, operand_of<T>(*input), operand_of<T>(*gate_weight), operand_of<T>(*up_weight)); };
    switch (item == 4 ? way_of.template operator()<float>() : way_of.template operator()<double>()) {
    case Way::rows: snprintf(name, sizeof(name), "gated_%s_rows%d", type, rows > 2 ? 4 : static_cast<int>(rows)); break;
    case Way::few: snprintf(name, sizeof(name), "gated_%s_few%d", type, few_rows_of(rows, hidden)); break;
    case Way::tiles: {
        const ForwardTile t = pick_forward_tile(item, rows, hidden, z.inner_row);
        snprintf(name, sizeof(name), "gated_%s_%dx%d%s", type, t.bm, t.bn, t.halves == 2 ? "_halves" : "");
        break;
    }
    case Way::products: snprintf(name, sizeof(name), "gated_%s_products", type); break;
    }
    return name;
}

ttamd_status ttamd_gated_linear_forward(int device, ttamd_dtype dtype, int activation, int64_t rows, int64_t inner, int64_t hidden,
                                        const ttamd_view2 *input, const ttamd_view2 *gate_weight, const ttamd_view2 *up_weight,
                                        const void *gate_bias, const void *up_bias, void *out, void *gate_out, void *up_out, void *workspace,
                                        size_t workspace_bytes, void *stream) {
    const char *const what = "gated_linear";
    if (ttamd_status s = check_gated(what, dtype, rows, inner, hidden)) return s;
    if (ttamd_status s = check_activation(what, activation)) return s;
    const size_t item = dtype_size(dtype);
    const bool work = rows > 0;
    if (ttamd_status s = check_view(what, "input", input, item, work)) return s;
    if (ttamd_status s = check_view(what, "gate weight", gate_weight, item, work)) return s;
    if (ttamd_status s = check_view(what, "up weight", up_weight, item, work)) return s;
    if (work && !out) {
        set_error("%s: NULL data pointer", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (!gate_out != !up_out) {
        set_error("%s: gate_out and up_out are given together or not at all", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    for (const void *q : {static_cast<const void *>(out), static_cast<const void *>(gate_out), static_cast<const void *>(up_out), gate_bias, up_bias})
        if (misaligned(q, item)) {
            set_error("%s: pointers must be aligned to the element size", what);
            return TTAMD_ERR_INVALID_ARGUMENT;
        }
    if (work) {
        const size_t need = sizes_of(dtype, rows, inner, hidden, false).bytes;
        if (ttamd_status s = check_workspace(what, workspace, workspace_bytes, need)) return s;
        const int64_t n = rows * hidden;
        if (ttamd_status s = check_disjoint(what,
                                            {dense_extent("out", out, n, item), dense_extent("gate_out", gate_out, n, item), dense_extent("up_out", up_out, n, item),
                                             dense_extent("the workspace", workspace, static_cast<int64_t>(need), 1)},
                                            {extent_of("input", *input, rows, inner, item), extent_of("gate weight", *gate_weight, inner, hidden, item),
                                             extent_of("up weight", *up_weight, inner, hidden, item), dense_extent("gate_bias", gate_bias, hidden, item),
                                             dense_extent("up_bias", up_bias, hidden, item)}))
            return s;
    }
    if (ttamd_status s = use_device(device)) return s;
    if (!work) return TTAMD_OK;
    const Pass p{device, activation, dtype, rows, inner, hidden, *input, *gate_weight, *up_weight, static_cast<char *>(workspace), stream};
    return dtype == TTAMD_F32 ? forward<float>(p, gate_bias, up_bias, out, gate_out, up_out)
                              : forward<double>(p, gate_bias, up_bias, out, gate_out, up_out);
}

ttamd_status ttamd_gated_linear_backward(int device, ttamd_dtype dtype, int activation, int64_t rows, int64_t inner, int64_t hidden,
                                         const void *grad_out, const ttamd_view2 *input, const ttamd_view2 *gate_weight,
                                         const ttamd_view2 *up_weight, const void *gate, const void *up, void *grad_input,
                                         void *grad_gate_weight, void *grad_up_weight, void *grad_gate_bias, void *grad_up_bias,
                                         void *workspace, size_t workspace_bytes, void *stream) {
    const char *const what = "gated_linear_backward";
    if (ttamd_status s = check_gated(what, dtype, rows, inner, hidden)) return s;
    if (ttamd_status s = check_activation(what, activation)) return s;
    const size_t item = dtype_size(dtype);
    const bool work = rows > 0;
    if (ttamd_status s = check_view(what, "input", input, item, work)) return s;
    if (ttamd_status s = check_view(what, "gate weight", gate_weight, item, work)) return s;
    if (ttamd_status s = check_view(what, "up weight", up_weight, item, work)) return s;
    if (!grad_gate_weight || !grad_up_weight || (work && (!grad_out || !gate || !up || !grad_input))) {
        set_error("%s: NULL data pointer", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    for (const void *q : {grad_out, gate, up, static_cast<const void *>(grad_input), static_cast<const void *>(grad_gate_weight),
                          static_cast<const void *>(grad_up_weight), static_cast<const void *>(grad_gate_bias), static_cast<const void *>(grad_up_bias)})
        if (misaligned(q, item)) {
            set_error("%s: pointers must be aligned to the element size", what);
            return TTAMD_ERR_INVALID_ARGUMENT;
        }
    size_t need = 0;
    if (work) {
        need = sizes_of(dtype, rows, inner, hidden, true).bytes;
        if (ttamd_status s = check_workspace(what, workspace, workspace_bytes, need)) return s;
    }
    const int64_t n = rows * hidden, w = inner * hidden;
    if (ttamd_status s = check_disjoint(what,
                                        {dense_extent("grad_input", grad_input, rows * inner, item), dense_extent("grad_gate_weight", grad_gate_weight, w, item),
                                         dense_extent("grad_up_weight", grad_up_weight, w, item), dense_extent("grad_gate_bias", grad_gate_bias, hidden, item),
                                         dense_extent("grad_up_bias", grad_up_bias, hidden, item), dense_extent("the workspace", workspace, static_cast<int64_t>(need), 1)},
                                        {dense_extent("grad_out", grad_out, n, item), extent_of("input", *input, rows, inner, item),
                                         extent_of("gate weight", *gate_weight, inner, hidden, item), extent_of("up weight", *up_weight, inner, hidden, item),
                                         dense_extent("gate", gate, n, item), dense_extent("up", up, n, item)}))
        return s;
    if (ttamd_status s = use_device(device)) return s;
    const Pass p{device, activation, dtype, rows, inner, hidden, *input, *gate_weight, *up_weight, static_cast<char *>(workspace), stream};
    return dtype == TTAMD_F32 ? backward<float>(p, grad_out, gate, up, grad_input, grad_gate_weight, grad_up_weight, grad_gate_bias, grad_up_bias)
                              : backward<double>(p, grad_out, gate, up, grad_input, grad_gate_weight, grad_up_weight, grad_gate_bias, grad_up_bias);
}

}  // extern "C"
