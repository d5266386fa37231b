// gated.h — what the two sources of the gated pair of Linear layers share: activations, kernel arguments, launchers.
#ifndef TTAMD_CSRC_GATED_H_
#define TTAMD_CSRC_GATED_H_

#include "common.h"

namespace ttamd {

constexpr int kSilu = TTAMD_ACT_SILU, kGelu = TTAMD_ACT_GELU, kRelu = TTAMD_ACT_RELU, kSigmoid = TTAMD_ACT_SIGMOID;

template <typename T>
__device__ __forceinline__ T sigmoid(T g) {
    if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
    else return 1.0 / (1.0 + exp(-g));
}
template <typename T>
__device__ __forceinline__ T normal_cdf(T g) {
    if constexpr (sizeof(T) == 4) return 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    else return 0.5 * (1.0 + erf(g * 0.70710678118654752));
}

// act(g).
template <typename T, int ACT>
__device__ __forceinline__ T activate(T g) {
    if constexpr (ACT == kRelu) {
        return g > T(0) ? g : T(0);
    } else if constexpr (ACT == kGelu) {
        return g * normal_cdf(g);
    } else {
        const T s = sigmoid(g);
        return ACT == kSigmoid ? s : g * s;
    }
}
// act(g) and act'(g).  relu's derivative is where(g < 0, 0, 1), as TensorRelu::backward has it (autograd/unary_ops.cpp:568-573).
template <typename T, int ACT>
__device__ __forceinline__ void activate(T g, T &value, T &slope) {
    if constexpr (ACT == kRelu) {
        value = g > T(0) ? g : T(0);
        slope = g < T(0) ? T(0) : T(1);
    } else if constexpr (ACT == kGelu) {
        const T cdf = normal_cdf(g);
        T density;
        if constexpr (sizeof(T) == 4) density = 0.3989422804014327f * expf(-0.5f * g * g);
        else density = 0.3989422804014327 * exp(-0.5 * g * g);
        value = g * cdf;
        slope = cdf + g * density;
    } else {
        const T s = sigmoid(g);
        value = ACT == kSigmoid ? s : g * s;
        slope = ACT == kSigmoid ? s * (T(1) - s) : s * (T(1) + g * (T(1) - s));
    }
}

// Operands of the tile kernels: row-major, 16-byte aligned, rows of whole 16-byte vectors.  Results are dense rows of the
// true sizes.
template <typename T>
struct GatedForward {
    const T *x, *wg, *wu;               // [rows, k], [k, w_cols]
    int64_t x_row, wg_row, wu_row;      // elements between rows
    int rows, k, w_cols, hidden, act;   // k, w_cols: whole vectors (what is beyond the true sizes holds zeros)
    const T *gate_bias, *up_bias;       // [hidden] or null
    T *out, *gate, *up;                 // [rows, hidden]; gate and up: both or neither
};
// How the backward products' reductions are cut: dx's two reductions of k each into x_splits chunks of x_chunk (0: both in
// one piece), the weights' reductions of `rows` into w_splits chunks of w_chunk (0: one piece).
struct GatedSplit {
    int tile;  // 64, or 128 for f32
    int x_splits, x_chunk, w_splits, w_chunk;
    int64_t x_parts, w_parts, b_parts;  // elements of the parts of dx, of dWg and dWu, of the bias gradients
};
GatedSplit plan_gated_split(size_t item, int64_t rows, int64_t inner, int64_t hidden, int64_t k);

template <typename T>
struct GatedBackward {
    const T *x, *wg, *wu;               // [rows, x_cols], [inner, k]
    int64_t x_row, wg_row, wu_row;
    const T *dg, *du;                   // [rows, k]
    int64_t d_row;
    int rows, inner, x_cols, hidden, k; // x_cols, k: whole vectors
    T *dx, *dwg, *dwu, *dbg, *dbu;      // [rows, inner], [inner, hidden], [hidden] or null
    GatedSplit split;
    T *x_part, *w_part, *b_part;        // [2 x_splits][rows, inner], [w_splits][2][inner, hidden], [w_splits][2][hidden]
};
// The tile of the forward grid: bm rows of x against bn / 2 columns of both weights, in `halves` parts of the reduction.
struct ForwardTile {
    int bm, bn, halves;
};
ForwardTile pick_forward_tile(size_t item, int64_t rows, int64_t hidden, int64_t k);

// A block of rows: k and w_cols are the true sizes, rows begin anywhere, hidden >= 2.  The estimate is its time in us.
int few_rows_of(int64_t rows, int64_t hidden);  // rows of a workgroup: 16 or 32
double few_rows_estimate(size_t item, int64_t rows, int64_t inner, int64_t hidden);
template <typename T>
ttamd_status launch_gated_few_rows(const GatedForward<T> &a, int device, hipStream_t st);
template <typename T>
ttamd_status launch_gated_forward_tiles(const GatedForward<T> &a, int device, hipStream_t st);
template <typename T>
ttamd_status launch_gated_backward_tiles(const GatedBackward<T> &a, int device, hipStream_t st);

}  // namespace ttamd

#endif  // TTAMD_CSRC_GATED_H_
