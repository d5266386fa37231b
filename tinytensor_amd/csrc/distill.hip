// distill.hip — distillation of a student's logits from a teacher's top logits, loss and gradient in one call (gfx950).
//
// With T the temperature, z the student's logits of a row, (i_j, t_j) the teacher's top slots and w the row's weight:
//   p = softmax over the row's valid slots of t / T,   q = softmax over all columns of z / T,
//   loss += w T^2 sum_j p_j (log p_j - log q_{i_j}),   dz_i = w T (q_i - sum of p_j over the slots with i_j = i).
// No counterpart in the reference; it stands beside nn::mse_loss (nn/loss.cpp:69-72) as ttamd_mse_loss does.
//
// Bound: HBM.  The logits are read once and the gradient is written once; what a kernel adds to that is a second read of
// the part of a row that it could not keep on the chip.
#include "common.h"

namespace ttamd {
namespace {

constexpr int kMaxTop = 1024;  // slots a row may have: their indices, probabilities and student logits are kept in LDS

template <typename T>
struct Num;
template <>
struct Num<float> {
    static constexpr int W = 4;  // elements of a 16-byte vector
    // rows of an odd length begin anywhere: the vectors are declared with their element's alignment, which the hardware's
    // 16-byte loads and stores accept
    typedef float vec_t __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float max_(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
    // exp(x / T) for x <= 0 as 2^(x * log2(e) / T): the difference to the row's largest logit is taken first, so the
    // factor's rounding (2^-24 of the exponent) only reaches entries far below the largest
    static __device__ __forceinline__ float exp_scaled(float x, float c) { return __builtin_amdgcn_exp2f(x * c); }
};
template <>
struct Num<double> {
    static constexpr int W = 2;
    typedef double vec_t __attribute__((ext_vector_type(2), aligned(8)));
    static __device__ __forceinline__ double max_(double a, double b) { return fmax(a, b); }
    static __device__ __forceinline__ double neg_inf() { return -__builtin_inf(); }
    static __device__ __forceinline__ double exp_scaled(double x, double c) { return exp(x * c); }
};

template <typename T>
struct DistillArgs {
    const T *z;
    int64_t z_row;        // elements between the rows of z
    const void *index;    // [rows, top] i32 or i64
    const T *teacher;     // [rows, top]
    const T *weight;      // [rows] or null: 1 / rows
    T *grad;              // [rows, cols]
    double *row_loss;     // [rows] scratch
    int64_t rows;
    int cols, top, index64;
    double temperature;
    T c;                  // factor of exp_scaled: log2(e) / T for float, 1 / T for double
    T uniform_weight;
};

// What a row's slots come to, in LDS.  p is 0 in a slot that does not count: an index outside the columns, a logit of -inf.
template <typename T>
struct Slots {
    T p[kMaxTop], z[kMaxTop];
    int index[kMaxTop];
};

template <typename T>
__device__ __forceinline__ T wave_max(T v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v = Num<T>::max_(v, __shfl_xor(v, d, 64));
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d, 64);
    return v;
}

template <typename T>
__device__ __forceinline__ int slot_index(const DistillArgs<T> &a, int64_t row, int j) {
    const int64_t at = row * a.top + j;
    const int64_t i = a.index64 ? static_cast<const int64_t *>(a.index)[at] : static_cast<const int32_t *>(a.index)[at];
    return i >= 0 && i < a.cols ? static_cast<int>(i) : -1;
}

// One wave reads the row's slots into `s` (probabilities, student logits, indices); false when none counts, and the row
// then contributes nothing.
template <typename T>
__device__ __forceinline__ bool read_slots(const DistillArgs<T> &a, int64_t row, int lane, Slots<T> &s) {
    const T *zr = a.z + row * a.z_row;
    T most = Num<T>::neg_inf();
    bool nan = false;
    for (int j = lane; j < a.top; j += 64) {
        const int i = slot_index(a, row, j);
        const T t = i >= 0 ? a.teacher[row * a.top + j] : Num<T>::neg_inf();
        s.index[j] = i;
        s.p[j] = t;
        s.z[j] = i >= 0 ? zr[i] : T(0);
        most = Num<T>::max_(most, t);
        nan = nan || t != t;
    }
    most = wave_max(most);
    if (most == Num<T>::neg_inf() && !__any(nan)) return false;
    T sum = T(0);
    for (int j = lane; j < a.top; j += 64) {
        const T e = s.index[j] >= 0 ? Num<T>::exp_scaled(s.p[j] - most, a.c) : T(0);
        s.p[j] = e;
        sum += e;
    }
    sum = wave_sum(sum);
    for (int j = lane; j < a.top; j += 64) s.p[j] /= sum;
    return true;
}

// One wave: T^2 sum_j p_j (log p_j - log q_j), log q_j = (z_j - m) / T - log(total); terms and sum in 64 bits.
template <typename T>
__device__ __forceinline__ double slots_loss(const DistillArgs<T> &a, int lane, const Slots<T> &s, T most, T total) {
    const double inv = 1.0 / a.temperature, log_total = log(static_cast<double>(total));
    double sum = 0;
    for (int j = lane; j < a.top; j += 64) {
        const double p = s.p[j];
        if (p != 0.0) sum += p * (log(p) - ((static_cast<double>(s.z[j]) - static_cast<double>(most)) * inv - log_total));  // (p = 0: the term is 0 whatever q is)
    }
    return a.temperature * a.temperature * wave_sum(sum);
}

// p summed over the slots with slot j's index (a teacher may name a column twice), in slot order.
template <typename T>
__device__ __forceinline__ T slot_share(const Slots<T> &s, int top, int j) {
    const int i = s.index[j];
    T sum = T(0);
    for (int k = 0; k < top; ++k) sum += s.index[k] == i ? s.p[k] : T(0);
    return sum;
}

template <typename T, int BT, bool MAX>
__device__ __forceinline__ T block_reduce(T v, T *lds) {
    constexpr int NW = BT / 64;
    v = MAX ? wave_max(v) : wave_sum(v);
    if constexpr (NW == 1) return v;
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    T r = lds[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) r = MAX ? Num<T>::max_(r, lds[i]) : r + lds[i];
    return r;
}

// A workgroup a row: largest logit, then the sum of the exponentials, then the gradient.
template <typename T, int BT>
__global__ void __launch_bounds__(BT) distill_row_kernel(DistillArgs<T> a) {
    using V = typename Num<T>::vec_t;
    constexpr int W = Num<T>::W;
    __shared__ Slots<T> slots;
    __shared__ T red[2][BT / 64];
    __shared__ int counts;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid % 64;
    const T *zr = a.z + row * a.z_row;
    T *gr = a.grad + row * a.cols;
    const int nvec = a.cols / W, tail0 = nvec * W;
    const T w = a.weight ? a.weight[row] : a.uniform_weight;
    if (tid < 64) {
        const bool on = w != T(0) && read_slots(a, row, lane, slots);
        if (tid == 0) counts = on;
    }
    __syncthreads();
    if (!counts) {  // a row that weighs nothing, or whose slots are all empty: no loss, no gradient, nothing read
        V zero;
#pragma unroll
        for (int k = 0; k < W; ++k) zero[k] = T(0);
        for (int v = tid; v < nvec; v += BT) reinterpret_cast<V *>(gr)[v] = zero;
        if (tail0 + tid < a.cols) gr[tail0 + tid] = T(0);
        if (tid == 0) a.row_loss[row] = 0.0;
        return;
    }
    T most = Num<T>::neg_inf();
    for (int v = tid; v < nvec; v += BT) {
        const V x = reinterpret_cast<const V *>(zr)[v];
#pragma unroll
        for (int k = 0; k < W; ++k) most = Num<T>::max_(most, x[k]);
    }
    if (tail0 + tid < a.cols) most = Num<T>::max_(most, zr[tail0 + tid]);
    most = block_reduce<T, BT, true>(most, red[0]);
    T total = T(0);
    for (int v = tid; v < nvec; v += BT) {
        const V x = reinterpret_cast<const V *>(zr)[v];
#pragma unroll
        for (int k = 0; k < W; ++k) total += Num<T>::exp_scaled(x[k] - most, a.c);
    }
    if (tail0 + tid < a.cols) total += Num<T>::exp_scaled(zr[tail0 + tid] - most, a.c);
    total = block_reduce<T, BT, false>(total, red[1]);
    const T wt = w * static_cast<T>(a.temperature), f = wt / total;
    for (int v = tid; v < nvec; v += BT) {
        V x = reinterpret_cast<const V *>(zr)[v];
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] = Num<T>::exp_scaled(x[k] - most, a.c) * f;
        reinterpret_cast<V *>(gr)[v] = x;
    }
    if (tail0 + tid < a.cols) gr[tail0 + tid] = Num<T>::exp_scaled(zr[tail0 + tid] - most, a.c) * f;
    if (tid < 64) {
        const double loss = slots_loss(a, lane, slots, most, total);
        if (tid == 0) a.row_loss[row] = static_cast<double>(w) * loss;
    }
    __syncthreads();  // the gradient's bulk comes first, the teacher's columns are written over it
    for (int j = tid; j < a.top; j += BT)
        if (slots.index[j] >= 0)
            gr[slots.index[j]] = Num<T>::exp_scaled(slots.z[j] - most, a.c) * f - wt * slot_share(slots, a.top, j);
}

// loss = sum of the rows' losses: a lane adds every 1024th, the lanes are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) distill_sum_kernel(const double *row_loss, int64_t rows, T *out) {
    __shared__ double red[16];
    double v = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) v += row_loss[r];
    v = block_reduce<double, 1024, false>(v, red);
    if (threadIdx.x == 0) out[0] = static_cast<T>(v);
}

template <typename T>
ttamd_status launch_distill(int64_t rows, int64_t cols, int64_t top, const void *input, int64_t input_row_stride, const void *index,
                            bool index64, const void *teacher, const void *weight, double temperature, void *loss_out, void *grad_out,
                            void *workspace, hipStream_t st) {
    if (rows > 0) {
        DistillArgs<T> a{};
        a.z = static_cast<const T *>(input);
        a.z_row = input_row_stride;
        a.index = index;
        a.index64 = index64;
        a.teacher = static_cast<const T *>(teacher);
        a.weight = static_cast<const T *>(weight);
        a.grad = static_cast<T *>(grad_out);
        a.row_loss = static_cast<double *>(workspace);
        a.rows = rows;
        a.cols = static_cast<int>(cols);
        a.top = static_cast<int>(top);
        a.temperature = temperature;
        a.c = static_cast<T>(sizeof(T) == 4 ? 1.4426950408889634 / temperature : 1.0 / temperature);
        a.uniform_weight = static_cast<T>(1.0 / static_cast<double>(rows));
        distill_row_kernel<T, 256><<<dim3(static_cast<unsigned>(rows)), 256, 0, st>>>(a);
        TTAMD_HIP_CHECK(hipGetLastError());
    }
    distill_sum_kernel<T><<<1, 1024, 0, st>>>(static_cast<const double *>(workspace), rows, static_cast<T *>(loss_out));
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

ttamd_status check_distill_shape(ttamd_dtype dtype, int64_t rows, int64_t cols, int64_t top) {
    if (dtype != TTAMD_F32 && dtype != TTAMD_F64) {
        set_error("distill_loss: floating point dtypes only");
        return TTAMD_ERR_UNSUPPORTED_DTYPE;
    }
    if (rows < 0 || cols < 1 || top < 1 || rows > 0x7fffffffLL || cols > 0x3fffffffLL || top > kMaxTop) {
        set_error("distill_loss: rows %lld, cols %lld, top %lld: fewer than 2^31 rows, 1 to 2^30 - 1 columns, 1 to %d teacher slots",
                  static_cast<long long>(rows), static_cast<long long>(cols), static_cast<long long>(top), kMaxTop);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    return TTAMD_OK;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" {

ttamd_status ttamd_distill_loss_workspace(ttamd_dtype dtype, int64_t rows, int64_t cols, int64_t top, size_t *bytes) {
    if (ttamd_status s = check_distill_shape(dtype, rows, cols, top)) return s;
    if (!bytes) {
        set_error("distill_loss: bytes is NULL");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    *bytes = static_cast<size_t>(rows) * sizeof(double);
    return TTAMD_OK;
}

ttamd_status ttamd_distill_loss(int device, ttamd_dtype dtype, ttamd_dtype index_dtype, int64_t rows, int64_t cols, int64_t top,
                                const void *input, int64_t input_row_stride, const void *teacher_index, const void *teacher_logit,
                                const void *row_weight, double temperature, void *loss_out, void *grad_input_out, void *workspace,
                                size_t workspace_bytes, void *stream) {
    size_t need = 0;
    if (ttamd_status s = ttamd_distill_loss_workspace(dtype, rows, cols, top, &need)) return s;
    if (index_dtype != TTAMD_I32 && index_dtype != TTAMD_I64) {
        set_error("distill_loss: teacher indices are i32 or i64 (dtype code %d)", static_cast<int>(index_dtype));
        return TTAMD_ERR_UNSUPPORTED_DTYPE;
    }
    if (!(temperature > 0) || !(temperature <= 1e30) || !(1 / temperature <= 1e30)) {
        set_error("distill_loss: temperature %g: expected a positive number between 1e-30 and 1e30", temperature);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    const size_t e = dtype_size(dtype), ie = dtype_size(index_dtype);
    if (rows > 0 && (input_row_stride < cols || input_row_stride > (int64_t(1) << 62) / rows / 8)) {
        set_error("distill_loss: row stride %lld of a matrix of %lld columns", static_cast<long long>(input_row_stride), static_cast<long long>(cols));
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (!loss_out || (rows > 0 && (!input || !teacher_index || !teacher_logit || !grad_input_out || !workspace))) {
        set_error("distill_loss: NULL data pointer");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(input, e) || misaligned(teacher_logit, e) || misaligned(row_weight, e) || misaligned(loss_out, e) ||
        misaligned(grad_input_out, e) || misaligned(teacher_index, ie) || misaligned(workspace, sizeof(double))) {
        set_error("distill_loss: pointers must be aligned to the element size, the workspace to 8 bytes");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (workspace_bytes < need) {
        set_error("distill_loss: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (rows > 0 && overlap(input, static_cast<size_t>((rows - 1) * input_row_stride + cols) * e, grad_input_out, static_cast<size_t>(rows * cols) * e)) {
        set_error("distill_loss: the gradient may not be written over the logits");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (ttamd_status s = use_device(device)) return s;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == TTAMD_F32)
        return launch_distill<float>(rows, cols, top, input, input_row_stride, teacher_index, index_dtype == TTAMD_I64, teacher_logit,
                                     row_weight, temperature, loss_out, grad_input_out, workspace, st);
    return launch_distill<double>(rows, cols, top, input, input_row_stride, teacher_index, index_dtype == TTAMD_I64, teacher_logit, row_weight,
                                  temperature, loss_out, grad_input_out, workspace, st);
}

}  // extern "C"
