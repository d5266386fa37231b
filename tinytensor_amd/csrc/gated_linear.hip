// gated_linear.hip — the gated pair of Linear layers of a feed-forward block, forward and backward (gfx950).
//
//   g = x . Wg + bg,  u = x . Wu + bu,  h = act(g) * u                          act: silu, gelu (erf), relu, sigmoid
//   dg = dh * u * act'(g),  du = dh * act(g),  dx = dg . Wg^T + du . Wu^T,  dW = x^T . d{g,u},  db = column sums of d{g,u}
// No counterpart in the reference; it stands beside nn::Linear (nn/linear.cpp:42-50) followed by an activation.
//
// Bound: the matrix cores for many rows (4 and 8 rows x inner x hidden flop), HBM (the weights) for a few.
#include "common.h"

namespace ttamd {
namespace {

constexpr int kSilu = 0, kGelu = 1, kRelu = 2, kSigmoid = 3;

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

// act(g) and act'(g).  relu's derivative is where(g < 0, 0, 1), as TensorRelu::backward has it (autograd/unary_ops.cpp:568-573).
template <typename T, int ACT>
__device__ __forceinline__ T activate(T g) {
    if constexpr (ACT == kRelu) return g > T(0) ? g : T(0);
    if constexpr (ACT == kGelu) return g * normal_cdf(g);
    const T s = sigmoid(g);
    return ACT == kSigmoid ? s : g * s;
}
template <typename T, int ACT>
__device__ __forceinline__ void activate(T g, T &value, T &slope) {
    if constexpr (ACT == kRelu) {
        value = g > T(0) ? g : T(0);
        slope = g < T(0) ? T(0) : T(1);
    } else if constexpr (ACT == kGelu) {
        const T cdf = normal_cdf(g);
        value = g * cdf;
        slope = cdf + g * (T(0.3989422804014327) * (sizeof(T) == 4 ? static_cast<T>(expf(static_cast<float>(T(-0.5) * g * g))) : static_cast<T>(exp(T(-0.5) * g * g))));
    } else {
        const T s = sigmoid(g);
        value = ACT == kSigmoid ? s : g * s;
        slope = ACT == kSigmoid ? s * (T(1) - s) : s * (T(1) + g * (T(1) - s));
    }
}

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

// dg = dh * u * act'(g) and du = dh * act(g) over n elements.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256) gated_slope_kernel(const T *__restrict__ dh, const T *__restrict__ gate, const T *__restrict__ up,
                                                          T *__restrict__ dg, T *__restrict__ du, int64_t n) {
    using V = typename VecOf<T>::type;
    constexpr int W = VEC ? VecOf<T>::W : 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, whole = n / W;
    const auto one = [&](int64_t i) {
        T value, slope;
        activate<T, ACT>(gate[i], value, slope);
        const T d = dh[i];
        dg[i] = d * up[i] * slope;
        du[i] = d * value;
    };
    for (int64_t i = first; i < whole; i += step) {
        if constexpr (VEC) {
            const V d = reinterpret_cast<const V *>(dh)[i], g = reinterpret_cast<const V *>(gate)[i], u = reinterpret_cast<const V *>(up)[i];
            V a, b;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                T value, slope;
                activate<T, ACT>(g[k], value, slope);
                a[k] = d[k] * u[k] * slope;
                b[k] = d[k] * value;
            }
            reinterpret_cast<V *>(dg)[i] = a;
            reinterpret_cast<V *>(du)[i] = b;
        } else {
            one(i);
        }
    }
    if (VEC && first < n - whole * W) one(whole * W + first);
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

template <typename T>
ttamd_status launch_slope(int act, const void *dh, const void *gate, const void *up, void *dg, void *du, int64_t n, hipStream_t st) {
    if (n == 0) return TTAMD_OK;
    const bool vec = aligned16({dh, gate, up, dg, du});
    const unsigned blocks = stream_blocks(vec ? n / VecOf<T>::W : n);
    for_activation(act, [&]<int ACT>() {
        const auto *d = static_cast<const T *>(dh), *g = static_cast<const T *>(gate), *u = static_cast<const T *>(up);
        if (vec) gated_slope_kernel<T, ACT, true><<<blocks, 256, 0, st>>>(d, g, u, static_cast<T *>(dg), static_cast<T *>(du), n);
        else gated_slope_kernel<T, ACT, false><<<blocks, 256, 0, st>>>(d, g, u, static_cast<T *>(dg), static_cast<T *>(du), n);
    });
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

struct GatedSizes {
    size_t item, hidden_matrix;  // bytes of an element; of a [rows, hidden] matrix, rounded up to 256
};

ttamd_status check_gated(const char *what, ttamd_dtype dtype, int64_t rows, int64_t inner, int64_t hidden, GatedSizes *out) {
    if (dtype != TTAMD_F32 && dtype != TTAMD_F64) {
        set_error("%s: floating point dtypes only", what);
        return TTAMD_ERR_UNSUPPORTED_DTYPE;
    }
    constexpr int64_t most = 0x7fffffffLL;
    if (rows < 0 || inner < 1 || hidden < 1 || rows > most || inner > most || hidden > most) {
        set_error("%s: rows %lld, inner %lld, hidden %lld: rows from 0, the others from 1, all below 2^31", what, static_cast<long long>(rows),
                  static_cast<long long>(inner), static_cast<long long>(hidden));
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    out->item = dtype_size(dtype);
    out->hidden_matrix = (static_cast<size_t>(rows) * static_cast<size_t>(hidden) * out->item + 255) / 256 * 256;
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
    if (v->offset < 0 || v->stride[0] < 0 || v->stride[1] < 0 || misaligned(v->data, item)) {
        set_error("%s: %s: negative offset or stride, or a pointer off the element size", what, name);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    return TTAMD_OK;
}

ttamd_view3 lift(const ttamd_view2 &v) { return {v.data, v.offset, {0, v.stride[0], v.stride[1]}}; }
ttamd_view3 lift_transposed(const ttamd_view2 &v) { return {v.data, v.offset, {0, v.stride[1], v.stride[0]}}; }

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" {

ttamd_status ttamd_gated_linear_workspace(ttamd_dtype dtype, int64_t rows, int64_t inner, int64_t hidden, int backward, size_t *bytes) {
    GatedSizes z;
    if (ttamd_status s = check_gated("gated_linear", dtype, rows, inner, hidden, &z)) return s;
    if (!bytes) {
        set_error("gated_linear: bytes is NULL");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    *bytes = 2 * z.hidden_matrix;  // g and u, or dg and du
    return TTAMD_OK;
}

ttamd_status ttamd_gated_linear_forward(int device, ttamd_dtype dtype, int activation, int64_t rows, int64_t inner, int64_t hidden,
                                        const ttamd_view2 *input, const ttamd_view2 *gate_weight, const ttamd_view2 *up_weight,
                                        const void *gate_bias, const void *up_bias, void *out, void *gate_out, void *up_out, void *workspace,
                                        size_t workspace_bytes, void *stream) {
    const char *const what = "gated_linear";
    GatedSizes z;
    if (ttamd_status s = check_gated(what, dtype, rows, inner, hidden, &z)) return s;
    if (ttamd_status s = check_activation(what, activation)) return s;
    const bool work = rows > 0;
    if (ttamd_status s = check_view(what, "input", input, z.item, work)) return s;
    if (ttamd_status s = check_view(what, "gate weight", gate_weight, z.item, work)) return s;
    if (ttamd_status s = check_view(what, "up weight", up_weight, z.item, work)) return s;
    if (work && (!out || (!workspace && !(gate_out && up_out)))) {
        set_error("%s: NULL data pointer", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (!gate_out != !up_out) {
        set_error("%s: gate_out and up_out are given together or not at all", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(out, z.item) || misaligned(gate_out, z.item) || misaligned(up_out, z.item) || misaligned(gate_bias, z.item) ||
        misaligned(up_bias, z.item) || misaligned(workspace, 16)) {
        set_error("%s: pointers must be aligned to the element size, the workspace to 16 bytes", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (workspace_bytes < 2 * z.hidden_matrix && !gate_out) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, 2 * z.hidden_matrix);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (ttamd_status s = use_device(device)) return s;
    if (!work) return TTAMD_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    void *g = gate_out ? gate_out : workspace;
    void *u = up_out ? up_out : static_cast<char *>(workspace) + z.hidden_matrix;
    const int R = static_cast<int>(rows), K = static_cast<int>(inner), H = static_cast<int>(hidden);
    const ttamd_view3 x = lift(*input), wg = lift(*gate_weight), wu = lift(*up_weight);
    ttamd_epilogue eg{}, eu{};
    eg.bias = gate_bias;
    eg.bias_mode = gate_bias ? 1 : 0;
    eu.bias = up_bias;
    eu.bias_mode = up_bias ? 1 : 0;
    if (ttamd_status s = ttamd_batched_matmul(device, dtype, 1, R, K, H, &x, &wg, g, &eg, stream)) return s;
    if (ttamd_status s = ttamd_batched_matmul(device, dtype, 1, R, K, H, &x, &wu, u, &eu, stream)) return s;
    const int64_t n = rows * hidden;
    return dtype == TTAMD_F32 ? launch_product<float>(activation, g, u, out, n, st) : launch_product<double>(activation, g, u, out, n, st);
}

ttamd_status ttamd_gated_linear_backward(int device, ttamd_dtype dtype, int activation, int64_t rows, int64_t inner, int64_t hidden,
                                         const void *grad_out, const ttamd_view2 *input, const ttamd_view2 *gate_weight,
                                         const ttamd_view2 *up_weight, const void *gate, const void *up, void *grad_input,
                                         void *grad_gate_weight, void *grad_up_weight, void *grad_gate_bias, void *grad_up_bias,
                                         void *workspace, size_t workspace_bytes, void *stream) {
    const char *const what = "gated_linear_backward";
    GatedSizes z;
    if (ttamd_status s = check_gated(what, dtype, rows, inner, hidden, &z)) return s;
    if (ttamd_status s = check_activation(what, activation)) return s;
    const bool work = rows > 0;
    if (ttamd_status s = check_view(what, "input", input, z.item, work)) return s;
    if (ttamd_status s = check_view(what, "gate weight", gate_weight, z.item, work)) return s;
    if (ttamd_status s = check_view(what, "up weight", up_weight, z.item, work)) return s;
    if (!grad_gate_weight || !grad_up_weight || (work && (!grad_out || !gate || !up || !grad_input || !workspace))) {
        set_error("%s: NULL data pointer", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    for (const void *p : {grad_out, gate, up, static_cast<const void *>(grad_input), static_cast<const void *>(grad_gate_weight),
                          static_cast<const void *>(grad_up_weight), static_cast<const void *>(grad_gate_bias), static_cast<const void *>(grad_up_bias)})
        if (misaligned(p, z.item)) {
            set_error("%s: pointers must be aligned to the element size", what);
            return TTAMD_ERR_INVALID_ARGUMENT;
        }
    if (work && (misaligned(workspace, 16) || workspace_bytes < 2 * z.hidden_matrix)) {
        set_error("%s: workspace of %zu bytes, %zu needed, aligned to 16", what, workspace_bytes, 2 * z.hidden_matrix);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (ttamd_status s = use_device(device)) return s;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int R = static_cast<int>(rows), K = static_cast<int>(inner), H = static_cast<int>(hidden);
    void *dg = workspace, *du = static_cast<char *>(workspace) + z.hidden_matrix;
    const int64_t n = rows * hidden;
    if (ttamd_status s = dtype == TTAMD_F32 ? launch_slope<float>(activation, grad_out, gate, up, dg, du, n, st)
                                            : launch_slope<double>(activation, grad_out, gate, up, dg, du, n, st))
        return s;
    // dx = dg . Wg^T, then += du . Wu^T; each weight's gradient with its bias gradient (no rows: zeros)
    const ttamd_view3 vg{dg, 0, {n, hidden, 1}}, vu{du, 0, {n, hidden, 1}};
    const ttamd_view3 xt = lift_transposed(*input), wgt = lift_transposed(*gate_weight), wut = lift_transposed(*up_weight);
    ttamd_epilogue add{}, eg{}, eu{};
    add.accumulate = 1;
    eg.rhs_colsum_out = grad_gate_bias;
    eu.rhs_colsum_out = grad_up_bias;
    if (work) {
        if (ttamd_status s = ttamd_batched_matmul(device, dtype, 1, R, H, K, &vg, &wgt, grad_input, nullptr, stream)) return s;
        if (ttamd_status s = ttamd_batched_matmul(device, dtype, 1, R, H, K, &vu, &wut, grad_input, &add, stream)) return s;
    }
    if (ttamd_status s = ttamd_batched_matmul(device, dtype, 1, K, R, H, &xt, &vg, grad_gate_weight, &eg, stream)) return s;
    return ttamd_batched_matmul(device, dtype, 1, K, R, H, &xt, &vu, grad_up_weight, &eu, stream);
}

}  // extern "C"
