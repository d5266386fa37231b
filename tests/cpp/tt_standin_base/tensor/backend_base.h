// backend_base.h — test-side stand-in for the reference's tinytensor/tensor/backend_base.h, for building
// test_adapter_amd where the reference tree is not present: an abstract class with a pure virtual for each member that
// backend_amd.h overrides, so that the adapter's code is compiled and called through a base reference.  It pins nothing
// about the reference's interface (tests/test_adapter_signatures.py does, where the tree is present).
#ifndef TT_STANDIN_BACKEND_BASE_H_
#define TT_STANDIN_BACKEND_BASE_H_

#include <tt/device.h>
#include <tt/random.h>
#include <tt/scalar.h>
#include <tt/tensor.h>

#include "tensor/storage_base.h"

#include <cstddef>
#include <cstdint>
#include <memory>
#include <optional>
#include <ostream>
#include <tuple>
#include <utility>
#include <vector>

namespace tinytensor {

// ---- signature families --------------------------------------------------------------------------------------
// element types of from_vec / to_vec (bool has only the const-reference from_vec: it is stored as uint8_t)
#define TT_BASE_VEC_TYPES(X) X(uint8_t) X(int16_t) X(int32_t) X(int64_t) X(float) X(double)

// Tensor f(const Tensor &tensor)
#define TT_BASE_TENSOR_TO_TENSOR(X)                                                                                     \
    X(min) X(argmin) X(max) X(argmax) X(sum)                                                                           \
    X(identity) X(negate) X(logical_not) X(abs) X(sign) X(log) X(log10) X(log2) X(log1p) X(exp) X(exp2) X(expm1)       \
    X(sqrt) X(sin) X(cos) X(tan) X(asin) X(acos) X(atan) X(sinh) X(cosh) X(tanh) X(asinh) X(acosh) X(atanh) X(erf)     \
    X(erfc) X(tgamma) X(lgamma) X(digamma) X(ceil) X(floor) X(round) X(isinf) X(isnan) X(isfinite)                     \
    X(sigmoid) X(log_sigmoid) X(hardsigmoid) X(relu) X(relu6) X(selu) X(silu) X(softsign)

// void f_(Tensor &tensor)
#define TT_BASE_TENSOR_INPLACE(X)                                                                                       \
    X(identity_) X(negate_) X(logical_not_) X(abs_) X(sign_) X(log_) X(log10_) X(log2_) X(log1p_) X(exp_) X(exp2_)     \
    X(expm1_) X(sqrt_) X(sin_) X(cos_) X(tan_) X(asin_) X(acos_) X(atan_) X(sinh_) X(cosh_) X(tanh_) X(asinh_)         \
    X(acosh_) X(atanh_) X(erf_) X(erfc_) X(tgamma_) X(lgamma_) X(digamma_) X(ceil_) X(floor_) X(round_)                \
    X(sigmoid_) X(log_sigmoid_) X(hardsigmoid_) X(relu_) X(relu6_) X(selu_) X(silu_) X(softsign_)

// Tensor f(const Tensor &lhs, const Tensor &rhs)
#define TT_BASE_BINARY(X)                                                                                               \
    X(eq) X(ne) X(lt) X(le) X(gt) X(ge) X(logical_or) X(logical_and) X(bitwise_or) X(bitwise_and) X(bitwise_xor)       \
    X(bitwise_left_shift) X(bitwise_right_shift) X(modulo) X(add) X(sub) X(mul) X(div) X(maximum) X(minimum) X(pow)    \
    X(batched_matmul)

// void f(Tensor &lhs, const Tensor &rhs)
#define TT_BASE_BINARY_INPLACE(X) X(assign) X(add_inplace) X(sub_inplace) X(mul_inplace) X(div_inplace)

// Tensor f(const Tensor &tensor, int dim)
#define TT_BASE_TENSOR_DIM(X) X(min) X(argmin) X(max) X(argmax) X(sum) X(all) X(any) X(softmax) X(log_softmax)

// distributions: Tensor f(const Tensor &a, [const Tensor &b,] Generator &gen) and the in-place forms
#define TT_BASE_DIST_ONE(X) X(bernoulli, p) X(geometric, p) X(poisson, lambda) X(exponential, lambda)
#define TT_BASE_DIST_TWO(X)                                                                                             \
    X(uniform_int, low, high) X(uniform_real, low, high) X(binomial, p, num_draws) X(normal, mu, std)                  \
    X(cauchy, loc, scale) X(lognormal, mu, std) X(weibull, scale, shape)

// pooling: Tensor f(input, kernel_size, stride, padding) and Tensor f_backward(grad_output, input, result, ...)
#define TT_BASE_POOLS(X) X(max_pool2d) X(min_pool2d) X(avg_pool2d)

class BackendBase {
public:
    using StoragePtr = std::unique_ptr<StorageBase>;
    virtual ~BackendBase() = default;

    // Tensor construction
    [[nodiscard]] virtual auto from_vec(const std::vector<bool> &data, int device_id) const -> StoragePtr = 0;
#define X(T)                                                                                        \
    [[nodiscard]] virtual auto from_vec(const std::vector<T> &data, int device_id) const -> StoragePtr = 0; \
    [[nodiscard]] virtual auto from_vec(std::vector<T> &&data, int device_id) const -> StoragePtr = 0;
    TT_BASE_VEC_TYPES(X)
#undef X
    [[nodiscard]] virtual auto from_scalar(Scalar scalar, int device_id) const -> StoragePtr = 0;
    [[nodiscard]] virtual auto full(const Scalar &value, std::size_t N, int device_id) const -> StoragePtr = 0;
    [[nodiscard]] virtual auto arange(std::size_t N, ScalarType dtype, int device_id) const -> StoragePtr = 0;

    // Conversion to vec
#define X(T) virtual void to_vec(const Tensor &tensor, std::vector<T> &data_out) const = 0;
    TT_BASE_VEC_TYPES(X)
#undef X

    // Getters
    [[nodiscard]] virtual auto item(const Tensor &tensor) const -> Scalar = 0;
    [[nodiscard]] virtual auto data_ptr(const Tensor &tensor) const -> uintptr_t = 0;

    // Indexing
    [[nodiscard]] virtual auto index_mask(const Tensor &input, const Tensor &mask, int N_mask) const -> Tensor = 0;
    [[nodiscard]] virtual auto index_indices(const Tensor &input, const Tensor &indices) const -> Tensor = 0;
    virtual void index_put_mask(Tensor &input, const Tensor &values, const Tensor &mask) const = 0;
    virtual void index_put_indices(Tensor &input, const Tensor &values, const Tensor &indices) const = 0;
    [[nodiscard]] virtual auto gather(const Tensor &input, const Tensor &indices, int idx) const -> Tensor = 0;

    // Casts, printing
    [[nodiscard]] virtual auto to(const Tensor &tensor, ScalarType dtype) const -> Tensor = 0;
    virtual auto print(std::ostream &os, const Tensor &tensor) const -> std::ostream & = 0;

    // Distributions
#define X(NAME, A)                                                                                 \
    [[nodiscard]] virtual auto NAME(const Tensor &A, Generator &gen) const -> Tensor = 0;            \
    virtual void NAME##_(Tensor &tensor, const Tensor &A, Generator &gen) const = 0;
    TT_BASE_DIST_ONE(X)
#undef X
#define X(NAME, A, B)                                                                              \
    [[nodiscard]] virtual auto NAME(const Tensor &A, const Tensor &B, Generator &gen) const -> Tensor = 0; \
    virtual void NAME##_(Tensor &tensor, const Tensor &A, const Tensor &B, Generator &gen) const = 0;
    TT_BASE_DIST_TWO(X)
#undef X

    // Binary operators (batched_matmul among them), their in-place forms and assign
#define X(NAME) [[nodiscard]] virtual auto NAME(const Tensor &lhs, const Tensor &rhs) const -> Tensor = 0;
    TT_BASE_BINARY(X)
#undef X
#define X(NAME) virtual void NAME(Tensor &lhs, const Tensor &rhs) const = 0;
    TT_BASE_BINARY_INPLACE(X)
#undef X

    // Reductions, unary operators and activations
#define X(NAME) [[nodiscard]] virtual auto NAME(const Tensor &tensor) const -> Tensor = 0;
    TT_BASE_TENSOR_TO_TENSOR(X)
#undef X
#define X(NAME) [[nodiscard]] virtual auto NAME(const Tensor &tensor, int dim) const -> Tensor = 0;
    TT_BASE_TENSOR_DIM(X)
#undef X
    [[nodiscard]] virtual auto all(const Tensor &tensor) const -> bool = 0;
    [[nodiscard]] virtual auto any(const Tensor &tensor) const -> bool = 0;
#define X(NAME) virtual void NAME(Tensor &tensor) const = 0;
    TT_BASE_TENSOR_INPLACE(X)
#undef X
    [[nodiscard]] virtual auto softplus(const Tensor &tensor, double beta, double threshold) const -> Tensor = 0;
    [[nodiscard]] virtual auto leaky_relu(const Tensor &tensor, double negative_slope) const -> Tensor = 0;
    [[nodiscard]] virtual auto elu(const Tensor &tensor, double alpha) const -> Tensor = 0;
    [[nodiscard]] virtual auto hardtanh(const Tensor &tensor, double min, double max) const -> Tensor = 0;
    virtual void softplus_(Tensor &tensor, double beta, double threshold) const = 0;
    virtual void leaky_relu_(Tensor &tensor, double negative_slope) const = 0;
    virtual void elu_(Tensor &tensor, double alpha) const = 0;
    virtual void hardtanh_(Tensor &tensor, double min, double max) const = 0;
    virtual void softmax_(Tensor &tensor, int dim) const = 0;
    virtual void log_softmax_(Tensor &tensor, int dim) const = 0;

    // Util/misc
    [[nodiscard]] virtual auto where(const Tensor &cond, const Tensor &lhs, const Tensor &rhs) const -> Tensor = 0;
    virtual void clamp_(Tensor &tensor, const Tensor &min, const Tensor &max) const = 0;

    // Convolution and pooling
    [[nodiscard]] virtual auto conv2d(
        const Tensor &input,
        const Tensor &weight,
        const std::optional<Tensor> &bias,
        int stride,
        int padding
    ) const -> Tensor = 0;
    [[nodiscard]] virtual auto conv2d_backward(
        const Tensor &grad_output,
        const Tensor &input,
        const Tensor &weight,
        const std::optional<Tensor> &bias,
        int stride,
        int padding
    ) const -> std::tuple<Tensor, Tensor, std::optional<Tensor>> = 0;
#define X(NAME)                                                                                                    \
    [[nodiscard]] virtual auto NAME(const Tensor &input, int kernel_size, int stride, int padding) const -> Tensor = 0; \
    [[nodiscard]] virtual auto NAME##_backward(                                                                            \
        const Tensor &grad_output,                                                                                 \
        const Tensor &input,                                                                                       \
        const Tensor &result,                                                                                      \
        int kernel_size,                                                                                           \
        int stride,                                                                                                \
        int padding                                                                                                \
    ) const -> Tensor = 0;
    TT_BASE_POOLS(X)
#undef X

    // Memory counters and devices
    [[nodiscard]] virtual auto current_memory_allocated(int device_id) const -> uint64_t = 0;
    [[nodiscard]] virtual auto total_memory_allocated(int device_id) const -> uint64_t = 0;
    [[nodiscard]] virtual auto get_device_count() const -> int = 0;
};


#undef TT_BASE_BINARY
#undef TT_BASE_BINARY_INPLACE
#undef TT_BASE_DIST_ONE
#undef TT_BASE_DIST_TWO
#undef TT_BASE_POOLS
#undef TT_BASE_TENSOR_DIM
#undef TT_BASE_TENSOR_INPLACE
#undef TT_BASE_TENSOR_TO_TENSOR
#undef TT_BASE_VEC_TYPES

}  // namespace tinytensor

#endif  // TT_STANDIN_BACKEND_BASE_H_
