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
constexpr int kLdsVecs = 8;    // vectors a lane may keep in LDS: 128 KB of the 160 KB for 1024 lanes, beside 20 KB of slots

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
    double *row_loss;     // [rows] scratch, or a place for the four rows of a wave
    T *loss;              // a launch of one workgroup writes the loss itself; null: distill_sum_kernel does
    int64_t rows, row0;   // row0: first row of the launch
    int cols, top, index64;
    double temperature;
    T c;                  // factor of exp_scaled: log2(e) / T for float, 1 / T for double
    T uniform_weight;
};

// What a row's slots come to, in LDS.  p is 0 in a slot that does not count: an index outside the columns, a logit of -inf.
// The arrays are padded to whole vectors with slots of no column.
template <typename T>
struct Slots {
    T *p, *z;
    int *index;
    static constexpr __host__ __device__ int64_t padded(int64_t top) { return (top + 3) / 4 * 4; }
    static size_t bytes(int64_t top) { return static_cast<size_t>(padded(top)) * (2 * sizeof(T) + sizeof(int)); }
    __device__ __forceinline__ Slots(void *lds, int top) : p(static_cast<T *>(lds)), z(p + padded(top)), index(reinterpret_cast<int *>(z + padded(top))) {}
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

// The slots in three steps, each lane with every BT-th of them, between the row's own reductions: what the indices, the
// teacher's and the student's logits are (returns the lane's largest teacher logit, NaN if one is NaN); the exponentials
// (returns their sum); the probabilities (returns T^2 sum_j p_j (log p_j - log q_j) with log q_j = (z_j - m) / T - log(total),
// terms and sum in 64 bits).
template <typename T, int BT>
__device__ __forceinline__ T slots_read(const DistillArgs<T> &a, int64_t row, const Slots<T> &s) {
    const T *zr = a.z + row * a.z_row;
    T most = Num<T>::neg_inf();
    bool nan = false;
    for (int j = threadIdx.x; j < Slots<T>::padded(a.top); j += BT) {
        const int i = j < a.top ? slot_index(a, row, j) : -1;
        const T t = i >= 0 ? a.teacher[row * a.top + j] : Num<T>::neg_inf();
        s.index[j] = i;
        s.p[j] = t;
        s.z[j] = i >= 0 ? zr[i] : T(0);
        most = Num<T>::max_(most, t);
        nan = nan || t != t;
    }
    return __any(nan) ? T(__builtin_nan("")) : wave_max(most);
}
template <typename T, int BT>
__device__ __forceinline__ T slots_exp(const DistillArgs<T> &a, const Slots<T> &s, T most) {
    T sum = T(0);
    for (int j = threadIdx.x; j < Slots<T>::padded(a.top); j += BT) {
        const T e = s.index[j] >= 0 ? Num<T>::exp_scaled(s.p[j] - most, a.c) : T(0);
        s.p[j] = e;
        sum += e;
    }
    return wave_sum(sum);
}
template <typename T, int BT>
__device__ __forceinline__ double slots_loss(const DistillArgs<T> &a, const Slots<T> &s, T sum, T most, double total) {
    const double inv = 1.0 / a.temperature, log_total = log(total);
    double loss = 0;
    for (int j = threadIdx.x; j < Slots<T>::padded(a.top); j += BT) {
        const T pj = s.p[j] / sum;
        s.p[j] = pj;
        const double p = s.index[j] >= 0 ? static_cast<double>(pj) : 0.0;
        if (p != 0.0) loss += p * (log(p) - ((static_cast<double>(s.z[j]) - static_cast<double>(most)) * inv - log_total));  // (p = 0: the term is 0 whatever q is)
    }
    return a.temperature * a.temperature * wave_sum(loss);
}

// The waves' values put together: largest (a NaN among them wins) or sum, in wave order.  `lds`: a place a wave.
template <typename T, int NW, bool MAX>
__device__ __forceinline__ T join_waves(const T *lds) {
    T r = lds[0];
    bool nan = r != r;
#pragma unroll
    for (int i = 1; i < NW; ++i) {
        if constexpr (MAX) {
            nan = nan || lds[i] != lds[i];
            r = Num<T>::max_(r, lds[i]);
        } else {
            r += lds[i];
        }
    }
    return MAX && nan ? T(__builtin_nan("")) : r;
}

// The teacher's columns of the gradient, over its bulk: w T (q - the p of all slots with this column, which a teacher may name
// twice).  Neighbouring lanes share a slot (as many as there are lanes for it, up to 16): each adds up a stretch of the
// slots, four a step, and the stretches are added in a fixed tree.
template <typename T, int BT>
__device__ __forceinline__ void write_slots(const DistillArgs<T> &a, const Slots<T> &s, T *grad, T most, T f, T wt, int c0, int c1, int c2) {
    typedef int idx4 __attribute__((ext_vector_type(4)));
    typedef T val4 __attribute__((ext_vector_type(4), aligned(16)));
    const int padded = static_cast<int>(Slots<T>::padded(a.top));
    int share = 1;
    while (share < 16 && 2 * share * a.top <= BT) share *= 2;
    const int stretch = (padded / 4 + share - 1) / share * 4, part = threadIdx.x & (share - 1);
    const int k0 = part * stretch, k1 = k0 + stretch < padded ? k0 + stretch : padded;
    for (int j0 = 0; j0 < a.top; j0 += BT / share) {  // (every lane takes part in the shuffles)
        const int j = j0 + threadIdx.x / share;
        const int i = j < a.top ? s.index[j] : -1;
        T sum = T(0);
        for (int k = k0; k < k1; k += 4) {
            const idx4 at = *reinterpret_cast<const idx4 *>(s.index + k);
            const val4 p = *reinterpret_cast<const val4 *>(s.p + k);
#pragma unroll
            for (int u = 0; u < 4; ++u) sum += at[u] == i ? p[u] : T(0);
        }
        for (int d = 1; d < share; d *= 2) sum += __shfl_xor(sum, d, 64);
        // columns of this workgroup: [c0, c1) and those from c2 on
        if (part == 0 && i >= 0 && ((i >= c0 && i < c1) || i >= c2)) grad[i] = Num<T>::exp_scaled(s.z[j] - most, a.c) * f - wt * sum;
    }
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

// One lane leaves a row's loss (the whole loss where there is one row).
template <typename T>
__device__ __forceinline__ void leave_loss(const DistillArgs<T> &a, int64_t row, double loss) {
    if (a.loss) a.loss[0] = static_cast<T>(loss);
    else a.row_loss[row] = loss;
}

// A row that weighs nothing, or whose slots are all empty: no loss, a gradient of zeros.
template <typename T, int BT>
__device__ __forceinline__ void empty_row(const DistillArgs<T> &a, int64_t row) {
    using V = typename Num<T>::vec_t;
    constexpr int W = Num<T>::W;
    T *gr = a.grad + row * a.cols;
    const int nvec = a.cols / W;
    V zero;
#pragma unroll
    for (int k = 0; k < W; ++k) zero[k] = T(0);
    for (int v = threadIdx.x; v < nvec; v += BT) reinterpret_cast<V *>(gr)[v] = zero;
    for (int i = nvec * W + threadIdx.x; i < a.cols; i += BT) gr[i] = T(0);
    if (threadIdx.x == 0) leave_loss(a, row, 0.0);
}

// A workgroup a row.  The row is requested once and stays: NV vectors of it in every lane's registers, `lds_vecs` more in
// the lane's own places in LDS, and only what is beyond both is read again for the sum and for the gradient (a row of
// 131072 floats just fits: 24 vectors in registers, of which the kernel spills 13 registers, and 8 in LDS; of the f64 forms the one
// of 24 vectors spills 42 registers, the one of 1024 lanes and 16 vectors 10).  Columns behind the row's last whole vector go one
// by one.
// NT: loads and stores that leave the caches alone, for matrices that would not stay in them anyway.
// Traffic is the floor's, read once and written once: 2048 x 32000 f32 with 64 slots 94 us (5.6 TB/s; a copy of 2 GiB
// reaches 4.9), 4096 x 131072 870 to 880 us (4.9 TB/s); as three reads and a write these took 199 and 1641 us.  Beyond the chip
// the third read remains: 1024 x 100003 f64 470 us of a floor of 334, 1024 x 151936 f32 279 of 254.
template <typename T, int BT, int NV, bool NT>
__global__ void __launch_bounds__(BT) distill_row_kernel(DistillArgs<T> a, int lds_vecs) {
    using V = typename Num<T>::vec_t;
    typedef T lds_t __attribute__((ext_vector_type(Num<T>::W)));
    constexpr int W = Num<T>::W;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    lds_t *const more = reinterpret_cast<lds_t *>(smem);  // [lds_vecs][BT]
    const Slots<T> slots(smem + static_cast<size_t>(lds_vecs) * BT * sizeof(lds_t), a.top);
    constexpr int NW = BT / 64;
    __shared__ T red[3][NW];
    __shared__ double total_of[NW], loss_of[NW];
    const int64_t row = a.row0 + blockIdx.x;
    const int tid = threadIdx.x, wave = tid / 64;
    const T *zr = a.z + row * a.z_row;
    T *gr = a.grad + row * a.cols;
    const int nvec = a.cols / W, tail = nvec * W + tid;
    const T w = a.weight ? a.weight[row] : a.uniform_weight;
    if (w == T(0)) {  // (the same for the whole workgroup)
        empty_row<T, BT>(a, row);
        return;
    }
    // (before the row is held: with the vectors in registers the longest rows would run out of them)
    const T tmost_wave = slots_read<T, BT>(a, row, slots);
    // Every lane requests its vectors before any is used.  A place behind the row's end repeats the last vector and is set
    // to -inf afterwards, which leaves the maximum alone and adds 0 to the sum: a branch around each load would wait for
    // each load.  (A row shorter than a vector comes here for its many slots; it requests its first column for nothing.)
    V held[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = tid + i * BT;
        if (nvec == 0) {
            held[i] = V{} + zr[0];
            continue;
        }
        const V *at = &reinterpret_cast<const V *>(zr)[v < nvec ? v : nvec - 1];
        if constexpr (NT) held[i] = __builtin_nontemporal_load(at);
        else held[i] = *at;
    }
    T last = tail < a.cols ? zr[tail] : Num<T>::neg_inf();
    const int lds_end = (NV + lds_vecs) * BT < nvec ? (NV + lds_vecs) * BT : nvec;
    T most = last;
    for (int v = NV * BT + tid; v < lds_end; v += BT) {
        const V x = reinterpret_cast<const V *>(zr)[v];
        lds_t y;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            y[k] = x[k];
            most = Num<T>::max_(most, x[k]);
        }
        more[v - NV * BT] = y;
    }
    for (int v = (NV + lds_vecs) * BT + tid; v < nvec; v += BT) {
        const V x = reinterpret_cast<const V *>(zr)[v];
#pragma unroll
        for (int k = 0; k < W; ++k) most = Num<T>::max_(most, x[k]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const bool in = tid + i * BT < nvec;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            held[i][k] = in ? held[i][k] : Num<T>::neg_inf();
            most = Num<T>::max_(most, held[i][k]);
        }
    }
    most = wave_max(most);
    if (tid % 64 == 0) {
        red[0][wave] = most;
        red[1][wave] = tmost_wave;
    }
    __syncthreads();
    most = join_waves<T, NW, true>(red[0]);
    // What is kept on the chip is added up in T, up to 128 exponentials a lane (vector by vector first, the 24-vector form would spill
    // four registers more: 4096 x 131072 f32 880 us against 868); what is beyond in 64 bits, for a lane may have 2^18 vectors there and
    // a running sum in 32 would round that often (2^22 columns, some large, the others just too small to count beside them: 2e-4 of
    // the sum was lost).
    T near = T(0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < W; ++k) {
            held[i][k] = Num<T>::exp_scaled(held[i][k] - most, a.c);
            near += held[i][k];
        }
    for (int v = NV * BT + tid; v < lds_end; v += BT) {
        lds_t x = more[v - NV * BT];
        T sum = T(0);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            x[k] = Num<T>::exp_scaled(x[k] - most, a.c);
            sum += x[k];
        }
        more[v - NV * BT] = x;
        near += sum;
    }
    double total = static_cast<double>(near);
    for (int v = (NV + lds_vecs) * BT + tid; v < nvec; v += BT) {
        const V x = reinterpret_cast<const V *>(zr)[v];
        T sum = T(0);
#pragma unroll
        for (int k = 0; k < W; ++k) sum += Num<T>::exp_scaled(x[k] - most, a.c);
        total += static_cast<double>(sum);
    }
    last = tail < a.cols ? Num<T>::exp_scaled(last - most, a.c) : T(0);
    total += static_cast<double>(last);
    total = wave_sum(total);
    if (tid % 64 == 0) total_of[wave] = total;
    __syncthreads();
    const T tmost = join_waves<T, NW, true>(red[1]);
    if (tmost == Num<T>::neg_inf()) {  // (no slot counts; the same for the whole workgroup)
        empty_row<T, BT>(a, row);
        return;
    }
    total = join_waves<double, NW, false>(total_of);
    const T wt = w * static_cast<T>(a.temperature), f = wt / static_cast<T>(total);
    const auto put = [&](int v, V x) {
        if constexpr (NT) __builtin_nontemporal_store(x, &reinterpret_cast<V *>(gr)[v]);
        else reinterpret_cast<V *>(gr)[v] = x;
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = tid + i * BT;
        if (v < nvec) put(v, held[i] * f);
    }
    for (int v = NV * BT + tid; v < lds_end; v += BT) {
        const lds_t x = more[v - NV * BT];
        V y;
#pragma unroll
        for (int k = 0; k < W; ++k) y[k] = x[k] * f;
        put(v, y);
    }
    for (int v = (NV + lds_vecs) * BT + tid; v < nvec; v += BT) {
        V x = reinterpret_cast<const V *>(zr)[v];
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] = Num<T>::exp_scaled(x[k] - most, a.c) * f;
        put(v, x);
    }
    if (tail < a.cols) gr[tail] = last * f;
    const T tsum_wave = slots_exp<T, BT>(a, slots, tmost);  // (now that the row's vectors have left the registers)
    if (tid % 64 == 0) red[2][wave] = tsum_wave;
    __syncthreads();
    const double loss = slots_loss<T, BT>(a, slots, join_waves<T, NW, false>(red[2]), most, total);
    if (tid % 64 == 0) loss_of[wave] = loss;
    __syncthreads();  // the gradient's bulk comes first, the teacher's columns are written over it
    if (tid == 0) leave_loss(a, row, static_cast<double>(w) * join_waves<double, NW, false>(loss_of));
    write_slots<T, BT>(a, slots, gr, most, f, wt, 0, a.cols, a.cols);
}

// Short rows: G lanes own a row, E columns each (lane l: columns l, l + G, ..), up to 64 slots.  Everything stays in
// registers; the slots go round the group one by one and the lane that holds a slot's column takes its share off.
template <typename T, int G, int E, int BT>
__global__ void __launch_bounds__(BT) distill_short_kernel(DistillArgs<T> a) {
    __shared__ double of_wave[BT / 64];
    constexpr int S = 64 / G;  // slots a lane
    const int64_t row_of = a.row0 + (static_cast<int64_t>(blockIdx.x) * BT + threadIdx.x) / G;
    const bool live = row_of < a.rows;
    const int64_t row = live ? row_of : a.rows - 1;  // (every lane takes part in the shuffles)
    const int lane = threadIdx.x % G;
    const T *zr = a.z + row * a.z_row;
    const T w = a.weight ? a.weight[row] : a.uniform_weight;
    T e[E], zs[S], t[S], p[S];
    int index[S];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = lane + i * G;
        e[i] = zr[c < a.cols ? c : a.cols - 1];
    }
    T tmost = Num<T>::neg_inf();
    int nan = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int j = lane + s * G;
        index[s] = -1;
        t[s] = Num<T>::neg_inf();
        if (j < a.top) {
            index[s] = slot_index(a, row, j);
            if (index[s] >= 0) t[s] = a.teacher[row * a.top + j];
        }
        zs[s] = T(0);
        if (s * G >= a.top) continue;  // (no lane has a slot here)
        zs[s] = zr[index[s] >= 0 ? index[s] : 0];
        tmost = Num<T>::max_(tmost, t[s]);
        nan |= t[s] != t[s];
    }
    T most = Num<T>::neg_inf();
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (lane + i * G >= a.cols) e[i] = Num<T>::neg_inf();
        most = Num<T>::max_(most, e[i]);
    }
#pragma unroll
    for (int d = G / 2; d > 0; d /= 2) {
        most = Num<T>::max_(most, __shfl_xor(most, d, G));
        tmost = Num<T>::max_(tmost, __shfl_xor(tmost, d, G));
        nan |= __shfl_xor(nan, d, G);
    }
    T total = T(0), ptotal = T(0);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        e[i] = Num<T>::exp_scaled(e[i] - most, a.c);
        if (lane + i * G >= a.cols) e[i] = T(0);
        total += e[i];
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
        p[s] = T(0);
        if (s * G >= a.top) continue;
        if (index[s] >= 0) p[s] = Num<T>::exp_scaled(t[s] - tmost, a.c);
        ptotal += p[s];
    }
#pragma unroll
    for (int d = G / 2; d > 0; d /= 2) {
        total += __shfl_xor(total, d, G);
        ptotal += __shfl_xor(ptotal, d, G);
    }
    const bool on = w != T(0) && (tmost != Num<T>::neg_inf() || nan);
    // log p_j - log q_j = ((t_j - tmost) - (z_j - most)) / T + log(total / ptotal): one logarithm in 64 bits for the whole row
    // instead of one a slot
    const double inv = 1.0 / a.temperature, shift = log(static_cast<double>(total) / static_cast<double>(ptotal));
    double loss = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (s * G >= a.top) continue;
        p[s] /= ptotal;
        const double pj = index[s] >= 0 ? static_cast<double>(p[s]) : 0.0;
        if (pj != 0.0)
            loss += pj * (((static_cast<double>(t[s]) - static_cast<double>(tmost)) - (static_cast<double>(zs[s]) - static_cast<double>(most))) * inv + shift);
    }
#pragma unroll
    for (int d = G / 2; d > 0; d /= 2) loss += __shfl_xor(loss, d, G);
    const T wt = w * static_cast<T>(a.temperature), f = wt / total;
    T share[E];
#pragma unroll
    for (int i = 0; i < E; ++i) share[i] = T(0);
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int n = a.top - s * G < G ? a.top - s * G : G;
        for (int k = 0; k < n; ++k) {
            const int c = __shfl(index[s], k, G);
            const T pk = __shfl(p[s], k, G);
#pragma unroll
            for (int i = 0; i < E; ++i) share[i] += c == lane + i * G ? pk : T(0);
        }
    }
    // the rows of a wave are added up here (its first row lives if any does)
    double own = live && on ? static_cast<double>(w) * a.temperature * a.temperature * loss : 0.0;
#pragma unroll
    for (int d = G; d < 64; d *= 2) own += __shfl_xor(own, d, 64);
    if (live) {
        if (threadIdx.x % 64 == 0 && !a.loss) a.row_loss[row / (64 / G)] = own;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int c = lane + i * G;
            if (c < a.cols) a.grad[row * a.cols + c] = on ? e[i] * f - wt * share[i] : T(0);
        }
    }
    if (!a.loss) return;  // (one workgroup: its waves' sums in order)
    if (threadIdx.x % 64 == 0) of_wave[threadIdx.x / 64] = own;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0;
        for (int w = 0; w < static_cast<int>(blockDim.x / 64); ++w) sum += of_wave[w];
        a.loss[0] = static_cast<T>(sum);
    }
}

// Few long rows: a workgroup has a part of a row, kPartVecs vectors a lane.  The first kernel leaves the part's largest
// logit and its sum of exponentials below that; the second joins the row's parts and writes the part's gradient, from
// logits that are still in a cache.
constexpr int kPartThreads = 256, kPartVecs = 4;

template <typename T>
struct PartSums {
    T most, total;
};

template <typename T>
__global__ void __launch_bounds__(kPartThreads) distill_part_kernel(DistillArgs<T> a, PartSums<T> *parts) {
    using V = typename Num<T>::vec_t;
    constexpr int W = Num<T>::W;
    __shared__ T red[2][kPartThreads / 64];
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x;
    if (a.weight && a.weight[row] == T(0)) return;  // (nobody reads its parts)
    const T *zr = a.z + row * a.z_row;
    const int nvec = a.cols / W, first = blockIdx.x * (kPartThreads * kPartVecs) + tid;
    const int tail = nvec * W + tid;
    V x[kPartVecs];
#pragma unroll
    for (int i = 0; i < kPartVecs; ++i) {
        const int v = first + i * kPartThreads;
        x[i] = reinterpret_cast<const V *>(zr)[v < nvec ? v : nvec - 1];
    }
    const T last = blockIdx.x == 0 && tail < a.cols ? zr[tail] : Num<T>::neg_inf();  // (the odd columns belong to part 0)
    T most = last;
#pragma unroll
    for (int i = 0; i < kPartVecs; ++i)
#pragma unroll
        for (int k = 0; k < W; ++k) {
            if (first + i * kPartThreads >= nvec) x[i][k] = Num<T>::neg_inf();
            most = Num<T>::max_(most, x[i][k]);
        }
    most = block_reduce<T, kPartThreads, true>(most, red[0]);
    const T base = most == Num<T>::neg_inf() ? T(0) : most;  // a part of nothing but -inf adds 0 to its row (a NaN stays one)
    T total = Num<T>::exp_scaled(last - base, a.c);
#pragma unroll
    for (int i = 0; i < kPartVecs; ++i)
#pragma unroll
        for (int k = 0; k < W; ++k) total += Num<T>::exp_scaled(x[i][k] - base, a.c);
    total = block_reduce<T, kPartThreads, false>(total, red[1]);
    if (tid == 0) parts[row * gridDim.x + blockIdx.x] = {most, total};
}

template <typename T>
__global__ void __launch_bounds__(kPartThreads) distill_join_kernel(DistillArgs<T> a, const PartSums<T> *parts) {
    using V = typename Num<T>::vec_t;
    constexpr int W = Num<T>::W, NW = kPartThreads / 64;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Slots<T> slots(smem, a.top);
    __shared__ T red[3][NW];
    __shared__ double total_of[NW], loss_of[NW];
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x, wave = tid / 64;
    const T *zr = a.z + row * a.z_row;
    T *gr = a.grad + row * a.cols;
    const int nvec = a.cols / W, first = blockIdx.x * (kPartThreads * kPartVecs) + tid;
    const int tail = nvec * W + tid;
    const T w = a.weight ? a.weight[row] : a.uniform_weight;
    const bool mine = blockIdx.x == 0;  // the row's loss and its columns behind the last whole vector
    V x[kPartVecs];
    T last = Num<T>::neg_inf(), most = Num<T>::neg_inf(), tmost = Num<T>::neg_inf(), tsum = T(0);
    double total = 0;  // of up to 2^18 parts: in 64 bits, as in distill_row_kernel
    if (w != T(0)) {  // (the same for the whole workgroup)
#pragma unroll
        for (int i = 0; i < kPartVecs; ++i) {
            const int v = first + i * kPartThreads;
            x[i] = reinterpret_cast<const V *>(zr)[v < nvec ? v : nvec - 1];
        }
        if (mine && tail < a.cols) last = zr[tail];
        const PartSums<T> *own = parts + row * gridDim.x;
        for (int i = tid; i < static_cast<int>(gridDim.x); i += kPartThreads) most = Num<T>::max_(most, own[i].most);
        most = wave_max(most);
        tmost = slots_read<T, kPartThreads>(a, row, slots);
        if (tid % 64 == 0) {
            red[0][wave] = most;
            red[1][wave] = tmost;
        }
        __syncthreads();
        most = join_waves<T, NW, true>(red[0]);
        tmost = join_waves<T, NW, true>(red[1]);
        for (int i = tid; i < static_cast<int>(gridDim.x); i += kPartThreads) total += static_cast<double>(own[i].total * Num<T>::exp_scaled(own[i].most - most, a.c));
        total = wave_sum(total);
        tsum = slots_exp<T, kPartThreads>(a, slots, tmost);
        if (tid % 64 == 0) {
            total_of[wave] = total;
            red[2][wave] = tsum;
        }
        __syncthreads();
        total = join_waves<double, NW, false>(total_of);
        tsum = join_waves<T, NW, false>(red[2]);
    }
    const bool on = w != T(0) && tmost != Num<T>::neg_inf();
    const T wt = w * static_cast<T>(a.temperature), f = wt / static_cast<T>(total);
#pragma unroll
    for (int i = 0; i < kPartVecs; ++i) {
        const int v = first + i * kPartThreads;
#pragma unroll
        for (int k = 0; k < W; ++k) x[i][k] = on ? Num<T>::exp_scaled(x[i][k] - most, a.c) * f : T(0);
        if (v < nvec) reinterpret_cast<V *>(gr)[v] = x[i];
    }
    if (mine && tail < a.cols) gr[tail] = on ? Num<T>::exp_scaled(last - most, a.c) * f : T(0);
    if (!on) {
        if (mine && tid == 0) a.row_loss[row] = 0.0;
        return;
    }
    const double loss = slots_loss<T, kPartThreads>(a, slots, tsum, most, total);
    if (tid % 64 == 0) loss_of[wave] = loss;
    __syncthreads();  // the bulk first, then the teacher's columns that lie in this part
    if (mine && tid == 0) a.row_loss[row] = static_cast<double>(w) * join_waves<double, NW, false>(loss_of);
    const int c0 = blockIdx.x * (kPartThreads * kPartVecs * W), c1 = c0 + kPartThreads * kPartVecs * W, whole = nvec * W;
    write_slots<T, kPartThreads>(a, slots, gr, most, f, wt, c0, c1 < whole ? c1 : whole, mine ? whole : a.cols);
}

// loss = sum of the rows' losses (or of what the rows of a wave came to: `n` of them): a lane adds every 1024th, the lanes are
// added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) distill_sum_kernel(const double *row_loss, int64_t n, T *out) {
    __shared__ double red[16];
    double v = 0;
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < n; r += 1024) v += row_loss[r];
    v = block_reduce<double, 1024, false>(v, red);
    if (threadIdx.x == 0) out[0] = static_cast<T>(v);
}

// Where the parts' sums begin in the workspace, behind the rows' losses, and how many parts a row is cut into (0: none).
size_t part_offset(int64_t rows) { return (static_cast<size_t>(rows) * sizeof(double) + 15) / 16 * 16; }

int64_t parts_of(size_t item, int64_t rows, int64_t cols) {
    const int64_t vec = 16 / static_cast<int64_t>(item), per = kPartThreads * kPartVecs * vec;
    const int64_t row_bytes = cols * static_cast<int64_t>(item);
    // (a third launch must pay: 16 x 131072 f32 21 us against 24 with a workgroup a row, 64 x 131072 21 against 33, 1 x 131072
    // f64 20 against 68; but 64 x 65000 f32 21 against 17, 200 x 131072 57 against 54)
    return rows <= 128 && row_bytes > 320 * 1024 ? (cols + per - 1) / per : 0;
}

// Rows of a few columns: 16 lanes each, four to a wave.  Rows of up to 1024 columns: a wave each (the slots go one by one:
// 4096 x 1000 f32 17 us with 16 of them, with 64 29 against 24).  0: others.
int short_lanes(int64_t cols, int64_t top) { return cols <= 64 && top <= 64 ? 16 : cols <= 1024 && top <= 32 ? 64 : 0; }

// Whether one workgroup has all rows: it adds up the loss too, which spares the second launch (64 x 60, 16 x 1000 and 1 x 30000
// f32 13.5 us a call against 15.7, host side included).  In f64 a CU's exponentials take longer: 8 x 1000 15.3 against 15.7,
// but 16 x 1000 24.9 against 15.8.
bool one_workgroup(size_t item, int64_t rows, int64_t cols, int64_t top) {
    const int lanes = short_lanes(cols, top);
    return lanes ? rows * lanes <= (lanes == 64 && item == 8 ? 512 : 1024) : rows == 1 && parts_of(item, rows, cols) == 0;
}

template <typename T, int G, int E>
void launch_short(const DistillArgs<T> &a, int64_t rows, hipStream_t st) {
    if (a.loss) distill_short_kernel<T, G, E, 1024><<<1, static_cast<unsigned>((rows * G + 63) / 64 * 64), 0, st>>>(a);
    else distill_short_kernel<T, G, E, 256><<<static_cast<unsigned>((rows + 256 / G - 1) / (256 / G)), 256, 0, st>>>(a);
}

template <typename T>
ttamd_status launch_some_rows(const DistillArgs<T> &a, int64_t rows, void *parts, hipStream_t st) {
    const size_t slots = Slots<T>::bytes(a.top);
    const int lanes = short_lanes(a.cols, a.top);
    if (lanes == 16) {
        launch_short<T, 16, 4>(a, rows, st);
    } else if (lanes == 64) {
        launch_short<T, 64, 16>(a, rows, st);
    } else if (const int64_t n = parts_of(sizeof(T), a.rows, a.cols)) {
        const dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(a.rows));
        distill_part_kernel<T><<<grid, kPartThreads, 0, st>>>(a, static_cast<PartSums<T> *>(parts));
        TTAMD_HIP_CHECK(hipGetLastError());
        distill_join_kernel<T><<<grid, kPartThreads, slots, st>>>(a, static_cast<const PartSums<T> *>(parts));
    } else {
        const int64_t nvec = a.cols / Num<T>::W;
        const auto run = [&](auto kernel, int threads, int held) -> ttamd_status {
            const int64_t left = nvec - static_cast<int64_t>(threads) * held;
            int64_t lds_vecs = left > 0 ? (left + threads - 1) / threads : 0;
            if (lds_vecs > kLdsVecs) lds_vecs = kLdsVecs;
            const size_t lds = static_cast<size_t>(lds_vecs) * threads * 16 + slots;
            // (the limit of the largest call, whichever comes first: calls of other threads may be between their two steps)
            const size_t most = static_cast<size_t>(kLdsVecs) * threads * 16 + Slots<T>::bytes(kMaxTop);
            if (lds > 48 * 1024)
                TTAMD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
            kernel<<<static_cast<unsigned>(rows), threads, lds, st>>>(a, static_cast<int>(lds_vecs));
            return TTAMD_OK;
        };
        // The smallest form that keeps the row: small workgroups share a CU and one's loads run under another's stores
        // (4096 x 8000 f32: 51 us with 256 x 8, 117 with 1024 x 8; 2048 x 64000: 214 with 1024 x 16, 294 with 256 x 32).
        // 24 vectors a lane only where they keep a row that 16 and LDS would not: they spill (rows beyond that, 1024 x 100003 f64:
        // 1.06 times as long with 24 as with 16).
        const auto pick = [&]<bool NT>() {
            if (nvec <= 256 * 4) return run(distill_row_kernel<T, 256, 4, NT>, 256, 4);
            if (nvec <= 256 * 8) return run(distill_row_kernel<T, 256, 8, NT>, 256, 8);
            if (nvec <= 512 * 8) return run(distill_row_kernel<T, 512, 8, NT>, 512, 8);
            if (nvec <= 512 * 16) return run(distill_row_kernel<T, 512, 16, NT>, 512, 16);
            if (nvec > 1024 * 24 && nvec <= 1024 * 32) return run(distill_row_kernel<T, 1024, 24, NT>, 1024, 24);
            return run(distill_row_kernel<T, 1024, 16, NT>, 1024, 16);
        };
        // Logits and gradient beyond 1.5 times the 256 MB Infinity Cache pass it by (2 x 262 MB: 97 us against 112;
        // 2 x 131 MB: 56 against 55, and there the next kernel finds part of the gradient in it).
        const bool beyond = static_cast<double>(a.rows) * a.cols * sizeof(T) > 192.0 * (1 << 20);
        if (ttamd_status s = beyond ? pick.template operator()<true>() : pick.template operator()<false>()) return s;
    }
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

// A launch holds fewer than 2^32 lanes: rows beyond kLaunchRows go to launches of their own.
constexpr int64_t kLaunchRows = int64_t(1) << 21;
template <typename T>
ttamd_status launch_rows(DistillArgs<T> a, void *parts, hipStream_t st) {
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += kLaunchRows)
        if (ttamd_status s = launch_some_rows(a, a.rows - a.row0 < kLaunchRows ? a.rows - a.row0 : kLaunchRows, parts, st)) return s;
    return TTAMD_OK;
}

template <typename T>
ttamd_status launch_distill(int64_t rows, int64_t cols, int64_t top, const void *input, int64_t input_row_stride, const void *index,
                            bool index64, const void *teacher, const void *weight, double temperature, void *loss_out, void *grad_out,
                            void *workspace, hipStream_t st) {
    const bool one = rows > 0 && one_workgroup(sizeof(T), rows, cols, top);
    if (rows > 0) {
        DistillArgs<T> a{};
        a.loss = one ? static_cast<T *>(loss_out) : nullptr;
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
        if (ttamd_status s = launch_rows(a, static_cast<char *>(workspace) + part_offset(rows), st)) return s;
    }
    if (one) return TTAMD_OK;
    const int64_t sums = short_lanes(cols, top) == 16 ? (rows + 3) / 4 : rows;
    distill_sum_kernel<T><<<1, 1024, 0, st>>>(static_cast<const double *>(workspace), sums, static_cast<T *>(loss_out));
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

ttamd_status check_distill_shape(ttamd_dtype dtype, int64_t rows, int64_t cols, int64_t top) {
    if (dtype != TTAMD_F32 && dtype != TTAMD_F64) {
        set_error("distill_loss: floating point dtypes only");
        return TTAMD_ERR_UNSUPPORTED_DTYPE;
    }
    if (rows < 0 || cols < 1 || top < 1 || rows > 0x7fffffffLL || cols > 0x3fffffffLL || rows * cols > int64_t(1) << 40 || top > kMaxTop) {
        set_error("distill_loss: rows %lld, cols %lld, top %lld: fewer than 2^31 rows, 1 to 2^30 - 1 columns, 2^40 elements at most, 1 to %d teacher slots",
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
    const size_t e = dtype_size(dtype);
    *bytes = part_offset(rows) + static_cast<size_t>(parts_of(e, rows, cols) * rows) * 2 * e;
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
        misaligned(grad_input_out, e) || misaligned(teacher_index, ie) || misaligned(workspace, 16)) {
        set_error("distill_loss: pointers must be aligned to the element size, the workspace to 16 bytes");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (workspace_bytes < need) {
        set_error("distill_loss: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (ttamd_status s = check_disjoint("distill_loss",
                                        {dense_extent("the gradient", grad_input_out, rows * cols, e), dense_extent("the loss", loss_out, 1, e),
                                         dense_extent("the workspace", workspace, static_cast<int64_t>(need), 1)},
                                        {{"the logits", input, rows, cols, input_row_stride, 1, e}, dense_extent("teacher_index", teacher_index, rows * top, ie),
                                         dense_extent("teacher_logit", teacher_logit, rows * top, e), dense_extent("row_weight", row_weight, rows, e)}))
        return s;
    if (ttamd_status s = use_device(device)) return s;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == TTAMD_F32)
        return launch_distill<float>(rows, cols, top, input, input_row_stride, teacher_index, index_dtype == TTAMD_I64, teacher_logit,
                                     row_weight, temperature, loss_out, grad_input_out, workspace, st);
    return launch_distill<double>(rows, cols, top, input, input_row_stride, teacher_index, index_dtype == TTAMD_I64, teacher_logit, row_weight,
                                  temperature, loss_out, grad_input_out, workspace, st);
}

}  // extern "C"
