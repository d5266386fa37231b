// gated_tiles.hip — the gated pair of Linear layers on the matrix cores: both products of the forward pass with their
// activation as one grid, and the three products of the backward pass as one grid; the forward pass of a few rows (gfx950).
//
// The grids are built from the tile engine of mfma_core.h.  Operands here are row-major with 16-byte aligned rows of whole 16-byte
// vectors; gated_linear.hip sees to that (it copies what is not) and picks between these kernels and separate products.
#include "gated.h"
#include "mfma_core.h"

#include <atomic>
#include <cmath>
#include <type_traits>

namespace ttamd {
namespace {

using namespace mfma;

// Stager of two matrices of the same size side by side (ROWS / 2 columns of each, contiguous along them): element (r, k) of
// the tile in LDS is column r / 2 of the first matrix for even r, of the second for odd r.  The engine reads neighbouring r
// as a pair and multiplies them into neighbouring blocks, so a lane ends up with both products of one column in its own
// registers, and the interleaving costs nothing: the two 16-byte vectors of a place are stored as two others.
template <typename T, int ROWS, int BK, int PF>
struct PairStager : TileLayout<T, ROWS, BK, false> {
    using L = TileLayout<T, ROWS, BK, false>;
    static constexpr int VEC = Mfma<T>::VK, HALF = ROWS / 2;
    using V = typename Vec<T, VEC>::type;
    static constexpr int kPF = PF;
    static constexpr int VPL = HALF / VEC;                 // vectors per line and matrix
    static constexpr int PS = HALF * BK / VEC / kThreads;  // passes per matrix
    static constexpr int P = 2 * PS;
    static_assert(HALF * BK / VEC % kThreads == 0, "tile must split evenly over the workgroup");

    V reg[PF][2][PS];
    uint32_t voff[2][PS];
    uint32_t k_step_b[2], k_off[2];
    __amdgpu_buffer_rsrc_t rsrc[2];
    int tid;
    static constexpr bool row_mask = false;  // whole vectors: one is inside the matrix or outside

    static __device__ __forceinline__ int line_of(int p, int tid) { return (p * kThreads + tid) / VPL; }
    static __device__ __forceinline__ int col_of(int p, int tid) { return ((p * kThreads + tid) % VPL) * VEC; }

    __device__ __forceinline__ void init(const T *first, const T *second, int tid_, int cols_left, int64_t s0, int64_t s1, int K) {
        tid = tid_;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int64_t s_k = m == 0 ? s0 : s1;
            rsrc[m] = make_rsrc(m == 0 ? first : second, (static_cast<int64_t>(K - 1) * s_k + cols_left) * static_cast<int64_t>(sizeof(T)));
            k_step_b[m] = static_cast<uint32_t>(s_k * BK * sizeof(T));
            k_off[m] = 0;
#pragma unroll
            for (int p = 0; p < PS; ++p) {
                const int line = line_of(p, tid), col = col_of(p, tid);
                voff[m][p] = col < cols_left ? static_cast<uint32_t>((col + line * s_k) * sizeof(T)) : kOob;
            }
        }
    }

    template <bool MASK, int SLOT = 0, bool UNIFORM_K = false>
    __device__ __forceinline__ void load(int k_left) {
        static_assert(!(MASK && UNIFORM_K), "a masked load relies on the range check of its whole offset");
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int p = 0; p < PS; ++p) {
                if constexpr (UNIFORM_K) {
                    reg[SLOT][m][p] = Vec<T, VEC>::load_at(rsrc[m], voff[m][p], k_off[m]);
                } else {
                    uint32_t off = voff[m][p] + k_off[m];
                    if constexpr (MASK) {
                        if (line_of(p, tid) >= k_left) off = kOob;
                    }
                    reg[SLOT][m][p] = Vec<T, VEC>::load(rsrc[m], off);
                    voff[m][p] += k_step_b[m];
                }
            }
        if constexpr (UNIFORM_K) {
            k_off[0] += k_step_b[0];
            k_off[1] += k_step_b[1];
        }
    }

    template <int SLOT = 0>
    __device__ __forceinline__ void store(T *lds) const {
#pragma unroll
        for (int p = 0; p < PS; ++p) {
            const int line = line_of(p, tid), col = col_of(p, tid);
            const V a = reg[SLOT][0][p], b = reg[SLOT][1][p];
            V lo, hi;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                lo[2 * j] = a[j];
                lo[2 * j + 1] = b[j];
                hi[2 * j] = a[VEC / 2 + j];
                hi[2 * j + 1] = b[VEC / 2 + j];
            }
            *reinterpret_cast<V *>(&lds[line * L::LD + 2 * col]) = lo;
            *reinterpret_cast<V *>(&lds[line * L::LD + 2 * col + VEC]) = hi;
        }
    }
};

// The finished tile: g + bg and u + bu go to gate / up where they are wanted, act(g) * u to out.  Rows of `cols` elements.
template <typename T, int ACT, class Engine>
__device__ __forceinline__ void store_gated(Engine &eng, const GatedForward<T> &a, int m0, int c0) {
    using MI = Mfma<T>;
    const int64_t first = static_cast<int64_t>(m0) * a.hidden + c0;
    const int rows = a.rows - m0 < Engine::kBM ? a.rows - m0 : Engine::kBM;
    const int cols = a.hidden - c0;
    const int64_t bytes = (static_cast<int64_t>(rows) * a.hidden - c0) * static_cast<int64_t>(sizeof(T));
    const __amdgpu_buffer_rsrc_t out = make_rsrc(a.out + first, bytes);
    // outputs that are not wanted are written through descriptors of zero length, whose stores the hardware drops
    const __amdgpu_buffer_rsrc_t gate = make_rsrc(a.gate ? a.gate + first : a.gate, a.gate ? bytes : 0);
    const __amdgpu_buffer_rsrc_t up = make_rsrc(a.gate ? a.up + first : a.up, a.gate ? bytes : 0);
    const int jcol = eng.lane % MI::MB;
#pragma unroll
    for (int pr = 0; pr < Engine::NBN / 2; ++pr) {
        const int n = Engine::FrB::index_of(eng.wn0, 2 * pr, jcol) / 2;  // even places: the first matrix
        const bool in = n < cols;
        const T bg = a.gate_bias && in ? a.gate_bias[c0 + n] : T(0), bu = a.up_bias && in ? a.up_bias[c0 + n] : T(0);
#pragma unroll
        for (int bm = 0; bm < Engine::NBM; ++bm) {
#pragma unroll
            for (int e = 0; e < MI::NACC; ++e) {
                const int m = Engine::FrA::index_of(eng.wm0, bm, MI::acc_row(e, eng.lane));
                const uint32_t off = in && m < rows ? static_cast<uint32_t>(m * a.hidden + n) * static_cast<uint32_t>(sizeof(T)) : kOob;
                const T g = eng.acc[bm][2 * pr][e] + bg, u = eng.acc[bm][2 * pr + 1][e] + bu;
                buffer_store(gate, off, g);
                buffer_store(up, off, u);
                buffer_store(out, off, activate<T, ACT>(g) * u);
            }
            __builtin_amdgcn_sched_barrier(0);  // (a block's results at a time: more would not fit the registers)
        }
    }
}

// BM rows of x against BN / 2 columns of both weights (the tiles of 256 rows spill 2 registers in f32, 8 in f64).  HALVES = 2: lanes 0-255 take the first half of the reduction, lanes
// 256-511 the second, each with buffers of its own (for grids of about a workgroup per CU, see gemm_mfma_dual_kernel); the
// halves have the same number of k tiles.
template <typename T, int BM, int BN, int BK, int WGM, int WGN, int PF, int HALVES>
__global__ void __launch_bounds__(HALVES *kThreads, BM * BN >= 256 * 256 || HALVES == 2 || (sizeof(T) == 8 && BM * BN >= 128 * 128) ? 1 : 2)
gated_forward_kernel(GatedForward<T> a, int tiles_m, int tiles_n, int k_half) {
    using StA = Stager<T, BM, BK, true, Mfma<T>::VK, PF>;
    using StB = PairStager<T, BN, BK, PF>;
    using Engine = TileEngine<T, BM, BN, BK, WGM, WGN, StA, StB>;
    static_assert(Engine::FrB::PAIRED, "neighbouring blocks hold the two products of a column");
    static_assert(HALVES == 1 || Engine::kAccPerLane * kThreads * sizeof(T) <= 2 * Engine::kLdsBytes, "the parked accumulators fit");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    const int half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kThreads));
    const int tid = threadIdx.x % kThreads;
    T *const smem = reinterpret_cast<T *>(smem_raw + half * Engine::kLdsBytes);
    int batch, tm, tn;
    decode_tile(remap_xcd(blockIdx.x, gridDim.x), tiles_m, tiles_n, batch, tm, tn);
    const int m0 = tm * BM, c0 = tn * (BN / 2), k0 = half * k_half;
    const int K = HALVES == 1 ? a.k : half == 0 ? k_half : a.k - k_half;
    StA sa;
    StB sb;
    sa.init(a.x + static_cast<int64_t>(m0) * a.x_row + k0, tid, a.rows - m0, a.x_row, 1, K);
    sb.init(a.wg + static_cast<int64_t>(k0) * a.wg_row + c0, a.wu + static_cast<int64_t>(k0) * a.wu_row + c0, tid, a.w_cols - c0, a.wg_row, a.wu_row, K);
    Engine eng;
    eng.init(tid);
    eng.run(sa, sb, smem, K, true);
    if constexpr (HALVES == 2) {
        __syncthreads();
        T *const exchange = reinterpret_cast<T *>(smem_raw);
        if (half == 1) eng.park_acc(exchange, tid);
        __syncthreads();
        if (half == 1) return;
        eng.add_parked_acc(exchange, tid);
    }
    switch (a.act) {
    case kSilu: store_gated<T, kSilu>(eng, a, m0, c0); break;
    case kGelu: store_gated<T, kGelu>(eng, a, m0, c0); break;
    case kRelu: store_gated<T, kRelu>(eng, a, m0, c0); break;
    default: store_gated<T, kSigmoid>(eng, a, m0, c0); break;
    }
}

// The backward pass's products as one grid of B x B tiles: first the tiles of dx = dg . Wg^T + du . Wu^T (two reductions one
// after the other), then those of dWg = x^T . dg and dWu = x^T . du, whose first rows of tiles also add up the vectors
// of dg / du that they stage: the bias gradients.  At least two workgroups share a CU, and one's first loads and stores run
// under the other's products; the long reductions of dx go first and the weights' tiles fill up beside them.  The f32 kernel of
// 128 x 128 tiles spills 48 registers, the accumulators set aside between dx's two reductions.
template <typename T, int B>
struct BackwardTile {
    static constexpr int BK = sizeof(T) == 4 && B == 64 ? 32 : 16;
    static constexpr int PF = B == 64 ? 2 : 1;
};

template <typename T, int B>
__device__ __forceinline__ void gated_dx_tile(const GatedBackward<T> &a, int item, int tiles, int tiles_n, T *smem) {
    constexpr int BK = BackwardTile<T, B>::BK, PF = BackwardTile<T, B>::PF, VK = Mfma<T>::VK;
    using St = Stager<T, B, BK, true, VK, PF>;
    using Engine = TileEngine<T, B, B, BK, 2, 2, St, St>;
    const int tid = threadIdx.x;
    const int part = item / tiles;  // of both reductions; 0 when they are not cut
    int batch, tm, tn;
    decode_tile(remap_xcd(item - part * tiles, tiles), tiles / tiles_n, tiles_n, batch, tm, tn);
    const int m0 = tm * B, n0 = tn * B;
    const int splits = a.split.x_splits;
    Engine eng;
    eng.init(tid);
    // The first reduction's result is set aside and added at the end: as exact as two products added up, where one run of both
    // through the accumulators would carry the roundings of twice the length.
    typename Engine::M::acc_t first[Engine::NBM][Engine::NBN];
#pragma unroll
    for (int i = 0; i < Engine::NBM; ++i)
#pragma unroll
        for (int j = 0; j < Engine::NBN; ++j) first[i][j] = eng.acc[i][j];
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        if (splits && s != part / splits) continue;
        if (s == 1 && !splits) {
            __syncthreads();  // every wave has read the first reduction's last tile
#pragma unroll
            for (int i = 0; i < Engine::NBM; ++i)
#pragma unroll
                for (int j = 0; j < Engine::NBN; ++j) {
                    first[i][j] = eng.acc[i][j];
#pragma unroll
                    for (int e = 0; e < Engine::M::NACC; ++e) eng.acc[i][j][e] = T(0);
                }
        }
        const int k0 = splits ? part % splits * a.split.x_chunk : 0;
        const int K = splits && a.k - k0 > a.split.x_chunk ? a.split.x_chunk : a.k - k0;
        const T *d = (s == 0 ? a.dg : a.du) + k0, *w = (s == 0 ? a.wg : a.wu) + k0;
        const int64_t w_row = s == 0 ? a.wg_row : a.wu_row;
        St sa, sb;
        sa.init(d + static_cast<int64_t>(m0) * a.d_row, tid, a.rows - m0, a.d_row, 1, K);
        sb.init(w + static_cast<int64_t>(n0) * w_row, tid, a.inner - n0, w_row, 1, K);
        eng.run(sa, sb, smem, K, true);
    }
#pragma unroll
    for (int i = 0; i < Engine::NBM; ++i)
#pragma unroll
        for (int j = 0; j < Engine::NBN; ++j) eng.acc[i][j] += first[i][j];
    T *const out = splits ? a.x_part + static_cast<int64_t>(part) * a.rows * a.inner : a.dx;
    store_tile_dense<T, true>(eng, out, a.rows, a.inner, m0, n0, static_cast<const T *>(nullptr), 0, 0, 0);
}

template <typename T, int B>
__device__ __forceinline__ void gated_dw_tile(const GatedBackward<T> &a, int item, int tiles, int tiles_n, T *smem) {
    constexpr int BK = BackwardTile<T, B>::BK, PF = BackwardTile<T, B>::PF, VK = Mfma<T>::VK;
    using StA = Stager<T, B, BK, false, VK, PF>;
    using StB = Stager<T, B, BK, false, VK, PF, true>;
    using Engine = TileEngine<T, B, B, BK, 2, 2, StA, StB>;
    static_assert(static_cast<size_t>(StB::kSumParts) * B * sizeof(T) <= Engine::kLdsBytes, "the operand sums fit the tile buffers");
    const int tid = threadIdx.x;
    const int which = item / tiles;  // 2 x chunk + (0: dWg, 1: dWu)
    const bool second = which & 1;
    int batch, tm, tn;
    decode_tile(remap_xcd(item - which * tiles, tiles), tiles / tiles_n, tiles_n, batch, tm, tn);
    const int m0 = tm * B, n0 = tn * B;
    const int splits = a.split.w_splits;
    const int r0 = splits ? which / 2 * a.split.w_chunk : 0;
    const int R = splits && a.rows - r0 > a.split.w_chunk ? a.split.w_chunk : a.rows - r0;
    T *bias = second ? a.dbu : a.dbg, *out = second ? a.dwu : a.dwg;
    if (splits) {
        bias = bias ? a.b_part + static_cast<int64_t>(which) * a.hidden : bias;
        out = a.w_part + static_cast<int64_t>(which) * a.inner * a.hidden;
    }
    StA sa;
    StB sb;
    sa.init(a.x + static_cast<int64_t>(r0) * a.x_row + m0, tid, a.x_cols - m0, 1, a.x_row, R);
    sb.init((second ? a.du : a.dg) + static_cast<int64_t>(r0) * a.d_row + n0, tid, a.k - n0, 1, a.d_row, R);
    sb.start_sums(bias && tm == 0);
    Engine eng;
    eng.init(tid);
    eng.run(sa, sb, smem, R, true);
    if (bias && tm == 0) {  // (workgroup-uniform) a lane's rows were added in order; the lanes of a column follow in lane order
        __syncthreads();
        *reinterpret_cast<typename StB::V *>(&smem[sb.sum_part() * B + sb.sum_row0()]) = sb.sum;
        __syncthreads();
        if (tid < B && n0 + tid < a.hidden) {
            T v = T(0);
#pragma unroll
            for (int r = 0; r < StB::kSumParts; ++r) v += smem[r * B + tid];
            bias[n0 + tid] = v;
        }
    }
    store_tile_dense<T, true>(eng, out, a.inner, a.hidden, m0, n0, static_cast<const T *>(nullptr), 0, 0, 0);
}

template <typename T, int B>
__global__ void __launch_bounds__(kThreads, 2) gated_backward_kernel(GatedBackward<T> a, int dx_items, int dx_tiles, int dx_tiles_n, int dw_tiles, int dw_tiles_n) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    T *const smem = reinterpret_cast<T *>(smem_raw);
    const int block = blockIdx.x;
    if (block < dx_items) gated_dx_tile<T, B>(a, block, dx_tiles, dx_tiles_n, smem);
    else gated_dw_tile<T, B>(a, block - dx_items, dw_tiles, dw_tiles_n, smem);
}

// out[i] = sum over p < parts of src[p * stride + i], p ascending; up to five such sums in a launch.
constexpr int kSums = 5;
template <typename T>
struct PartSum {
    const T *src;
    T *out;
    int64_t n, stride;
    int parts, blocks;
};
template <typename T>
struct PartSums {
    PartSum<T> job[kSums];
};
template <typename T>
__global__ void __launch_bounds__(256) gated_add_parts_kernel(PartSums<T> a) {
    constexpr int W = Mfma<T>::VK;
    typedef T near_t __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    int block = blockIdx.x;
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
        const PartSum<T> &j = a.job[k];
        if (block < j.blocks) {
            const int64_t i = (static_cast<int64_t>(block) * 256 + threadIdx.x) * W;
            if (i + W <= j.n) {
                near_t v = {};
#pragma unroll 4
                for (int p = 0; p < j.parts; ++p) v += *reinterpret_cast<const near_t *>(j.src + p * j.stride + i);
                *reinterpret_cast<near_t *>(j.out + i) = v;
            } else {
                for (int64_t e = i; e < j.n; ++e) {
                    T v = T(0);
                    for (int p = 0; p < j.parts; ++p) v += j.src[p * j.stride + e];
                    j.out[e] = v;
                }
            }
            return;
        }
        block -= j.blocks;
    }
}

// A block of rows (a batch of requests in step, a short prompt): too few for tiles of 64 rows, more than the vector units
// want.  A workgroup owns 32 columns of both weights and 16 or 32 rows, and its NW waves share out the reduction in groups of
// 64 / MB x VK k, every NW-th to a wave: a lane loads 16 bytes of a row of x and the rows of the weights that meet them,
// straight into the registers that the matrix instructions read (lane group h of a group takes k = VK h .. VK h + VK - 1, of
// x and weights alike, so the order inside a group does not matter).  Weights are read once, there is no barrier until the end;
// the waves' sums are added up through LDS in wave order, and the same lanes apply biases and activation: one launch.
// Columns behind the last are moved back onto it (they come out twice, the same); rows behind the last repeat it and are dropped.
// Bound: HBM with 16 rows (16 x 2048 x 8192 f32 22.6 us, 5.9 TB/s with what the caches keep; separate products 48; 8 x 2048 x
// 8192 22 against 36 on the vector units), the matrix cores next to it with 32 (32 x 2048 x 8192 32 us against 75;
// 64 x 2048 x 2048 20 against 47; f64 33 x 2048 x 2048 23 against 52).
// Blocks of 16 x 16 f32: half the matrix instructions' time of 32 x 32 for up to 16 rows.
struct Mfma16 {
    static constexpr int MB = 16, VK = 4, NACC = 4;
    using acc_t = float __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ acc_t mma(float a, float b, acc_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int acc_row(int e, int lane) { return 4 * (lane / 16) + e; }
};
template <typename T, class MI, int RB>
struct FewShape {
    static constexpr int CB = 32 / MI::MB;                  // blocks of columns: neighbouring columns of a lane
    static constexpr int E = RB * CB * MI::NACC;            // elements a lane and matrix
    static constexpr int NW = E * sizeof(T) > 64 ? 8 : 16;  // 128 KB of parts
    static constexpr size_t kLds = static_cast<size_t>(NW) * 2 * E * 64 * sizeof(T);
    static constexpr int kRows = RB * MI::MB;
};

template <typename T, class MI, int RB, int ACT>
__global__ void __launch_bounds__((FewShape<T, MI, RB>::NW * 64)) gated_few_kernel(GatedForward<T> a) {
    using S = FewShape<T, MI, RB>;
    constexpr int MB = MI::MB, VK = MI::VK, CB = S::CB, E = S::E, NW = S::NW, kGroup = 64 / MB * VK;
    typedef T xvec_t __attribute__((ext_vector_type(VK), aligned(sizeof(T))));
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    T *const part = reinterpret_cast<T *>(smem_raw);  // [NW][2][E][64]
    const int tid = threadIdx.x, lane = tid % 64, l = lane % MB, h = lane / MB;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int c0 = blockIdx.x * 32, m0 = blockIdx.y * S::kRows;
    const auto col_of = [&](int place, int cb) {  // the column that a lane's place holds
        const int at = c0 + place * CB;
        return (at + CB <= a.hidden ? at : a.hidden - CB) + cb;
    };
    const T *xr[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        const int m = m0 + r * MB + l;
        xr[r] = a.x + (m < a.rows ? m : a.rows - 1) * a.x_row + h * VK;
    }
    const T *wg = a.wg + h * VK * a.wg_row + col_of(l, 0), *wu = a.wu + h * VK * a.wu_row + col_of(l, 0);
    typename MI::acc_t acc[2][RB][CB];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
                for (int e = 0; e < MI::NACC; ++e) acc[m][r][c][e] = T(0);
    typedef T wvec_t __attribute__((ext_vector_type(CB), aligned(sizeof(T))));
    xvec_t x[RB];
    wvec_t w[2][VK];
    const auto load = [&](int64_t k) {
#pragma unroll
        for (int r = 0; r < RB; ++r) x[r] = *reinterpret_cast<const xvec_t *>(xr[r] + k);
#pragma unroll
        for (int j = 0; j < VK; ++j) {
            w[0][j] = *reinterpret_cast<const wvec_t *>(wg + (k + j) * a.wg_row);
            w[1][j] = *reinterpret_cast<const wvec_t *>(wu + (k + j) * a.wu_row);
        }
    };
    const auto multiply = [&] {
#pragma unroll
        for (int j = 0; j < VK; ++j)
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int c = 0; c < CB; ++c) acc[m][r][c] = MI::mma(x[r][j], w[m][j][c], acc[m][r][c]);
    };
    // A wave's next group is requested once the last one has been multiplied; the other waves' loads fill the time.  (Two to
    // four groups in flight a wave: 1.4 times as long at 32 x 2048 x 8192 f32.)
    const int groups = a.k / kGroup;
    if (wave < groups) {
        load(static_cast<int64_t>(wave) * kGroup);
        int g = wave;
        for (; g + NW < groups; g += NW) {
            multiply();
            __builtin_amdgcn_sched_barrier(0);
            load(static_cast<int64_t>(g + NW) * kGroup);
            __builtin_amdgcn_sched_barrier(0);
        }
        multiply();
    }
    if (groups * kGroup < a.k && wave == groups % NW) {  // the last k, one by one; zeros on both sides behind them
        const int k = groups * kGroup;
#pragma unroll
        for (int j = 0; j < VK; ++j) {
            const bool in = k + h * VK + j < a.k;
#pragma unroll
            for (int r = 0; r < RB; ++r) x[r][j] = in ? xr[r][k + j] : T(0);
            const wvec_t zero = {};
            w[0][j] = in ? *reinterpret_cast<const wvec_t *>(wg + (k + j) * a.wg_row) : zero;
            w[1][j] = in ? *reinterpret_cast<const wvec_t *>(wu + (k + j) * a.wu_row) : zero;
        }
        multiply();
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
                for (int e = 0; e < MI::NACC; ++e) part[((wave * 2 + m) * E + (r * CB + c) * MI::NACC + e) * 64 + lane] = acc[m][r][c][e];
    __syncthreads();
#pragma unroll
    for (int e = wave; e < E; e += NW) {
        const int r = e / (CB * MI::NACC), c = e / MI::NACC % CB;
        const int row = m0 + r * MB + MI::acc_row(e % MI::NACC, lane), col = col_of(l, c);
        T g = T(0), u = T(0);
#pragma unroll
        for (int v = 0; v < NW; ++v) {
            g += part[((v * 2 + 0) * E + e) * 64 + lane];
            u += part[((v * 2 + 1) * E + e) * 64 + lane];
        }
        if (a.gate_bias) g += a.gate_bias[col];
        if (a.up_bias) u += a.up_bias[col];
        if (row >= a.rows) continue;
        const int64_t to = static_cast<int64_t>(row) * a.hidden + col;
        if (a.gate) {
            a.gate[to] = g;
            a.up[to] = u;
        }
        a.out[to] = activate<T, ACT>(g) * u;
    }
}

template <typename T, class MI, int RB, int ACT>
ttamd_status run_few(const GatedForward<T> &a, int device, hipStream_t st) {
    using S = FewShape<T, MI, RB>;
    static_assert(S::kLds <= 160 * 1024, "LDS of a CU");
    auto kernel = gated_few_kernel<T, MI, RB, ACT>;
    static std::atomic<bool> configured[kMaxDevices] = {};
    if (!configured[device].load(std::memory_order_acquire)) {
        TTAMD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kLds)));
        configured[device].store(true, std::memory_order_release);
    }
    kernel<<<dim3(static_cast<unsigned>((a.hidden + 31) / 32), static_cast<unsigned>((a.rows + S::kRows - 1) / S::kRows)), S::NW * 64, S::kLds, st>>>(a);
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

template <typename T, int BM, int BN, int BK, int WGM, int WGN, int PF, int HALVES>
ttamd_status run_forward(const GatedForward<T> &a, int device, hipStream_t st) {
    using StA = Stager<T, BM, BK, true, Mfma<T>::VK, PF>;
    using StB = PairStager<T, BN, BK, PF>;
    constexpr size_t lds = HALVES * TileEngine<T, BM, BN, BK, WGM, WGN, StA, StB>::kLdsBytes;
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    auto kernel = gated_forward_kernel<T, BM, BN, BK, WGM, WGN, PF, HALVES>;
    if (lds > 48 * 1024) {  // raising the dynamic LDS limit: once per kernel and device
        static std::atomic<bool> configured[kMaxDevices] = {};
        if (!configured[device].load(std::memory_order_acquire)) {
            TTAMD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
            configured[device].store(true, std::memory_order_release);
        }
    }
    const int tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.hidden + BN / 2 - 1) / (BN / 2);
    constexpr int VK = Mfma<T>::VK;
    const int k_half = HALVES == 1 ? a.k : ((a.k + 1) / 2 + VK - 1) / VK * VK;
    kernel<<<static_cast<unsigned>(static_cast<int64_t>(tiles_m) * tiles_n), HALVES * kThreads, lds, st>>>(a, tiles_m, tiles_n, k_half);
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

// Whether two halves of a reduction have the same number of k tiles (they share the engine's barriers).
template <typename T>
bool halves_match(int64_t k, int bk) {
    constexpr int VK = Mfma<T>::VK;
    const int64_t lower = ((k + 1) / 2 + VK - 1) / VK * VK;
    return k > lower && (lower + bk - 1) / bk == (k - lower + bk - 1) / bk;
}

}  // namespace

// 16 rows a workgroup while each finds a CU of its own, else 32 (32 x 4000 x 512 f32 35 us against 55 with 32; 32 x 2048 x 8192 42
// with 16 against 32).
int few_rows_of(int64_t rows, int64_t hidden) { return rows <= 16 || (rows + 15) / 16 * ((hidden + 31) / 32) <= 256 ? 16 : 32; }

double few_rows_estimate(size_t item, int64_t rows, int64_t inner, int64_t hidden) {
    const int block = few_rows_of(rows, hidden);
    const int64_t rounds = ((rows + block - 1) / block * ((hidden + 31) / 32) + 255) / 256;
    const double a_k = item == 4 ? (block == 16 ? 7.5e-3 : 13e-3) : (block == 16 ? 9e-3 : 17e-3);
    return static_cast<double>(rounds) * (a_k * static_cast<double>(inner) + 3);
}

template <typename T>
ttamd_status launch_gated_few_rows(const GatedForward<T> &a, int device, hipStream_t st) {
    const auto run = [&]<class MI, int RB>() -> ttamd_status {
        switch (a.act) {
        case kSilu: return run_few<T, MI, RB, kSilu>(a, device, st);
        case kGelu: return run_few<T, MI, RB, kGelu>(a, device, st);
        case kRelu: return run_few<T, MI, RB, kRelu>(a, device, st);
        default: return run_few<T, MI, RB, kSigmoid>(a, device, st);
        }
    };
    using MI = std::conditional_t<sizeof(T) == 4, Mfma16, Mfma<T>>;
    static_assert(MI::MB == 16);
    return few_rows_of(a.rows, a.hidden) == 16 ? run.template operator()<MI, 1>() : run.template operator()<MI, 2>();
}

// The tile whose workgroups, dealt to 256 CUs, are done first: workgroups of the fullest CU x tile area / the share of the
// peak that the tile reaches (measured at inner = 1024: f32 64 x 128 0.83, 128 x 128 0.84 alone on its CU and 0.90 from two
// on, 256 x 128 0.90 and 0.925; f64 64 x 64 0.70 alone and 0.84, 128 x 128 0.89, 256 x 128 0.91).
ForwardTile pick_forward_tile(size_t item, int64_t rows, int64_t hidden, int64_t k) {
    const bool f32 = item == 4;
    const auto per_cu = [&](int bm, int bn) { return ((rows + bm - 1) / bm * ((hidden + bn / 2 - 1) / (bn / 2)) + 255) / 256; };
    const auto cost = [&](int bm, int bn, double alone, double shared) {
        const int64_t n = per_cu(bm, bn);
        return static_cast<double>(n) * bm * bn / (n == 1 ? alone : shared);
    };
    const double small = f32 ? cost(64, 128, 0.83, 0.83) : cost(64, 64, 0.70, 0.84);
    const double large = f32 ? cost(128, 128, 0.84, 0.90) : cost(128, 128, 0.89, 0.89);
    const double xl = f32 ? cost(256, 128, 0.90, 0.925) : cost(256, 128, 0.91, 0.91);
    if (xl < large && xl < small) return {256, 128, 1};
    if (large < small) return {128, 128, 1};
    if (!f32) return {64, 64, 1};
    // a workgroup alone on its CU: two halves of the reduction cover each other's waits (1024 x 784 x 1024: 31.2 -> 30.5 us)
    return {64, 128, per_cu(64, 128) == 1 && k >= 256 && halves_match<float>(k, 32) ? 2 : 1};
}

template <typename T>
ttamd_status launch_gated_forward_tiles(const GatedForward<T> &a, int device, hipStream_t st) {
    const ForwardTile tile = pick_forward_tile(sizeof(T), a.rows, a.hidden, a.k);
    if (tile.bm == 256) return run_forward<T, 256, 128, 16, 2, 2, 1, 1>(a, device, st);
    if (tile.bm == 128) return run_forward<T, 128, 128, 16, 2, 2, 1, 1>(a, device, st);
    if constexpr (sizeof(T) == 4) {
        if (tile.halves == 2) return run_forward<float, 64, 128, 32, 2, 2, 2, 2>(a, device, st);
        return run_forward<float, 64, 128, 32, 2, 2, 2, 1>(a, device, st);
    } else {
        return run_forward<double, 64, 64, 16, 2, 2, 2, 1>(a, device, st);
    }
}

// Reductions are cut into equal chunks where their tiles alone would load the CUs unevenly: of the tile sizes and numbers of
// chunks tried, those that are done first by this estimate, in units of one k of a 64 x 64 tile (15 ns on a CU in f32, 30 in
// f64).  The tiles are dealt to 256 CUs in order, dx's first; a tile costs its reduction and 70 units of first loads and
// stores; a 128 x 128 tile (f32) costs 3.7 times as much a k; cut reductions cost a launch (200) and the traffic of their
// parts.  Against whole reductions: 16 x 1024 x 4096 154 -> 46 us forward and backward, 4096 x 256 x 512 134 -> 73.
GatedSplit plan_gated_split(size_t item, int64_t rows, int64_t inner, int64_t hidden, int64_t k) {
    const int64_t x_bytes = 2 * rows * inner * static_cast<int64_t>(item), w_bytes = 2 * inner * hidden * static_cast<int64_t>(item);
    constexpr int64_t kMostBytes = int64_t(64) << 20, kShortest = 192;
    const auto chunk_of = [](int64_t reduction, int n) { return ((reduction + n - 1) / n + 31) / 32 * 32; };  // (whole k tiles of either type)
    double best = 0;
    int best_b = 0, best_x = 0, best_w = 1;
    for (int B = 64; B <= (item == 4 ? 128 : 64); B *= 2) {
        const int64_t dx = (rows + B - 1) / B * ((inner + B - 1) / B), dw = 2 * ((inner + B - 1) / B) * ((hidden + B - 1) / B);
        const double unit = B == 64 ? 1.0 : 3.7, once = B == 64 ? 70.0 : 160.0;
        const double share = B == 64 && item == 4 ? 3 : 2;  // workgroups that a CU holds
        for (int sx = 0; sx <= 32; sx = sx ? 2 * sx : 1) {  // 0: both reductions of a dx tile in one piece
            if (sx > 0 && ((sx > 1 && chunk_of(k, sx) < kShortest) || sx * x_bytes > kMostBytes)) break;
            const double lx = once + unit * (sx ? static_cast<double>(chunk_of(k, sx)) : 2.0 * k);
            const int64_t nx = dx * (sx ? 2 * sx : 1);
            // CUs hold nx / 256 tiles of dx, the first nx % 256 of them one more; the weights' tiles go where there is room
            const double low = static_cast<double>(nx / 256) * lx, high = nx % 256 ? low + lx : low;
            const int64_t many = nx % 256, few = 256 - many;
            for (int sw = 1; sw <= 32; sw *= 2) {
                if (sw > 1 && (chunk_of(rows, sw) < kShortest || sw * w_bytes > kMostBytes)) break;
                // (32-bit offsets: prefer pieces of rows that the tiles can reach)
                if ((chunk_of(rows, sw) + 64) * (k > inner ? k : inner) * static_cast<int64_t>(item) > 0x7fffffffLL && 2 * sw <= 32 && 2 * sw * w_bytes <= kMostBytes) continue;
                const double lw = once + unit * static_cast<double>(sw > 1 ? chunk_of(rows, sw) : rows);
                const int64_t nw = dw * sw;
                double end = (nx * lx + nw * lw) / 256;
                if (end < high) end = high;
                for (int tries = 0; tries < 64; ++tries) {
                    const double a = std::floor((end - low) / lw + 1e-9), b = std::floor((end - high) / lw + 1e-9);
                    if (few * a + many * b >= nw) break;
                    const double next_low = low + (a + 1) * lw, next_high = high + (b + 1) * lw;
                    end = many && next_high < next_low ? next_high : next_low;
                }
                // The workgroups of a CU share it: a dx tile proceeds at 1 / share of its rate while weights' tiles are left to
                // fill the other places, and what is left of it then runs on after everything else has ended.
                const double filled = (few * (share - nx / 256) + many * (share - nx / 256 - 1)) / share;
                const double until = filled > 0 ? nw * lw / filled : share * lx;
                if (nx < 256 * share && until < share * lx) {
                    const double after = until + (nx / 256 + (many ? 1 : 0)) * (lx - until / share);
                    if (end < after) end = after;
                }
                const double parts = (sx ? static_cast<double>(sx) * x_bytes : 0.0) + (sw > 1 ? static_cast<double>(sw) * w_bytes : 0.0);
                if (parts > 0) end += 200 + 2 * parts / 4e12 / (item == 4 ? 15e-9 : 30e-9);
                if (!best_b || end < best) {
                    best = end;
                    best_b = B;
                    best_x = sx;
                    best_w = sw;
                }
            }
        }
    }
    GatedSplit s{};
    s.tile = best_b;
    if (best_x > 0) {
        s.x_chunk = static_cast<int>(chunk_of(k, best_x));
        s.x_splits = static_cast<int>((k + s.x_chunk - 1) / s.x_chunk);
    }
    if (best_w > 1) {
        s.w_chunk = static_cast<int>(chunk_of(rows, best_w));
        s.w_splits = static_cast<int>((rows + s.w_chunk - 1) / s.w_chunk);
    }
    s.x_parts = 2 * s.x_splits * rows * inner;
    s.w_parts = 2 * s.w_splits * inner * hidden;
    s.b_parts = 2 * s.w_splits * hidden;
    return s;
}

template <typename T>
ttamd_status launch_gated_backward_tiles(const GatedBackward<T> &a, int device, hipStream_t st) {
    constexpr int VK = Mfma<T>::VK;
    const GatedSplit &sp = a.split;
    const auto run = [&]<int B>() -> ttamd_status {
        constexpr int BK = BackwardTile<T, B>::BK, PF = BackwardTile<T, B>::PF;
        const int dx_n = (a.inner + B - 1) / B, dx = (a.rows + B - 1) / B * dx_n, dx_items = dx * (sp.x_splits ? 2 * sp.x_splits : 1);
        const int dw_n = (a.hidden + B - 1) / B, dw = (a.inner + B - 1) / B * dw_n, dw_items = dw * (sp.w_splits ? 2 * sp.w_splits : 2);
        using StK = Stager<T, B, BK, true, VK, PF>;
        using StM = Stager<T, B, BK, false, VK, PF>;
        constexpr size_t lds_k = TileEngine<T, B, B, BK, 2, 2, StK, StK>::kLdsBytes, lds_m = TileEngine<T, B, B, BK, 2, 2, StM, StM>::kLdsBytes;
        constexpr size_t lds = lds_k > lds_m ? lds_k : lds_m;
        static_assert(lds <= 48 * 1024, "within the default dynamic LDS limit");
        gated_backward_kernel<T, B><<<static_cast<unsigned>(dx_items + dw_items), kThreads, lds, st>>>(a, dx_items, dx, dx_n, dw, dw_n);
        TTAMD_HIP_CHECK(hipGetLastError());
        return TTAMD_OK;
    };
    if constexpr (sizeof(T) == 4) {
        if (sp.tile == 128) {
            if (ttamd_status s = run.template operator()<128>()) return s;
        } else if (ttamd_status s = run.template operator()<64>()) {
            return s;
        }
    } else {
        if (ttamd_status s = run.template operator()<64>()) return s;
    }
    PartSums<T> sums{};
    unsigned blocks = 0;
    const auto add = [&](int k, const T *src, T *out, int64_t n, int64_t stride, int parts) {
        if (!parts || !out) return;
        sums.job[k] = {src, out, n, stride, parts, static_cast<int>((n + 256 * VK - 1) / (256 * VK))};
        blocks += sums.job[k].blocks;
    };
    const int64_t x_n = static_cast<int64_t>(a.rows) * a.inner, w_n = static_cast<int64_t>(a.inner) * a.hidden;
    add(0, a.x_part, a.dx, x_n, x_n, 2 * sp.x_splits);
    add(1, a.w_part, a.dwg, w_n, 2 * w_n, sp.w_splits);
    add(2, a.w_part + w_n, a.dwu, w_n, 2 * w_n, sp.w_splits);
    add(3, a.b_part, a.dbg, a.hidden, 2 * a.hidden, sp.w_splits);
    add(4, a.b_part + a.hidden, a.dbu, a.hidden, 2 * a.hidden, sp.w_splits);
    if (blocks) {
        gated_add_parts_kernel<T><<<blocks, 256, 0, st>>>(sums);
        TTAMD_HIP_CHECK(hipGetLastError());
    }
    return TTAMD_OK;
}

template ttamd_status launch_gated_few_rows<float>(const GatedForward<float> &, int, hipStream_t);
template ttamd_status launch_gated_few_rows<double>(const GatedForward<double> &, int, hipStream_t);
template ttamd_status launch_gated_forward_tiles<float>(const GatedForward<float> &, int, hipStream_t);
template ttamd_status launch_gated_forward_tiles<double>(const GatedForward<double> &, int, hipStream_t);
template ttamd_status launch_gated_backward_tiles<float>(const GatedBackward<float> &, int, hipStream_t);
template ttamd_status launch_gated_backward_tiles<double>(const GatedBackward<double> &, int, hipStream_t);

}  // namespace ttamd
