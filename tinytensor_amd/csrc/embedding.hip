// embedding.hip — rows of a table looked up by token, scaled, and the table's gradient (gfx950).
//
//   out[i] = scale * table[index[i]]            (an index outside the table: a row of zeros)
//   dtable[v] = scale * sum of dy[i] over the positions i with index[i] = v, in groups of ordered positions
// No counterpart in the reference; the layer stands in front of nn::Linear (nn/linear.cpp:42-50).
//
// Bound: HBM in both directions.  The gradient of a token is a sum over positions that lie anywhere, so the positions are
// first put in the order of their tokens (embedding_order_kernel), then every run of equal tokens is added up
// (embedding_sum_kernel, embedding_join_kernel): each row of dy is read once, each row of the gradient written once, and
// the order of every sum is fixed by the indices alone -- no atomics on floating point values.
#include "common.h"

namespace ttamd {
namespace {

template <typename T>
struct Row;
template <>
struct Row<float> {
    static constexpr int W = 4;
    typedef float vec_t __attribute__((ext_vector_type(4), aligned(4)));  // (rows of any length begin anywhere)
};
template <>
struct Row<double> {
    static constexpr int W = 2;
    typedef double vec_t __attribute__((ext_vector_type(2), aligned(8)));
};

template <bool I64>
__device__ __forceinline__ int64_t load_index(const void *index, int64_t i) {
    if constexpr (I64) return static_cast<const int64_t *>(index)[i];
    else return static_cast<const int32_t *>(index)[i];
}

// A wave sets a row to zero; the last vector is moved back to end with the row.
template <typename T>
__device__ __forceinline__ void zero_row(T *row, int64_t dim, int lane) {
    using V = typename Row<T>::vec_t;
    constexpr int W = Row<T>::W;
    if (dim < W) {
        if (lane < dim) row[lane] = T(0);
        return;
    }
    for (int64_t d = lane * W; d < dim; d += 64 * W) *reinterpret_cast<V *>(row + (d + W <= dim ? d : dim - W)) = V{};
}

// ---- forward ----------------------------------------------------------------------------------------------------------
// 2^lanes_log lanes own a row and walk it in vectors.  A row whose length is no multiple of the vector ends in a vector
// that is moved back to end with the row: its first elements are written twice, with the same values.  VEC = false: one
// element at a time, for tables whose columns are not neighbours (a transposed view) and rows shorter than a vector.
template <typename T, bool I64, bool VEC, bool NT>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const T *__restrict__ table, int64_t row_stride, int64_t col_stride,
                                                                const void *__restrict__ index, int64_t count, int64_t vocab, int64_t dim,
                                                                T scale, T *__restrict__ out, int lanes_log) {
    constexpr int W = VEC ? Row<T>::W : 1;
    using V = typename Row<T>::vec_t;
    const int lanes = 1 << lanes_log;
    const int64_t step = (static_cast<int64_t>(gridDim.x) * 256) >> lanes_log;
    const int lane = threadIdx.x & (lanes - 1);
    const int64_t nvec = (dim + W - 1) / W;
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> lanes_log; i < count; i += step) {
        const int64_t v = load_index<I64>(index, i);
        const bool ok = v >= 0 && v < vocab;
        const T *src = table + (ok ? v : 0) * row_stride;
        T *dst = out + i * dim;
#pragma unroll 4
        for (int64_t u = lane; u < nvec; u += lanes) {
            if constexpr (VEC) {
                const int64_t at = u * W + W <= dim ? u * W : dim - W;
                V x = {};
                if (ok) x = *reinterpret_cast<const V *>(src + at) * scale;
                if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<V *>(dst + at));
                else *reinterpret_cast<V *>(dst + at) = x;
            } else {
                dst[u] = ok ? src[u * col_stride] * scale : T(0);
            }
        }
    }
}

// ---- gradient: the order of the positions ------------------------------------------------------------------------------
// Workgroup b owns the tokens v with v % buckets == b (neighbouring tokens, often equally frequent, go to different
// workgroups) and finds its positions by reading every index: count * 4 or 8 bytes out of L2 a workgroup, which for all
// but the shortest rows is less than the time the rows themselves take, and spares the passes of a sort over the device.
// A stable counting sort: wave w counts the tokens in the w-th sixteenth of the positions (the count of a (token, wave)
// pair does not depend on the order of the additions), the counts are summed up in (token, wave) order, and the waves
// walk their positions again and hand out the places.  What lies in lower buckets is counted on the same walk, so the
// workgroups' places need no second kernel either.
// The order is by (bucket, token); all that the sums need is that equal tokens lie together.
constexpr int kOrderWaves = 16;
constexpr int kOrderThreads = 64 * kOrderWaves;
constexpr int kOrderTokens = 512;  // tokens of a bucket at most: their (token, wave) counters fill 32 KB of LDS

struct OrderArgs {
    const void *index;
    int64_t count, vocab;
    int bucket_log;   // log2 of the number of buckets
    int tokens;       // tokens a bucket has room for: ceil(vocab / buckets)
    int32_t *position, *token;  // [count] in the order of the tokens
    int32_t *total;   // [0]: positions whose index lies in the table; [1], [2]: 0
    uint8_t *absent;  // [buckets][tokens] 1 for a token that no position has, or null
};

constexpr int kBatch = 8;  // loads of 64 indices in flight: with one at a time a scan of 60000 indices took 27 us of waiting

constexpr int kListed = 252;  // positions of its bucket that a wave keeps in LDS; a wave that finds more reads its share again
// Counters, lists and the waves' sums together stay within the 64 KB that a launch may have without raising a limit.
static_assert(kOrderWaves * (kOrderTokens * sizeof(int32_t) + kListed * sizeof(int2) + 2 * sizeof(int32_t)) <= 64 * 1024, "LDS of the order kernel");

// The next kBatch x 64 positions of a wave's share: lane l's u-th token is that of position i0 + 64 u + l; -1 where there is
// none, or where the index names no row.
template <bool I64>
__device__ __forceinline__ void load_batch(const OrderArgs &a, int64_t i0, int64_t last, int lane, int (&v)[kBatch]) {
    int64_t x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const int64_t i = i0 + u * 64 + lane;
        x[u] = load_index<I64>(a.index, i < last ? i : last - 1);
    }
    const uint32_t vocab = static_cast<uint32_t>(a.vocab);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const uint32_t lo = static_cast<uint32_t>(x[u]);
        const bool small = !I64 || static_cast<uint64_t>(x[u]) >> 32 == 0;
        v[u] = small && lo < vocab ? static_cast<int>(lo) : -1;
    }
    if (i0 + kBatch * 64 > last) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (i0 + u * 64 + lane >= last) v[u] = -1;
    }
}

template <bool I64>
__global__ void __launch_bounds__(kOrderThreads) embedding_order_kernel(OrderArgs a) {
    extern __shared__ int32_t counters[];  // [tokens][kOrderWaves]
    __shared__ int32_t wave_sum[kOrderWaves], below_sum[kOrderWaves];
    __shared__ int2 listed[kOrderWaves][kListed];  // (position, token) in the order of the positions
    const int tid = threadIdx.x, lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int buckets = 1 << a.bucket_log, mine = blockIdx.x;
    const int cells = a.tokens * kOrderWaves;
    for (int i = tid; i < cells; i += kOrderThreads) counters[i] = 0;
    __syncthreads();
    const int64_t per = (a.count + kOrderWaves - 1) / kOrderWaves;
    const int64_t first = wave * per, last = first + per < a.count ? first + per : a.count;
    // Every workgroup looks at every index, so what a look costs counts: a comparison with the vocabulary, two with the
    // bucket, the rest on the scalar unit (30000 indices: 21 us with per-lane counts and a second scan).
    int below = 0, found = 0;
    int v[kBatch];
    for (int64_t i0 = first; i0 < last; i0 += kBatch * 64) {
        load_batch<I64>(a, i0, last, lane, v);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            // (-1 & (buckets - 1) is the last bucket, so it is told apart by its sign)
            const int b = v[u] < 0 ? buckets : v[u] & (buckets - 1);
            below += __popcll(__ballot(b < mine));
            const uint64_t in = __ballot(b == mine);
            if (in) {
                const int at = found + __popcll(in & ((1ull << lane) - 1));
                if (b == mine) {
                    atomicAdd(&counters[(v[u] >> a.bucket_log) * kOrderWaves + wave], 1);
                    if (at < kListed) listed[wave][at] = make_int2(static_cast<int>(i0 + u * 64 + lane), v[u]);
                }
                found += __popcll(in);
            }
        }
    }
    if (lane == 0) below_sum[wave] = below;
    __syncthreads();
    // exclusive sums over the cells: a thread adds up its share of neighbouring cells, the threads' totals are added in order
    const int share = (cells + kOrderThreads - 1) / kOrderThreads;
    const int c0 = tid * share, c1 = c0 + share < cells ? c0 + share : cells;
    int own = 0;
    for (int i = c0; i < c1; ++i) own += counters[i];
    int run = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(run, d, 64);
        if (lane >= d) run += o;
    }
    if (lane == 63) wave_sum[wave] = run;
    __syncthreads();
    int base = 0, in_bucket = 0;
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) {
        base += below_sum[w];
        in_bucket += wave_sum[w];
    }
    if (mine == buckets - 1 && tid == 0) {
        a.total[0] = base + in_bucket;
        a.total[1] = a.total[2] = 0;  // (the sums' lists of crossing runs)
    }
    int at = base + run - own;
    for (int w = 0; w < wave; ++w) at += wave_sum[w];
    for (int i = c0; i < c1; ++i) {
        const int n = counters[i];
        counters[i] = at;
        at += n;
    }
    __syncthreads();
    // Which tokens nothing has: a token's run is empty when its first cell and the next token's begin at one place.
    if (a.absent) {
        const int end = base + in_bucket;
        for (int t = tid; t < a.tokens; t += kOrderThreads)
            a.absent[static_cast<int64_t>(mine) * a.tokens + t] = counters[t * kOrderWaves] == (t + 1 < a.tokens ? counters[(t + 1) * kOrderWaves] : end);
    }
    __syncthreads();  // the cells are moved on from here
    const auto place = [&](bool in, int position, int token) {
        const int t = token >> a.bucket_log;
        uint64_t left = __ballot(in);
        while (left) {  // a round for each different token among the 64 positions
            const int lead = __builtin_ctzll(left);
            const int which = __builtin_amdgcn_readlane(t, lead);
            const uint64_t same = __ballot(in && t == which);
            const int cell = which * kOrderWaves + wave;
            const int next = counters[cell];
            if (in && t == which) {
                const int p = next + __popcll(same & ((1ull << lane) - 1));
                a.position[p] = position;
                a.token[p] = token;
            }
            if (lane == lead) counters[cell] = next + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the other lanes read the cell in a later round
            left &= ~same;
        }
    };
    if (found <= kListed) {
        for (int k = 0; k < found; k += 64) {
            const bool in = k + lane < found;
            const int2 e = in ? listed[wave][k + lane] : make_int2(0, 0);
            place(in, e.x, e.y);
        }
        return;
    }
    for (int64_t i0 = first; i0 < last; i0 += kBatch * 64) {
        load_batch<I64>(a, i0, last, lane, v);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            place(v[u] >= 0 && (v[u] & (buckets - 1)) == mine, static_cast<int>(i0 + u * 64 + lane), v[u]);
    }
}

// ---- gradient: the sums ------------------------------------------------------------------------------------------------
// A wave adds up the rows of a chunk of ordered positions, 64 vectors of columns wide.  A run of equal tokens that lies
// inside goes to the gradient; the part of one that began before is left in partial[2 c], of one that goes on in
// partial[2 c + 1].  Sums are held in 64 bits: the conversions cost nothing beside the loads, and a frequent token's sum
// over tens of thousands of rows keeps its last bits.
// Chunks of 64 positions leave a quarter of the parts of chunks of 16, but a quarter of the waves: plan_backward.
constexpr int kRows = 8;       // rows in flight ahead of those that are being added
constexpr int kZeroRows = 16;  // table rows a wave looks after when it fills those of absent tokens
constexpr int kJoinWaves = 16;
constexpr int kLongRun = 24;   // parts from which a whole workgroup joins a run

template <typename T>
struct SumArgs {
    const T *dy;
    T *grad;
    double *partial;  // [2 * chunks][dim]
    const int32_t *position, *token;
    int32_t *total;   // [0]: ordered positions; [1]: runs of few parts in `crossing`; [2]: runs of kLongRun and more
    int4 *crossing;   // [list] runs that begin in a chunk and go on: the chunk, the number of its parts, its token; those of
                      // few parts from the front, the others from the back
    int64_t list;     // chunks
    int64_t dim;
    int chunk;  // positions a chunk: 16 or 64
    double scale;
    int accumulate;
    // rows of absent tokens, set to zero by the workgroups behind the chunks' (none when accumulating)
    const uint8_t *absent;
    int bucket_log, tokens;
    int64_t vocab;
};

template <typename T, int W, bool NT = false>
__device__ __forceinline__ void load_row(const T *p, T (&x)[W]) {
    if constexpr (W == 1) {
        x[0] = *p;
    } else {
        typename Row<T>::vec_t v;
        if constexpr (NT) v = __builtin_nontemporal_load(reinterpret_cast<const typename Row<T>::vec_t *>(p));
        else v = *reinterpret_cast<const typename Row<T>::vec_t *>(p);
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] = v[k];
    }
}

template <typename T, int W>
__device__ __forceinline__ void write_gradient(const SumArgs<T> &a, int64_t token, int64_t col, const double (&sum)[W]) {
    T *g = a.grad + token * a.dim + col;
    T x[W];
    if (a.accumulate) load_row<T, W>(g, x);
#pragma unroll
    for (int k = 0; k < W; ++k) x[k] = static_cast<T>(a.accumulate ? static_cast<double>(x[k]) + sum[k] * a.scale : sum[k] * a.scale);
    if constexpr (W == 1) {
        *g = x[0];
    } else {
        typename Row<T>::vec_t v;
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = x[k];
        *reinterpret_cast<typename Row<T>::vec_t *>(g) = v;
    }
}

template <typename T, int W>
__device__ __forceinline__ void write_partial(const SumArgs<T> &a, int64_t part, int64_t col, const double (&sum)[W]) {
    double *p = a.partial + part * a.dim + col;
    if constexpr (W == 1) {
        *p = sum[0];
    } else {
#pragma unroll
        for (int k = 0; k < W; k += 2) {
            Row<double>::vec_t v;
            v[0] = sum[k];
            v[1] = sum[k + 1];
            *reinterpret_cast<Row<double>::vec_t *>(p + k) = v;
        }
    }
}

// A wave sets the rows of those among kZeroRows tokens to zero that nothing has (bucket by bucket, as `absent` lists them).
// It rides in the sums' launch: on its own the fill (131 MB of a 32000 x 1024 f32 table) held up the sums for 17 us, here
// its stores run under their loads.
template <typename T>
__device__ __forceinline__ void zero_absent(const SumArgs<T> &a, int64_t q0, int lane) {
    const int64_t all = static_cast<int64_t>(a.tokens) << a.bucket_log;
    const int64_t q = q0 + lane;
    const bool here = lane < kZeroRows && q < all;
    uint64_t left = __ballot(here && a.absent[here ? q : 0] != 0);
    while (left) {
        const int64_t at = q0 + __builtin_ctzll(left);
        left &= left - 1;
        const int64_t bucket = at / a.tokens;
        const int64_t row = ((at - bucket * a.tokens) << a.bucket_log) + bucket;
        if (row < a.vocab) zero_row(a.grad + row * a.dim, a.dim, lane);
    }
}

template <typename T, int W, bool NT>
__global__ void __launch_bounds__(64) embedding_sum_kernel(SumArgs<T> a) {
    const int64_t c = blockIdx.x;
    if (c >= a.list) {
        zero_absent(a, ((c - a.list) * gridDim.y + blockIdx.y) * kZeroRows, static_cast<int>(threadIdx.x));
        return;
    }
    const int total = a.total[0];
    const int64_t s0 = c * a.chunk;
    if (s0 >= total) return;
    const int n = total - s0 < a.chunk ? static_cast<int>(total - s0) : a.chunk;
    const int lane = threadIdx.x;
    // A row's last vector is moved back to end with the row: its first columns are then summed and written twice, the same
    // way.  (Lanes beyond the row's end stay and work on its last columns: every lane's position is read by the others.)
    const int64_t at = (static_cast<int64_t>(blockIdx.y) * 64 + lane) * W, col = at + W <= a.dim ? at : a.dim - W;
    const bool live = at < a.dim;
    // lane l knows the l-th position and token; lanes n and beyond repeat the last one
    const int mine = lane < n ? lane : n - 1;
    const int position = a.position[s0 + mine], token = a.token[s0 + mine];
    const int before = c > 0 ? a.token[s0 - 1] : -1;
    const int after = s0 + n < total ? a.token[s0 + n] : -1;
    T x[2][kRows][W];
    const auto load = [&](int i0, T (&to)[kRows][W]) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            load_row<T, W, NT>(a.dy + static_cast<int64_t>(__builtin_amdgcn_readlane(position, i0 + i)) * a.dim + col, to[i]);
    };
    double sum[W];
#pragma unroll
    for (int k = 0; k < W; ++k) sum[k] = 0;
    int cur = __builtin_amdgcn_readfirstlane(token);
    bool head = before == cur;
    const auto add = [&](int i0, const T (&from)[kRows][W]) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i0 + i >= n) break;
            const int t = __builtin_amdgcn_readlane(token, i0 + i);
            if (t != cur) {
                if (live) {
                    if (head) write_partial<T, W>(a, 2 * c, col, sum);
                    else write_gradient<T, W>(a, cur, col, sum);
                }
                head = false;
                cur = t;
#pragma unroll
                for (int k = 0; k < W; ++k) sum[k] = 0;
            }
#pragma unroll
            for (int k = 0; k < W; ++k) sum[k] += static_cast<double>(from[i][k]);
        }
    };
    load(0, x[0]);
    for (int i0 = 0; i0 < n; i0 += 2 * kRows) {  // (n <= 64 lanes: the lanes named below exist)
        load(i0 + kRows, x[1]);
        add(i0, x[0]);
        if (i0 + 2 * kRows < n) load(i0 + 2 * kRows, x[0]);
        add(i0 + kRows, x[1]);
    }
    if (!head && after == cur && blockIdx.y == 0) {
        // the following chunks that begin with the token: a block of neighbours, found by doubling and halving
        const int64_t chunks = (static_cast<int64_t>(total) + a.chunk - 1) / a.chunk;
        int64_t lo = c + 1, hi = c + 2;  // chunk lo begins with it
        while (hi < chunks && a.token[hi * a.chunk] == cur) {
            lo = hi;
            hi = c + 2 * (hi - c);
        }
        if (hi > chunks) hi = chunks;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (a.token[mid * a.chunk] == cur) lo = mid;
            else hi = mid;
        }
        if (lane == 0) {
            const int parts = static_cast<int>(lo - c + 1);
            const int64_t place = parts < kLongRun ? atomicAdd(&a.total[1], 1) : a.list - 1 - atomicAdd(&a.total[2], 1);
            a.crossing[place] = make_int4(static_cast<int>(c), parts, cur, 0);
        }
    }
    if (!live) return;
    if (head || after == cur) write_partial<T, W>(a, 2 * c + (head ? 0 : 1), col, sum);
    else write_gradient<T, W>(a, cur, col, sum);
}

// The sum of parts p0 .. p1 - 1 of the run that begins in chunk c.
template <typename T, int W>
__device__ __forceinline__ void add_parts(const SumArgs<T> &a, int64_t c, int64_t p0, int64_t p1, int64_t col, double (&sum)[W]) {
#pragma unroll
    for (int k = 0; k < W; ++k) sum[k] = 0;
#pragma unroll 8
    for (int64_t p = p0; p < p1; ++p) {
        const double *src = a.partial + (p == 0 ? 2 * c + 1 : 2 * (c + p)) * a.dim + col;
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += src[k];
    }
}

// The run that begins in chunk c and goes on: its parts are partial[2 c + 1] and partial[2 j] of the following chunks j
// that begin with its token.  A wave joins a run of few parts, a workgroup one of many, whose waves add
// contiguous shares, and the shares' sums are added in order.  (The f32 vector form keeps eight parts of four doubles in flight and
// spills 20 registers.)  The runs come in the order in which their chunks were listed,
// which changes from call to call and no result with it.
template <typename T, int W>
__global__ void __launch_bounds__(64 * kJoinWaves) embedding_join_kernel(SumArgs<T> a) {
    __shared__ double waves[kJoinWaves][64 * W];
    const int runs = a.total[1], long_runs = a.total[2];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t at = (static_cast<int64_t>(blockIdx.y) * 64 + lane) * W, col = at + W <= a.dim ? at : a.dim - W;
    const bool live = at < a.dim;
    double sum[W];
    for (int r = blockIdx.x; r < long_runs; r += gridDim.x) {
        const int4 run = a.crossing[a.list - 1 - r];
        const int per = (run.y + kJoinWaves - 1) / kJoinWaves;
        const int p0 = wave * per, p1 = p0 + per < run.y ? p0 + per : run.y;
        add_parts<T, W>(a, run.x, p0, live ? p1 : p0, col, sum);
#pragma unroll
        for (int k = 0; k < W; ++k) waves[wave][lane * W + k] = sum[k];
        __syncthreads();
        if (wave == 0 && live) {
            for (int v = 1; v < kJoinWaves; ++v)
#pragma unroll
                for (int k = 0; k < W; ++k) sum[k] += waves[v][lane * W + k];
            write_gradient<T, W>(a, run.z, col, sum);
        }
        __syncthreads();
    }
    for (int r = blockIdx.x * kJoinWaves + wave; r < runs; r += gridDim.x * kJoinWaves) {
        const int4 run = a.crossing[r];
        if (!live) continue;
        add_parts<T, W>(a, run.x, 0, run.y, col, sum);
        write_gradient<T, W>(a, run.z, col, sum);
    }
}

// ---- gradient of few positions: one launch -------------------------------------------------------------------------------
// With kFew positions at most a wave holds every index in two registers a lane and finds the positions of a token by two
// comparisons, so each wave sees to its kZeroRows rows of the table by itself: sums in the order of the positions, zeros where
// there is none.  (17 positions, 1096 rows of 97 doubles: three launches and their workspace take the host 18 us, one 12.)
constexpr int kFew = 128;
template <typename T, int W, bool I64>
__global__ void __launch_bounds__(64) embedding_few_kernel(SumArgs<T> a, const void *index, int count) {
    const int lane = threadIdx.x;
    int v[kFew / 64];
#pragma unroll
    for (int u = 0; u < kFew / 64; ++u) {
        const int i = u * 64 + lane;
        const int64_t x = i < count ? load_index<I64>(index, i) : -1;
        v[u] = x >= 0 && x < a.vocab ? static_cast<int>(x) : -1;
    }
    const int64_t at = (static_cast<int64_t>(blockIdx.y) * 64 + lane) * W, col = at + W <= a.dim ? at : a.dim - W;
    const bool live = at < a.dim;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kZeroRows, last = first + kZeroRows < a.vocab ? first + kZeroRows : a.vocab;
    for (int64_t row = first; row < last; ++row) {
        uint64_t with[kFew / 64], any = 0;
#pragma unroll
        for (int u = 0; u < kFew / 64; ++u) any |= with[u] = __ballot(v[u] == static_cast<int>(row));
        if (!any) {
            if (live && !a.accumulate) {
#pragma unroll
                for (int k = 0; k < W; ++k) a.grad[row * a.dim + col + k] = T(0);
            }
            continue;
        }
        double sum[W];
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] = 0;
#pragma unroll
        for (int u = 0; u < kFew / 64; ++u)
            while (with[u]) {  // four rows in flight
                T x[4][W];
                const uint64_t four = with[u];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int p = with[u] ? __builtin_ctzll(with[u]) : __builtin_ctzll(four);
                    with[u] &= with[u] - 1;
                    load_row<T, W>(a.dy + static_cast<int64_t>(u * 64 + p) * a.dim + col, x[i]);
                }
                const int n = __popcll(four);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < n) {
#pragma unroll
                        for (int k = 0; k < W; ++k) sum[k] += static_cast<double>(x[i][k]);
                    }
            }
        if (live) write_gradient<T, W>(a, row, col, sum);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------
struct BackwardPlan {
    int bucket_log, tokens, chunk;
    int64_t chunks;
    size_t position, token, total, crossing, absent, partial, bytes;  // byte offsets into the workspace
};

BackwardPlan plan_backward(size_t item, int64_t count, int64_t vocab, int64_t dim) {
    BackwardPlan p{};
    // 256 buckets, a workgroup for each CU; more where a bucket's tokens would not fit the counters, fewer for tiny tables
    p.bucket_log = 8;
    while (p.bucket_log > 0 && (int64_t(1) << (p.bucket_log - 1)) >= vocab) --p.bucket_log;
    while ((vocab + (int64_t(1) << p.bucket_log) - 1) >> p.bucket_log > kOrderTokens) ++p.bucket_log;
    p.tokens = static_cast<int>((vocab + (int64_t(1) << p.bucket_log) - 1) >> p.bucket_log);
    const int64_t slab = 64 * (16 / static_cast<int64_t>(item));
    p.chunk = count / 64 * ((dim + slab - 1) / slab) >= 2048 ? 64 : 16;
    p.chunks = (count + p.chunk - 1) / p.chunk;
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    p.position = 0;
    p.token = p.position + up(static_cast<size_t>(count) * 4);
    p.total = p.token + up(static_cast<size_t>(count) * 4);
    p.crossing = p.total + 256;
    p.absent = p.crossing + up(static_cast<size_t>(p.chunks) * sizeof(int4));
    p.partial = p.absent + up(static_cast<size_t>(p.tokens) << p.bucket_log);
    p.bytes = p.partial + static_cast<size_t>(2 * p.chunks) * static_cast<size_t>(dim) * sizeof(double);
    return p;
}

template <typename T>
ttamd_status launch_forward(int64_t count, int64_t vocab, int64_t dim, const void *index, bool index64, const void *table,
                            int64_t row_stride, int64_t col_stride, double scale, void *out, hipStream_t st) {
    const bool vec = col_stride == 1 && dim >= Row<T>::W;
    const int64_t nvec = vec ? (dim + Row<T>::W - 1) / Row<T>::W : dim;
    int lanes_log = 0;
    while (lanes_log < 6 && (int64_t(1) << lanes_log) < nvec) ++lanes_log;
    const int64_t blocks = ((count << lanes_log) + 255) / 256;
    const dim3 grid(static_cast<unsigned>(blocks < (1 << 22) ? blocks : (1 << 22)));
    const auto run = [&](auto kernel) {
        kernel<<<grid, 256, 0, st>>>(static_cast<const T *>(table), row_stride, col_stride, index, count, vocab, dim, static_cast<T>(scale),
                                     static_cast<T *>(out), lanes_log);
    };
    // a result beyond half of the 256 MB Infinity Cache is stored past it (65536 x 512 f32: 32.9 -> 30.1 us)
    const bool beyond = static_cast<double>(count) * dim * sizeof(T) >= 128.0 * (1 << 20);
    if (vec && beyond) index64 ? run(embedding_forward_kernel<T, true, true, true>) : run(embedding_forward_kernel<T, false, true, true>);
    else if (vec) index64 ? run(embedding_forward_kernel<T, true, true, false>) : run(embedding_forward_kernel<T, false, true, false>);
    else index64 ? run(embedding_forward_kernel<T, true, false, false>) : run(embedding_forward_kernel<T, false, false, false>);
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

template <typename T>
ttamd_status launch_backward(int64_t count, int64_t vocab, int64_t dim, const void *grad_out, const void *index, bool index64, double scale,
                             int accumulate, void *grad, void *workspace, hipStream_t st) {
    // (columns that two lanes write may not be added to what is there twice)
    const bool vec = accumulate ? dim % Row<T>::W == 0 : dim >= Row<T>::W;
    const int w = vec ? Row<T>::W : 1;
    const int64_t slabs = (dim + 64 * w - 1) / (64 * w);
    if (count <= kFew) {
        const SumArgs<T> a{static_cast<const T *>(grad_out), static_cast<T *>(grad), nullptr, nullptr, nullptr, nullptr, nullptr, 0, dim, 0, scale,
                           accumulate, nullptr, 0, 0, vocab};
        const dim3 grid(static_cast<unsigned>((vocab + kZeroRows - 1) / kZeroRows), static_cast<unsigned>(slabs));
        const auto run = [&](auto kernel) { kernel<<<grid, 64, 0, st>>>(a, index, static_cast<int>(count)); };
        if (vec) index64 ? run(embedding_few_kernel<T, Row<T>::W, true>) : run(embedding_few_kernel<T, Row<T>::W, false>);
        else index64 ? run(embedding_few_kernel<T, 1, true>) : run(embedding_few_kernel<T, 1, false>);
        TTAMD_HIP_CHECK(hipGetLastError());
        return TTAMD_OK;
    }
    const BackwardPlan p = plan_backward(sizeof(T), count, vocab, dim);
    char *ws = static_cast<char *>(workspace);
    uint8_t *absent = accumulate ? nullptr : reinterpret_cast<uint8_t *>(ws + p.absent);
    const OrderArgs o{index, count, vocab, p.bucket_log, p.tokens, reinterpret_cast<int32_t *>(ws + p.position),
                      reinterpret_cast<int32_t *>(ws + p.token), reinterpret_cast<int32_t *>(ws + p.total), absent};
    const size_t lds = static_cast<size_t>(p.tokens) * kOrderWaves * sizeof(int32_t);
    if (index64) embedding_order_kernel<true><<<1u << p.bucket_log, kOrderThreads, lds, st>>>(o);
    else embedding_order_kernel<false><<<1u << p.bucket_log, kOrderThreads, lds, st>>>(o);
    TTAMD_HIP_CHECK(hipGetLastError());
    const SumArgs<T> a{static_cast<const T *>(grad_out), static_cast<T *>(grad), reinterpret_cast<double *>(ws + p.partial), o.position,
                       o.token, o.total, reinterpret_cast<int4 *>(ws + p.crossing), p.chunks, dim, p.chunk, scale, accumulate,
                       absent, p.bucket_log, p.tokens, vocab};
    const int64_t fill = accumulate ? 0 : ((static_cast<int64_t>(p.tokens) << p.bucket_log) + kZeroRows * slabs - 1) / (kZeroRows * slabs);
    const dim3 grid(static_cast<unsigned>(p.chunks + fill), static_cast<unsigned>(slabs));
    // rows beyond half of the 256 MB Infinity Cache are loaded past it (65536 x 1024 f32: 216 -> 187 us in all; 8192 x 1024:
    // 44.3 without, 45.3 with)
    const bool beyond = static_cast<double>(count) * dim * sizeof(T) > 128.0 * (1 << 20);
    if (vec && beyond) embedding_sum_kernel<T, Row<T>::W, true><<<grid, 64, 0, st>>>(a);
    else if (vec) embedding_sum_kernel<T, Row<T>::W, false><<<grid, 64, 0, st>>>(a);
    else embedding_sum_kernel<T, 1, false><<<grid, 64, 0, st>>>(a);
    TTAMD_HIP_CHECK(hipGetLastError());
    const int64_t groups = (p.chunks + kJoinWaves - 1) / kJoinWaves;
    const dim3 join(static_cast<unsigned>(groups < 256 ? groups : 256), grid.y);
    if (vec) embedding_join_kernel<T, Row<T>::W><<<join, 64 * kJoinWaves, 0, st>>>(a);
    else embedding_join_kernel<T, 1><<<join, 64 * kJoinWaves, 0, st>>>(a);
    TTAMD_HIP_CHECK(hipGetLastError());
    return TTAMD_OK;
}

ttamd_status check_shape(const char *what, ttamd_dtype dtype, int64_t count, int64_t vocab, int64_t dim) {
    if (dtype != TTAMD_F32 && dtype != TTAMD_F64) {
        set_error("%s: floating point dtypes only", what);
        return TTAMD_ERR_UNSUPPORTED_DTYPE;
    }
    // (the column slabs of a row are a grid's second dimension: dim / 64 below 2^16)
    if (count < 0 || vocab < 1 || dim < 1 || count > 0x7fffffffLL || vocab > (int64_t(1) << 28) || dim > (1 << 21)) {
        set_error("%s: count %lld, vocab %lld, dim %lld: fewer than 2^31 indices, 1 to 2^28 rows of 1 to 2^21 elements", what,
                  static_cast<long long>(count), static_cast<long long>(vocab), static_cast<long long>(dim));
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    return TTAMD_OK;
}

ttamd_status check_index_dtype(const char *what, ttamd_dtype index_dtype) {
    if (index_dtype == TTAMD_I32 || index_dtype == TTAMD_I64) return TTAMD_OK;
    set_error("%s: indices are i32 or i64 (dtype code %d)", what, static_cast<int>(index_dtype));
    return TTAMD_ERR_UNSUPPORTED_DTYPE;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" {

ttamd_status ttamd_embedding_forward(int device, ttamd_dtype dtype, ttamd_dtype index_dtype, int64_t count, int64_t vocab, int64_t dim,
                                     const void *index, const void *table, int64_t row_stride, int64_t col_stride, double scale, void *out,
                                     void *stream) {
    const char *const what = "embedding";
    if (ttamd_status s = check_shape(what, dtype, count, vocab, dim)) return s;
    if (ttamd_status s = check_index_dtype(what, index_dtype)) return s;
    if (row_stride < 0 || col_stride < 0 || row_stride > (int64_t(1) << 32) || col_stride > (int64_t(1) << 32)) {
        set_error("%s: strides %lld, %lld of the table: 0 to 2^32", what, static_cast<long long>(row_stride), static_cast<long long>(col_stride));
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    const size_t e = dtype_size(dtype);
    if (count > 0 && (!index || !table || !out)) {
        set_error("%s: NULL data pointer", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(table, e) || misaligned(out, e) || misaligned(index, dtype_size(index_dtype))) {
        set_error("%s: pointers must be aligned to the element size", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (ttamd_status s = check_disjoint(what, {dense_extent("the result", out, count * dim, e)},
                                        {{"the table", table, vocab, dim, row_stride, col_stride, e}, dense_extent("the indices", index, count, dtype_size(index_dtype))}))
        return s;
    if (ttamd_status s = use_device(device)) return s;
    if (count == 0) return TTAMD_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool i64 = index_dtype == TTAMD_I64;
    if (dtype == TTAMD_F32) return launch_forward<float>(count, vocab, dim, index, i64, table, row_stride, col_stride, scale, out, st);
    return launch_forward<double>(count, vocab, dim, index, i64, table, row_stride, col_stride, scale, out, st);
}

ttamd_status ttamd_embedding_backward_workspace(ttamd_dtype dtype, int64_t count, int64_t vocab, int64_t dim, size_t *bytes) {
    if (ttamd_status s = check_shape("embedding_backward", dtype, count, vocab, dim)) return s;
    if (!bytes) {
        set_error("embedding_backward: bytes is NULL");
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    // Each of vocab / kOrderTokens workgroups looks at every index: half a second's work at this bound.
    if (count > kFew && vocab > (1 << 17) && count > (int64_t(1) << 48) / vocab) {
        set_error("embedding_backward: %lld positions of a table of %lld rows: beyond 2^17 rows, positions x rows up to 2^48",
                  static_cast<long long>(count), static_cast<long long>(vocab));
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    *bytes = count <= kFew ? 0 : plan_backward(dtype_size(dtype), count, vocab, dim).bytes;
    return TTAMD_OK;
}

ttamd_status ttamd_embedding_backward(int device, ttamd_dtype dtype, ttamd_dtype index_dtype, int64_t count, int64_t vocab, int64_t dim,
                                      const void *grad_out, const void *index, double scale, int accumulate, void *grad_table,
                                      void *workspace, size_t workspace_bytes, void *stream) {
    const char *const what = "embedding_backward";
    size_t need = 0;
    if (ttamd_status s = ttamd_embedding_backward_workspace(dtype, count, vocab, dim, &need)) return s;
    if (ttamd_status s = check_index_dtype(what, index_dtype)) return s;
    const size_t e = dtype_size(dtype);
    if (!grad_table || (need > 0 && !workspace) || (count > 0 && (!index || !grad_out))) {
        set_error("%s: NULL data pointer", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(grad_out, e) || misaligned(grad_table, e) || misaligned(index, dtype_size(index_dtype)) || (need > 0 && misaligned(workspace, 16))) {
        set_error("%s: pointers must be aligned to the element size, the workspace to 16 bytes", what);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
        return TTAMD_ERR_INVALID_ARGUMENT;
    }
    if (ttamd_status s = check_disjoint(what, {dense_extent("the gradient", grad_table, vocab * dim, e), dense_extent("the workspace", workspace, static_cast<int64_t>(need), 1)},
                                        {dense_extent("grad_out", grad_out, count * dim, e), dense_extent("the indices", index, count, dtype_size(index_dtype))}))
        return s;
    if (ttamd_status s = use_device(device)) return s;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool i64 = index_dtype == TTAMD_I64;
    if (dtype == TTAMD_F32) return launch_backward<float>(count, vocab, dim, grad_out, index, i64, scale, accumulate, grad_table, workspace, st);
    return launch_backward<double>(count, vocab, dim, grad_out, index, i64, scale, accumulate, grad_table, workspace, st);
}

}  // extern "C"
