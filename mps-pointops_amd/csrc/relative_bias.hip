// The bias that is learned by buckets of the relative position, as a dense
// tensor: out[h][i][j] = table[bucket(N - Q + i - j)][h], and its gradient.
//
// Both are bound by memory: the forward writes H Q N values, the backward
// reads them, each once.  The forward's blocks work out the few offsets of
// their rows once, in LDS, and copy from there.  In the backward a thread
// walks down a few neighbouring diagonals, whose offset does not change, so
// that the sums stay in registers and have a fixed order; each block adds its
// diagonals by bucket, and a second kernel the blocks.
//
// 16 x 2048 x 2048, float32 (268 MB each way): 42 us forward, 48 and 4 backward,
// 6.4 and 5.5 TB/s with what the last-level cache takes; a large copy has 4.7 to 5.1.
#include <algorithm>

#include "attention.hpp"

namespace pointops {
namespace attn {

bool read_buckets(const int32_t* edges, int n, int count, int64_t most, Buckets* out) {
    if (edges == nullptr || n < 1 || n > 255 || (count != n + 1 && count != 2 * (n + 1))) return false;
    out->n = n;
    out->count = count;
    for (int i = 0; i < n; ++i) {
        if (edges[i] < 1 || edges[i] > most || (i > 0 && edges[i] < edges[i - 1])) return false;
        out->edge[i] = edges[i];
    }
    return true;
}

namespace {

constexpr int kBiasRows = 64;    // of a block, or fewer where there are few blocks
constexpr int kBiasCols = 1024;  // of a block

// Threads write 16 bytes each along a row, at any alignment, and its last
// values one by one.
template <typename T>
__global__ __launch_bounds__(kThreads) void relative_bias_kernel(const Buckets bk, const T* __restrict__ table,
                                                                 T* __restrict__ out, int H, int Q, int N,
                                                                 int col_blocks, int block_rows) {
    constexpr int VEC = kPerFrag<T>, kWide = kBiasCols / VEC, kStep = kThreads / kWide;
    __shared__ int edges[255];
    __shared__ T values[kBiasRows + kBiasCols + VEC];  // entry x: offset base + rows - 1 - x
    const int h = blockIdx.x / col_blocks, j0 = static_cast<int>(blockIdx.x % col_blocks) * kBiasCols;
    const int i0 = blockIdx.y * block_rows, rows = min(block_rows, Q - i0), cols = min(kBiasCols, N - j0);
    const int base = N - Q + i0 - j0;  // offset of the first row and column
    for (int x = threadIdx.x; x < bk.n; x += kThreads) edges[x] = bk.edge[x];
    __syncthreads();
    for (int x = threadIdx.x; x < rows + cols - 1; x += kThreads)
        values[x] = table[static_cast<int64_t>(bucket_of(bk, edges, base + rows - 1 - x)) * H + h];
    __syncthreads();
    const int c = static_cast<int>(threadIdx.x) % kWide * VEC;
    if (c >= cols) return;
    for (int row = threadIdx.x / kWide; row < rows; row += kStep) {
        T* const dst = out + (static_cast<int64_t>(h) * Q + i0 + row) * N + j0 + c;
        T v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = values[rows - 1 - row + c + e];
        if (c + VEC <= cols) {
            typedef int words __attribute__((ext_vector_type(4), aligned(2)));
            words w;
            __builtin_memcpy(&w, v, sizeof w);
            *reinterpret_cast<words*>(dst) = w;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (c + e < cols) dst[e] = v[e];
        }
    }
}

constexpr int kDiagonals = 4;   // neighbouring ones of a thread
constexpr int kDiagRows = 64;   // rows of a block, or fewer where there are few blocks
constexpr int kDiagSpan = kThreads * kDiagonals;

// kDiagonals values at any address, read past the caches' order of use: what
// the forward has just written fills them, and the gradient is read once (16 x
// 2048 x 2048, float32, aligned rows: 87 us with ordinary loads, 52 with these; 48 =
// 5.5 TB/s since the buckets' bounds come from LDS).
template <typename T>
struct Values {
    T e[kDiagonals];
};
template <typename T>
__device__ __forceinline__ Values<T> read_once(const T* p) {
    typedef int words __attribute__((ext_vector_type(kDiagonals * sizeof(T) / 4), aligned(alignof(T))));
    return __builtin_bit_cast(Values<T>, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
}

// A thread's diagonals hold key less row = c .. c + 3, down the block's rows;
// part[h][block][bucket].
template <typename T>
__global__ __launch_bounds__(kThreads) void relative_bias_grad_kernel(const Buckets bk, const T* __restrict__ grad,
                                                                      int64_t stride_h, int64_t stride_i,
                                                                      float* __restrict__ part, int Q, int N, int block_rows) {
    __shared__ float sums[kDiagSpan];  // by falling diagonal, so rising offset
    const int h = blockIdx.z, i0 = blockIdx.y * block_rows, i_end = min(Q, i0 + block_rows);
    // The block's diagonals: those that meet its rows are -(i_end - 1) .. N - 1 - i0.
    const int c0 = static_cast<int>(blockIdx.x) * kDiagSpan - (i_end - 1);
    const int c = c0 + static_cast<int>(threadIdx.x) * kDiagonals;
    float sum[kDiagonals] = {};
    const T* const src = grad + h * stride_h + c;
    // Rows where some, and where all, of the diagonals lie inside.
    const int some = max(i0, -c - (kDiagonals - 1)), some_end = min(i_end, N - c);
    const int all = min(max(i0, -c), some_end), all_end = max(all, min(i_end, N - c - (kDiagonals - 1)));
    auto edge = [&](int from, int to) {
        for (int i = from; i < to; ++i)
#pragma unroll
            for (int e = 0; e < kDiagonals; ++e)
                if (c + e + i >= 0 && c + e + i < N) sum[e] += to_float(src[i * stride_i + i + e]);
    };
    edge(some, all);
#pragma unroll 8
    for (int i = all; i < all_end; ++i) {
        const auto v = read_once<T>(src + i * stride_i + i);
#pragma unroll
        for (int e = 0; e < kDiagonals; ++e) sum[e] += to_float(v.e[e]);
    }
    edge(all_end, some_end);
#pragma unroll
    for (int e = 0; e < kDiagonals; ++e) sums[kDiagSpan - 1 - (threadIdx.x * kDiagonals + e)] = sum[e];
    __syncthreads();
    // Diagonal c has offset N - Q - c: entry 0 is diagonal c0 + kDiagSpan - 1.
    const int64_t block = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
    float* const dst = part + (h * static_cast<int64_t>(gridDim.x) * gridDim.y + block) * bk.count;
    add_buckets(bk, bk.edge, sums, kDiagSpan, c0 + kDiagSpan - 1 - (N - Q), dst);
}

// The same where every row starts at a multiple of 16 bytes: a thread reads
// aligned pieces of V values, the same columns for V rows and V columns further
// for the next V, so that 2 V - 1 diagonals stay in its registers; its
// neighbour's share of them is added at the end.  16 x 2048 x 2048, float32: 48 us,
// where the kernel above took 60 to this one's 52.
template <typename T>
__global__ __launch_bounds__(kThreads) void relative_bias_grad_aligned_kernel(const Buckets bk, const T* __restrict__ grad,
                                                                              int64_t stride_h, int64_t stride_i,
                                                                              float* __restrict__ part, int Q, int N,
                                                                              int block_rows) {
    constexpr int V = kPerFrag<T>, kSpan = kThreads * V + V - 1;
    __shared__ float sums[kSpan];  // by falling diagonal, so rising offset
    const int h = blockIdx.z, i0 = blockIdx.y * block_rows, rows = min(block_rows, Q - i0);
    // Columns at the block's first row: from -block_rows on.
    const int first = static_cast<int>(blockIdx.x) * kThreads * V - block_rows;
    const int c0 = first + static_cast<int>(threadIdx.x) * V;
    float sum[2 * V - 1] = {};
    const T* const src = grad + h * stride_h + i0 * stride_i;
#pragma unroll 2
    for (int r = 0; r < block_rows; r += V) {
        const int col = c0 + r;
        i32x4 v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = i32x4{0, 0, 0, 0};
            if (col >= 0 && col < N && r + i < rows) v[i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(src + (r + i) * stride_i + col));
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e - i + V - 1] += element<T>(v[i], e);
    }
    // Column less row, both from the block's first: c0 - (V - 1) .. c0 + V - 1;
    // entry 0 is the last thread's last.
    float* const mine = sums + kSpan - 1 - (V - 1) - static_cast<int>(threadIdx.x) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) mine[-e] = sum[e + V - 1];
    if (threadIdx.x == 0) {
#pragma unroll
        for (int e = 1; e < V; ++e) mine[e] = 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int e = 1; e < V; ++e) mine[e] += sum[V - 1 - e];
    __syncthreads();
    // A diagonal c (column less the tensor's row) has offset N - Q - c.
    const int64_t block = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
    float* const dst = part + (h * static_cast<int64_t>(gridDim.x) * gridDim.y + block) * bk.count;
    add_buckets(bk, bk.edge, sums, kSpan, first + kThreads * V - 1 - i0 - (N - Q), dst);
}

// 32 lanes of parts for each of 8 buckets of a head.
constexpr int kJoinBuckets = 8;
template <typename T>
__global__ __launch_bounds__(kThreads) void join_buckets_kernel(const float* __restrict__ part, int B, int64_t blocks,
                                                                int count, const T* __restrict__ bias, T* __restrict__ grad) {
    constexpr int kLanes = 32, kBuckets = kJoinBuckets;
    __shared__ float sums[kLanes][kBuckets];
    const int H = gridDim.x, h = blockIdx.x, x = threadIdx.x % kBuckets, y = threadIdx.x / kBuckets;
    const int bucket = blockIdx.y * kBuckets + x;
    float all = 0.f;
    if (bucket < count)
        for (int b = 0; b < B; ++b) {
            const float* const src = part + (static_cast<int64_t>(b) * H + h) * blocks * count + bucket;
#pragma unroll 8
            for (int64_t i = y; i < blocks; i += kLanes) all += src[i * count];
        }
    sums[y][x] = all;
    __syncthreads();
    if (y == 0 && bucket < count) {
        all = sums[0][x];
#pragma unroll
        for (int i = 1; i < kLanes; ++i) all += sums[i][x];
        const int64_t at = static_cast<int64_t>(bucket) * H + h;
        if (bias != nullptr && to_float(bias[at]) == -kInf) all = 0.f;
        grad[at] = from_float<T>(all);
    }
}

template <typename T>
hipError_t launch_bias(const Buckets& bk, const void* table, void* out, int H, int Q, int N, hipStream_t stream) {
    const int col_blocks = (N + kBiasCols - 1) / kBiasCols;
    const int64_t x = static_cast<int64_t>(col_blocks) * H;
    const int rows = x * ((Q + kBiasRows - 1) / kBiasRows) >= 512 ? kBiasRows : kBiasRows / 8;
    const int64_t y = (static_cast<int64_t>(Q) + rows - 1) / rows;
    if (x > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(relative_bias_kernel<T>, dim3(static_cast<uint32_t>(x), static_cast<uint32_t>(y)), dim3(kThreads), 0,
                       stream, bk, static_cast<const T*>(table), static_cast<T*>(out), H, Q, N, col_blocks, rows);
    return hipGetLastError();
}

// Rows of a block, and the blocks of `span` columns and those rows.
int diagonal_rows(int64_t H, int64_t Q, int64_t N) {
    return H * ((Q + kDiagRows - 1) / kDiagRows) * ((N + kDiagSpan - 1) / kDiagSpan) >= 512 ? kDiagRows : kDiagRows / 4;
}
dim3 diagonal_grid(int64_t H, int64_t Q, int64_t N, int64_t span) {
    const int64_t rows = diagonal_rows(H, Q, N);
    return dim3(static_cast<uint32_t>((N + rows + span - 1) / span), static_cast<uint32_t>((Q + rows - 1) / rows),
                static_cast<uint32_t>(H));
}

// Sizes that the kernels' launches hold.
constexpr int64_t kMostRows = 65535 * int64_t(kBiasRows);  // a grid's second dimension
constexpr int64_t kBiasLimit = int64_t(1) << 22;
static_assert(kBiasRows == kDiagRows, "one limit for both directions");
bool bias_sizes(int64_t Q, int64_t N, int64_t H, int32_t type) {
    return Q >= 0 && N >= 0 && H >= 0 && Q <= kMostRows && N < kBiasLimit && H <= 65535 && type >= POINTOPS_F32 &&
           type <= POINTOPS_BF16;
}

}  // namespace

hipError_t join_buckets(const float* part, int B, int H, int64_t blocks, int count, int type, const void* bias, void* grad,
                        hipStream_t stream) {
    const dim3 grid(H, (count + kJoinBuckets - 1) / kJoinBuckets);
    switch (type) {
        case POINTOPS_F32:
            hipLaunchKernelGGL(join_buckets_kernel<float>, grid, dim3(kThreads), 0, stream, part, B, blocks, count,
                               static_cast<const float*>(bias), static_cast<float*>(grad));
            break;
        case POINTOPS_F16:
            hipLaunchKernelGGL(join_buckets_kernel<f16>, grid, dim3(kThreads), 0, stream, part, B, blocks, count,
                               static_cast<const f16*>(bias), static_cast<f16*>(grad));
            break;
        default:
            hipLaunchKernelGGL(join_buckets_kernel<bf16>, grid, dim3(kThreads), 0, stream, part, B, blocks, count,
                               static_cast<const bf16*>(bias), static_cast<bf16*>(grad));
    }
    return hipGetLastError();
}

}  // namespace attn
}  // namespace pointops

extern "C" {

hipError_t pointops_relative_bias(const void* table, const int32_t* edges, int32_t n_edges, int32_t buckets, int32_t type,
                                  void* out, int64_t H, int64_t Q, int64_t N, hipStream_t stream) {
    using namespace pointops::attn;
    Buckets bk;
    if (!bias_sizes(Q, N, H, type) || !read_buckets(edges, n_edges, buckets, int64_t(1) << 30, &bk))
        return hipErrorInvalidValue;
    if (H == 0 || Q == 0 || N == 0) return hipSuccess;
    if (table == nullptr || out == nullptr) return hipErrorInvalidValue;
    const int h = static_cast<int>(H), q = static_cast<int>(Q), n = static_cast<int>(N);
    switch (type) {
        case POINTOPS_F32: return launch_bias<float>(bk, table, out, h, q, n, stream);
        case POINTOPS_F16: return launch_bias<f16>(bk, table, out, h, q, n, stream);
        default: return launch_bias<bf16>(bk, table, out, h, q, n, stream);
    }
}

size_t pointops_relative_bias_backward_workspace_bytes(int64_t H, int64_t Q, int64_t N, int32_t buckets) {
    using namespace pointops::attn;
    if (!bias_sizes(Q, N, H, POINTOPS_F32) || Q == 0 || N == 0 || buckets < 0) return 0;
    const dim3 grid = diagonal_grid(H, Q, N, kDiagSpan);  // the narrowest blocks
    return static_cast<size_t>(H) * grid.x * grid.y * buckets * sizeof(float);
}

hipError_t pointops_relative_bias_backward(const void* grad, int64_t stride_h, int64_t stride_i, const int32_t* edges,
                                           int32_t n_edges, int32_t buckets, int32_t type, void* grad_table,
                                           void* workspace, int64_t H, int64_t Q, int64_t N, hipStream_t stream) {
    using namespace pointops::attn;
    Buckets bk;
    if (!bias_sizes(Q, N, H, type) || !read_buckets(edges, n_edges, buckets, int64_t(1) << 30, &bk))
        return hipErrorInvalidValue;
    if (H == 0) return hipSuccess;
    if (grad_table == nullptr || (Q > 0 && N > 0 && (grad == nullptr || workspace == nullptr))) return hipErrorInvalidValue;
    const int h = static_cast<int>(H), q = static_cast<int>(Q), n = static_cast<int>(N);
    float* const part = static_cast<float*>(workspace);
    if (Q == 0 || N == 0) return join_buckets(nullptr, 0, h, 0, bk.count, type, nullptr, grad_table, stream);
    const int per = type == POINTOPS_F32 ? 4 : 8;
    const bool aligned = reinterpret_cast<uintptr_t>(grad) % 16 == 0 && stride_h % per == 0 && stride_i % per == 0 && N % per == 0;
    const dim3 grid = diagonal_grid(H, Q, N, aligned ? kThreads * per : kDiagSpan);
    auto sums = [&](auto zero) {
        using T = decltype(zero);
        auto* const kernel = aligned ? relative_bias_grad_aligned_kernel<T> : relative_bias_grad_kernel<T>;
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, bk, static_cast<const T*>(grad), stride_h, stride_i, part,
                           q, n, diagonal_rows(H, Q, N));
        return hipGetLastError();
    };
    const hipError_t err = type == POINTOPS_F32 ? sums(float{}) : type == POINTOPS_F16 ? sums(f16{}) : sums(bf16{});
    if (err != hipSuccess) return err;
    return join_buckets(part, 1, h, static_cast<int64_t>(grid.x) * grid.y, bk.count, type, nullptr, grad_table, stream);
}

}  // extern "C"
