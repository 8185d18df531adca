// The bias that is learned by buckets of the relative position, as a dense
// tensor: out[h][i][j] = table[bucket(N - Q + i - j)][h], and its gradient.
//
// Both are bound by memory: the forward writes H Q N values, the backward
// reads them, each once.  The forward's blocks work out the few offsets of
// their rows once, in LDS, and copy from there.  In the backward a thread
// walks down a few neighbouring diagonals, whose offset does not change, so
// that the sums stay in registers and have a fixed order; a second kernel adds
// the diagonals of each bucket.
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

constexpr int kBiasRows = 64;    // of a block
constexpr int kBiasCols = 1024;  // of a block

// VEC values a store (rows are a multiple of that).
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void relative_bias_kernel(const Buckets bk, const T* __restrict__ table,
                                                                 T* __restrict__ out, int H, int Q, int N,
                                                                 int col_blocks) {
    __shared__ int edges[255];
    __shared__ T values[kBiasRows + kBiasCols];  // of offset base + kBiasRows - 1 - x
    const int h = blockIdx.x / col_blocks, j0 = static_cast<int>(blockIdx.x % col_blocks) * kBiasCols;
    const int i0 = blockIdx.y * kBiasRows, rows = min(kBiasRows, Q - i0), cols = min(kBiasCols, N - j0);
    const int base = N - Q + i0 - j0;  // offset of the first row and column
    for (int x = threadIdx.x; x < bk.n; x += kThreads) edges[x] = bk.edge[x];
    __syncthreads();
    for (int x = threadIdx.x; x < rows + cols - 1; x += kThreads)
        values[x] = table[static_cast<int64_t>(bucket_of(bk, edges, base + rows - 1 - x)) * H + h];
    __syncthreads();
    T* const dst = out + (static_cast<int64_t>(h) * Q + i0) * N + j0;
    const int per = cols / VEC;
    // Threads along a row, then down the rows.
    const int wide = kBiasCols / VEC, step = max(1, kThreads / wide);
    for (int row = threadIdx.x / wide; row < rows; row += step)
        for (int c = threadIdx.x % wide; c < per; c += kThreads) {
            T v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = values[rows - 1 - row + c * VEC + e];
            __builtin_memcpy(__builtin_assume_aligned(dst + static_cast<int64_t>(row) * N + c * VEC, VEC * sizeof(T)), v,
                             sizeof v);
        }
}

constexpr int kDiagonals = 4;   // neighbouring ones of a thread
constexpr int kDiagRows = 128;  // rows of a block

// part[h][row block][offset + Q - 1]: a thread's diagonals hold key less row
// = c .. c + 3.
template <typename T>
__global__ __launch_bounds__(kThreads) void relative_bias_grad_kernel(const T* __restrict__ grad, int64_t stride_h,
                                                                      int64_t stride_i, float* __restrict__ part, int Q,
                                                                      int N) {
    const int h = blockIdx.z, i0 = blockIdx.y * kDiagRows, i_end = min(Q, i0 + kDiagRows);
    const int entries = Q + N - 1;
    const int c = static_cast<int>(blockIdx.x * kThreads + threadIdx.x) * kDiagonals - (Q - 1);
    if (c >= N) return;
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
        T v[kDiagonals];
        __builtin_memcpy(v, src + i * stride_i + i, sizeof v);
#pragma unroll
        for (int e = 0; e < kDiagonals; ++e) sum[e] += to_float(v[e]);
    }
    edge(all_end, some_end);
    float* const dst = part + (static_cast<int64_t>(h) * gridDim.y + blockIdx.y) * entries;
#pragma unroll
    for (int e = 0; e < kDiagonals; ++e)
        if (c + e < N) dst[N - 1 - (c + e)] = sum[e];  // offset N - Q - c
}

// One block a bucket and head.
template <typename T>
__global__ __launch_bounds__(kThreads) void bucket_sums_kernel(const Buckets bk, const float* __restrict__ part, int B,
                                                               int blocks, int entries, int zero,
                                                               T* __restrict__ grad) {
    __shared__ float waves[kWaves];
    const int H = gridDim.x, h = blockIdx.x, bucket = blockIdx.y, side = bk.n + 1, e = bucket % side;
    const bool two_sided = bk.count > side, later = bucket >= side;
    // The bucket's distances, then its entries.  The last one of a side has no
    // end; the first also takes later keys that have no buckets of their own.
    const int d_low = e == 0 ? 0 : bk.edge[e - 1];
    int64_t low, high;
    if (later) {
        low = e == bk.n ? 0 : static_cast<int64_t>(zero) - (bk.edge[e] - 1);
        high = static_cast<int64_t>(zero) - max(d_low, 1);
    } else {
        low = e == 0 && !two_sided ? 0 : static_cast<int64_t>(zero) + d_low;
        high = e == bk.n ? entries - 1 : static_cast<int64_t>(zero) + bk.edge[e] - 1;
    }
    low = max(low, int64_t(0));
    high = min(high, static_cast<int64_t>(entries) - 1);
    float all = 0.f;
    if (low <= high) {
        const int64_t count = high - low + 1, total = count * blocks;
        for (int b = 0; b < B; ++b) {
            const float* const src = part + (static_cast<int64_t>(b) * H + h) * blocks * entries + low;
            int64_t at = threadIdx.x;
            int64_t block = at / count, rest = at % count;
            const int64_t step = kThreads / count, left = kThreads % count;
            for (; at < total; at += kThreads) {
                all += src[block * entries + rest];
                block += step;
                rest += left;
                if (rest >= count) {
                    rest -= count;
                    ++block;
                }
            }
        }
    }
    all = wave_sum(all);
    if (lane_id() == 0) waves[threadIdx.x / kWave] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        float sum = 0.f;
        for (int w = 0; w < kWaves; ++w) sum += waves[w];
        grad[static_cast<int64_t>(bucket) * H + h] = from_float<T>(sum);
    }
}

template <typename T>
hipError_t launch_bias(const Buckets& bk, const void* table, void* out, int H, int Q, int N, hipStream_t stream) {
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    const int col_blocks = (N + kBiasCols - 1) / kBiasCols;
    const int64_t x = static_cast<int64_t>(col_blocks) * H, y = (static_cast<int64_t>(Q) + kBiasRows - 1) / kBiasRows;
    if (x > INT32_MAX || y > 65535) return hipErrorInvalidValue;
    const dim3 grid(static_cast<uint32_t>(x), static_cast<uint32_t>(y));
    const T* const src = static_cast<const T*>(table);
    T* const dst = static_cast<T*>(out);
    if (N % VEC == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0)
        hipLaunchKernelGGL((relative_bias_kernel<T, VEC>), grid, dim3(kThreads), 0, stream, bk, src, dst, H, Q, N, col_blocks);
    else
        hipLaunchKernelGGL((relative_bias_kernel<T, 1>), grid, dim3(kThreads), 0, stream, bk, src, dst, H, Q, N, col_blocks);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_diagonals(const void* grad, int64_t stride_h, int64_t stride_i, float* part, int H, int Q, int N,
                            hipStream_t stream) {
    const int per = kThreads * kDiagonals;
    const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(Q) + N - 1 + per - 1) / per),
                    static_cast<uint32_t>((Q + kDiagRows - 1) / kDiagRows), static_cast<uint32_t>(H));
    hipLaunchKernelGGL(relative_bias_grad_kernel<T>, grid, dim3(kThreads), 0, stream, static_cast<const T*>(grad), stride_h,
                       stride_i, part, Q, N);
    return hipGetLastError();
}

// Sizes that the kernels' launches hold.
constexpr int64_t kBiasLimit = int64_t(1) << 22;
bool bias_sizes(int64_t Q, int64_t N, int64_t H, int32_t type) {
    return Q >= 0 && N >= 0 && H >= 0 && Q < kBiasLimit && N < kBiasLimit && H <= 65535 && type >= POINTOPS_F32 &&
           type <= POINTOPS_BF16;
}

}  // namespace

hipError_t bucket_sums(const Buckets& bk, const float* part, int B, int H, int blocks, int entries, int zero, int type,
                       void* grad, hipStream_t stream) {
    const dim3 grid(H, bk.count);
    switch (type) {
        case POINTOPS_F32:
            hipLaunchKernelGGL(bucket_sums_kernel<float>, grid, dim3(kThreads), 0, stream, bk, part, B, blocks, entries, zero,
                               static_cast<float*>(grad));
            break;
        case POINTOPS_F16:
            hipLaunchKernelGGL(bucket_sums_kernel<f16>, grid, dim3(kThreads), 0, stream, bk, part, B, blocks, entries, zero,
                               static_cast<f16*>(grad));
            break;
        default:
            hipLaunchKernelGGL(bucket_sums_kernel<bf16>, grid, dim3(kThreads), 0, stream, bk, part, B, blocks, entries, zero,
                               static_cast<bf16*>(grad));
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

size_t pointops_relative_bias_backward_workspace_bytes(int64_t H, int64_t Q, int64_t N) {
    using namespace pointops::attn;
    if (!bias_sizes(Q, N, H, POINTOPS_F32) || Q == 0 || N == 0) return 0;
    return static_cast<size_t>(H) * ((Q + kDiagRows - 1) / kDiagRows) * (Q + N - 1) * sizeof(float);
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
    if (Q == 0 || N == 0) return bucket_sums(bk, nullptr, 0, h, 0, 0, 0, type, grad_table, stream);
    hipError_t err;
    switch (type) {
        case POINTOPS_F32: err = launch_diagonals<float>(grad, stride_h, stride_i, part, h, q, n, stream); break;
        case POINTOPS_F16: err = launch_diagonals<f16>(grad, stride_h, stride_i, part, h, q, n, stream); break;
        default: err = launch_diagonals<bf16>(grad, stride_h, stride_i, part, h, q, n, stream);
    }
    if (err != hipSuccess) return err;
    return bucket_sums(bk, part, 1, h, (q + kDiagRows - 1) / kDiagRows, q + n - 1, q - 1, type, grad_table, stream);
}

}  // extern "C"
