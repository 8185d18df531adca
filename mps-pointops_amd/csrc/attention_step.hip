// Attention of one or a few new queries over a cache: the queries stand at the
// last positions of their cloud's length and see the keys before them, within
// the window, and the first ones.
//
// Bound by reading the part of the cache that is seen, once: all query heads
// of a key head (and all new queries) share one pass as up to 32 columns of
// the matrix products.  Each wave takes 32 keys at a time for itself, keys
// straight from memory into the product's registers, values through its own
// piece of LDS (for the transposing read), without a barrier in the loop.  The
// keys are split over the block's waves and, where the batch is small, over
// blocks, whose maxima, sums and outputs (32-bit) a second kernel joins.
//
// As the products wait for memory, 16-bit weights keep their bits: values are
// multiplied by the rounded weights and by what the rounding left, so that outputs
// carry the result's rounding alone (float16's fill its range for it; bfloat16, error against 64 bits over one
// rounding's: 1.35 -> 1.0; 4 x 65536 keys, 32 heads over 8 of 128, 166.8 -> 168.7 us,
// 4 x 2048, 8 heads over 2 of 64, window 512, 12.1 -> 12.6).
#include <algorithm>

#include "attention.hpp"

namespace pointops {
namespace attn {
namespace {

constexpr int kTile = 32;  // keys of a wave at a time; queries of a block

// Waves of a block: 8 where all that is seen is 32 tiles or fewer, which are
// then one block's work and need no join, 4 otherwise (4 x 65536 keys, 32 heads
// over 8 of 128, bfloat16: 171 us by 4 waves, 183 by 8) and for 32-bit values,
// whose tiles take twice the LDS.
constexpr int kShortTiles = 32;

// The tiles that a block of rows sees: the first keys', then the window's.
struct Tiles {
    int first, low, count;
    __device__ __forceinline__ int key(int index) const {
        return (index < first ? index : index - first + low) * kTile;
    }
};

template <typename T, int DP, bool VEC, int WAVES>
__global__ __launch_bounds__(kWave * WAVES, sizeof(T) == 4 ? 1 : 2) void attention_step_kernel(
    const Args a, T* __restrict__ out, float* __restrict__ part, int row_blocks, int splits) {
    using TileT = Tile<T, DP>;
    constexpr int kWaves = WAVES, kThreads = kWave * kWaves;
    constexpr int kOut = DP / 32, kPerRow = DP * static_cast<int>(sizeof(T)) / 16, kPieces = kTile * kPerRow / kWave;
    constexpr int kSumStride = DP + 4;
    constexpr int kTileBytes = kTile * TileT::kStride;
    constexpr int kSumBytes = kTile * kSumStride * 4;
    __shared__ char lds[kWaves * kTileBytes > kSumBytes ? kWaves * kTileBytes : kSumBytes];
    __shared__ float tops[kWaves][kTile], totals[kWaves][kTile];
    extern __shared__ float table[];  // [buckets][32 rows], then the buckets of 0 .. reach, then the edges

    const int lane = lane_id(), half = lane / 32, col = lane % 32, wave = uniform(threadIdx.x / kWave);
    const int group = a.H / a.G, total = a.Q * group;
    const uint32_t blk = blockIdx.x;
    const int split = static_cast<int>(blk % splits);
    const int unit = static_cast<int>(blk / splits), r0 = unit % row_blocks * kTile;
    const int bg = unit / row_blocks, b = bg / a.G, g = bg % a.G;
    const int len = a.length(b), shift = len - a.Q;
    const int rows = min(kTile, total - r0);

    const int p_first = max(shift + r0 / group, 0), p_last = shift + (r0 + rows - 1) / group;
    Tiles tiles{0, 0, 0};
    if (p_first <= p_last) {
        tiles.first = (seen_first(a, p_last, len) + kTile - 1) / kTile;
        tiles.low = max(tiles.first, seen_low(a, p_first) / kTile);
        tiles.count = max(tiles.first, tiles.first + p_last / kTile + 1 - tiles.low);
    }
    const int begin = static_cast<int>(static_cast<int64_t>(tiles.count) * split / splits);
    const int end = static_cast<int>(static_cast<int64_t>(tiles.count) * (split + 1) / splits);

    const int r = r0 + col, i = r / group, h = g * group + r % group, p = shift + i;
    const bool mine = col < rows;
    const Seen seen = mine ? seen_by(a, p, len) : Seen{0, 0, 0};

    const T* const k = a.k.at<T>(b, g);
    const T* const v = a.v.at<T>(b, g);
    i32x4 kr[TileT::kChunks], vr[kPieces];
    auto fetch = [&](int index) {
        const int j0 = tiles.key(index);
        const int j = j0 + col;
#pragma unroll
        for (int c = 0; c < TileT::kChunks; ++c) {
            kr[c] = i32x4{0, 0, 0, 0};
            if (j < len) kr[c] = load_row<T, VEC>(k + j * a.k.n, (2 * c + half) * kPerFrag<T>, a.D);
        }
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int at = x * kWave + lane, jv = j0 + at / kPerRow;
            vr[x] = i32x4{0, 0, 0, 0};
            if (jv < len) vr[x] = load_row<T, VEC>(v + jv * a.v.n, at % kPerRow * kPerFrag<T>, a.D);
        }
    };
    int index = begin + wave;
    if (index < end) fetch(index);

    i32x4 q[TileT::kChunks];
#pragma unroll
    for (int c = 0; c < TileT::kChunks; ++c) {
        q[c] = i32x4{0, 0, 0, 0};
        if (mine) q[c] = load_row<T, VEC>(a.q.at<T>(b, h) + i * a.q.n, (2 * c + half) * kPerFrag<T>, a.D);
    }
    const bool biased = a.bias != nullptr;
    uint8_t* const ids = reinterpret_cast<uint8_t*>(table + a.bk.count * kTile);
    float far = 0.f;
    if (biased) {
        int* const edges = reinterpret_cast<int*>(ids + (a.reach + 4) / 4 * 4);
        for (int x = threadIdx.x; x < a.bk.n; x += kThreads) edges[x] = a.bk.edge[x];
        for (int x = threadIdx.x; x < a.bk.count * kTile; x += kThreads) {
            const int rr = min(r0 + x % kTile, total - 1);
            table[x] = bias_log2(to_float(static_cast<const T*>(a.bias)[static_cast<int64_t>(x / kTile) * a.H + g * group + rr % group]));
        }
        __syncthreads();
        for (int x = threadIdx.x; x <= a.reach; x += kThreads) ids[x] = static_cast<uint8_t>(bucket_of(a.bk, edges, x));
        __syncthreads();
        far = table[a.bk.n * kTile + col];
    }
    auto bias_at = [&](int offset, int column) {
        return table[ids[min(max(offset, 0), a.reach)] * kTile + column];
    };

    char* const vtile = lds + wave * kTileBytes;
    f32x16 o[kOut] = {};
    float m = -kInf, l = 0.f;
    for (; index < end; index += kWaves) {
        const int j0 = tiles.key(index);
        f32x16 s = {};
#pragma unroll
        for (int c = 0; c < TileT::kChunks; ++c) s = mma<T>(kr[c], q[c], s);
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int at = x * kWave + lane;
            *reinterpret_cast<i32x4*>(vtile + at / kPerRow * TileT::kStride + at % kPerRow * 16) = vr[x];
        }
        if (index + kWaves < end) fetch(index + kWaves);
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] *= a.scale_log2;
        const int j = j0 + 4 * half;
        if (biased) {
            if (p_first - (j0 + kTile - 1) >= a.reach) {
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] += far;
            } else {
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] += bias_at(p - (j + 8 * (x / 4) + x % 4), col);
            }
        }
#pragma unroll
        for (int x = 0; x < 16; ++x)
            if (!seen(j + 8 * (x / 4) + x % 4)) s[x] = -kInf;
        float top = s[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) top = fmaxf(top, s[x]);
        top = halves_max(top);
        if (ballot(top - m > kMostLog<T>) != 0) {
            const float next = fmaxf(m, reference_of<T>(top));
            const float keep = m == next ? 1.f : exp2_fast(m - next);
            m = next;
            l *= keep;
#pragma unroll
            for (int d = 0; d < kOut; ++d)
#pragma unroll
                for (int x = 0; x < 16; ++x) o[d][x] *= keep;
        }
        const float base = m == -kInf ? 0.f : m;
        float w[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            w[x] = exp2_fast(s[x] - base);
            l += w[x];
        }
        lanes_exchange();
#pragma unroll
        for (int c = 0; c < 16 / kPerFrag<T>; ++c) {
            const i32x4 f = as_fragment<T>(&w[c * kPerFrag<T>]);
            i32x4 rest;
            if constexpr (sizeof(T) == 2) {
                float left[kPerFrag<T>];
#pragma unroll
                for (int e = 0; e < kPerFrag<T>; ++e) left[e] = w[c * kPerFrag<T> + e] - element<T>(f, e);
                rest = as_fragment<T>(left);
            }
#pragma unroll
            for (int d = 0; d < kOut; ++d) {
                const i32x4 values = TileT::columns(vtile, c * TileT::kRowsPerFrag, 32 * d);
                o[d] = mma<T>(values, f, o[d]);
                if constexpr (sizeof(T) == 2) o[d] = mma<T>(values, rest, o[d]);
            }
        }
        lanes_exchange();
    }
    l = halves_sum(l);

    // The waves' parts, brought to their common maximum and added in order.
    if (half == 0) {
        tops[wave][col] = m;
        totals[wave][col] = l;
    }
    __syncthreads();  // also: the tiles' LDS is free
    float top = tops[0][col], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, tops[w][col]);
    const float base = top == -kInf ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += totals[w][col] * exp2_fast(tops[w][col] - base);
    const float mine_by = exp2_fast(m - base);
    float* const sums = reinterpret_cast<float*>(lds);
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave && mine) {
#pragma unroll
            for (int d = 0; d < kOut; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f32x4* const at = reinterpret_cast<f32x4*>(sums + col * kSumStride + 32 * d + 8 * e + 4 * half);
                    f32x4 x = w == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : *at;
#pragma unroll
                    for (int f = 0; f < 4; ++f) x[f] = __builtin_fmaf(o[d][4 * e + f], mine_by, x[f]);
                    *at = x;
                }
        }
        __syncthreads();
    }
    // Rows of the block, 8 a wave: out, or the split's part of it.
    if (half == 0 && wave == 0) {
        tops[0][col] = top;
        totals[0][col] = sum;
    }
    __syncthreads();
    for (int row = wave; row < rows; row += kWaves) {
        const int ii = (r0 + row) / group, hh = g * group + (r0 + row) % group;
        float x0 = lane < a.D ? sums[row * kSumStride + lane] : 0.f;
        float x1 = lane + kWave < a.D ? sums[row * kSumStride + lane + kWave] : 0.f;
        float lm = tops[0][row], ll = totals[0][row];
        // A sum of weights that is NaN comes from a seen pair, and all of its row is NaN as it
        // lies, but where a bias of -inf masks that pair.
        const bool whole = ll != ll;
        bool masks = false;
        if (whole && biased)
            for (int x = lane; x < a.bk.count; x += kWave) masks |= table[x * kTile + row] == -kInf;
        const bool n0 = whole || !finite(x0), n1 = whole || !finite(x1);
        if (ll == 0.f) {
            x0 = x1 = 0.f;
        } else if (whole ? ballot(masks) != 0 : ballot(n0 || n1) != 0) {
            CarefulRow<T> c(a, b, g, a.q.at<T>(b, hh) + ii * a.q.n);
            const Seen sees = seen_by(a, shift + ii, len);
            bool done = false;
            for (int t = begin; t < end && !done; ++t)
                for (int j = tiles.key(t); j < tiles.key(t) + kTile && !done; ++j)
                    if (sees(j)) {
                        c.add(j, biased ? bias_at(shift + ii - j, row) : 0.f);
                        done = whole ? c.l != c.l : c.settled(n0, n1);
                    }
            c.replace(whole, n0, n1, x0, x1, lm, ll);
        }
        if (splits == 1) {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
            T* const dst = out + ((static_cast<int64_t>(b) * a.Q + ii) * a.H + hh) * a.D;
            if (lane < a.D) dst[lane] = from_float<T>(x0 * inv);
            if (lane + kWave < a.D) dst[lane + kWave] = from_float<T>(x1 * inv);
        } else {
            // (unit, split, row): maximum, sum, D values
            float* const dst = part + ((static_cast<int64_t>(unit) * splits + split) * kTile + row) * (a.D + 2);
            if (lane == 0) {
                dst[0] = lm;
                dst[1] = ll;
            }
            if (lane < a.D) dst[2 + lane] = x0;
            if (lane + kWave < a.D) dst[2 + lane + kWave] = x1;
        }
    }
}

// One wave a row: the splits' parts, brought to their common maximum.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_step_join_kernel(const Args a, const float* __restrict__ part,
                                                                       T* __restrict__ out, int row_blocks, int splits) {
    const int lane = lane_id(), group = a.H / a.G, total = a.Q * group;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;  // (b, g, row)
    if (id >= static_cast<int64_t>(a.B) * a.G * total) return;
    const int row = static_cast<int>(id % total);
    const int64_t bg = id / total;
    const int b = static_cast<int>(bg / a.G), g = static_cast<int>(bg % a.G);
    const int width = a.D + 2;
    const float* const src = part + ((bg * row_blocks + row / kTile) * splits * kTile + row % kTile) * width;
    const int64_t step = static_cast<int64_t>(kTile) * width;
    float top = -kInf;
    for (int s = lane; s < splits; s += kWave) top = fmaxf(top, src[s * step]);
    top = wave_max(top);
    const float base = top == -kInf ? 0.f : top;
    const int c0 = min(lane, a.D - 1), c1 = min(lane + kWave, a.D - 1);
    // The splits' mean; all sums are 2^-above of what they are by the maximum.
    auto mean = [&](float above, float& x0, float& x1) {
        float sum = x0 = x1 = 0.f;
        for (int first = 0; first < splits; first += kWave) {
            // A lane's split: its factor; then the splits' rows one after another.
            const int s = first + lane;
            float by = 0.f;
            if (s < splits) {
                by = exp2_fast(src[s * step] - base - above);
                sum = __builtin_fmaf(src[s * step + 1], by, sum);
            }
            const int count = min(kWave, splits - first);
            const float* const rows = src + first * step + 2;
            constexpr int kAtOnce = 8;
            for (int i = 0; i < count; i += kAtOnce) {
                float y0[kAtOnce], y1[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const int64_t at = min(i + k, count - 1) * step;
                    y0[k] = rows[at + c0];
                    y1[k] = rows[at + c1];
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const float f = i + k < count ? i2f(readlane(f2i(by), min(i + k, count - 1))) : 0.f;
                    x0 = __builtin_fmaf(y0[k], f, x0);
                    x1 = __builtin_fmaf(y1[k], f, x1);
                }
            }
        }
        sum = wave_sum(sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        x0 *= inv;
        x1 *= inv;
    };
    float x0, x1;
    mean(0.f, x0, x1);
    if (ballot(!finite(x0) || !finite(x1)) != 0) {
        // Values near the largest, of which a mean is finite and a sum need not be.
        float y0, y1;
        mean(30.f, y0, y1);
        x0 = finite(x0) ? x0 : y0;
        x1 = finite(x1) ? x1 : y1;
    }
    T* const dst = out + ((static_cast<int64_t>(b) * a.Q + row / group) * a.H + g * group + row % group) * a.D;
    if (lane < a.D) dst[lane] = from_float<T>(x0);
    if (lane + kWave < a.D) dst[lane + kWave] = from_float<T>(x1);
}

struct Plan {
    int row_blocks, waves, splits;
};

// Splits of the keys that give every compute unit four blocks, with at least
// two tiles a wave.  By the cache's size: the lengths are on the device, and a call
// does not wait for it (4 clouds of 500 tokens, 32 heads over 8 of 128: 24 us in a cache
// of 65536, 16 in one of 512).
Plan plan_of(const Args& a, int type) {
    const int64_t rows = static_cast<int64_t>(a.Q) * (a.H / a.G), row_blocks = (rows + kTile - 1) / kTile;
    const int64_t all = (static_cast<int64_t>(a.N) + kTile - 1) / kTile;
    const int64_t window = (static_cast<int64_t>(a.window) + a.Q - 1) / kTile + 2 + (a.sinks + kTile - 1) / kTile;
    const int64_t tiles = std::min(all, window), units = std::max<int64_t>(1, row_blocks * a.B * a.G);
    if (type != POINTOPS_F32 && tiles <= kShortTiles) return {static_cast<int>(row_blocks), 8, 1};
    const int64_t splits = std::min((1024 + units - 1) / units, tiles / 8);
    return {static_cast<int>(row_blocks), 4, static_cast<int>(std::max<int64_t>(1, splits))};
}

size_t workspace_of(const Args& a, int type) {
    const Plan p = plan_of(a, type);
    if (p.splits == 1) return 0;
    return static_cast<size_t>(a.B) * a.G * p.row_blocks * p.splits * kTile * (a.D + 2) * sizeof(float);
}

template <typename T>
hipError_t step(const Args& a, int type, void* out, void* workspace, hipStream_t stream) {
    const Plan plan = plan_of(a, type);
    const int64_t blocks = static_cast<int64_t>(a.B) * a.G * plan.row_blocks * plan.splits;
    const int64_t rows = static_cast<int64_t>(a.B) * a.H * a.Q;
    if (blocks > INT32_MAX || (rows + kWaves - 1) / kWaves > INT32_MAX) return hipErrorInvalidValue;
    const size_t lds = a.bias == nullptr ? 0 : 4 * (a.bk.count * kTile) + (a.reach + 4) / 4 * 4 + 4 * a.bk.n;
    const bool vec = vector_rows<T>(a.q, a.D) && vector_rows<T>(a.k, a.D) && vector_rows<T>(a.v, a.D);
    float* const part = static_cast<float*>(workspace);
    const hipError_t err = with_width(a.D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        auto launch = [&](auto* kernel, int waves) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kWave * waves), lds, stream, a,
                               static_cast<T*>(out), part, plan.row_blocks, plan.splits);
        };
        if constexpr (sizeof(T) == 2) {
            if (plan.waves == 8) {
                launch(vec ? attention_step_kernel<T, DP, true, 8> : attention_step_kernel<T, DP, false, 8>, 8);
                return hipGetLastError();
            }
        }
        launch(vec ? attention_step_kernel<T, DP, true, 4> : attention_step_kernel<T, DP, false, 4>, 4);
        return hipGetLastError();
    });
    if (err != hipSuccess || plan.splits == 1) return err;
    hipLaunchKernelGGL(attention_step_join_kernel<T>, dim3(static_cast<uint32_t>((rows + kWaves - 1) / kWaves)),
                       dim3(kThreads), 0, stream, a, part, static_cast<T*>(out), plan.row_blocks, plan.splits);
    return hipGetLastError();
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" {

size_t pointops_attention_step_workspace_bytes(const pointops_attention* in) {
    using namespace pointops::attn;
    Args a;
    return read_args(in, &a) && a.H > 0 ? workspace_of(a, in->type) : 0;
}

hipError_t pointops_attention_step(const pointops_attention* in, void* out, void* workspace, hipStream_t stream) {
    using namespace pointops::attn;
    Args a;
    if (!read_args(in, &a)) return hipErrorInvalidValue;
    if (a.B == 0 || a.H == 0 || a.Q == 0) return hipSuccess;
    if (!a.causal || (a.bias != nullptr && a.bk.count != a.bk.n + 1)) return hipErrorInvalidValue;
    if (static_cast<int64_t>(a.Q) * (a.H / a.G) > (int64_t(1) << 30)) return hipErrorInvalidValue;
    if (in->q == nullptr || out == nullptr || (in->N > 0 && (in->k == nullptr || in->v == nullptr)))
        return hipErrorInvalidValue;
    if (workspace == nullptr && workspace_of(a, in->type) != 0) return hipErrorInvalidValue;
    switch (in->type) {
        case POINTOPS_F32: return step<float>(a, in->type, out, workspace, stream);
        case POINTOPS_F16: return step<f16>(a, in->type, out, workspace, stream);
        default: return step<bf16>(a, in->type, out, workspace, stream);
    }
}

}  // extern "C"
