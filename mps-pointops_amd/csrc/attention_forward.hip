// Attention within a window of the order, with first keys that stay visible:
// the forward pass.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  s_ij = scale q_i k_j + bias(i - j)
//
// over the keys j that query i sees.  One pass: a block of 4 waves holds 128
// queries (32 a wave, one a lane column) with their running maximum, sum and
// output in registers and takes its keys 64 (32 bits: 32) at a time through
// LDS; tiles that no query of the block sees are never read, and masks are
// applied only where a tile's edge runs through the window.  Scores, maxima,
// sums and outputs are 32-bit; the weights p are rounded to the values' type
// for the second product, as its matrix instruction takes them.
//
// Bound by the operands' reads from LDS and the products, which take as long as each
// other and of which two waves a SIMD overlap a part: the matrix cores are busy for
// 37 % of a compute unit's busy cycles, LDS for 37 % (every earlier key: 33 and 33 %).
// 16384 queries, 8 heads over 2 of 128, window 2048, bfloat16, takes 170 to 177 us, 733
// to 765 T/s of the pairs seen (a large library product: 1204); every earlier key at 2 x
// 4096 queries, 8 heads of 128, 118 to 128 us.  32 queries a wave keep their output and operands in
// registers beside a whole tile's scores; with the tiles in two LDS buffers one
// barrier a tile is left.
#include "attention.hpp"

namespace pointops {
namespace attn {

bool read_args(const pointops_attention* in, Args* out) {
    const int64_t limit = (int64_t(1) << 30) - 1024;  // sums of two positions fit an int
    if (in == nullptr || out == nullptr) return false;
    if (in->B < 0 || in->Q < 0 || in->N < 0 || in->H < 0 || in->G < 0 || in->D < 1 || in->D > kMaxHead) return false;
    if (in->B > limit || in->Q > limit || in->N > limit || in->H > limit || in->G > limit) return false;
    if (in->type < POINTOPS_F32 || in->type > POINTOPS_BF16) return false;
    if (in->H > 0 && (in->G < 1 || in->H % in->G != 0)) return false;
    if (in->window < 1 || in->sinks < 0) return false;
    if (in->lengths != nullptr && in->length_bits != 32 && in->length_bits != 64) return false;
    Args& a = *out;
    a.q = {in->q, in->q_stride[0], in->q_stride[1], in->q_stride[2]};
    a.k = {in->k, in->k_stride[0], in->k_stride[1], in->k_stride[2]};
    a.v = {in->v, in->v_stride[0], in->v_stride[1], in->v_stride[2]};
    a.bias = in->bias;
    a.lengths = in->lengths;
    a.length_bits = in->length_bits;
    a.B = static_cast<int>(in->B);
    a.Q = static_cast<int>(in->Q);
    a.N = static_cast<int>(in->N);
    a.H = static_cast<int>(in->H);
    a.G = static_cast<int>(in->G);
    a.D = static_cast<int>(in->D);
    a.window = static_cast<int>(in->window > in->N + 1 ? in->N + 1 : in->window);
    a.sinks = static_cast<int>(in->sinks > in->N ? in->N : in->sinks);
    a.causal = in->causal != 0;
    a.scale = in->scale;
    a.scale_log2 = in->scale * kLog2e;
    a.reach = 0;
    a.bk.n = a.bk.count = 0;
    if (in->bias != nullptr) {
        if (!read_buckets(in->edges, in->n_edges, in->buckets, kMaxReach, &a.bk)) return false;
        a.reach = a.bk.edge[a.bk.n - 1];
    }
    return true;
}

namespace {

// n0, n1: whether this lane's columns are needed; whole: so is lse (else it stays, as
// the sum of the weights has not met masked pairs).
template <typename T>
__device__ __forceinline__ void careful_row(const Args& a, int b, int h, int i, int len, const float* table, bool whole,
                                            bool n0, bool n1, T* out, float* lse) {
    const int lane = lane_id(), p = i + a.N - a.Q;
    const Seen seen = seen_by(a, p, len);
    CarefulRow<T> row(a, b, h / (a.H / a.G), a.q.at<T>(b, h) + i * a.q.n);
    n0 = n0 && row.d0;
    n1 = n1 && row.d1;
    auto settled = [&](int j) {
        const int off = min(max(p - j, -a.reach), a.reach);
        row.add(j, a.bias != nullptr ? table[off + a.reach + kMargin] : 0.f);
        return whole ? row.l != row.l : row.settled(n0, n1);  // (then all that follows is NaN)
    };
    bool done = false;
    for (int j = 0; j < seen.first && !done; ++j) done = settled(j);
    for (int j = max(seen.low, seen.first); j < seen.low + seen.count && !done; ++j) done = settled(j);
    const float inv = row.l == 0.f ? 0.f : 1.f / row.l;
    if (n0) out[lane] = from_float<T>(row.o0 * inv);
    if (n1) out[lane + kWave] = from_float<T>(row.o1 * inv);
    if (whole && lane == 0 && lse != nullptr) *lse = row.l == 0.f ? kInf : row.m + log2f(row.l);
}

template <typename T, int DP, bool VEC, bool BIAS, int SPLIT>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 384 ? 1 : 2) void attention_forward_kernel(const Args a, T* __restrict__ out,
                                                                        float* __restrict__ lse_out) {
    using TileT = Tile<T, DP>;
    constexpr int TK = Cut<T, SPLIT>::kInnerRows, kSub = Cut<T, SPLIT>::kSub, kRows = Cut<T, SPLIT>::kRows, kOut = DP / 32;
    constexpr int kTileBytes = TK * TileT::kStride;
    extern __shared__ char lds[];  // two pairs of a key and a value tile, the bias's table
    float* const table = reinterpret_cast<float*>(lds + 4 * kTileBytes);

    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / kWave);
    const int wave_row = 32 * (wave % (kWaves / SPLIT)), sub = wave / (kWaves / SPLIT) * kSub;  // its rows, its pieces
    const int blocks = (a.Q + kRows - 1) / kRows;
    const Place at = place(a.B * a.H, blocks);
    const int b = at.outer / a.H, h = at.outer % a.H, g = h / (a.H / a.G);
    const int i0 = folded(at.inner, blocks) * kRows;
    const int len = a.length(b), shift = a.N - a.Q;

    // The block's rows that exist, by position, and the tiles that they see.
    const int rows = min(kRows, a.Q - i0);
    const Walk walk(a, max(i0 + shift, 0), min(i0 + shift + rows, len) - 1, len, TK);

    // This wave's rows.
    const int w0 = i0 + wave_row + shift;  // position of its first row
    const int w_count = min(32, i0 + rows - (i0 + wave_row));
    const int w_first = max(w0, 0), w_last = min(w0 + w_count, len) - 1;
    const bool w_any = w_first <= w_last, w_whole = w_any && w0 >= 0 && w0 + w_count <= len;
    const int row = i0 + wave_row + lane % 32, p = row + shift;
    const Seen seen = seen_by(a, p, len);

    const T* const k = a.k.at<T>(b, g);
    const T* const v = a.v.at<T>(b, g);
    Stage<T, DP, TK, VEC> ks, vs;
    int t = walk.begin();
    if (t < walk.end) {
        ks.load(k, a.k.n, t * TK, len, a.D);
        vs.load(v, a.v.n, t * TK, len, a.D);
    }
    const bool biased = BIAS && (VEC || a.bias != nullptr);  // rows that are not aligned have one kernel for both
    if (biased) fill_bias<T>(a, h, table, reinterpret_cast<int*>(table + bias_entries(a.reach)));
    i32x4 q[TileT::kChunks];
    {
        const T* src = a.q.at<T>(b, h) + row * a.q.n;
#pragma unroll
        for (int c = 0; c < TileT::kChunks; ++c) {
            q[c] = i32x4{0, 0, 0, 0};
            if (row < a.Q) q[c] = load_row<T, VEC>(src, (2 * c + half) * kPerFrag<T>, a.D);
        }
    }
    if (t < walk.end) {
        ks.store(lds);
        vs.store(lds + kTileBytes);
    }
    __syncthreads();

    // Scores as the products leave them, in units of 1 / factor: a bias needs
    // them scaled, and a negative scale turns their order.
    const bool scaled = biased || !(a.scale > 0.f);
    const float factor = scaled ? 1.f : a.scale_log2;
    f32x16 o[kOut] = {};
    float m = -kInf, l = 0.f;  // the maximum so far (scaled; see kSlack) and this half-wave's sum
    char* ktile = lds;
    while (t < walk.end) {
        char* const vtile = ktile + kTileBytes;
        const int j0 = t * TK;
        t = walk.after(t);
        if (t < walk.end) {
            ks.load(k, a.k.n, t * TK, len, a.D);
            vs.load(v, a.v.n, t * TK, len, a.D);
        }
        const bool meets = w_any && ((j0 <= seen_high(a, w_last, len) && j0 + TK > seen_low(a, w_first)) ||
                                     j0 < seen_first(a, w_last, len));
        if (meets) {
            const bool whole = w_whole && ((j0 + TK - 1 <= seen_high(a, w_first, len) && j0 >= seen_low(a, w_last)) ||
                                           j0 + TK <= seen_first(a, w_first, len));
            f32x16 s[kSub];
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                RowFrags<T, DP> f;
                f.load(ktile, 32 * (sub + u));
                keep_order();
                s[u] = f.times(q);
            }
            ColumnFrags<T, DP> vf[2];  // of this chunk of keys and the next
            vf[0].load(vtile, 32 * sub);
            keep_order();
            if (scaled) {
#pragma unroll
                for (int u = 0; u < kSub; ++u) s[u] *= a.scale_log2;
            }
            if (biased) {
                const int near = w0 - j0;  // offset of the wave's first row and the tile's first key
                if (near - (TK - 1) >= a.reach || near + 31 <= -a.reach) {
                    const float far = table[near > 0 ? bias_entries(a.reach) - 1 : 0];
#pragma unroll
                    for (int u = 0; u < kSub; ++u) s[u] += far;
                } else {
                    const float* from = table + near - 32 * sub + lane % 32 - 4 * half + a.reach + kMargin;
#pragma unroll
                    for (int u = 0; u < kSub; ++u)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[u][r] += from[-(32 * u + 8 * (r / 4) + r % 4)];
                }
            }
            if (!whole) {
                const int j = j0 + 32 * sub + 4 * half;
#pragma unroll
                for (int u = 0; u < kSub; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!seen(j + 32 * u + 8 * (r / 4) + r % 4)) s[u][r] = -kInf;
            }
            float top = s[0][0];
#pragma unroll
            for (int u = 0; u < kSub; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
            top = halves_max(top) * factor;
            if (ballot(top > m + kSlack) != 0) {
                const float next = fmaxf(m, top);
                const float keep = m == next ? 1.f : exp2_fast(m - next);
                m = next;
                l *= keep;
#pragma unroll
                for (int d = 0; d < kOut; ++d) o[d] *= keep;
            }
            const float base = m == -kInf ? 0.f : m;
            // A chunk's weights are formed while the products of the one before run.
            constexpr int kPer = 16 / kPerFrag<T>, kSteps = kSub * kPer;
            i32x4 x[2];
            auto weigh = [&](int c) {
                float w[kPerFrag<T>];
#pragma unroll
                for (int r = 0; r < kPerFrag<T>; ++r) {
                    w[r] = exp2_fast(__builtin_fmaf(s[c / kPer][c % kPer * kPerFrag<T> + r], factor, -base));
                    l += w[r];
                }
                x[c % 2] = as_fragment<T>(w);
            };
            weigh(0);
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                if (c + 1 < kSteps) vf[(c + 1) % 2].load(vtile, 32 * sub + (c + 1) * TileT::kRowsPerFrag);
                keep_order();
                vf[c % 2].add(x[c % 2], o);
                if (c + 1 < kSteps) weigh(c + 1);
            }
        }
        ktile = ktile == lds ? lds + 2 * kTileBytes : lds;
        if (t < walk.end) {
            ks.store(ktile);
            vs.store(ktile + kTileBytes);
        }
        __syncthreads();
    }

    if constexpr (SPLIT == 2) {
        // The later half's sums, brought to the pair's common maximum.
        float* const other = reinterpret_cast<float*>(lds) + wave % 2 * (16 * kOut + 2) * kWave;
        if (wave >= 2) {
            put_sums(other + 2 * kWave, o);
            other[lane] = m;
            other[kWave + lane] = l;
        }
        __syncthreads();
        if (wave >= 2) return;
        const float m2 = other[lane], top = fmaxf(m, m2), base = top == -kInf ? 0.f : top;
        const float keep = exp2_fast(m - base), by = exp2_fast(m2 - base);
        m = top;
        l = l * keep + other[kWave + lane] * by;
        get_sums(other + 2 * kWave, o, keep, by);
    }
    l = halves_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float lse = l == 0.f ? kInf : m + log2f(l);
    float odd = lse == kInf ? 0.f : lse * 0.f;  // NaN where anything is not finite
#pragma unroll
    for (int d = 0; d < kOut; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[d][r] *= inv;
            odd += o[d][r] * 0.f;
        }
    uint64_t bad = ballot(row < a.Q && odd != 0.f);
    bad = (bad | bad >> 32) & 0xffffffffu;
    if (row < a.Q) {
        T* const dst = out + ((static_cast<int64_t>(b) * a.Q + row) * a.H + h) * a.D;
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) store4<T, VEC>(dst, 32 * d + 8 * e + 4 * half, a.D, o[d], 4 * e);
        if (half == 0 && lse_out != nullptr) lse_out[(static_cast<int64_t>(b) * a.H + h) * a.Q + row] = lse;
    }
    if (bad == 0) return;
    // A sum of weights that is NaN comes from a seen pair, and all of its row is NaN as it
    // lies, but where a bias of -inf masks that pair.
    bool masks = false;
    if (biased)
        for (int x = lane; x < bias_entries(a.reach); x += kWave) masks |= table[x] == -kInf;
    masks = ballot(masks) != 0;
    const uint64_t odd_o = odd_values(o);
    __threadfence();  // what is written again comes behind the rows' stores
    while (bad != 0) {
        const int r = __builtin_ctzll(bad);
        bad &= bad - 1;
        const float sum = i2f(readlane(f2i(l), r));
        if (sum != sum && !masks) continue;
        const int i = i0 + wave_row + r;
        const bool whole = sum != sum;
        careful_row<T>(a, b, h, i, sum == 0.f ? 0 : len, table, whole, whole || odd_value(odd_o, r, lane),
                       whole || odd_value(odd_o, r, lane + kWave), out + ((static_cast<int64_t>(b) * a.Q + i) * a.H + h) * a.D,
                       lse_out == nullptr ? nullptr : lse_out + (static_cast<int64_t>(b) * a.H + h) * a.Q + i);
    }
}

template <typename T>
hipError_t forward(const pointops_attention* in, const Args& a, void* out, float* lse, hipStream_t stream) {
    const bool vec = vector_rows<T>(a.q, a.D) && vector_rows<T>(a.k, a.D) && vector_rows<T>(a.v, a.D);
    return with_width(in->D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        const bool bias = a.bias != nullptr;
        const bool split = kSplits<T, DP> && vec && few_blocks((in->Q + kOuter - 1) / kOuter * in->B * in->H);
        const int64_t rows = split ? kOuter / 2 : kOuter, blocks = (in->Q + rows - 1) / rows * in->B * in->H;
        if (blocks > INT32_MAX) return hipErrorInvalidValue;
        const size_t tiles = static_cast<size_t>(4) * (split ? Cut<T, 2>::kInnerRows : kInner<T>) * Tile<T, DP>::kStride;
        const size_t lds = tiles + (bias ? 4 * (bias_entries(a.reach) + a.bk.n) : 0);
        const dim3 grid(static_cast<uint32_t>(blocks));
        const int which = !vec ? 0 : (bias ? 1 : 2) + (split ? 2 : 0);
        auto* kernel = which == 0   ? attention_forward_kernel<T, DP, false, true, 1>
                       : which == 1 ? attention_forward_kernel<T, DP, true, true, 1>
                                    : attention_forward_kernel<T, DP, true, false, 1>;
        if constexpr (kSplits<T, DP>)
            if (split) kernel = bias ? attention_forward_kernel<T, DP, true, true, 2> : attention_forward_kernel<T, DP, true, false, 2>;
        if (lds > kLdsFree) {
            static std::atomic<uint64_t> allowed[5];
            const hipError_t err = allow_lds(kernel, allowed[which], tiles + 4 * (bias_entries(kMaxReach) + 255));
            if (err != hipSuccess) return err;
        }
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, stream, a, static_cast<T*>(out), lse);
        return hipGetLastError();
    });
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" hipError_t pointops_attention_forward(const pointops_attention* in, void* out, float* lse,
                                                 hipStream_t stream) {
    using namespace pointops::attn;
    Args a;
    if (!read_args(in, &a)) return hipErrorInvalidValue;
    if (in->B == 0 || in->H == 0 || in->Q == 0) return hipSuccess;
    if (in->q == nullptr || out == nullptr || (in->N > 0 && (in->k == nullptr || in->v == nullptr)))
        return hipErrorInvalidValue;
    switch (in->type) {
        case POINTOPS_F32: return forward<float>(in, a, out, lse, stream);
        case POINTOPS_F16: return forward<f16>(in, a, out, lse, stream);
        default: return forward<bf16>(in, a, out, lse, stream);
    }
}
