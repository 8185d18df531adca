// The root-mean-square norm of each head's query and key with the rotation by
// the token's position, in one pass over both, and its gradients.
//
//   r = rsqrt(mean x^2 + eps), y = x r w;
//   out[i] = y[i] cos[i] - y[i + R/2] sin[i], out[i + R/2] = y[i + R/2] cos[i] + y[i] sin[i]
//   (i < R/2), out[i] = y[i] from R on.
//   dy: the rotation's transpose of dout;  dw = sum over rows of dy x r;
//   dx = r (dy w - x r mean(dy w x r)).
//
// Bound by memory: every value is read once and written once.  A row (token
// and head) is held by 1 to 64 neighbouring lanes, each with two pieces of up
// to 16 bytes: values i and i + R/2 of rotated ones, so that no lane needs
// another's, or two pieces of the others.  Where a part is no multiple of the
// piece, its last piece starts earlier: two lanes then hold the same values and
// write the same results, and one of them leaves them out of the sums.  A group
// of lanes keeps its columns for all its heads and tokens: the angles are read
// once a token, the weights once, and the weights' gradients are summed in
// registers, then over a block, then over all, in a fixed order.
#include <algorithm>

#include "attention.hpp"

namespace pointops {
namespace attn {
namespace {

struct NormArgs {
    Rows q, k;
    const void *wq, *wk;
    const float *cos, *sin;
    int64_t angle_b, angle_n;
    int64_t tokens;  // B N
    int64_t step;    // tokens that are in work at a time
    int slices;      // groups of lanes that share a token's heads
    int N, H, G, D, R;
    float eps, inv_d;
};

template <typename T, int VEC>
struct Piece {
    float v[VEC];
    __device__ __forceinline__ void load(const T* p, bool there) {
        T raw[VEC] = {};
        if (there) __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = to_float(raw[e]);
    }
    __device__ __forceinline__ void store(T* p, bool there) const {
        T raw[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) raw[e] = from_float<T>(v[e]);
        if (there) __builtin_memcpy(p, raw, sizeof raw);
    }
};

// Columns of unit `unit`: its two pieces' first columns, and how many values at
// their start are the piece's before.  A piece that does not exist is at D.
template <int VEC>
struct Columns {
    int a, b, skip_a, skip_b;
    bool turned;
    __host__ __device__ Columns(int unit, int D, int R) {
        const int half = R / 2, turning = (half + VEC - 1) / VEC;
        turned = unit < turning;
        if (turned) {
            a = unit * VEC < half - VEC ? unit * VEC : half - VEC;
            b = half + a;
            skip_a = skip_b = unit * VEC - a;
            return;
        }
        const int at = 2 * (unit - turning) * VEC, rest = D - R;
        a = at >= rest ? rest : at < rest - VEC ? at : rest - VEC;
        b = at + VEC >= rest ? rest : at + VEC < rest - VEC ? at + VEC : rest - VEC;
        skip_a = at - a;
        skip_b = at + VEC - b;
        a += R;
        b += R;
    }
};

// A lane's place: its slice of the heads, its pieces' columns, its token.
template <typename T, int VEC, int L>
struct Place {
    Columns<VEC> col;
    int slice;
    bool has_a, has_b;
    int b, n, step_b, step_n;
    int64_t token;

    __device__ __forceinline__ explicit Place(const NormArgs& a) : col(threadIdx.x % L, a.D, a.R) {
        const int64_t group = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L;
        slice = static_cast<int>(group % a.slices);
        token = group / a.slices;
        if (token >= a.step) token = a.tokens;  // groups behind the last whole set
        has_a = col.a < a.D;
        has_b = col.b < a.D;
        b = static_cast<int>(token / a.N);
        n = static_cast<int>(token % a.N);
        step_b = static_cast<int>(a.step / a.N);
        step_n = static_cast<int>(a.step % a.N);
    }
    __device__ __forceinline__ void next(const NormArgs& a) {
        token += a.step;
        b += step_b;
        n += step_n;
        if (n >= a.N) {
            n -= a.N;
            ++b;
        }
    }
    // Head `head` of q's, then of k's, as it comes and as a row of the contiguous results.
    __device__ __forceinline__ const T* in(const Rows& q, const Rows& k, int H, int head) const {
        return head < H ? q.at<T>(b, head) + n * q.n : k.at<T>(b, head - H) + n * k.n;
    }
    __device__ __forceinline__ T* out(T* q, T* k, const NormArgs& a, int head) const {
        return head < a.H ? q + (token * a.H + head) * a.D : k + (token * a.G + head - a.H) * a.D;
    }
};

template <typename W, int VEC>
struct Weights {
    Piece<W, VEC> a, b;
    __device__ __forceinline__ void load(const void* w, const Columns<VEC>& col, bool has_a, bool has_b) {
        const bool given = w != nullptr;
        a.load(static_cast<const W*>(w) + col.a, given && has_a);
        b.load(static_cast<const W*>(w) + col.b, given && has_b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            a.v[e] = given ? a.v[e] : 1.f;
            b.v[e] = given ? b.v[e] : 1.f;
        }
    }
};

constexpr int kAhead = 2;  // heads whose values are asked for at once

// By value: a conditional of two array elements would choose an address.
__device__ __forceinline__ float pick(bool first, float x, float y) { return first ? x : y; }

// The sum of x y over the row, each value once.
template <int VEC>
__device__ __forceinline__ float row_part(const float (&xa)[VEC], const float (&ya)[VEC], const float (&xb)[VEC],
                                          const float (&yb)[VEC], const Columns<VEC>& col) {
    const uint32_t keep_a = ~0u << col.skip_a, keep_b = ~0u << col.skip_b;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        sum = __builtin_fmaf((keep_a >> e & 1) != 0 ? xa[e] : 0.f, ya[e], sum);
        sum = __builtin_fmaf((keep_b >> e & 1) != 0 ? xb[e] : 0.f, yb[e], sum);
    }
    return sum;
}

template <typename T, typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_kernel(const NormArgs a, T* __restrict__ q_out, T* __restrict__ k_out) {
    Place<T, VEC, L> at(a);
    const Columns<VEC> col = at.col;
    const int heads = a.H + a.G;
    Weights<W, VEC> wq, wk;
    wq.load(a.wq, col, at.has_a, at.has_b);
    wk.load(a.wk, col, at.has_a, at.has_b);
    for (; at.token < a.tokens; at.next(a)) {
        Piece<float, VEC> c, s;
        const int64_t angle = at.b * a.angle_b + at.n * a.angle_n + col.a;
        c.load(a.cos + angle, col.turned);
        s.load(a.sin + angle, col.turned);
        for (int first = at.slice; first < heads; first += kAhead * a.slices) {
            Piece<T, VEC> xa[kAhead], xb[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int head = first + u * a.slices;
                const T* const x = at.in(a.q, a.k, a.H, head);
                xa[u].load(x + col.a, at.has_a && head < heads);
                xb[u].load(x + col.b, at.has_b && head < heads);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int head = first + u * a.slices;
                const float sum = row_part<VEC>(xa[u].v, xa[u].v, xb[u].v, xb[u].v, col);
                const float r = __builtin_amdgcn_rsqf(group_sum<L>(sum) * a.inv_d + a.eps);
                const bool is_q = head < a.H;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float ya = xa[u].v[e] * r * pick(is_q, wq.a.v[e], wk.a.v[e]);
                    const float yb = xb[u].v[e] * r * pick(is_q, wq.b.v[e], wk.b.v[e]);
                    xa[u].v[e] = col.turned ? ya * c.v[e] - yb * s.v[e] : ya;
                    xb[u].v[e] = col.turned ? yb * c.v[e] + ya * s.v[e] : yb;
                }
                T* const out = at.out(q_out, k_out, a, head);
                xa[u].store(out + col.a, at.has_a && head < heads);
                xb[u].store(out + col.b, at.has_b && head < heads);
            }
        }
    }
}

template <typename T, typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_grad_kernel(const NormArgs a, const Rows gq, const Rows gk,
                                                                T* __restrict__ dq, T* __restrict__ dk,
                                                                float* __restrict__ part) {
    __shared__ float sums[kThreads / L][2 * L * VEC];  // a group's columns: its first pieces, then its second
    Place<T, VEC, L> at(a);
    const Columns<VEC> col = at.col;
    const int heads = a.H + a.G;
    Weights<W, VEC> wq, wk;
    wq.load(a.wq, col, at.has_a, at.has_b);
    wk.load(a.wk, col, at.has_a, at.has_b);
    float sa[2][VEC] = {}, sb[2][VEC] = {};  // q's and k's
    for (; at.token < a.tokens; at.next(a)) {
        Piece<float, VEC> c, s;
        const int64_t angle = at.b * a.angle_b + at.n * a.angle_n + col.a;
        c.load(a.cos + angle, col.turned);
        s.load(a.sin + angle, col.turned);
        for (int first = at.slice; first < heads; first += kAhead * a.slices) {
            Piece<T, VEC> xa[kAhead], xb[kAhead], ga[kAhead], gb[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int head = first + u * a.slices;
                const T* const x = at.in(a.q, a.k, a.H, head);
                const T* const g = at.in(gq, gk, a.H, head);
                xa[u].load(x + col.a, at.has_a && head < heads);
                xb[u].load(x + col.b, at.has_b && head < heads);
                ga[u].load(g + col.a, at.has_a && head < heads);
                gb[u].load(g + col.b, at.has_b && head < heads);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int head = first + u * a.slices;
                const bool is_q = head < a.H;
                float ua[VEC], ub[VEC];  // dy w
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float da = col.turned ? ga[u].v[e] * c.v[e] + gb[u].v[e] * s.v[e] : ga[u].v[e];
                    const float db = col.turned ? gb[u].v[e] * c.v[e] - ga[u].v[e] * s.v[e] : gb[u].v[e];
                    ga[u].v[e] = da;
                    gb[u].v[e] = db;
                    ua[e] = da * pick(is_q, wq.a.v[e], wk.a.v[e]);
                    ub[e] = db * pick(is_q, wq.b.v[e], wk.b.v[e]);
                }
                const float sum = row_part<VEC>(xa[u].v, xa[u].v, xb[u].v, xb[u].v, col);
                const float along = row_part<VEC>(xa[u].v, ua, xb[u].v, ub, col);
                const float r = __builtin_amdgcn_rsqf(group_sum<L>(sum) * a.inv_d + a.eps);
                const float mean = group_sum<L>(along) * r * a.inv_d;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float na = xa[u].v[e] * r, nb = xb[u].v[e] * r;
                    const float ta = ga[u].v[e] * na, tb = gb[u].v[e] * nb;
                    sa[0][e] += is_q ? ta : 0.f;
                    sb[0][e] += is_q ? tb : 0.f;
                    sa[1][e] += is_q ? 0.f : ta;
                    sb[1][e] += is_q ? 0.f : tb;
                    xa[u].v[e] = r * (ua[e] - na * mean);
                    xb[u].v[e] = r * (ub[e] - nb * mean);
                }
                // Of a row of one value the difference leaves eps r^2 alone, which rounding would bury.
                if constexpr (VEC == 1 && L == 1)
                    if (a.D == 1) xa[u].v[0] = r * r * r * a.eps * ua[0];
                T* const out = at.out(dq, dk, a, head);
                xa[u].store(out + col.a, at.has_a && head < heads);
                xb[u].store(out + col.b, at.has_b && head < heads);
            }
        }
    }
    if (part == nullptr) return;
    // part (blocks, q or k, columns in the lanes' order)
    constexpr int kColumns = 2 * L * VEC;
    const int group = threadIdx.x / L, unit = threadIdx.x % L;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sums[group][unit * VEC + e] = sa[which][e];
            sums[group][(L + unit) * VEC + e] = sb[which][e];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kColumns; i += kThreads) {
            float all = 0.f;
#pragma unroll 8
            for (int gr = 0; gr < kThreads / L; ++gr) all += sums[gr][i];
            part[(static_cast<int64_t>(blockIdx.x) * 2 + which) * kColumns + i] = all;
        }
    }
}

// dw from the blocks' parts: a block for 16 columns, 16 lanes of blocks each.
template <typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_weight_kernel(const float* __restrict__ part, int blocks, int D, int R,
                                                                  W* __restrict__ dwq, W* __restrict__ dwk) {
    constexpr int kColumns = 2 * L * VEC, kAcross = 16, kLanes = kThreads / kAcross;
    __shared__ float sums[kLanes][kAcross];
    const int x = threadIdx.x % kAcross, y = threadIdx.x / kAcross, id = blockIdx.x * kAcross + x;
    float all = 0.f;
    if (id < 2 * kColumns) {
#pragma unroll 8
        for (int b = y; b < blocks; b += kLanes) all += part[static_cast<int64_t>(b) * 2 * kColumns + id];
    }
    sums[y][x] = all;
    __syncthreads();
    if (y != 0 || id >= 2 * kColumns) return;
    for (int i = 1; i < kLanes; ++i) all += sums[i][x];
    const int i = id % kColumns, e = i % VEC, unit = i / VEC % L;
    const Columns<VEC> col(unit, D, R);
    const bool second = i >= L * VEC;
    const int at = (second ? col.b : col.a) + e;
    W* const dst = id < kColumns ? dwq : dwk;
    // A value that two pieces hold is the first one's.
    if (dst != nullptr && (second ? col.b : col.a) < D && e >= (second ? col.skip_b : col.skip_a)) dst[at] = from_float<W>(all);
}

constexpr int64_t kBlocks = 2048;

struct Shape {
    int vec, lanes, slices;
    int64_t blocks, step;
};

// The widest pieces that the rotated half and the rest hold, and blocks enough
// to fill the card (each keeps its sums until its end).  A wave takes
// neighbouring heads of a token, or all of its heads at once where the whole
// call is small and its latency counts.
Shape shape_of(const pointops_qk_norm& in) {
    const int half = static_cast<int>(in.R / 2), rest = static_cast<int>(in.D - in.R);
    Shape s;
    s.vec = in.type == POINTOPS_F32 ? 4 : 8;
    while ((half > 0 && s.vec > half) || (rest > 0 && s.vec > rest)) s.vec /= 2;
    const int units = (half + s.vec - 1) / s.vec + ((rest + s.vec - 1) / s.vec + 1) / 2;
    s.lanes = 1;
    while (s.lanes < units) s.lanes *= 2;
    const int64_t tokens = in.B * in.N, heads = in.H + in.G, groups = kThreads / s.lanes;
    const bool small = tokens * heads * s.lanes <= (1 << 18);
    s.slices = static_cast<int>(small ? heads : std::min<int64_t>(heads, kWave / s.lanes));
    s.blocks = std::min(kBlocks, (tokens * s.slices + groups - 1) / groups);
    s.blocks = std::max(s.blocks, (s.slices + groups - 1) / groups);
    s.step = std::min(tokens, s.blocks * groups / s.slices);
    return s;
}

bool valid(const pointops_qk_norm* in) {
    const int64_t limit = int64_t(1) << 30;
    return in != nullptr && in->B >= 0 && in->N >= 0 && in->H >= 0 && in->G >= 0 && in->B < limit && in->N < limit &&
           in->H < limit && in->G < limit && in->D >= 1 && in->D <= kMaxHead && in->R >= 0 && in->R <= in->D &&
           in->R % 2 == 0 && in->type >= POINTOPS_F32 && in->type <= POINTOPS_BF16 &&
           (in->weight_type == POINTOPS_F32 || in->weight_type == in->type);
}

NormArgs args_of(const pointops_qk_norm& in, const Shape& s) {
    NormArgs a;
    a.q = {in.q, in.q_stride[0], in.q_stride[1], in.q_stride[2]};
    a.k = {in.k, in.k_stride[0], in.k_stride[1], in.k_stride[2]};
    a.wq = in.q_weight;
    a.wk = in.k_weight;
    a.cos = in.cos;
    a.sin = in.sin;
    a.angle_b = in.angle_stride[0];
    a.angle_n = in.angle_stride[1];
    a.tokens = in.B * in.N;
    a.step = s.step;
    a.slices = s.slices;
    a.N = static_cast<int>(in.N);
    a.H = static_cast<int>(in.H);
    a.G = static_cast<int>(in.G);
    a.D = static_cast<int>(in.D);
    a.R = static_cast<int>(in.R);
    a.eps = in.eps;
    a.inv_d = 1.f / static_cast<float>(in.D);
    return a;
}

// f(T, W, VEC, L) for the call's types and shape.
template <typename F>
hipError_t with_shape(const pointops_qk_norm& in, const Shape& s, F f) {
    auto lanes = [&](auto t, auto w, auto vec) {
        constexpr int VEC = decltype(vec)::value;
        switch (s.lanes) {  // a row is at most 128 values
            case 1: return f(t, w, vec, std::integral_constant<int, 1>{});
            case 2: return f(t, w, vec, std::integral_constant<int, 2>{});
            case 4: return f(t, w, vec, std::integral_constant<int, 4>{});
            case 8: return f(t, w, vec, std::integral_constant<int, 8>{});
            case 16: return f(t, w, vec, std::integral_constant<int, 16>{});
            case 32: if constexpr (VEC <= 4) return f(t, w, vec, std::integral_constant<int, 32>{}); break;
            case 64: if constexpr (VEC <= 2) return f(t, w, vec, std::integral_constant<int, 64>{}); break;
        }
        return hipErrorInvalidValue;
    };
    auto vecs = [&](auto t, auto w) {
        switch (s.vec) {
            case 1: return lanes(t, w, std::integral_constant<int, 1>{});
            case 2: return lanes(t, w, std::integral_constant<int, 2>{});
            case 4: return lanes(t, w, std::integral_constant<int, 4>{});
            case 8: if constexpr (sizeof(t) == 2) return lanes(t, w, std::integral_constant<int, 8>{}); break;
        }
        return hipErrorInvalidValue;
    };
    const bool own = in.weight_type == in.type;
    switch (in.type) {
        case POINTOPS_F32: return vecs(float{}, float{});
        case POINTOPS_F16: return own ? vecs(f16{}, f16{}) : vecs(f16{}, float{});
        default: return own ? vecs(bf16{}, bf16{}) : vecs(bf16{}, float{});
    }
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" {

hipError_t pointops_qk_norm_rotate(const pointops_qk_norm* in, void* q_out, void* k_out, hipStream_t stream) {
    using namespace pointops::attn;
    using namespace pointops;
    if (!valid(in)) return hipErrorInvalidValue;
    if (in->B == 0 || in->N == 0 || in->H + in->G == 0) return hipSuccess;
    if ((in->H > 0 && (in->q == nullptr || q_out == nullptr)) || (in->G > 0 && (in->k == nullptr || k_out == nullptr)) ||
        (in->R > 0 && (in->cos == nullptr || in->sin == nullptr)))
        return hipErrorInvalidValue;
    const Shape s = shape_of(*in);
    if (s.blocks > INT32_MAX) return hipErrorInvalidValue;
    const NormArgs a = args_of(*in, s);
    return with_shape(*in, s, [&](auto t, auto w, auto vec, auto lanes) {
        using T = decltype(t);
        using W = decltype(w);
        hipLaunchKernelGGL((qk_norm_kernel<T, W, decltype(vec)::value, decltype(lanes)::value>),
                           dim3(static_cast<uint32_t>(s.blocks)), dim3(kThreads), 0, stream, a, static_cast<T*>(q_out),
                           static_cast<T*>(k_out));
        return hipGetLastError();
    });
}

size_t pointops_qk_norm_rotate_backward_workspace_bytes(const pointops_qk_norm* in) {
    using namespace pointops::attn;
    if (!valid(in) || in->B == 0 || in->N == 0 || in->H + in->G == 0) return 0;
    // For each block, q's and k's columns: at most 256 each.
    return static_cast<size_t>(std::max(kBlocks, in->H + in->G)) * 2 * 256 * sizeof(float);
}

hipError_t pointops_qk_norm_rotate_backward(const pointops_qk_norm* in, const void* q_grad, const int64_t* q_grad_stride,
                                            const void* k_grad, const int64_t* k_grad_stride, void* dq, void* dk, void* dq_weight,
                                            void* dk_weight, void* workspace, hipStream_t stream) {
    using namespace pointops::attn;
    using namespace pointops;
    if (!valid(in)) return hipErrorInvalidValue;
    if ((dq_weight != nullptr && in->q_weight == nullptr) || (dk_weight != nullptr && in->k_weight == nullptr))
        return hipErrorInvalidValue;
    if (in->B == 0 || in->N == 0 || in->H + in->G == 0) return hipSuccess;
    if ((in->H > 0 && (in->q == nullptr || dq == nullptr || q_grad == nullptr || q_grad_stride == nullptr)) ||
        (in->G > 0 && (in->k == nullptr || dk == nullptr || k_grad == nullptr || k_grad_stride == nullptr)) ||
        (in->R > 0 && (in->cos == nullptr || in->sin == nullptr)))
        return hipErrorInvalidValue;
    const bool sums = dq_weight != nullptr || dk_weight != nullptr;
    if (sums && workspace == nullptr) return hipErrorInvalidValue;
    Rows gq{}, gk{};
    if (q_grad_stride != nullptr) gq = {q_grad, q_grad_stride[0], q_grad_stride[1], q_grad_stride[2]};
    if (k_grad_stride != nullptr) gk = {k_grad, k_grad_stride[0], k_grad_stride[1], k_grad_stride[2]};
    const Shape s = shape_of(*in);
    if (s.blocks > INT32_MAX) return hipErrorInvalidValue;
    const NormArgs a = args_of(*in, s);
    float* const part = sums ? static_cast<float*>(workspace) : nullptr;
    return with_shape(*in, s, [&](auto t, auto w, auto vec, auto lanes) {
        using T = decltype(t);
        using W = decltype(w);
        constexpr int VEC = decltype(vec)::value, L = decltype(lanes)::value;
        hipLaunchKernelGGL((qk_norm_grad_kernel<T, W, VEC, L>), dim3(static_cast<uint32_t>(s.blocks)), dim3(kThreads), 0,
                           stream, a, gq, gk, static_cast<T*>(dq), static_cast<T*>(dk), part);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess || !sums) return err;
        hipLaunchKernelGGL((qk_norm_weight_kernel<W, VEC, L>), dim3((4 * L * VEC + 15) / 16), dim3(kThreads), 0, stream, part,
                           static_cast<int>(s.blocks), a.D, a.R, static_cast<W*>(dq_weight), static_cast<W*>(dk_weight));
        return hipGetLastError();
    });
}

}  // extern "C"
