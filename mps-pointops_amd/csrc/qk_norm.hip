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
// another's, or two pieces of the others.  A lane keeps its head and columns
// for all its tokens, and with them the weights and their gradient's sums, in
// registers; the sums of a block, then of all, are added in a fixed order.
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
    int N, H, G, D, R;
    float eps, inv_d;
};

template <typename T, int VEC>
struct Piece {
    static constexpr int kAlign = VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16;
    float v[VEC];
    __device__ __forceinline__ void load(const T* p, bool there) {
        if (there) {
            T raw[VEC];
            __builtin_memcpy(raw, __builtin_assume_aligned(p, kAlign), sizeof raw);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = to_float(raw[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = 0.f;
        }
    }
    __device__ __forceinline__ void store(T* p, bool there) const {
        T raw[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) raw[e] = from_float<T>(v[e]);
        if (there) __builtin_memcpy(__builtin_assume_aligned(p, kAlign), raw, sizeof raw);
    }
};

// A lane's place: its head, its pieces' columns, its first token.
template <typename T, int VEC, int L>
struct Place {
    int head, col_a, col_b;  // head: q's, then k's
    bool turned, has_a, has_b, is_q;
    int b, n, step_b, step_n;
    int64_t token;

    __device__ __forceinline__ explicit Place(const NormArgs& a) {
        const int64_t group = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L;
        const int unit = threadIdx.x % L, heads = a.H + a.G;
        head = static_cast<int>(group % heads);
        token = group / heads;
        is_q = head < a.H;
        if (token >= a.step) token = a.tokens;  // groups behind the last whole set
        const int half = a.R / 2, turning = half / VEC;
        turned = unit < turning;
        col_a = turned ? unit * VEC : a.R + 2 * (unit - turning) * VEC;
        col_b = turned ? half + unit * VEC : col_a + VEC;
        has_a = col_a < a.D;
        has_b = col_b < a.D;
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
    __device__ __forceinline__ const T* in(const Rows& q, const Rows& k, int H) const {
        return is_q ? q.at<T>(b, head) + n * q.n : k.at<T>(b, head - H) + n * k.n;
    }
    // Row of the contiguous output.
    __device__ __forceinline__ T* out(T* q, T* k, const NormArgs& a) const {
        return is_q ? q + (token * a.H + head) * a.D : k + (token * a.G + head - a.H) * a.D;
    }
};

template <typename W, int VEC>
__device__ __forceinline__ void load_weight(Piece<W, VEC>& p, const void* w, int col, bool there) {
    if (w != nullptr) {
        p.load(static_cast<const W*>(w) + col, there);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p.v[e] = there ? 1.f : 0.f;
    }
}

template <typename T, typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_kernel(const NormArgs a, T* __restrict__ q_out, T* __restrict__ k_out) {
    Place<T, VEC, L> at(a);
    Piece<W, VEC> wa, wb;
    load_weight(wa, at.is_q ? a.wq : a.wk, at.col_a, at.has_a);
    load_weight(wb, at.is_q ? a.wq : a.wk, at.col_b, at.has_b);
    for (; at.token < a.tokens; at.next(a)) {
        const T* const x = at.in(a.q, a.k, a.H);
        Piece<T, VEC> xa, xb;
        Piece<float, VEC> c, s;
        xa.load(x + at.col_a, at.has_a);
        xb.load(x + at.col_b, at.has_b);
        const int64_t angle = at.b * a.angle_b + at.n * a.angle_n + at.col_a;
        c.load(a.cos + angle, at.turned);
        s.load(a.sin + angle, at.turned);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum = __builtin_fmaf(xa.v[e], xa.v[e], __builtin_fmaf(xb.v[e], xb.v[e], sum));
        const float r = __builtin_amdgcn_rsqf(group_sum<L>(sum) * a.inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float ya = xa.v[e] * r * wa.v[e], yb = xb.v[e] * r * wb.v[e];
            xa.v[e] = at.turned ? ya * c.v[e] - yb * s.v[e] : ya;
            xb.v[e] = at.turned ? yb * c.v[e] + ya * s.v[e] : yb;
        }
        T* const out = at.out(q_out, k_out, a);
        xa.store(out + at.col_a, at.has_a);
        xb.store(out + at.col_b, at.has_b);
    }
}

template <typename T, typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_grad_kernel(const NormArgs a, const Rows gq, const Rows gk,
                                                                T* __restrict__ dq, T* __restrict__ dk,
                                                                float* __restrict__ part) {
    __shared__ float sums[kThreads / L][2 * L * VEC];  // a group's columns: its first pieces, then its second
    __shared__ bool of_q[kThreads / L];
    Place<T, VEC, L> at(a);
    Piece<W, VEC> wa, wb;
    load_weight(wa, at.is_q ? a.wq : a.wk, at.col_a, at.has_a);
    load_weight(wb, at.is_q ? a.wq : a.wk, at.col_b, at.has_b);
    float sa[VEC] = {}, sb[VEC] = {};
    for (; at.token < a.tokens; at.next(a)) {
        const T* const x = at.in(a.q, a.k, a.H);
        const T* const g = at.in(gq, gk, a.H);
        Piece<T, VEC> xa, xb, ga, gb;
        Piece<float, VEC> c, s;
        xa.load(x + at.col_a, at.has_a);
        xb.load(x + at.col_b, at.has_b);
        ga.load(g + at.col_a, at.has_a);
        gb.load(g + at.col_b, at.has_b);
        const int64_t angle = at.b * a.angle_b + at.n * a.angle_n + at.col_a;
        c.load(a.cos + angle, at.turned);
        s.load(a.sin + angle, at.turned);
        float sum = 0.f, along = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sum = __builtin_fmaf(xa.v[e], xa.v[e], __builtin_fmaf(xb.v[e], xb.v[e], sum));
            const float da = at.turned ? ga.v[e] * c.v[e] + gb.v[e] * s.v[e] : ga.v[e];
            const float db = at.turned ? gb.v[e] * c.v[e] - ga.v[e] * s.v[e] : gb.v[e];
            ga.v[e] = da;
            gb.v[e] = db;
            along = __builtin_fmaf(da * wa.v[e], xa.v[e], __builtin_fmaf(db * wb.v[e], xb.v[e], along));
        }
        const float r = __builtin_amdgcn_rsqf(group_sum<L>(sum) * a.inv_d + a.eps);
        const float mean = group_sum<L>(along) * r * a.inv_d;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float ua = xa.v[e] * r, ub = xb.v[e] * r;
            sa[e] = __builtin_fmaf(ga.v[e], ua, sa[e]);
            sb[e] = __builtin_fmaf(gb.v[e], ub, sb[e]);
            xa.v[e] = r * (ga.v[e] * wa.v[e] - ua * mean);
            xb.v[e] = r * (gb.v[e] * wb.v[e] - ub * mean);
        }
        // Of a row of one value the difference leaves eps r^2 alone, which rounding would bury.
        if constexpr (VEC == 1 && L == 1)
            if (a.D == 1) xa.v[0] = r * r * r * a.eps * ga.v[0] * wa.v[0];
        T* const out = at.out(dq, dk, a);
        xa.store(out + at.col_a, at.has_a);
        xb.store(out + at.col_b, at.has_b);
    }
    if (part == nullptr) return;
    const int group = threadIdx.x / L, unit = threadIdx.x % L;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        sums[group][unit * VEC + e] = sa[e];
        sums[group][(L + unit) * VEC + e] = sb[e];
    }
    if (unit == 0) of_q[group] = at.is_q;
    __syncthreads();
    // part (blocks, q or k, columns in the lanes' order)
    constexpr int kColumns = 2 * L * VEC;
    for (int i = threadIdx.x; i < 2 * kColumns; i += kThreads) {
        const bool q = i < kColumns;
        float all = 0.f;
        for (int gr = 0; gr < kThreads / L; ++gr)
            if (of_q[gr] == q) all += sums[gr][i % kColumns];
        part[static_cast<int64_t>(blockIdx.x) * 2 * kColumns + i] = all;
    }
}

// dw from the blocks' parts: one wave a column, the blocks over its lanes.
template <typename W>
__global__ __launch_bounds__(kThreads) void qk_norm_weight_kernel(const float* __restrict__ part, int blocks, int L, int VEC,
                                                                  int D, int R, W* __restrict__ dwq, W* __restrict__ dwk) {
    const int id = blockIdx.x * kWaves + threadIdx.x / kWave, columns = 2 * L * VEC;
    if (id >= 2 * columns) return;
    const int i = id % columns, piece = i / (L * VEC), unit = i / VEC % L, e = i % VEC;
    const int half = R / 2, turning = half / VEC;
    const int col = (unit < turning ? unit * VEC + piece * half : R + (2 * (unit - turning) + piece) * VEC) + e;
    float all = 0.f;
    for (int b = lane_id(); b < blocks; b += kWave) all += part[static_cast<int64_t>(b) * 2 * columns + id];
    all = wave_sum(all);
    W* const dst = id < columns ? dwq : dwk;
    if (lane_id() == 0 && col < D && dst != nullptr) dst[col] = from_float<W>(all);
}

constexpr int64_t kBlocks = 2048;

struct Shape {
    int vec, lanes;
    int64_t blocks, step;
};

// The widest pieces that all rows, the rotated half and the rest allow, and
// blocks enough to fill the card (each keeps its sums until its end).
Shape shape_of(const pointops_qk_norm& in, int64_t extra_alignment) {
    const int size = in.type == POINTOPS_F32 ? 4 : 2;
    int64_t bits = static_cast<int64_t>(16 / size) | (in.R / 2) | (in.D - in.R) | extra_alignment;
    for (int i = 0; i < 3; ++i) bits |= in.q_stride[i] | in.k_stride[i];
    bits |= reinterpret_cast<uintptr_t>(in.q) / size | reinterpret_cast<uintptr_t>(in.k) / size;
    if (in.R > 0)
        bits |= in.angle_stride[0] | in.angle_stride[1] | reinterpret_cast<uintptr_t>(in.cos) / 4 |
                reinterpret_cast<uintptr_t>(in.sin) / 4;
    Shape s;
    s.vec = static_cast<int>(bits & -bits);
    const int64_t rest = (in.D - in.R) / s.vec, units = in.R / 2 / s.vec + (rest + 1) / 2;
    s.lanes = 1;
    while (s.lanes < units) s.lanes *= 2;
    const int64_t tokens = in.B * in.N, heads = in.H + in.G, groups = kThreads / s.lanes;
    s.blocks = std::min(kBlocks, (tokens * heads + groups - 1) / groups);
    s.blocks = std::max(s.blocks, (heads + groups - 1) / groups);
    s.step = std::min(tokens, s.blocks * groups / heads);
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
            case 16: if constexpr (VEC <= 4) return f(t, w, vec, std::integral_constant<int, 16>{}); break;
            case 32: if constexpr (VEC <= 2) return f(t, w, vec, std::integral_constant<int, 32>{}); break;
            case 64: if constexpr (VEC <= 1) return f(t, w, vec, std::integral_constant<int, 64>{}); break;
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

bool weights_aligned(const pointops_qk_norm& in) {
    return reinterpret_cast<uintptr_t>(in.q_weight) % 16 == 0 && reinterpret_cast<uintptr_t>(in.k_weight) % 16 == 0;
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
    const Shape s = shape_of(*in, weights_aligned(*in) ? 0 : 1);
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
    // For each block, q's and k's columns: at most 128 each, whatever the pieces' width.
    return static_cast<size_t>(std::max(kBlocks, in->H + in->G)) * 2 * 128 * sizeof(float);
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
    const int size = in->type == POINTOPS_F32 ? 4 : 2;
    Rows gq{}, gk{};
    int64_t bits = weights_aligned(*in) ? 0 : 1;
    if (q_grad_stride != nullptr) {
        gq = {q_grad, q_grad_stride[0], q_grad_stride[1], q_grad_stride[2]};
        bits |= gq.b | gq.n | gq.h | static_cast<int64_t>(reinterpret_cast<uintptr_t>(q_grad) / size);
    }
    if (k_grad_stride != nullptr) {
        gk = {k_grad, k_grad_stride[0], k_grad_stride[1], k_grad_stride[2]};
        bits |= gk.b | gk.n | gk.h | static_cast<int64_t>(reinterpret_cast<uintptr_t>(k_grad) / size);
    }
    const Shape s = shape_of(*in, bits);
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
        hipLaunchKernelGGL(qk_norm_weight_kernel<W>, dim3((4 * L * VEC + kWaves - 1) / kWaves), dim3(kThreads), 0, stream,
                           part, static_cast<int>(s.blocks), L, VEC, a.D, a.R, static_cast<W*>(dq_weight),
                           static_cast<W*>(dk_weight));
        return hipGetLastError();
    });
}

}  // extern "C"
