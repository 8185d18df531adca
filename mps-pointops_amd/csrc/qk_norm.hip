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
// of lanes keeps its head and columns for all its tokens: the weights and the
// sums for their gradients stay in registers, and are added over a block, then
// over all, in a fixed order.
//
// At 32 x 4096 tokens, 4 + 4 heads of 32, float32: 55 us (5.1 TB/s of what it
// must move; a large copy reaches 5.15) and 85 + 5 us for the gradients (4.9).
// At 65537 tokens, 12 + 3 heads of 80 (60 rotated), float16, which are 6 lanes
// of 8: 79 us (4.2 TB/s) and 110 + 7 (4.4); with one piece of 4 bytes a lane,
// as the parts' common divisor would have it, 133 and 305.
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
    int units;       // lanes of a row that have columns
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

// A lane's place: its head (of q's, then of k's) and its pieces' columns for
// the whole call, and the tokens it goes through.  Lanes behind the last unit
// read the first columns, add nothing and write nothing.
template <typename T, int VEC, int L>
struct Place {
    Columns<VEC> col;
    int head;
    bool is_q, has_a, has_b;
    int n;
    int64_t token, b;

    __device__ __forceinline__ explicit Place(const NormArgs& a) : col(threadIdx.x % L, a.D, a.R) {
        const int64_t group = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L;
        const int heads = a.H + a.G;
        head = static_cast<int>(group % heads);
        token = group / heads;
        if (token >= a.step) token = a.tokens;  // groups behind the last whole set
        is_q = head < a.H;
        const bool used = static_cast<int>(threadIdx.x % L) < a.units;
        has_a = used && col.a < a.D;
        has_b = used && col.b < a.D;
        if (!has_a) {
            col.a = 0;
            col.skip_a = VEC;
        }
        if (!has_b) {
            col.b = 0;
            col.skip_b = VEC;
        }
        b = token / a.N;
        n = static_cast<int>(token % a.N);
    }
    // On to the next token; whether it is in another batch than step / N further.
    __device__ __forceinline__ bool next(const NormArgs& a) {
        token += a.step;
        n += static_cast<int>(a.step % a.N);
        const bool wrapped = n >= a.N;
        n -= wrapped ? a.N : 0;
        return wrapped;
    }
};

// A row's place in a tensor, moved on with its token.
struct Cursor {
    int64_t at, step, wrap;  // elements; wrap: what a change of batch adds
    __device__ __forceinline__ Cursor(int64_t b, int64_t n, int64_t stride_b, int64_t stride_n, const NormArgs& a)
        : at(b * stride_b + n * stride_n),
          step(a.step / a.N * stride_b + a.step % a.N * stride_n),
          wrap(stride_b - a.N * stride_n) {}
    __device__ __forceinline__ void next(bool wrapped) { at += step + (wrapped ? wrap : 0); }
};

template <typename W, int VEC>
struct Weights {
    Piece<W, VEC> a, b;
    __device__ __forceinline__ Weights(const void* w, const Columns<VEC>& col) {
        const bool given = w != nullptr;
        a.load(static_cast<const W*>(w) + col.a, given);
        b.load(static_cast<const W*>(w) + col.b, given);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            a.v[e] = given ? a.v[e] : 1.f;
            b.v[e] = given ? b.v[e] : 1.f;
        }
    }
};


// The pieces with what another lane counts left out.
template <int VEC>
__device__ __forceinline__ void counted(const float (&x)[VEC], int skip, float (&out)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = e >= skip ? x[e] : 0.f;
}

template <typename T, typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_kernel(const NormArgs a, T* __restrict__ q_out, T* __restrict__ k_out) {
    Place<T, VEC, L> at(a);
    const Columns<VEC> col = at.col;
    const Rows& rows = at.is_q ? a.q : a.k;
    const int head = at.is_q ? at.head : at.head - a.H, count = at.is_q ? a.H : a.G;
    const T* const x = static_cast<const T*>(rows.p) + head * rows.h;
    T* const out = (at.is_q ? q_out : k_out) + static_cast<int64_t>(head) * a.D;
    Cursor in(at.b, at.n, rows.b, rows.n, a), angle(at.b, at.n, a.angle_b, a.angle_n, a);
    const Weights<W, VEC> w(at.is_q ? a.wq : a.wk, col);
    const int64_t width = static_cast<int64_t>(count) * a.D;
    while (at.token < a.tokens) {
        Piece<T, VEC> xa, xb;
        Piece<float, VEC> c, s;
        xa.load(x + in.at + col.a, true);
        xb.load(x + in.at + col.b, true);
        c.load(a.cos + angle.at + col.a, col.turned);
        s.load(a.sin + angle.at + col.a, col.turned);
        float ca[VEC], cb[VEC], sum = 0.f;
        counted<VEC>(xa.v, col.skip_a, ca);
        counted<VEC>(xb.v, col.skip_b, cb);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum = __builtin_fmaf(ca[e], ca[e], __builtin_fmaf(cb[e], cb[e], sum));
        const float r = __builtin_amdgcn_rsqf(group_sum<L>(sum) * a.inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float ya = xa.v[e] * (r * w.a.v[e]), yb = xb.v[e] * (r * w.b.v[e]);
            const float ta = __builtin_fmaf(ya, c.v[e], -(yb * s.v[e]));
            const float tb = __builtin_fmaf(yb, c.v[e], ya * s.v[e]);
            xa.v[e] = col.turned ? ta : ya;
            xb.v[e] = col.turned ? tb : yb;
        }
        T* const dst = out + at.token * width;
        xa.store(dst + col.a, at.has_a);
        xb.store(dst + col.b, at.has_b);
        const bool wrapped = at.next(a);
        in.next(wrapped);
        angle.next(wrapped);
    }
}

template <typename T, typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_grad_kernel(const NormArgs a, const Rows gq, const Rows gk,
                                                                T* __restrict__ dq, T* __restrict__ dk,
                                                                float* __restrict__ part) {
    __shared__ float sums[kThreads / L][2 * L * VEC];  // a group's columns: its first pieces, then its second
    __shared__ int kinds[kThreads / L];
    Place<T, VEC, L> at(a);
    const Columns<VEC> col = at.col;
    const Rows& rows = at.is_q ? a.q : a.k;
    const Rows& grads = at.is_q ? gq : gk;
    const int head = at.is_q ? at.head : at.head - a.H, count = at.is_q ? a.H : a.G;
    const T* const x = static_cast<const T*>(rows.p) + head * rows.h;
    const T* const g = static_cast<const T*>(grads.p) + head * grads.h;
    T* const out = (at.is_q ? dq : dk) + static_cast<int64_t>(head) * a.D;
    Cursor in(at.b, at.n, rows.b, rows.n, a), from(at.b, at.n, grads.b, grads.n, a), angle(at.b, at.n, a.angle_b, a.angle_n, a);
    const Weights<W, VEC> w(at.is_q ? a.wq : a.wk, col);
    const int64_t width = static_cast<int64_t>(count) * a.D;
    float sa[VEC] = {}, sb[VEC] = {};
    while (at.token < a.tokens) {
        Piece<T, VEC> xa, xb, ga, gb;
        Piece<float, VEC> c, s;
        xa.load(x + in.at + col.a, true);
        xb.load(x + in.at + col.b, true);
        ga.load(g + from.at + col.a, true);
        gb.load(g + from.at + col.b, true);
        c.load(a.cos + angle.at + col.a, col.turned);
        s.load(a.sin + angle.at + col.a, col.turned);
        float ca[VEC], cb[VEC], ua[VEC], ub[VEC];  // x counted once, dy w
        counted<VEC>(xa.v, col.skip_a, ca);
        counted<VEC>(xb.v, col.skip_b, cb);
        float sum = 0.f, along = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float da = __builtin_fmaf(ga.v[e], c.v[e], gb.v[e] * s.v[e]);
            const float db = __builtin_fmaf(gb.v[e], c.v[e], -(ga.v[e] * s.v[e]));
            ga.v[e] = col.turned ? da : ga.v[e];
            gb.v[e] = col.turned ? db : gb.v[e];
            ua[e] = ga.v[e] * w.a.v[e];
            ub[e] = gb.v[e] * w.b.v[e];
            sum = __builtin_fmaf(ca[e], ca[e], __builtin_fmaf(cb[e], cb[e], sum));
            along = __builtin_fmaf(ca[e], ua[e], __builtin_fmaf(cb[e], ub[e], along));
        }
        const float r = __builtin_amdgcn_rsqf(group_sum<L>(sum) * a.inv_d + a.eps);
        const float mean = group_sum<L>(along) * r * a.inv_d;
        const float back = mean * r * r;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sa[e] = __builtin_fmaf(ga.v[e], xa.v[e] * r, sa[e]);
            sb[e] = __builtin_fmaf(gb.v[e], xb.v[e] * r, sb[e]);
            xa.v[e] = __builtin_fmaf(ua[e], r, -(xa.v[e] * back));
            xb.v[e] = __builtin_fmaf(ub[e], r, -(xb.v[e] * back));
        }
        // Of a row of one value the difference leaves eps r^2 alone, which rounding would bury.
        if constexpr (VEC == 1 && L == 1)
            if (a.D == 1) xa.v[0] = r * r * r * a.eps * ua[0];
        T* const dst = out + at.token * width;
        xa.store(dst + col.a, at.has_a);
        xb.store(dst + col.b, at.has_b);
        const bool wrapped = at.next(a);
        in.next(wrapped);
        from.next(wrapped);
        angle.next(wrapped);
    }
    if (part == nullptr) return;
    // part (blocks, q or k, columns in the lanes' order)
    constexpr int kColumns = 2 * L * VEC;
    const int group = threadIdx.x / L, unit = threadIdx.x % L;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        sums[group][unit * VEC + e] = sa[e];
        sums[group][(L + unit) * VEC + e] = sb[e];
    }
    if (unit == 0) kinds[group] = at.is_q ? 0 : 1;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * kColumns; i += kThreads) {
        float all = 0.f;
#pragma unroll 8
        for (int gr = 0; gr < kThreads / L; ++gr) all += kinds[gr] == i / kColumns ? sums[gr][i % kColumns] : 0.f;
        part[static_cast<int64_t>(blockIdx.x) * 2 * kColumns + i] = all;
    }
}

// dw from the blocks' parts: a block for 8 columns, 32 lanes of blocks each.
template <typename W, int VEC, int L>
__global__ __launch_bounds__(kThreads) void qk_norm_weight_kernel(const float* __restrict__ part, int blocks, int D, int R,
                                                                  W* __restrict__ dwq, W* __restrict__ dwk) {
    constexpr int kColumns = 2 * L * VEC, kAcross = 8, kLanes = kThreads / kAcross;
    __shared__ float sums[kLanes][kAcross];
    const int x = threadIdx.x % kAcross, y = threadIdx.x / kAcross, id = blockIdx.x * kAcross + x;
    float all = 0.f;
    if (id < 2 * kColumns) {
#pragma unroll 16
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
    int vec, units, lanes;
    int64_t blocks, step;
};

// The widest pieces that the rotated half and the rest hold, and blocks enough
// to fill the card (each keeps its sums until its end).
Shape shape_of(const pointops_qk_norm& in) {
    const int half = static_cast<int>(in.R / 2), rest = static_cast<int>(in.D - in.R);
    Shape s;
    s.vec = in.type == POINTOPS_F32 ? 4 : 8;
    while ((half > 0 && s.vec > half) || (rest > 0 && s.vec > rest)) s.vec /= 2;
    s.units = (half + s.vec - 1) / s.vec + ((rest + s.vec - 1) / s.vec + 1) / 2;
    s.lanes = 1;
    while (s.lanes < s.units) s.lanes *= 2;
    const int64_t tokens = in.B * in.N, heads = std::max<int64_t>(1, in.H + in.G), groups = kThreads / s.lanes;
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
    a.units = s.units;
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
    const bool sums = dq_weight != nullptr || dk_weight != nullptr;
    const bool none = in->B == 0 || in->N == 0 || in->H + in->G == 0;
    if (none && !sums) return hipSuccess;
    if (!none && ((in->H > 0 && (in->q == nullptr || dq == nullptr || q_grad == nullptr || q_grad_stride == nullptr)) ||
        (in->G > 0 && (in->k == nullptr || dk == nullptr || k_grad == nullptr || k_grad_stride == nullptr)) ||
        (in->R > 0 && (in->cos == nullptr || in->sin == nullptr))))
        return hipErrorInvalidValue;
    if (!none && sums && workspace == nullptr) return hipErrorInvalidValue;
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
        if (!none) {
            hipLaunchKernelGGL((qk_norm_grad_kernel<T, W, VEC, L>), dim3(static_cast<uint32_t>(s.blocks)), dim3(kThreads), 0,
                               stream, a, gq, gk, static_cast<T*>(dq), static_cast<T*>(dk), part);
            const hipError_t err = hipGetLastError();
            if (err != hipSuccess || !sums) return err;
        }
        hipLaunchKernelGGL((qk_norm_weight_kernel<W, VEC, L>), dim3((4 * L * VEC + 7) / 8), dim3(kThreads), 0, stream, part,
                           none ? 0 : static_cast<int>(s.blocks), a.D, a.R, static_cast<W*>(dq_weight), static_cast<W*>(dk_weight));
        return hipGetLastError();
    });
}

}  // extern "C"
