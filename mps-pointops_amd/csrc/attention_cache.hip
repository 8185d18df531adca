// Attention of new tokens over caches and a common start: the calls, how the keys are cut
// into parts, and the kernel that joins them.
#include "attention_cache.hpp"

namespace pointops {
namespace attn {

#define POINTOPS_FORM(T, F) \
    extern template hipError_t launch_cache_form<T, F>(const CacheArgs&, const CachePlan&, void*, float*, hipStream_t);
POINTOPS_FORM(float, kAligned)
POINTOPS_FORM(float, kAny)
POINTOPS_FORM(float, kEight)
POINTOPS_FORM(float, kFour)
POINTOPS_FORM(f16, kAligned)
POINTOPS_FORM(f16, kAny)
POINTOPS_FORM(f16, kEight)
POINTOPS_FORM(f16, kFour)
POINTOPS_FORM(bf16, kAligned)
POINTOPS_FORM(bf16, kAny)
POINTOPS_FORM(bf16, kEight)
POINTOPS_FORM(bf16, kFour)
#undef POINTOPS_FORM

namespace {

struct JoinArgs {
    int B, Q, H, G, D, group, per, width;
    int start_rows, own_rows, start_blocks, own_blocks, start_splits, own_splits;
    int64_t start_floats;
};

// One wave a row: its parts, of the start's keys and of its own, brought to their common
// maximum and added in order.  The first ones' values are asked for beside the maxima.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_cache_join_kernel(const JoinArgs a, const float* __restrict__ parts,
                                                                        T* __restrict__ out) {
    const int lane = lane_id(), width = a.width;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;  // (g, b, row)
    const int64_t all = static_cast<int64_t>(a.B) * a.per, in_g = id % all;
    if (id >= a.G * all) return;
    const int g = static_cast<int>(id / all), b = static_cast<int>(in_g / a.per), row = static_cast<int>(in_g % a.per);
    // Of each kind: the row's first part, and from one to the next.
    const int64_t start_unit = static_cast<int64_t>(g) * a.start_blocks + in_g / a.start_rows;
    const int64_t own_unit = (static_cast<int64_t>(b) * a.G + g) * a.own_blocks + row / a.own_rows;
    const float* const start = parts + (start_unit * a.start_splits * a.start_rows + in_g % a.start_rows) * width;
    const float* const own = parts + a.start_floats + (own_unit * a.own_splits * a.own_rows + row % a.own_rows) * width;
    const int start_step = a.start_rows * width, own_step = a.own_rows * width;
    const int count = a.start_splits + a.own_splits;
    auto part = [&](int s) {
        return s < a.start_splits ? start + static_cast<int64_t>(s) * start_step
                                  : own + static_cast<int64_t>(s - a.start_splits) * own_step;
    };
    const int c0 = 4 + min(lane, a.D - 1), c1 = 4 + min(lane + kWave, a.D - 1);
    constexpr int kAtOnce = 16;
    float y0[kAtOnce], y1[kAtOnce];
    auto ask = [&](int from) {  // (past the end: the last one again, for which the factor is not used)
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const float* const at = part(min(from + k, count - 1));
            y0[k] = at[c0];
            y1[k] = at[c1];
        }
    };
    ask(0);
    float top = -kInf;
    for (int s = lane; s < count; s += kWave) top = fmaxf(top, part(s)[0]);
    top = wave_max(top);
    const float less = top == -kInf ? 0.f : top;
    float sum = 0.f, x0 = 0.f, x1 = 0.f;
    for (int from = 0; from < count; from += kWave) {
        // A lane's part: its factor; then the parts' rows one after another.
        const int s = from + lane;
        float by = 0.f;
        if (s < count) {
            by = exp2_fast(part(s)[0] - less);
            sum = __builtin_fmaf(part(s)[1], by, sum);
        }
        const int some = min(kWave, count - from);
        for (int i = 0; i < some; i += kAtOnce) {
            if (from + i > 0) ask(from + i);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (i + k < some) {
                    const float f = i2f(readlane(f2i(by), i + k));
                    x0 = __builtin_fmaf(y0[k], f, x0);
                    x1 = __builtin_fmaf(y1[k], f, x1);
                }
            }
        }
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* const dst = out + ((static_cast<int64_t>(b) * a.Q + row / a.group) * a.H + g * a.group + row % a.group) * a.D;
    if (lane < a.D) dst[lane] = from_float<T>(x0 * inv);
    if (lane + kWave < a.D) dst[lane + kWave] = from_float<T>(x1 * inv);
}

int size_of(int type) { return type == POINTOPS_F32 ? 4 : 2; }

bool read_keys(const pointops_keys& in, const pointops_cache_attention& call, Kept* out) {
    if (in.N < 0 || in.N > (int64_t(1) << 30) - 1024) return false;
    Kept& k = *out;
    k = {};
    k.tokens = static_cast<int>(in.N);
    if (in.N == 0) return true;
    k.k = static_cast<const char*>(in.k);
    k.v = static_cast<const char*>(in.v);
    if (call.bits == 0) {
        const int64_t size = size_of(call.type);
        k.kb = in.k_stride[0] * size;
        k.kn = in.k_stride[1] * size;
        k.kh = in.k_stride[2] * size;
        k.vb = in.v_stride[0] * size;
        k.vn = in.v_stride[1] * size;
        k.vh = in.v_stride[2] * size;
        return true;
    }
    const int64_t row = padded(static_cast<int>(call.D)) * call.bits / 8, scales = padded(static_cast<int>(call.D)) / kGroup;
    k.k_scales = in.k_scales;
    k.v_scales = in.v_scales;
    k.kb = k.vb = in.k_stride[0] * row;
    k.kn = k.vn = row;
    k.kh = k.vh = in.k_stride[2] * row;
    k.sb = in.k_stride[0] * scales;
    k.sh = in.k_stride[2] * scales;
    return true;
}

bool read_call(const pointops_cache_attention* in, CacheArgs* out) {
    const int64_t limit = (int64_t(1) << 30) - 1024;  // sums of two positions fit an int
    if (in == nullptr) return false;
    if (in->B < 0 || in->Q < 0 || in->H < 0 || in->G < 0 || in->D < 1 || in->D > kMaxHead) return false;
    if (in->B > limit || in->Q > limit || in->H > limit || in->G > limit) return false;
    if (in->type < POINTOPS_F32 || in->type > POINTOPS_BF16) return false;
    if (in->bits != 0 && in->bits != 8 && in->bits != 4) return false;
    if (in->H > 0 && (in->G < 1 || in->H % in->G != 0)) return false;
    if (in->window < 1 || in->sinks < 0) return false;
    if (in->lengths != nullptr && in->length_bits != 32 && in->length_bits != 64) return false;
    CacheArgs& a = *out;
    if (!read_keys(in->start, *in, &a.start) || !read_keys(in->own, *in, &a.own)) return false;
    const int64_t keys = static_cast<int64_t>(a.start.tokens) + a.own.tokens;
    if (keys > limit || in->B * in->Q > limit || in->B * in->Q * in->H > limit) return false;
    a.q = {in->q, in->q_stride[0], in->q_stride[1], in->q_stride[2]};
    a.q_vec = false;
    a.bias = in->bias;
    a.lengths = in->lengths;
    a.length_bits = in->length_bits;
    a.B = static_cast<int>(in->B);
    a.Q = static_cast<int>(in->Q);
    a.H = static_cast<int>(in->H);
    a.G = static_cast<int>(in->G);
    a.D = static_cast<int>(in->D);
    a.window = static_cast<int>(std::min(in->window, keys + 1));
    a.sinks = static_cast<int>(std::min(in->sinks, keys));
    a.scale_log2 = in->scale * kLog2e;
    a.reach = 0;
    a.bk.n = a.bk.count = 0;
    if (in->bias != nullptr) {
        if (!read_buckets(in->edges, in->n_edges, in->buckets, kMaxReach, &a.bk)) return false;
        if (a.bk.count != a.bk.n + 1) return false;
        a.reach = a.bk.edge[a.bk.n - 1];
    }
    return true;
}

// (Strides in bytes.  A tile of up to 64 rows lies within 2 GiB behind its first.)
bool pieces(const void* p, int64_t b, int64_t n, int64_t h) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && b % 16 == 0 && n % 16 == 0 && h % 16 == 0 && n >= 0 && n < (1 << 25);
}
bool pieces(const Kept& k) { return k.tokens == 0 || (pieces(k.k, k.kb, k.kn, k.kh) && pieces(k.v, k.vb, k.vn, k.vh)); }

// Rows that 16-byte reads serve: a row's reads stay inside it, as D is a multiple of a piece.
int form_of(const pointops_cache_attention& in, CacheArgs* a) {
    const int64_t size = size_of(in.type);
    const bool whole = in.D * size % 16 == 0;
    a->q_vec = whole && pieces(a->q.p, a->q.b * size, a->q.n * size, a->q.h * size);
    if (in.bits != 0) return in.bits;
    return whole && pieces(a->start) && pieces(a->own) ? kAligned : kAny;
}

// Where what a sequence's rows see are so many tiles at most, and so many of all sequences (whose
// blocks each read the start's keys), one launch of whole rows is shorter than parts and their join.
constexpr int kDirectTiles = 40, kDirectWork = 16384;

// Parts that give every compute unit the two blocks that its registers hold (4 x 65536 tokens in
// 8 bits: 98 us by 512 blocks, 104 by 1024 in two rounds), at least two tiles a wave; the start's and the caches' as their work is to each other.  By
// the caches' sizes: the lengths are on the device, and a call does not wait for it.
CachePlan plan_of(const CacheArgs& a, int form) {
    CachePlan p = {};
    const int64_t per = static_cast<int64_t>(a.Q) * (a.H / a.G), all = per * a.B;
    const bool some = a.start.tokens != 0;
    const int64_t seen = (static_cast<int64_t>(a.window) + a.Q - 1) / kKeys + 2 + (a.sinks + kKeys - 1) / kKeys;
    auto tiles = [&](int tokens) { return std::min<int64_t>((static_cast<int64_t>(tokens) + kKeys - 1) / kKeys, seen); };
    const int64_t start_tiles = tiles(a.start.tokens), own_tiles = tiles(a.own.tokens);
    // (A window over both sees no more than one over either.)
    const int64_t all_tiles = std::min(start_tiles + own_tiles, seen + 1);
    if (form == kAny) p.shape = kTwoTwo;
    else if (per <= 16 && all_tiles <= kDirectTiles && all_tiles * a.B * a.G <= kDirectWork) p.shape = kDirect;
    else if (per > 16) p.shape = some && all > 32 ? kPairsTwo : kTwoTwo;
    else if (!some || all <= 16) p.shape = kOne;
    else p.shape = all <= 32 ? kTwo : kPairs;
    const ShapeRows rows = kShapeRows[p.shape];
    p.start_rows = 16 * rows.cols * rows.row_waves;
    p.own_rows = 16 * rows.own_cols;
    auto blocks = [](int64_t rows, int each) { return static_cast<int>((rows + each - 1) / each); };
    p.own_blocks = blocks(per, p.own_rows);
    p.own_units = static_cast<int64_t>(a.B) * a.G * p.own_blocks;
    if (p.shape == kDirect) {
        p.own_splits = 1;
        p.direct = true;
        return p;
    }
    p.start_blocks = blocks(all, p.start_rows);
    p.start_units = some ? static_cast<int64_t>(a.G) * p.start_blocks : 0;
    const double start_work = static_cast<double>(p.start_units) * start_tiles * std::max(1, rows.row_waves);
    const double own_work = static_cast<double>(p.own_units) * own_tiles;
    const double target = 512, sum = std::max(1.0, start_work + own_work);
    auto splits = [&](double work, int64_t units, int64_t count) {
        const int64_t wanted = static_cast<int64_t>(target * (work / sum) / std::max<int64_t>(1, units) + 0.999);
        return static_cast<int>(std::max<int64_t>(1, std::min(wanted, count / (2 * kStepWaves))));
    };
    p.start_splits = p.start_units == 0 ? 0 : splits(start_work, p.start_units, start_tiles);
    p.own_splits = splits(own_work, p.own_units, own_tiles);
    p.direct = p.start_splits == 0 && p.own_splits == 1;
    p.start_floats = p.start_units * p.start_splits * p.start_rows * part_width(padded(a.D));
    return p;
}

size_t workspace_of(const CacheArgs& a, const CachePlan& p) {
    if (p.direct) return 0;
    return sizeof(float) * (p.start_floats + p.own_units * p.own_splits * p.own_rows * part_width(padded(a.D)));
}

template <typename T>
hipError_t cache_step(const CacheArgs& a, int form, void* out, void* workspace, hipStream_t stream) {
    const CachePlan plan = plan_of(a, form);
    if (workspace == nullptr && workspace_of(a, plan) != 0) return hipErrorInvalidValue;
    const int64_t blocks = plan.start_units * plan.start_splits + plan.own_units * plan.own_splits;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;
    float* const parts = static_cast<float*>(workspace);
    const auto launch = form == kAligned ? launch_cache_form<T, kAligned>
                        : form == kAny   ? launch_cache_form<T, kAny>
                        : form == kEight ? launch_cache_form<T, kEight>
                                         : launch_cache_form<T, kFour>;
    const hipError_t err = launch(a, plan, out, parts, stream);
    if (err != hipSuccess || plan.direct) return err;
    const int64_t rows = static_cast<int64_t>(a.B) * a.Q * a.H;
    const JoinArgs join = {a.B, a.Q, a.H, a.G, a.D, a.H / a.G, a.Q * (a.H / a.G), part_width(padded(a.D)), plan.start_rows, plan.own_rows,
                           plan.start_blocks, plan.own_blocks, plan.start_splits, plan.own_splits, plan.start_floats};
    hipLaunchKernelGGL(attention_cache_join_kernel<T>, dim3(static_cast<uint32_t>((rows + kWaves - 1) / kWaves)),
                       dim3(kThreads), 0, stream, join, static_cast<const float*>(parts), static_cast<T*>(out));
    return hipGetLastError();
}

bool kept_aligned(const Kept& k, int D) {
    return k.tokens == 0 || (pieces(k) && codes_aligned(k.k, k.k_scales, D) && codes_aligned(k.v, k.v_scales, D));
}

bool no_keys(const pointops_keys& k, int bits) {
    return k.N > 0 && (k.k == nullptr || k.v == nullptr || (bits != 0 && (k.k_scales == nullptr || k.v_scales == nullptr)));
}

}  // namespace
}  // namespace attn
}  // namespace pointops

extern "C" {

size_t pointops_cache_attention_step_workspace_bytes(const pointops_cache_attention* in) {
    using namespace pointops::attn;
    CacheArgs a;
    if (!read_call(in, &a) || a.B == 0 || a.H == 0 || a.Q == 0) return 0;
    const int form = form_of(*in, &a);
    return workspace_of(a, plan_of(a, form));
}

hipError_t pointops_cache_attention_step(const pointops_cache_attention* in, void* out, void* workspace, hipStream_t stream) {
    using namespace pointops::attn;
    CacheArgs a;
    if (!read_call(in, &a)) return hipErrorInvalidValue;
    if (a.B == 0 || a.H == 0 || a.Q == 0) return hipSuccess;
    if (in->q == nullptr || out == nullptr || no_keys(in->start, in->bits) || no_keys(in->own, in->bits)) return hipErrorInvalidValue;
    if (in->bits != 0 && (!kept_aligned(a.start, a.D) || !kept_aligned(a.own, a.D))) return hipErrorInvalidValue;
    const int form = form_of(*in, &a);
    switch (in->type) {
        case POINTOPS_F32: return cache_step<float>(a, form, out, workspace, stream);
        case POINTOPS_F16: return cache_step<f16>(a, form, out, workspace, stream);
        default: return cache_step<bf16>(a, form, out, workspace, stream);
    }
}

}  // extern "C"
