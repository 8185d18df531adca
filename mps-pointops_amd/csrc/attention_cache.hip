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
    Divisor all, per, group;  // rows of a key head, of a sequence's, heads of a key head
    int rows, Q, H, G, D;
    Parts start, own;
};

// One wave a row: its parts, of the start's keys and of its own.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_cache_join_kernel(const JoinArgs a, const float* __restrict__ parts,
                                                                        T* __restrict__ out, uint32_t first_block) {
    const int width = part_width(padded(a.D)), id = uniform(static_cast<int>((first_block + blockIdx.x) * kWaves + threadIdx.x / kWave));  // (g, b, row)
    if (id >= a.rows) return;
    const int g = a.all.of_row(id), in_g = id - g * static_cast<int>(a.all.d);
    const int b = a.per.of_row(in_g), row = in_g - b * static_cast<int>(a.per.d), i = a.group.of_row(row);
    auto join = [&](RowSum sum) {
        sum.add(a.start.first(parts, g, in_g, width), static_cast<int64_t>(a.start.rows) * width, a.start.splits, a.D);
        sum.add(a.own.first(parts + a.start.floats, b * a.G + g, row, width), static_cast<int64_t>(a.own.rows) * width, a.own.splits, a.D);
        sum.divide();
        return sum;
    };
    RowSum sum = join({});
    if (ballot(!finite(sum.x0) || !finite(sum.x1)) != 0) {
        // Values near the largest, of which a mean is finite and a sum need not be.
        RowSum low;
        low.above = 30.f;
        low = join(low);
        sum.x0 = finite(sum.x0) ? sum.x0 : low.x0;
        sum.x1 = finite(sum.x1) ? sum.x1 : low.x1;
    }
    const int h = g * static_cast<int>(a.group.d) + row - i * static_cast<int>(a.group.d);
    sum.write(out + ((static_cast<int64_t>(b) * a.Q + i) * a.H + h) * a.D, a.D);
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
    a.group = Divisor::of(in->H > 0 ? in->H / in->G : 1);
    a.per = Divisor::of(in->H > 0 && in->Q > 0 ? in->H / in->G * in->Q : 1);
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

// Rows that 16-byte reads serve: a row's reads stay inside it, as D is a multiple of a piece.  Where one
// tensor's are not, all of a call's are read value by value, by kernels of 32 rows a wave that do not
// share a start's keys (64 behind 16384, bfloat16, width 124: 773 us, 128: 66; 20: 131, 24: 43; 8 behind
// 1024, window 512, width 60: 27.5, 64: 8.0).
int form_of(const pointops_cache_attention& in, CacheArgs* a) {
    const int64_t size = size_of(in.type);
    const bool whole = in.D * size % 16 == 0;
    a->q_vec = whole && pieces(a->q.p, a->q.b * size, a->q.n * size, a->q.h * size);
    if (in.bits != 0) return in.bits;
    return whole && pieces(a->start) && pieces(a->own) ? kAligned : kAny;
}

// LDS of a start's block whose waves share their keys: two sets of tiles (or the sums), the bias.
size_t pairs_lds(const CacheArgs& a, int type, int form) {
    const bool words = form == kAligned && type == POINTOPS_F32, streamed = form == kAligned && !words;
    const size_t bytes = padded(a.D) * (words ? 4 : 2), stride = streamed ? bytes : bytes + (bytes == 256 ? 48 : 16), key_waves = kStepWaves / kShapeRows[kPairs].row_waves;
    const size_t rows = kShapeRows[kPairs].start(), tiles = 4 * kKeys * key_waves * stride, sums = rows * part_width(padded(a.D)) * 4;
    return std::max(tiles, sums) + 2 * key_waves * rows * 4 + bias_lds(a, static_cast<int>(rows));
}

// Where what a sequence's rows see are so many tiles at most, and so many of all sequences (whose
// blocks each read the start's keys), one launch of whole rows: a call of parts waits for the host 4.5 us
// longer, for its workspace and its join.  4 sequences, 32 heads over 8 of 128, by one launch and by
// parts: over 8 bits and 16 tiles 10.6 and 14.1 us, 32 tiles 13.3 and 14.1, 40 tiles 14.6 and 14.3;
// bfloat16 14.7 and 19.3, 17.4 and 19.2, 20.9 and 19.0.  Recorded in a graph, where the host does not
// count, parts are shorter from about 20 tiles on (8 bits 10.5 and 10.9, 13.6 and 11.1, 14.5 and 11.1), and
// over float32 tensors, whose tiles take three times as long, they are everywhere (24 and 18, 41 and
// 19, 49 and 20).  64 sequences of 40 tiles in 8 bits (20480 of all key heads): 38 and 32.
constexpr int kDirectTiles = 40, kDirectWork = 16384;

// Parts that give every compute unit two blocks, at least two tiles a wave; the start's and
// the caches' as their work is to each other.  Kernels over codes of 16-bit queries would hold three;
// by 256, 512, 768 and 1024 blocks: 4 x 65536 tokens in 8 bits 88, 90, 92, 91 us, 32 x 8192 under float16
// in 8 bits 90, 89, 103, 93, in 4 bits 64, 56, 55, 62; 64 behind 65536, bfloat16, 166, 133, 145, 146.  By the caches' sizes: the lengths are on the device, and
// a call does not wait for it.
CachePlan plan_of(const CacheArgs& a, int type, int form) {
    CachePlan p = {};
    const int64_t per = a.per.d, all = per * a.B, width = part_width(padded(a.D));
    const int64_t seen = (static_cast<int64_t>(a.window) + a.Q - 1) / kKeys + 2 + (a.sinks + kKeys - 1) / kKeys;
    auto tiles = [&](int tokens) { return std::min<int64_t>((static_cast<int64_t>(tokens) + kKeys - 1) / kKeys, seen); };
    const int64_t start_tiles = tiles(a.start.tokens), own_tiles = tiles(a.own.tokens);
    // (A window over both sees no more than one over either.)
    const int64_t both = std::min(start_tiles + own_tiles, seen + 1), heads = static_cast<int64_t>(a.B) * a.G;
    const bool some = a.start.tokens != 0, pairs = pairs_lds(a, type, form) <= kMostLds;
    if (form == kAny) p.shape = kTwoTwo;
    else if (per <= 16 && both <= kDirectTiles && both * heads <= kDirectWork) p.shape = kDirect;
    else if (per > 16) p.shape = some && all > 32 && pairs ? kPairsTwo : kTwoTwo;
    else if (!some || all <= 16) p.shape = kOne;
    else p.shape = all > 32 && pairs ? kPairs : kTwo;
    const ShapeRows rows = kShapeRows[p.shape];
    auto cut = [&](Parts& parts, int each, int64_t rows, int64_t heads) {
        while ((1 << parts.shift) < each) ++parts.shift;
        parts.blocks = static_cast<int>((rows + each - 1) / each);
        parts.rows = static_cast<int>(std::min<int64_t>(each, rows));
        parts.units = heads * parts.blocks;
    };
    cut(p.own, rows.own(), per, heads);
    p.own.splits = 1;
    if (p.shape == kDirect) return p;
    if (some) cut(p.start, rows.start(), all, a.G);
    const double start_work = static_cast<double>(p.start.units) * start_tiles * rows.row_waves;
    const double own_work = static_cast<double>(p.own.units) * own_tiles, sum = std::max(1.0, start_work + own_work);
    auto split = [&](Parts& parts, double work, int64_t count) {
        const int64_t wanted = static_cast<int64_t>(512 * (work / sum) / std::max<int64_t>(1, parts.units) + 0.999);
        parts.splits = static_cast<int>(std::max<int64_t>(1, std::min(wanted, count / (2 * kStepWaves))));
        parts.floats = parts.units * parts.splits * parts.rows * width;
    };
    if (some) split(p.start, start_work, start_tiles);
    split(p.own, own_work, own_tiles);
    p.joined = some || p.own.splits > 1;
    return p;
}

size_t workspace_of(const CachePlan& p) { return sizeof(float) * (p.start.floats + (p.joined ? p.own.floats : 0)); }

template <typename T>
hipError_t cache_step(const CacheArgs& a, int type, int form, void* out, void* workspace, hipStream_t stream) {
    const CachePlan plan = plan_of(a, type, form);
    if (workspace == nullptr && workspace_of(plan) != 0) return hipErrorInvalidValue;
    if (plan.start.units * plan.start.splits + plan.own.units * plan.own.splits > INT32_MAX) return hipErrorInvalidValue;
    float* const parts = static_cast<float*>(workspace);
    const auto launch = form == kAligned ? launch_cache_form<T, kAligned>
                        : form == kAny   ? launch_cache_form<T, kAny>
                        : form == kEight ? launch_cache_form<T, kEight>
                                         : launch_cache_form<T, kFour>;
    const hipError_t err = launch(a, plan, out, parts, stream);
    if (err != hipSuccess || !plan.joined) return err;
    const int64_t rows = static_cast<int64_t>(a.B) * a.Q * a.H;  // (at most 2^30)
    const JoinArgs join = {Divisor::of(rows / a.G), a.per, a.group, static_cast<int>(rows), a.Q, a.H, a.G, a.D, plan.start, plan.own};
    return in_launches(static_cast<uint32_t>((rows + kWaves - 1) / kWaves), [&](uint32_t first, uint32_t count) {
        hipLaunchKernelGGL(attention_cache_join_kernel<T>, dim3(count), dim3(kThreads), 0, stream, join,
                           static_cast<const float*>(parts), static_cast<T*>(out), first);
    });
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
    return workspace_of(plan_of(a, in->type, form));
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
        case POINTOPS_F32: return cache_step<float>(a, in->type, form, out, workspace, stream);
        case POINTOPS_F16: return cache_step<f16>(a, in->type, form, out, workspace, stream);
        default: return cache_step<bf16>(a, in->type, form, out, workspace, stream);
    }
}

}  // extern "C"
