// Rotary positions: each pair of channels of a row is turned by position * frequency, forwards or back (the gradient).
//
// Bound by HBM: every value is read once and written once. The angles belong to a token, not to a head, so a CTA takes a few
// tokens and a run of heads, works out the tokens' sines and cosines once into shared memory and turns all the heads' rows by them.
// position * frequency passes 2^24 for far positions, where f32 has lost the angle: the product and its reduction to one turn are
// made in f64 (one product, rint and difference a pair and token), the sine and cosine of what is left, within half a turn, in f32.
// Next come the issue slots (two thirds taken): rows and units are stepped to, and a CTA's heads are of one pair of tensors (with the L2 flushed before
// each pass 57.7 us for 60.4, the gradient below 22.9 for 25.6).
// 2 x 8192 tokens, 32 + 8 heads of 128 bf16 channels: 56 to 59 us, 5.7 to 6.0 TB/s, 86 to 91 % of the copy rate; 3 x 1001 f32 tokens, 16 + 16 heads, half of each
// turned: 21 us, 4.7 TB/s; one token of 32 sequences: 5.4 us, a launch.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "dfgpu_cache.h"

namespace dfgpu {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kRopeTable = 2048;      // (cosine, sine) pairs of a CTA: 16 KiB
constexpr int64_t kRopeMaxD = 1024;

struct RopeSide {
    const void* x;
    void* y;
    int64_t x_stride[3], y_stride[3];   // batch, head, token
    int32_t heads, in_place;            // in_place: channels that are not turned stay where they are
};
struct RopeArgs {
    RopeSide side[2];
    const void* positions;
    const float* frequencies;
    int64_t position_batch, position_token, frequency_stride;
    int32_t positions_wide, seq, tiles, token_shift;   // a CTA's tokens: 1 << token_shift
    int32_t first_side, heads_per_cta, half, turning, units, pitch;   // first_side: runs of heads of the first pair of tensors; units of V pairs (half) or V channels (interleaved) a row; pitch: of a token in the table
    int32_t rows_on, units_on;                         // kRopeThreads units on: whole rows, and the units beyond
    FastDivisor by_units, by_tiles;
    float scale, sign;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// One unit of a row: V pairs as two vectors (i and i + half), or with INTERLEAVED V channels as one (V = 1: one pair as two values).
template <typename T, int V, bool INTERLEAVED>
struct RopeUnit {
    static constexpr bool kTwo = !INTERLEAVED || V == 1;
    static constexpr int kPairs = kTwo ? V : V / 2;
    Pack<T, V> first, second;
    T* to;
    int32_t table;     // the first pair's place in the table; -1: channels to copy, -2: nothing
    int32_t apart;     // elements from the first vector to the second

    // row: (head of the run, token of the CTA); x, y: of the run's first head and the CTA's first token
    __device__ __forceinline__ void load(const RopeArgs& a, const RopeSide& s, const T* x, T* y, int row, int rows, int unit, int tokens) {
        table = -2;
        const int local = row & ((1 << a.token_shift) - 1), head = row >> a.token_shift;
        const bool turns = unit < a.turning;
        if (row >= rows || local >= tokens || (!turns && s.in_place)) return;
        const int channel = turns ? (INTERLEAVED ? unit * (V == 1 ? 2 : V) : unit * V) : 2 * a.half + (unit - a.turning) * V;
        apart = INTERLEAVED ? 1 : a.half;
        const T* from = x + head * s.x_stride[1] + local * s.x_stride[2] + channel;
        to = y + head * s.y_stride[1] + local * s.y_stride[2] + channel;
        table = turns ? local * a.pitch + unit : -1;
        first = *reinterpret_cast<const Pack<T, V>*>(from);
        if (kTwo && turns) second = *reinterpret_cast<const Pack<T, V>*>(from + apart);
    }
    __device__ __forceinline__ void turn_and_store(const RopeArgs& a, const float2* angles) {
        if (table == -2) return;
        if (table >= 0) {
#pragma unroll
            for (int p = 0; p < kPairs; ++p) {
                const float2 cs = angles[table + p * a.turning];   // (pair p of neighbouring units side by side)
                T& one = kTwo ? first.v[p] : first.v[2 * p];
                T& two = kTwo ? second.v[p] : first.v[(2 * p + 1) % V];
                const float x1 = widen(one), x2 = widen(two);
                one = narrow<T>(__fmaf_rn(x1, cs.x, -(x2 * cs.y)));
                two = narrow<T>(__fmaf_rn(x2, cs.x, x1 * cs.y));
            }
            if (kTwo) *reinterpret_cast<Pack<T, V>*>(to + apart) = second;
        }
        *reinterpret_cast<Pack<T, V>*>(to) = first;
    }
};

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads)
rope_kernel(RopeArgs a) {
    using Unit = RopeUnit<T, V, INTERLEAVED>;
    extern __shared__ float2 angles[];
    const int tile = static_cast<int>(blockIdx.x);
    const int batch_index = static_cast<int>(fast_divide(static_cast<uint32_t>(tile), a.by_tiles));
    const int token0 = (tile - batch_index * a.tiles) << a.token_shift;
    // A CTA's heads are of one pair of tensors, so that all of its addresses share their strides.
    const bool second_side = static_cast<int>(blockIdx.y) >= a.first_side;
    const RopeSide s = second_side ? a.side[1] : a.side[0];
    const int head0 = (static_cast<int>(blockIdx.y) - (second_side ? a.first_side : 0)) * a.heads_per_cta;
    const int rows = min(a.heads_per_cta, s.heads - head0) << a.token_shift, tokens = a.seq - token0;
    const T* x = static_cast<const T*>(s.x) + batch_index * s.x_stride[0] + head0 * s.x_stride[1] + token0 * s.x_stride[2];
    T* y = static_cast<T*>(s.y) + batch_index * s.y_stride[0] + head0 * s.y_stride[1] + token0 * s.y_stride[2];
    chain_begin();
    int row = static_cast<int>(fast_divide(threadIdx.x, a.by_units)), unit = static_cast<int>(threadIdx.x) - row * a.units;
    Unit now, next;
    now.load(a, s, x, y, row, rows, unit, tokens);   // (on its way while the angles are worked out)
    for (int i = threadIdx.x; i < a.half << a.token_shift; i += kRopeThreads) {
        const int local = i & ((1 << a.token_shift) - 1), pair = i >> a.token_shift;
        if (token0 + local < a.seq) {
            const int64_t at = batch_index * a.position_batch + (token0 + local) * a.position_token;
            const int64_t position = a.positions_wide ? static_cast<const int64_t*>(a.positions)[at] : static_cast<int64_t>(static_cast<const int32_t*>(a.positions)[at]);
            const double turns = static_cast<double>(position) * static_cast<double>(a.frequencies[pair * a.frequency_stride]) * 0.15915494309189533577;
            float sine, cosine;
            sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sine, &cosine);
            const int unit = pair / Unit::kPairs;
            angles[local * a.pitch + (pair - unit * Unit::kPairs) * a.turning + unit] = make_float2(cosine * a.scale, sine * a.scale * a.sign);
        }
    }
    __syncthreads();
    while (row < rows) {
        row += a.rows_on, unit += a.units_on;
        if (unit >= a.units) unit -= a.units, ++row;
        next.load(a, s, x, y, row, rows, unit, tokens);
        now.turn_and_store(a, angles);
        now = next;
    }
}

bool aligned(const void* pointer, int64_t bytes) { return (reinterpret_cast<uintptr_t>(pointer) & static_cast<uintptr_t>(bytes - 1)) == 0; }

int check_side(const dfgpu_tensor& x, const dfgpu_tensor& y, const dfgpu_tensor& reference, const char* name) {
    if (!valid_tensor(x) || !valid_tensor(y) || x.rank != 4 || y.rank != 4) return fail(kInvalidShape, "ROPE: %s must have rank 4 and positive extents", name);
    for (int i = 0; i < 4; ++i) {
        if (x.dim[i] != y.dim[i]) return fail(kInvalidShape, "ROPE: input and output of %s differ in extent", name);
        if (i != 1 && x.dim[i] != reference.dim[i]) return fail(kInvalidShape, "ROPE: X and X2 differ in batch, length or head dimension");
    }
    if (x.dtype != DFGPU_F32 && x.dtype != DFGPU_F16 && x.dtype != DFGPU_BF16) return fail(kUnsupported, "ROPE: %s must be FLOAT, HALF or BFLOAT16", name);
    if (x.dtype != y.dtype || x.dtype != reference.dtype) return fail(kUnsupported, "ROPE: all tensors that are turned have one type");
    if (x.stride[3] != 1 || y.stride[3] != 1) return fail(kInvalidLayout, "ROPE: the head dimension must have unit stride");
    for (int i = 0; i < 3; ++i)
        if (y.dim[i] > 1 && y.stride[i] == 0) return fail(kInvalidLayout, "ROPE: the output of %s overlaps itself", name);
    return kOk;
}

// Values to a vector by the descriptors alone: 16 bytes, 8, or one value.
int vector_width(const dfgpu_rope_params& p) {
    const int bytes = dtype_bytes(p.x.dtype);
    const int64_t half = p.frequencies.dim[3];
    for (int width = 16 / bytes; width * bytes >= 8; width /= 2) {
        bool fits = p.x.dim[3] % width == 0 && (2 * half) % width == 0 && (p.interleaved || half % width == 0);
        for (const dfgpu_tensor* t : {&p.x, &p.y, &p.x2, &p.y2})
            for (int i = 0; i < 3 && t->rank; ++i) fits = fits && (t->dim[i] == 1 || t->stride[i] % width == 0);
        if (fits) return width;
    }
    return 1;
}

int check_rope(const dfgpu_rope_params& p, int& width) {
    int status = check_side(p.x, p.y, p.x, "X");
    if (!status && (p.x2.rank || p.y2.rank)) status = check_side(p.x2, p.y2, p.x, "X2");
    if (status) return status;
    if (!valid_tensor(p.positions) || p.positions.rank != 4 || (p.positions.dim[0] != 1 && p.positions.dim[0] != p.x.dim[0]) || p.positions.dim[1] != 1 ||
        p.positions.dim[2] != p.x.dim[2] || p.positions.dim[3] != 1)
        return fail(kInvalidShape, "ROPE: positions must be [B or 1, 1, S, 1]");
    if (p.positions.dtype != DFGPU_I32 && p.positions.dtype != DFGPU_I64) return fail(kUnsupported, "ROPE: positions must be INT32 or INT64");
    if (!valid_tensor(p.frequencies) || p.frequencies.rank != 4 || p.frequencies.dim[0] != 1 || p.frequencies.dim[1] != 1 || p.frequencies.dim[2] != 1)
        return fail(kInvalidShape, "ROPE: frequencies must be [1, 1, 1, R/2]");
    if (p.frequencies.dtype != DFGPU_F32) return fail(kUnsupported, "ROPE: frequencies must be FLOAT");
    if (2 * p.frequencies.dim[3] > p.x.dim[3]) return fail(kInvalidShape, "ROPE: two channels for each frequency are more than the head dimension");
    if (p.x.dim[3] > kRopeMaxD) return fail(kUnsupported, "ROPE: head dimension above %lld", static_cast<long long>(kRopeMaxD));
    const int64_t heads = p.x.dim[1] + (p.x2.rank ? p.x2.dim[1] : 0);
    if (heads > 65535 || p.x.dim[2] >= (1ll << 30) || p.x.dim[0] * p.x.dim[2] >= (1ll << 31)) return fail(kUnsupported, "ROPE: too many heads or tokens");
    if (p.kernel < DFGPU_ROPE_AUTO || p.kernel > DFGPU_ROPE_SCALAR) return fail(kInvalidArgument, "ROPE: unknown kernel id %d", p.kernel);
    width = p.kernel == DFGPU_ROPE_SCALAR ? 1 : vector_width(p);
    if (p.kernel == DFGPU_ROPE_VECTOR && width == 1) return fail(kUnsupported, "ROPE: the vector kernel needs extents and strides of whole 8-byte vectors");
    return kOk;
}

template <typename T, int V>
void launch_rope(const RopeArgs& a, bool interleaved, dim3 grid, size_t shared, cudaStream_t stream) {
    launch_chained(interleaved ? rope_kernel<T, V, true> : rope_kernel<T, V, false>, grid, dim3(kRopeThreads), shared, stream, a);
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_rope(const dfgpu_rope_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "ROPE: null params");
    int width;
    const int status = check_rope(*p, width);
    if (status) return status;
    info->kernel = width > 1 ? DFGPU_ROPE_VECTOR : DFGPU_ROPE_SCALAR;
    info->launches = 1;
    info->scratch_bytes = 0;
    return kOk;
}

extern "C" int dfgpu_rope(const dfgpu_rope_params* p, void* const* tensors, void* scratch, void* stream) {
    (void)scratch;
    if (!p || !tensors) return fail(kInvalidArgument, "ROPE: null params");
    int width;
    const int status = check_rope(*p, width);
    if (status) return status;
    const bool two = p->x2.rank != 0;
    for (int i = 0; i < (two ? 6 : 4); ++i)
        if (!tensors[i]) return fail(kInvalidArgument, "ROPE: port %d is null", i);
    if (two && (tensors[1] == tensors[5] || tensors[0] == tensors[5] || tensors[1] == tensors[4])) return fail(kInvalidArgument, "ROPE: the output of one pair is a tensor of the other");
    const int bytes = dtype_bytes(p->x.dtype);
    RopeArgs a{};
    for (int s = 0; s < (two ? 2 : 1); ++s) {
        const dfgpu_tensor &x = s ? p->x2 : p->x, &y = s ? p->y2 : p->y;
        RopeSide& side = a.side[s];
        side.x = tensors[s ? 4 : 0];
        side.y = tensors[s ? 5 : 1];
        if (!aligned(side.x, bytes) || !aligned(side.y, bytes)) return fail(kInvalidArgument, "ROPE: a tensor is not aligned to its type");
        bool same = true;
        for (int i = 0; i < 3; ++i) {
            side.x_stride[i] = x.dim[i] == 1 ? 0 : x.stride[i];
            side.y_stride[i] = y.dim[i] == 1 ? 0 : y.stride[i];
            same = same && side.x_stride[i] == side.y_stride[i];
        }
        if (side.x == side.y && !same) return fail(kInvalidLayout, "ROPE: in place, input and output have the same strides");
        side.in_place = side.x == side.y;
        side.heads = static_cast<int>(x.dim[1]);
        while (width > 1 && !(aligned(side.x, width * bytes) && aligned(side.y, width * bytes))) {
            if (p->kernel == DFGPU_ROPE_VECTOR && width * bytes <= 8) return fail(kInvalidArgument, "ROPE: the vector kernel needs tensors on 8-byte boundaries");
            width = width * bytes > 8 ? width / 2 : 1;
        }
    }
    if (!aligned(tensors[2], p->positions.dtype == DFGPU_I64 ? 8 : 4) || !aligned(tensors[3], 4)) return fail(kInvalidArgument, "ROPE: positions or frequencies are not aligned to their type");
    a.positions = tensors[2];
    a.positions_wide = p->positions.dtype == DFGPU_I64;
    a.position_batch = p->positions.dim[0] == 1 ? 0 : p->positions.stride[0];
    a.position_token = p->positions.stride[2];
    a.frequencies = static_cast<const float*>(tensors[3]);
    a.frequency_stride = p->frequencies.stride[3];
    a.scale = p->scale;
    a.sign = p->inverse ? -1.0f : 1.0f;
    a.seq = static_cast<int>(p->x.dim[2]);
    a.half = static_cast<int>(p->frequencies.dim[3]);
    const int pairs = p->interleaved && width > 1 ? width / 2 : width;   // of a unit
    a.turning = a.half / pairs;
    a.units = a.turning + (static_cast<int>(p->x.dim[3]) - 2 * a.half) / width;
    a.by_units = make_fast_divisor(static_cast<uint32_t>(a.units));
    a.pitch = a.half + a.turning;   // (eight units of a token and the next token's do not meet in the same banks)
    // Up to eight tokens a CTA, so that a long run of heads shares each token's sines; then as few heads as give each thread eight units.
    // (One unit a thread, all else being equal: 108 us for 60 with 2 x 8192 tokens of 40 heads of 128 bf16 channels, 16.1 for 13.2 with 2048, 7.5 for 7.6 with
    // 512: the sines cost more than the CTAs gain.)
    while (a.token_shift < 3 && (1 << a.token_shift) < a.seq && (a.pitch << (a.token_shift + 1)) <= kRopeTable) ++a.token_shift;
    a.tiles = (a.seq + (1 << a.token_shift) - 1) >> a.token_shift;
    a.by_tiles = make_fast_divisor(static_cast<uint32_t>(a.tiles));
    const int64_t tiles = p->x.dim[0] * a.tiles;
    a.heads_per_cta = std::min(std::max(a.side[0].heads, a.side[1].heads), (8 * kRopeThreads - 1) / (a.units << a.token_shift) + 1);
    a.first_side = (a.side[0].heads + a.heads_per_cta - 1) / a.heads_per_cta;
    a.rows_on = kRopeThreads / a.units, a.units_on = kRopeThreads % a.units;
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(a.first_side + (a.side[1].heads + a.heads_per_cta - 1) / a.heads_per_cta));
    const size_t shared = sizeof(float2) * static_cast<size_t>(a.pitch << a.token_shift);
    const bool interleaved = p->interleaved != 0;
    cudaStream_t on = as_stream(stream);
    if (p->x.dtype == DFGPU_F32) {
        if (width == 4) launch_rope<float, 4>(a, interleaved, grid, shared, on);
        else if (width == 2) launch_rope<float, 2>(a, interleaved, grid, shared, on);
        else launch_rope<float, 1>(a, interleaved, grid, shared, on);
    } else if (p->x.dtype == DFGPU_F16) {
        if (width == 8) launch_rope<__half, 8>(a, interleaved, grid, shared, on);
        else if (width == 4) launch_rope<__half, 4>(a, interleaved, grid, shared, on);
        else launch_rope<__half, 1>(a, interleaved, grid, shared, on);
    } else {
        if (width == 8) launch_rope<__nv_bfloat16, 8>(a, interleaved, grid, shared, on);
        else if (width == 4) launch_rope<__nv_bfloat16, 4>(a, interleaved, grid, shared, on);
        else launch_rope<__nv_bfloat16, 1>(a, interleaved, grid, shared, on);
    }
    return check_launch("ROPE");
}

extern "C" int dfgpu_rope_frequencies(const dfgpu_rope_scaling* s, float* frequencies, float* magnitude) {
    if (!s || !frequencies) return fail(kInvalidArgument, "ROPE frequencies: null argument");
    if (s->rotary < 2 || s->rotary % 2 != 0) return fail(kInvalidShape, "ROPE frequencies: the rotary extent must be even and positive");
    if (s->kind < DFGPU_ROPE_SCALING_NONE || s->kind > DFGPU_ROPE_SCALING_BANDS) return fail(kInvalidArgument, "ROPE frequencies: unknown scaling %d", s->kind);
    if (!(s->base > 1.0) || !std::isfinite(s->base)) return fail(kInvalidValue, "ROPE frequencies: the base must be above 1");
    const bool borders = s->kind == DFGPU_ROPE_SCALING_RAMP || s->kind == DFGPU_ROPE_SCALING_BANDS;
    if (s->kind != DFGPU_ROPE_SCALING_NONE && (!(s->factor >= 1.0) || !std::isfinite(s->factor))) return fail(kInvalidValue, "ROPE frequencies: the factor must be at least 1");
    if (borders && (!(s->original > 0.0) || !std::isfinite(s->original) || !(s->low > 0.0) || !(s->high > s->low) || !std::isfinite(s->high)))
        return fail(kInvalidValue, "ROPE frequencies: original must be positive and 0 < low < high");
    if (s->kind == DFGPU_ROPE_SCALING_BASE && s->rotary < 4) return fail(kInvalidShape, "ROPE frequencies: scaling the base needs more than one pair");
    const double pi = 3.14159265358979323846;
    double base = s->base;
    if (s->kind == DFGPU_ROPE_SCALING_BASE) base *= std::pow(s->factor, static_cast<double>(s->rotary) / (s->rotary - 2));
    double from = 0.0, until = 0.0;   // RAMP: pair numbers
    if (s->kind == DFGPU_ROPE_SCALING_RAMP) {
        auto pair_at = [&](double turns) { return s->rotary * std::log(s->original / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
        from = std::fmax(std::floor(pair_at(s->high)), 0.0);
        until = std::fmin(std::ceil(pair_at(s->low)), s->rotary - 1.0);
        if (until <= from) until = from + 0.001;   // (a step)
    }
    for (int i = 0; i < s->rotary / 2; ++i) {
        double f = std::pow(base, -2.0 * i / s->rotary);
        if (s->kind == DFGPU_ROPE_SCALING_LINEAR) f /= s->factor;
        if (borders) {
            const double turns = s->original * f / (2.0 * pi);
            const double kept = s->kind == DFGPU_ROPE_SCALING_RAMP ? 1.0 - (i - from) / (until - from) : (turns - s->low) / (s->high - s->low);
            const double share = std::fmin(std::fmax(kept, 0.0), 1.0);
            f = f / s->factor * (1.0 - share) + f * share;
        }
        frequencies[i] = static_cast<float>(f);
    }
    if (magnitude) *magnitude = s->kind == DFGPU_ROPE_SCALING_RAMP ? static_cast<float>(0.1 * std::log(s->factor) + 1.0) : 1.0f;
    return kOk;
}

// 1: rotary positions, cache append, cache attention, page bookkeeping.
extern "C" int dfgpu_cache_abi_version(void) { return 1; }
