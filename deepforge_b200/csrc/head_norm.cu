// RMS norms of query and key heads with their gains and rotary positions in one pass, and the gradients of all three.
//
// A row is one token's head, D channels. It is taken by a group of lanes that hold it in registers between its sum of squares and its result
// (pairs that turn together lie in one lane), so that it is read once and written once: HBM is what bounds both kernels, and close behind it the chain of instructions of
// a row, which few warps hide (registers hold the angles and the gradients' sums). 2 x 8192 tokens of 32 + 8 heads of 128 bf16 channels 58 us (the bytes alone 51); gradients of
// 4 x 2048 such tokens 51.5 (38.5), of 3 x 1001 f32 tokens with gains of every head 37.3 (22.6), the sums of dgain among them (6, half of it behind the first kernel's end).
// Token by token as slices of one buffer 60 and 52; with 16-bit gains 60; f32 rows 57 (51). With gains of every head, which a row takes from shared memory, 79 (f32 rows 61) and gradients 105; half of
// a head turned as halves apart, where a unit of what stays has half the bytes, 86 and 82. Outside the vectors a warp takes a row value by value or twice: 2 x 2048 tokens of 66 channels 79 (6.6), of 128 off
// the boundaries 83 (12.8), gradients 146 and 271; of 4 + 1 heads of 1024 channels 38 (12.8), gradients 159.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

constexpr int kNormThreads = 128, kNormWarps = kNormThreads / 32;
constexpr int kNormTable = 2048;      // (cosine, sine) pairs of a CTA, forward: 16 KiB
constexpr int kNormGains = 8 * 1024;     // bytes of gains of heads, forward
constexpr int kNormShared = 18 * 1024;   // bytes of a CTA's table, gradient: with the rows on their way within 48 KiB
constexpr int64_t kNormMaxD = 1024;

struct NormSide {
    const void* x;
    const void* dy;                   // (gradient)
    void* out;                        // Y or dX
    const void* gain;                 // null: ones
    float* partial;                   // (gradient: sums of dgain, null where it is not wanted)
    int64_t x_stride[3], dy_stride[3], out_stride[3];   // batch, head, token
    int64_t gain_head;
    int32_t gain_type, heads, per_head;   // per_head: sums of dgain go out for each head
    int32_t runs, first_run;          // (gradient) of heads: those that hold some of these
};
struct NormArgs {
    NormSide side[2];
    Positions at;
    int32_t seq, tokens, tiles, token_shift;   // tokens: of all sequences; a CTA's: 1 << token_shift
    int32_t heads_per_cta;                     // of both pairs of tensors in a row
    int32_t gain_floats;                       // (forward) room for gains in shared memory
    int32_t d, half, turning, units;           // units of V pairs (half) or V channels (interleaved, or not turned) a row
    int32_t group_shift;                       // lanes of a row: 1 << group_shift
    FastDivisor by_tiles, by_seq, by_d;
    float scale, epsilon, gain_offset, inverse_d;
};

__device__ __forceinline__ float gain_at(const NormSide& s, float offset, int64_t at) {
    if (!s.gain) return 1.0f;
    if (s.gain_type == DFGPU_F32) return static_cast<const float*>(s.gain)[at] + offset;
    if (s.gain_type == DFGPU_F16) return __half2float(static_cast<const __half*>(s.gain)[at]) + offset;
    return bf16_bits_to_f32(static_cast<const uint16_t*>(s.gain)[at]) + offset;
}

__device__ __forceinline__ uint32_t narrow_two(__nv_bfloat16*, float lo, float hi) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&pair);
}
__device__ __forceinline__ uint32_t narrow_two(__half*, float lo, float hi) {
    const __half2 pair = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&pair);
}
__device__ __forceinline__ uint64_t minus2(uint64_t v) { return v ^ 0x8000000080000000ull; }
__device__ __forceinline__ float sum2(uint64_t v) {
    float lo, hi;
    unpack2(v, lo, hi);
    return lo + hi;
}

// One unit of a row: V pairs as two vectors (i and i + half), or with INTERLEAVED V channels as one (V = 1: one pair as two values); of channels that do not
// turn, V as one. In registers the pairs' first values are `one`, the second `two`, two neighbouring pairs to a register pair, which one instruction takes.
template <typename T, int V, bool INTERLEAVED>
struct NormUnit {
    static constexpr bool kTwo = !INTERLEAVED || V == 1;
    static constexpr int kPairs = kTwo ? V : V / 2, kPacks = (kPairs + 1) / 2, kQuad = kPairs < 4 ? kPairs : 4;
    static constexpr int kPerLane = V == 1 ? 0 : (16 / static_cast<int>(sizeof(T))) / kPairs;   // units that hold 32 bytes
    static __device__ __forceinline__ int channel(const NormArgs& a, int unit) {
        return unit < a.turning ? (INTERLEAVED ? unit * (V == 1 ? 2 : V) : unit * V) : 2 * a.half + (unit - a.turning) * V;
    }
    static __device__ __forceinline__ int apart(const NormArgs& a) { return INTERLEAVED ? 1 : a.half; }
    // of value `half` (0, 1) of pack k: its place in a vector
    static constexpr __device__ int place(int k, int half, bool second) { return kTwo ? 2 * k + half : 4 * k + 2 * half + (second ? 1 : 0); }
};
template <int PACKS>
struct Values {
    uint64_t one[PACKS], two[PACKS];
};
template <typename T, int V, bool INTERLEAVED>
struct RawUnit {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using In = Values<Form::kPacks>;
    Pack<T, V> first, second;
    __device__ __forceinline__ void load(const T* from, int apart, bool turns) {
        first = *reinterpret_cast<const Pack<T, V>*>(from);
#pragma unroll
        for (int i = 0; i < V; ++i) second.v[i] = narrow<T>(0.0f);
        if (Form::kTwo && turns) second = *reinterpret_cast<const Pack<T, V>*>(from + apart);
    }
    __device__ __forceinline__ In values() const {
        In v;
#pragma unroll
        for (int k = 0; k < Form::kPacks; ++k) {
            if constexpr (V == 1) {
                v.one[k] = pack2(widen(first.v[0]), 0.0f);
                v.two[k] = pack2(widen(second.v[0]), 0.0f);
            } else if constexpr (Form::kTwo) {
                v.one[k] = pack2(widen(first.v[2 * k]), widen(first.v[2 * k + 1]));
                v.two[k] = pack2(widen(second.v[2 * k]), widen(second.v[2 * k + 1]));
            } else {
                v.one[k] = pack2(widen(first.v[4 * k]), widen(first.v[4 * k + 2]));
                v.two[k] = pack2(widen(first.v[4 * k + 1]), widen(first.v[4 * k + 3]));
            }
        }
        return v;
    }
    static __device__ __forceinline__ void store(T* to, int apart, bool turns, const In& v) {
        Pack<T, V> out[2];
#pragma unroll
        for (int k = 0; k < Form::kPacks; ++k) {
            float a0, a1, b0, b1;
            unpack2(v.one[k], a0, a1);
            unpack2(v.two[k], b0, b1);
            if constexpr (V == 1) {
                out[0].v[0] = narrow<T>(a0);
                out[1].v[0] = narrow<T>(b0);
            } else if constexpr (sizeof(T) == 2) {
                uint32_t* words[2] = {reinterpret_cast<uint32_t*>(&out[0]), reinterpret_cast<uint32_t*>(&out[1])};
                if constexpr (Form::kTwo) {
                    words[0][k] = narrow_two(static_cast<T*>(nullptr), a0, a1);
                    words[1][k] = narrow_two(static_cast<T*>(nullptr), b0, b1);
                } else {
                    words[0][2 * k] = narrow_two(static_cast<T*>(nullptr), a0, b0);
                    words[0][2 * k + 1] = narrow_two(static_cast<T*>(nullptr), a1, b1);
                }
            } else if constexpr (Form::kTwo) {
                out[0].v[2 * k] = a0, out[0].v[2 * k + 1] = a1;
                out[1].v[2 * k] = b0, out[1].v[2 * k + 1] = b1;
            } else {
                out[0].v[4 * k] = a0, out[0].v[4 * k + 1] = b0;
                out[0].v[4 * k + 2] = a1, out[0].v[4 * k + 3] = b1;
            }
        }
        *reinterpret_cast<Pack<T, V>*>(to) = out[0];
        if constexpr (Form::kTwo) {
            if (turns) *reinterpret_cast<Pack<T, V>*>(to + apart) = out[1];
        }
    }
};
template <typename Form, int V>
__device__ __forceinline__ void load_gains(const NormArgs& a, const NormSide& s, int head, int channel, bool live, bool turns, Values<Form::kPacks>& gain) {
    const int apart = Form::kTwo ? Form::apart(a) : 0;
    const int64_t base = head * s.gain_head + channel;
#pragma unroll
    for (int k = 0; k < Form::kPacks; ++k) {
        float g[2][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const bool there = live && (V > 1 || half == 0);
            g[0][half] = there ? gain_at(s, a.gain_offset, base + Form::place(k, half, false)) : 0.0f;
            g[1][half] = there && (!Form::kTwo || turns) ? gain_at(s, a.gain_offset, base + apart + Form::place(k, half, true)) : 0.0f;
        }
        gain.one[k] = pack2(g[0][0], g[0][1]);
        gain.two[k] = pack2(g[1][0], g[1][1]);
    }
}
// Gains as f32 in shared memory (by all threads; the barrier behind the angles' is its too): of all heads together, or of `heads` from head0 on. And a lane's part of
// them: `shared` is the head's there, or null.
__device__ __forceinline__ void fill_gains(const NormArgs& a, const NormSide& s, float* to, int head0, int heads) {
    const int count = (s.gain_head ? heads : 1) * a.d;
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kNormThreads) {
        const int head = static_cast<int>(fast_divide(static_cast<uint32_t>(i), a.by_d));
        to[i] = gain_at(s, a.gain_offset, (head0 + head) * s.gain_head + (i - head * a.d));
    }
}
template <typename Form, int V>
__device__ __forceinline__ void take_gains(const NormArgs& a, const NormSide& s, const float* shared, int head, int channel, bool live, bool turns, Values<Form::kPacks>& gain) {
    if (!shared) return load_gains<Form, V>(a, s, head, channel, live, turns, gain);
    gain = Values<Form::kPacks>{};
    if (!live) return;
    const float* first = shared + channel;
#pragma unroll
    for (int k = 0; k < Form::kPacks; ++k) {
        if constexpr (Form::kTwo) {
            gain.one[k] = reinterpret_cast<const uint64_t*>(first)[k];
            if (turns) gain.two[k] = reinterpret_cast<const uint64_t*>(first + Form::apart(a))[k];
        } else {
            const float4 four = reinterpret_cast<const float4*>(first)[k];
            gain.one[k] = pack2(four.x, four.z);
            gain.two[k] = pack2(four.y, four.w);
        }
    }
}
// The table of a token: cosines of all pairs, then sines, those of a unit's pairs in vectors of kQuad, vectors of neighbouring units side by side.
template <typename Form>
__device__ __forceinline__ int angle_place(const NormArgs& a, int unit, int quad) { return (quad * a.turning + unit) * Form::kQuad; }
// A thread's part of the tables of 1 << token_shift tokens: one token's, whose position it holds, pair by pair. The angle is reduced to one turn in 64 bits. f32 rows take sine
// and cosine of the f32 nearest to it and what that leaves out; 16-bit ones those of the special function unit, which are off by 2^-21.4, and 1.9e-7 of the angle.
template <typename T, typename Form>
__device__ __forceinline__ void fill_angles(const NormArgs& a, float* angles, int local, bool live, int64_t batch, int64_t token) {
    if (!live || a.half == 0) return;
    const int64_t at = batch * a.at.batch + token * a.at.token;
    const double position = a.at.wide ? static_cast<double>(static_cast<const int64_t*>(a.at.positions)[at]) : static_cast<double>(static_cast<const int32_t*>(a.at.positions)[at]);
    float* table = angles + local * 2 * a.half;
    for (int pair = threadIdx.x >> a.token_shift; pair < a.half; pair += kNormThreads >> a.token_shift) {
        const double turns = position * static_cast<double>(a.at.frequencies[pair * a.at.frequency_stride]) * 0.15915494309189533577;
        const double rest = turns - rint(turns);
        float sine, cosine;
        if constexpr (sizeof(T) == 4) {
            const float halves = static_cast<float>(2.0 * rest), more = 3.14159265f * static_cast<float>(2.0 * rest - static_cast<double>(halves));
            sincospif(halves, &sine, &cosine);
            const float first = cosine;
            cosine = __fmaf_rn(-sine, more, cosine);
            sine = __fmaf_rn(first, more, sine);
        } else {
            __sincosf(static_cast<float>(6.283185307179586 * rest), &sine, &cosine);
        }
        const int unit = pair / Form::kPairs, within = pair - unit * Form::kPairs, place = angle_place<Form>(a, unit, within / Form::kQuad) + within % Form::kQuad;
        table[place] = cosine * a.scale;
        table[a.half + place] = sine * a.scale;
    }
}
template <typename Form>
__device__ __forceinline__ void get_angles(const float* table, int place, int step, uint64_t (&out)[Form::kPacks]) {
    if constexpr (Form::kQuad == 4) {
#pragma unroll
        for (int q = 0; q < Form::kPacks / 2; ++q) {
            const float4 four = *reinterpret_cast<const float4*>(table + place + q * step);
            out[2 * q] = pack2(four.x, four.y);
            out[2 * q + 1] = pack2(four.z, four.w);
        }
    } else if constexpr (Form::kQuad == 2) {
        const float2 two = *reinterpret_cast<const float2*>(table + place);
        out[0] = pack2(two.x, two.y);
    } else {
        out[0] = pack2(table[place], 0.0f);
    }
}
// The pairs of a unit by a token's angles; BACK: the other way.
template <typename Form, bool BACK>
__device__ __forceinline__ void turn_unit(const NormArgs& a, const float* table, int unit, Values<Form::kPacks>& v) {
    uint64_t cosine[Form::kPacks], sine[Form::kPacks];
    const int place = angle_place<Form>(a, unit, 0), step = a.turning * Form::kQuad;
    get_angles<Form>(table, place, step, cosine);
    get_angles<Form>(table + a.half, place, step, sine);
#pragma unroll
    for (int k = 0; k < Form::kPacks; ++k) {
        const uint64_t one = v.one[k], two = v.two[k], back = minus2(sine[k]);
        v.one[k] = fma2(one, cosine[k], mul2(two, BACK ? sine[k] : back));
        v.two[k] = fma2(two, cosine[k], mul2(one, BACK ? back : sine[k]));
    }
}
__device__ __forceinline__ float sum_over(float v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__device__ __forceinline__ float inverse_root(float v) { return sizeof(T) == 4 ? __frsqrt_rn(v) : rsqrtf(v); }   // (the other is off by 2^-23 and a little, which 16 bits do not show)

// What a lane has of every row: up to 32 bytes.
template <typename Form, int U>
struct Share {
    int channel[U], unit[U];
    bool there[U], turns[U];
    __device__ __forceinline__ Share(const NormArgs& a, int lane) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            unit[j] = lane + (j << a.group_shift);
            there[j] = unit[j] < a.units;
            turns[j] = unit[j] < a.turning;
            channel[j] = Form::channel(a, unit[j]);
        }
    }
};

// Rows on their way: a thread copies its own vectors into shared memory (16 or 8 bytes each, asynchronously) and reads none but those, so nothing waits for
// another thread, and what is in flight takes no registers. What is not wanted becomes zeros.
template <typename T, int V, bool INTERLEAVED, int STAGES, int TENSORS>
struct Ring {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Vector = Pack<T, V>;
    static constexpr int U = Form::kPerLane, kSlots = (Form::kTwo ? 2 : 1) * U, kBytes = static_cast<int>(sizeof(Vector)) * kSlots * TENSORS * STAGES * kNormThreads;
    Vector* own;   // [stage][tensor][slot][thread]
    int filling = 0, reading = 0;
    __device__ __forceinline__ explicit Ring(void* shared) : own(static_cast<Vector*>(shared) + threadIdx.x) {}
    __device__ __forceinline__ Vector* slot(int stage, int tensor, int i) const { return own + ((stage * TENSORS + tensor) * kSlots + i) * kNormThreads; }
    static __device__ __forceinline__ void copy(Vector* to, const T* from, bool wanted) {
        const uint32_t bytes = wanted ? static_cast<uint32_t>(sizeof(Vector)) : 0u;
        if constexpr (sizeof(Vector) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(__cvta_generic_to_global(from)), "r"(bytes) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(to)), "l"(__cvta_generic_to_global(from)), "r"(bytes) : "memory");
    }
    // One row of each tensor: `from` is an address that may be read, wanted or not.
    __device__ __forceinline__ void fill(const Share<Form, U>& share, int apart, const T* const (&from)[TENSORS], bool wanted) {
#pragma unroll
        for (int t = 0; t < TENSORS; ++t)
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const bool first = wanted && share.there[j], second = first && share.turns[j];
                copy(slot(filling, t, j), first ? from[t] + share.channel[j] : from[t], first);
                if constexpr (Form::kTwo) copy(slot(filling, t, U + j), second ? from[t] + share.channel[j] + apart : from[t], second);
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
        filling = filling + 1 == STAGES ? 0 : filling + 1;
    }
    // The oldest row that was not taken yet, of which STAGES - 1 are on their way.
    __device__ __forceinline__ void take(RawUnit<T, V, INTERLEAVED> (&rows)[TENSORS][U]) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
#pragma unroll
        for (int t = 0; t < TENSORS; ++t)
#pragma unroll
            for (int j = 0; j < U; ++j) {
                rows[t][j].first = *slot(reading, t, j);
                if constexpr (Form::kTwo) rows[t][j].second = *slot(reading, t, U + j);
            }
        reading = reading + 1 == STAGES ? 0 : reading + 1;
    }
    // A unit of the first tensor's row that was taken last: nothing goes into its place before the next row but one is asked for.
    __device__ __forceinline__ RawUnit<T, V, INTERLEAVED> taken(int j) const {
        RawUnit<T, V, INTERLEAVED> row;
        const int stage = reading == 0 ? STAGES - 1 : reading - 1;
        row.first = *slot(stage, 0, j);
        if constexpr (Form::kTwo) row.second = *slot(stage, 0, U + j);
        return row;
    }
    // What is still on its way is waited for and not taken.
    __device__ __forceinline__ void drain() {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        reading = filling;
    }
};
constexpr int kForwardStages = 4, kGradientStages = 3;   // (gradients of 4 x 2048 bf16 tokens 51.8 us; two stages 61.2, four 52.2; of 3 x 1001 f32 tokens 38.0, 38.1 and 43.0)

// ---- forward: a CTA takes a few tokens of one sequence and a run of heads of both pairs of tensors, which share the tokens' angles -----------------------
// A group of lanes has one token and walks the heads, so that the angles stay in registers, multiplied by the gains already.
// OF_HEADS: some gains are those of each head.
template <typename T, int V, bool INTERLEAVED, bool OF_HEADS>
__global__ void __launch_bounds__(kNormThreads, 6)
head_norm_kernel(const __grid_constant__ NormArgs a) {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Raw = RawUnit<T, V, INTERLEAVED>;
    constexpr int U = Form::kPerLane;
    extern __shared__ __align__(16) float angles[];
    const int tile = static_cast<int>(blockIdx.x);
    const int batch_index = static_cast<int>(fast_divide(static_cast<uint32_t>(tile), a.by_tiles));
    const int token0 = (tile - batch_index * a.tiles) << a.token_shift, tokens = a.seq - token0, mask = (1 << a.token_shift) - 1;
    const int lanes = 1 << a.group_shift, group = threadIdx.x >> a.group_shift, groups = kNormThreads >> a.group_shift;
    const int local = group & mask, first_head = group >> a.token_shift, step = groups >> a.token_shift;   // (no more tokens than groups)
    const Share<Form, U> share(a, threadIdx.x & (lanes - 1));
    const int apart = Form::apart(a), run0 = static_cast<int>(blockIdx.y) * a.heads_per_cta, run1 = run0 + a.heads_per_cta;
    const bool live = local < tokens;
    int which = run0 < a.side[0].heads ? 0 : 1, head = 0, heads = 0;   // of the pair of tensors that is at hand: heads of the run
    const T* x = nullptr;
    T* y = nullptr;
    auto begin = [&] {
        const NormSide& s = a.side[which];
        const int before = which ? a.side[0].heads : 0, head0 = max(run0 - before, 0);
        head = head0 + first_head;
        heads = min(run1 - before, s.heads);
        x = static_cast<const T*>(s.x) + batch_index * s.x_stride[0] + head * s.x_stride[1] + (token0 + local) * s.x_stride[2];
        y = static_cast<T*>(s.out) + batch_index * s.out_stride[0] + head * s.out_stride[1] + (token0 + local) * s.out_stride[2];
    };
    // gains of both pairs of tensors, of each the CTA's heads' or one
    float* const first_gains = angles + ((2 * a.half) << a.token_shift);
    const int first_heads = max(min(run1, a.side[0].heads) - run0, 0), second_head0 = max(run0 - a.side[0].heads, 0), second_heads = max(min(run1 - a.side[0].heads, a.side[1].heads) - second_head0, 0);
    float* const second_gains = first_gains + (a.side[0].gain_head ? first_heads : 1) * a.d;
    Ring<T, V, INTERLEAVED, kForwardStages, 1> ring(first_gains + a.gain_floats);
    int64_t x_step = 0;
    auto start = [&] {   // the first rows of the pair of tensors at hand
        x_step = step * a.side[which].x_stride[1];
#pragma unroll
        for (int i = 0; i + 1 < kForwardStages; ++i) {
            const bool wanted = live && head + i * step < heads;
            const T* const from[1] = {wanted ? x + i * x_step : static_cast<const T*>(a.side[which].x)};
            ring.fill(share, apart, from, wanted);
        }
    };
    begin();
    chain_begin();
    start();   // (on their way while the angles are worked out)
    fill_gains(a, a.side[0], first_gains, run0, first_heads);
    if (second_heads) fill_gains(a, a.side[1], second_gains, second_head0, second_heads);
    const int filled = threadIdx.x & mask;
    fill_angles<T, Form>(a, angles, filled, filled < tokens, batch_index, token0 + filled);
    __syncthreads();
    for (;;) {
        const NormSide& s = a.side[which];
        const int64_t y_step = step * s.out_stride[1];
        Values<Form::kPacks> along[U], across[U];   // what a pair's own value and the other one are multiplied by
#pragma unroll
        for (int j = 0; j < U; ++j) {               // (by the gains already, where all heads have the same)
            Values<Form::kPacks> gain;
#pragma unroll
            for (int k = 0; k < Form::kPacks; ++k) gain.one[k] = gain.two[k] = pack2(1.0f, 1.0f);
            if (!OF_HEADS || !s.gain_head) take_gains<Form, V>(a, s, which ? second_gains : first_gains, 0, share.channel[j], share.there[j], share.turns[j], gain);
            along[j] = gain;
            across[j] = Values<Form::kPacks>{};
            if (!share.turns[j]) continue;
            uint64_t cosine[Form::kPacks], sine[Form::kPacks];
            const float* table = angles + local * 2 * a.half;
            const int place = angle_place<Form>(a, share.unit[j], 0), stride = a.turning * Form::kQuad;
            get_angles<Form>(table, place, stride, cosine);
            get_angles<Form>(table + a.half, place, stride, sine);
#pragma unroll
            for (int k = 0; k < Form::kPacks; ++k) {
                along[j].one[k] = mul2(gain.one[k], cosine[k]);
                along[j].two[k] = mul2(gain.two[k], cosine[k]);
                across[j].one[k] = minus2(mul2(gain.two[k], sine[k]));
                across[j].two[k] = mul2(gain.one[k], sine[k]);
            }
        }
        // (whole warps stay together: a warp's groups have heads side by side)
        while (__any_sync(0xffffffffu, head < heads)) {
            const bool own = live && head < heads, later = live && head + (kForwardStages - 1) * step < heads;
            Raw now[1][U];
            ring.take(now);
            const T* const from[1] = {later ? x + (kForwardStages - 1) * x_step : static_cast<const T*>(s.x)};
            ring.fill(share, apart, from, later);
            Values<Form::kPacks> v[U];
            uint64_t squares = 0;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                v[j] = now[0][j].values();
#pragma unroll
                for (int k = 0; k < Form::kPacks; ++k) squares = fma2(v[j].two[k], v[j].two[k], fma2(v[j].one[k], v[j].one[k], squares));
            }
            const float r = inverse_root<T>(__fmaf_rn(sum_over(sum2(squares), lanes), a.inverse_d, a.epsilon));
            const uint64_t both = pack2(r, r);
            // (r first: a gain may take a row past f32's range whose r is 0)
            const float* of_head = OF_HEADS && s.gain_head ? (which ? second_gains - second_head0 * a.d : first_gains - run0 * a.d) + min(head, heads - 1) * a.d : nullptr;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                Values<Form::kPacks> gain;
                if (of_head) take_gains<Form, V>(a, s, of_head, 0, share.channel[j], share.there[j], share.turns[j], gain);
#pragma unroll
                for (int k = 0; k < Form::kPacks; ++k) {
                    uint64_t one = mul2(v[j].one[k], both), two = mul2(v[j].two[k], both);
                    if (of_head) {
                        one = mul2(one, gain.one[k]);
                        two = mul2(two, gain.two[k]);
                    }
                    v[j].one[k] = fma2(one, along[j].one[k], mul2(two, across[j].one[k]));
                    v[j].two[k] = fma2(two, along[j].two[k], mul2(one, across[j].two[k]));
                }
                if (own && share.there[j]) Raw::store(y + share.channel[j], apart, share.turns[j], v[j]);
            }
            // Side by side, channels that do not turn have a neighbour that is no partner, and 0 of it is NaN where it is an infinity. Such a row has an r of 0, and these channels are stored once
            // more without it (asked for every value, rows of gains of each head took 4 to 6 % longer, those of 4-value vectors 11).
            if (!Form::kTwo && r == 0.0f && own) {
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    if (share.turns[j] || !share.there[j]) continue;
                    v[j] = ring.taken(j).values();
                    Values<Form::kPacks> gain;
                    if (of_head) take_gains<Form, V>(a, s, of_head, 0, share.channel[j], true, false, gain);
#pragma unroll
                    for (int k = 0; k < Form::kPacks; ++k) {
                        v[j].one[k] = mul2(mul2(v[j].one[k], both), of_head ? gain.one[k] : along[j].one[k]);
                        v[j].two[k] = mul2(mul2(v[j].two[k], both), of_head ? gain.two[k] : along[j].two[k]);
                    }
                    Raw::store(y + share.channel[j], apart, false, v[j]);
                }
            }
            head += step;
            x += x_step;
            y += y_step;
        }
        ring.drain();
        if (which == 1 || run1 <= a.side[0].heads || a.side[1].heads == 0) return;
        which = 1;
        begin();
        start();
    }
}

// Single values, and rows longer than a warp's registers: a row is a whole warp's and read a second time (from the cache).
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kNormThreads)
head_norm_long_kernel(const __grid_constant__ NormArgs a) {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Raw = RawUnit<T, V, INTERLEAVED>;
    extern __shared__ __align__(16) float angles[];
    const int tile = static_cast<int>(blockIdx.x);
    const int batch_index = static_cast<int>(fast_divide(static_cast<uint32_t>(tile), a.by_tiles));
    const int token0 = (tile - batch_index * a.tiles) << a.token_shift, tokens = a.seq - token0, mask = (1 << a.token_shift) - 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int apart = Form::apart(a), run0 = static_cast<int>(blockIdx.y) * a.heads_per_cta, run1 = run0 + a.heads_per_cta;
    chain_begin();
    const int filled = threadIdx.x & mask;
    fill_angles<T, Form>(a, angles, filled, filled < tokens, batch_index, token0 + filled);
    __syncthreads();
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const NormSide& s = a.side[which];
        const int before = which ? a.side[0].heads : 0, head0 = max(run0 - before, 0), heads = min(run1 - before, s.heads) - head0;
        if (heads <= 0) continue;
        const T* x = static_cast<const T*>(s.x) + batch_index * s.x_stride[0] + head0 * s.x_stride[1] + token0 * s.x_stride[2];
        T* y = static_cast<T*>(s.out) + batch_index * s.out_stride[0] + head0 * s.out_stride[1] + token0 * s.out_stride[2];
        for (int row = warp; row < heads << a.token_shift; row += kNormWarps) {
            const int local = row & mask, head = row >> a.token_shift;
            if (local >= tokens) continue;   // (a whole warp's row)
            const T* from = x + head * s.x_stride[1] + local * s.x_stride[2];
            T* to = y + head * s.out_stride[1] + local * s.out_stride[2];
            uint64_t squares = 0;
            for (int unit = lane; unit < a.units; unit += 32) {
                Raw raw;
                raw.load(from + Form::channel(a, unit), apart, unit < a.turning);
                const Values<Form::kPacks> v = raw.values();
#pragma unroll
                for (int k = 0; k < Form::kPacks; ++k) squares = fma2(v.two[k], v.two[k], fma2(v.one[k], v.one[k], squares));
            }
            const float r = inverse_root<T>(__fmaf_rn(sum_over(sum2(squares), 32), a.inverse_d, a.epsilon));
            const uint64_t both = pack2(r, r);
            for (int unit = lane; unit < a.units; unit += 32) {
                const bool turns = unit < a.turning;
                const int channel = Form::channel(a, unit);
                Raw raw;
                raw.load(from + channel, apart, turns);
                Values<Form::kPacks> v = raw.values(), gain;
                load_gains<Form, V>(a, s, s.gain_head ? head0 + head : 0, channel, true, turns, gain);
#pragma unroll
                for (int k = 0; k < Form::kPacks; ++k) {
                    v.one[k] = mul2(mul2(v.one[k], both), gain.one[k]);
                    v.two[k] = mul2(mul2(v.two[k], both), gain.two[k]);
                }
                if (turns) turn_unit<Form, false>(a, angles + local * 2 * a.half, unit, v);
                Raw::store(to + channel, apart, turns, v);
            }
        }
    }
}

// ---- gradients: a CTA takes tokens of all sequences in a row and a run of heads ------------------------------------------------------------------------
// u turned back, squares and v x of a unit, added to the sums that the row needs.
template <typename Form>
__device__ __forceinline__ void add_unit(const Values<Form::kPacks>& x, const Values<Form::kPacks>& u, const Values<Form::kPacks>& gain, uint64_t& squares, uint64_t& product) {
#pragma unroll
    for (int k = 0; k < Form::kPacks; ++k) {
        squares = fma2(x.two[k], x.two[k], fma2(x.one[k], x.one[k], squares));
        product = fma2(mul2(u.two[k], gain.two[k]), x.two[k], fma2(mul2(u.one[k], gain.one[k]), x.one[k], product));
    }
}
// dX of a unit in u's place, and the terms of dgain onto `sums`.
template <typename Form>
__device__ __forceinline__ void finish_unit(const Values<Form::kPacks>& x, Values<Form::kPacks>& u, const Values<Form::kPacks>& gain, float r, float along, Values<Form::kPacks>& sums) {
    const uint64_t both = pack2(r, r), back = pack2(-along, -along);
#pragma unroll
    for (int k = 0; k < Form::kPacks; ++k) {
        sums.one[k] = fma2(u.one[k], mul2(x.one[k], both), sums.one[k]);
        sums.two[k] = fma2(u.two[k], mul2(x.two[k], both), sums.two[k]);
        u.one[k] = mul2(both, fma2(x.one[k], back, mul2(u.one[k], gain.one[k])));
        u.two[k] = mul2(both, fma2(x.two[k], back, mul2(u.two[k], gain.two[k])));
    }
}
// A token's places in X, dY and dX.
struct TokenPlaces {
    int64_t x, dy, out;
    __device__ __forceinline__ TokenPlaces(const NormArgs& a, const NormSide& s, int token) {
        const int b = static_cast<int>(fast_divide(static_cast<uint32_t>(token), a.by_seq)), t = token - b * a.seq;
        x = b * s.x_stride[0] + t * s.x_stride[2];
        dy = b * s.dy_stride[0] + t * s.dy_stride[2];
        out = b * s.out_stride[0] + t * s.out_stride[2];
    }
};
// (gradient: tokens of all sequences in a row)
template <typename T, typename Form>
__device__ __forceinline__ void fill_angles_of(const NormArgs& a, float* angles, int token0, int tokens) {
    const int local = threadIdx.x & ((1 << a.token_shift) - 1), token = token0 + min(local, tokens - 1), b = static_cast<int>(fast_divide(static_cast<uint32_t>(token), a.by_seq));
    fill_angles<T, Form>(a, angles, local, local < tokens, b, token - b * a.seq);
}
// The values of a lane's share, met over the groups of its warp, to channels at `to`.
template <typename Form, int U, int V>
__device__ __forceinline__ void put_sums(const NormArgs& a, const Share<Form, U>& share, const Values<Form::kPacks> (&sums)[U], float* to) {
    const int lanes = 1 << a.group_shift;
    const bool first_group = (threadIdx.x & 31) < lanes;
    const int apart = Form::kTwo ? Form::apart(a) : 0;
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
        for (int k = 0; k < Form::kPacks; ++k) {
            float v[2][2];
            unpack2(sums[j].one[k], v[0][0], v[0][1]);
            unpack2(sums[j].two[k], v[1][0], v[1][1]);
#pragma unroll
            for (int second = 0; second < 2; ++second)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float sum = v[second][half];
                    for (int o = lanes; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (first_group && share.there[j] && (!second || !Form::kTwo || share.turns[j])) to[share.channel[j] + (second ? apart : 0) + Form::place(k, half, second != 0)] = sum;
                }
        }
}

// PER_HEAD: each warp has heads of its own, with their gains, and walks the tokens, whose angles are in the table; the sums of dgain go out with each head.
// Otherwise a group of lanes has one token, its angles in registers, and walks the heads; all have one sum.
// (CTAs on an SM, against registers: bf16 four 51.8 us, three 60.2, five 70.3 with spills; f32 six 38.0, five 40.5, four 40.6, seven 39.1)
template <typename T, int V, bool INTERLEAVED, bool PER_HEAD>
__global__ void __launch_bounds__(kNormThreads, sizeof(T) == 4 ? 6 : 4)
head_norm_grad_kernel(const __grid_constant__ NormArgs a) {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Raw = RawUnit<T, V, INTERLEAVED>;
    constexpr int U = Form::kPerLane;
    extern __shared__ __align__(16) float angles[];
    __shared__ int64_t places[3][32];                                 // (PER_HEAD) of the tokens in X, dY, dX
    const int tile = static_cast<int>(blockIdx.x), token0 = tile << a.token_shift, tokens = min(a.tokens - token0, 1 << a.token_shift);
    const int run0 = static_cast<int>(blockIdx.y) * a.heads_per_cta, run1 = run0 + a.heads_per_cta;
    const int warp = threadIdx.x >> 5, lanes = 1 << a.group_shift, apart = Form::apart(a);
    const Share<Form, U> share(a, threadIdx.x & (lanes - 1));
    const int group = PER_HEAD ? (threadIdx.x & 31) >> a.group_shift : threadIdx.x >> a.group_shift, groups = (PER_HEAD ? 32 : kNormThreads) >> a.group_shift;
    const int local = PER_HEAD ? 0 : group & ((1 << a.token_shift) - 1);   // (no more tokens than groups)
    const bool own_token = local < tokens;
    float* gains = angles + ((2 * a.half) << a.token_shift);   // of both pairs of tensors
    float* meeting = gains + 2 * a.d;                          // where the rows are on their way, and the warps' sums afterwards
    Ring<T, V, INTERLEAVED, kGradientStages, 2> ring(meeting);
    Raw rows[2][U];   // of X and dY, at hand
    Values<Form::kPacks> gain[U], sums[U], cosine[U], sine[U];   // (the angles, not PER_HEAD: `one` alone)
    bool first = true;
    chain_begin();
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const NormSide& s = a.side[which];
        const int before = which ? a.side[0].heads : 0, head0 = max(run0 - before, 0), heads = min(run1 - before, s.heads) - head0;
        if (heads <= 0) continue;
        const bool sums_wanted = s.partial != nullptr;
        const T* x = static_cast<const T*>(s.x) + head0 * s.x_stride[1];
        const T* dy = static_cast<const T*>(s.dy) + head0 * s.dy_stride[1];
        T* dx = static_cast<T*>(s.out) + head0 * s.out_stride[1];
#pragma unroll
        for (int j = 0; j < U; ++j) sums[j] = Values<Form::kPacks>{};
        auto fill = [&](const T* from_x, const T* from_dy, bool wanted) {
            const T* const from[2] = {wanted ? from_x : static_cast<const T*>(s.x), wanted ? from_dy : static_cast<const T*>(s.dy)};
            ring.fill(share, apart, from, wanted);
        };
        auto gains_of = [&](int head) {
#pragma unroll
            for (int j = 0; j < U; ++j) take_gains<Form, V>(a, s, s.gain_head ? nullptr : gains + which * a.d, head, share.channel[j], share.there[j], share.turns[j], gain[j]);
        };
        auto angles_and_gains = [&] {   // (once)
            if (!first) return;
            first = false;
            for (int i = 0; i < 2; ++i)
                if (a.side[i].heads && !a.side[i].gain_head) fill_gains(a, a.side[i], gains + i * a.d, 0, 1);
            fill_angles_of<T, Form>(a, angles, token0, tokens);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < U; ++j) {
#pragma unroll
                for (int k = 0; k < Form::kPacks; ++k) {
                    cosine[j].one[k] = pack2(1.0f, 1.0f);
                    sine[j].one[k] = 0;
                }
                if (PER_HEAD || !share.turns[j] || !own_token) continue;   // (behind the last token there are no angles: zeros stay zeros in the sums)
                const float* table = angles + local * 2 * a.half;
                const int place = angle_place<Form>(a, share.unit[j], 0), stride = a.turning * Form::kQuad;
                get_angles<Form>(table, place, stride, cosine[j].one);
                get_angles<Form>(table + a.half, place, stride, sine[j].one);
            }
        };
        // The row at hand: u turned back, both sums, dX to `to`, and the terms of dgain.
        auto row = [&](T* to, const float* table, bool live) {
            Values<Form::kPacks> v[U], u[U];
            uint64_t squares2 = 0, product2 = 0;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                v[j] = rows[0][j].values();
                u[j] = rows[1][j].values();
                if constexpr (PER_HEAD) {
                    if (share.turns[j]) turn_unit<Form, true>(a, table, share.unit[j], u[j]);
                } else if (share.turns[j]) {   // (elsewhere an infinity times a sine of 0 would be the neighbour's NaN, or that of the sum)
#pragma unroll
                    for (int k = 0; k < Form::kPacks; ++k) {
                        const uint64_t one = u[j].one[k], two = u[j].two[k];
                        u[j].one[k] = fma2(one, cosine[j].one[k], mul2(two, sine[j].one[k]));
                        u[j].two[k] = fma2(two, cosine[j].one[k], mul2(one, minus2(sine[j].one[k])));
                    }
                }
                add_unit<Form>(v[j], u[j], gain[j], squares2, product2);
            }
            float squares = sum2(squares2), product = sum2(product2);
            for (int o = 1; o < lanes; o <<= 1) {
                squares += __shfl_xor_sync(0xffffffffu, squares, o);
                product += __shfl_xor_sync(0xffffffffu, product, o);
            }
            const float r = live ? inverse_root<T>(__fmaf_rn(squares, a.inverse_d, a.epsilon)) : 0.0f;
            const float along = r * r * (product * a.inverse_d);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                finish_unit<Form>(v[j], u[j], gain[j], r, along, sums[j]);
                if (live && share.there[j]) Raw::store(to + share.channel[j], apart, share.turns[j], u[j]);
            }
        };
        bool fresh = true;
        if constexpr (PER_HEAD) {
            if (!first) __syncthreads();   // (the other pair's places are not needed any more)
            if (threadIdx.x < tokens) {
                const TokenPlaces of(a, s, token0 + static_cast<int>(threadIdx.x));
                places[0][threadIdx.x] = of.x;
                places[1][threadIdx.x] = of.dy;
                places[2][threadIdx.x] = of.out;
            }
            __syncthreads();
            int head = warp, base = 0, ahead = warp, ahead_base = 0;   // at hand, and the next to be fetched
            auto fetch = [&] {
                const int token = ahead_base + group;
                const bool wanted = ahead < heads && token < tokens;
                const int at = wanted ? token : 0;
                fill(x + ahead * s.x_stride[1] + places[0][at], dy + ahead * s.dy_stride[1] + places[1][at], wanted);
                if ((ahead_base += groups) >= tokens) {
                    ahead_base = 0;
                    ahead += kNormWarps;
                }
            };
#pragma unroll
            for (int i = 0; i + 1 < kGradientStages; ++i) fetch();   // (on their way while the angles are worked out)
            angles_and_gains();
            while (head < heads) {
                const int token = min(base + group, tokens - 1);
                const bool live = base + group < tokens, last = base + groups >= tokens;
                ring.take(rows);
                fetch();
                if (fresh) gains_of(head0 + head);
                fresh = last && s.gain_head != 0;
                row(dx + head * s.out_stride[1] + places[2][token], angles + token * 2 * a.half, live);
                if (last && sums_wanted) put_sums<Form, U, V>(a, share, sums, s.partial + (static_cast<int64_t>(tile) * s.heads + head0 + head) * a.d);
                if (last) {
#pragma unroll
                    for (int j = 0; j < U; ++j) sums[j] = Values<Form::kPacks>{};
                }
                base += groups;
                if (last) {
                    base = 0;
                    head += kNormWarps;
                }
            }
            ring.drain();
        } else {
            const int step = groups >> a.token_shift;
            const TokenPlaces of(a, s, token0 + (own_token ? local : 0));
            int head = group >> a.token_shift;
            x += of.x + head * s.x_stride[1];
            dy += of.dy + head * s.dy_stride[1];
            dx += of.out + head * s.out_stride[1];
            const int64_t x_step = step * s.x_stride[1], dy_step = step * s.dy_stride[1], dx_step = step * s.out_stride[1];
#pragma unroll
            for (int i = 0; i + 1 < kGradientStages; ++i) fill(x + i * x_step, dy + i * dy_step, own_token && head + i * step < heads);   // (on their way while the angles are worked out)
            angles_and_gains();
            while (__any_sync(0xffffffffu, head < heads)) {
                if (fresh) gains_of(head0 + min(head, heads - 1));
                fresh = s.gain_head != 0;
                ring.take(rows);
                fill(x + (kGradientStages - 1) * x_step, dy + (kGradientStages - 1) * dy_step, own_token && head + (kGradientStages - 1) * step < heads);
                row(dx, nullptr, own_token && head < heads);
                head += step;
                x += x_step;
                dy += dy_step;
                dx += dx_step;
            }
            ring.drain();
            if (!sums_wanted) continue;
            __syncthreads();   // (no rows are on their way any more)
            put_sums<Form, U, V>(a, share, sums, meeting + warp * a.d);
            __syncthreads();
            const int64_t sum_row = static_cast<int64_t>(tile) * s.runs + (static_cast<int>(blockIdx.y) - s.first_run);
            for (int c = threadIdx.x; c < a.d; c += kNormThreads) {
                float sum = meeting[c];
#pragma unroll
                for (int w = 1; w < kNormWarps; ++w) sum += meeting[w * a.d + c];
                s.partial[sum_row * a.d + c] = sum;
            }
            if (which == 0) __syncthreads();   // (before rows are on their way again)
        }
    }
}

// Single values, and rows longer than a warp's registers: a row is a whole warp's and read a second time (from the caches); sums of dgain are in shared memory.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kNormThreads)
head_norm_grad_long_kernel(const __grid_constant__ NormArgs a) {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Raw = RawUnit<T, V, INTERLEAVED>;
    extern __shared__ __align__(16) float angles[];                   // the table, and each warp's sums behind it
    const int tile = static_cast<int>(blockIdx.x), token0 = tile << a.token_shift, tokens = min(a.tokens - token0, 1 << a.token_shift);
    const int run0 = static_cast<int>(blockIdx.y) * a.heads_per_cta, run1 = run0 + a.heads_per_cta;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, apart = Form::apart(a);
    chain_begin();
    fill_angles_of<T, Form>(a, angles, token0, tokens);
    __syncthreads();
    float* meeting = angles + ((2 * a.half) << a.token_shift);
    float* sums = meeting + warp * a.d;   // (a lane's channels are its own)
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const NormSide& s = a.side[which];
        const int before = which ? a.side[0].heads : 0, head0 = max(run0 - before, 0), heads = min(run1 - before, s.heads) - head0;
        if (heads <= 0) continue;
        const bool sums_wanted = s.partial != nullptr;
        for (int c = lane; c < a.d; c += 32) sums[c] = 0.0f;
        __syncwarp();
        for (int head = warp; head < heads; head += kNormWarps) {
            for (int local = 0; local < tokens; ++local) {
                const TokenPlaces of(a, s, token0 + local);
                const T* from_x = static_cast<const T*>(s.x) + (head0 + head) * s.x_stride[1] + of.x;
                const T* from_dy = static_cast<const T*>(s.dy) + (head0 + head) * s.dy_stride[1] + of.dy;
                T* to = static_cast<T*>(s.out) + (head0 + head) * s.out_stride[1] + of.out;
                float r = 0.0f, along = 0.0f;
                uint64_t squares = 0, product = 0;
                for (int pass = 0; pass < 2; ++pass) {
                    for (int unit = lane; unit < a.units; unit += 32) {
                        const bool turns = unit < a.turning;
                        const int channel = Form::channel(a, unit);
                        Raw raw_x, raw_dy;
                        raw_x.load(from_x + channel, apart, turns);
                        raw_dy.load(from_dy + channel, apart, turns);
                        const Values<Form::kPacks> v = raw_x.values();
                        Values<Form::kPacks> u = raw_dy.values(), gain, terms{};
                        load_gains<Form, V>(a, s, s.gain_head ? head0 + head : 0, channel, true, turns, gain);
                        if (turns) turn_unit<Form, true>(a, angles + local * 2 * a.half, unit, u);
                        if (pass == 0) {
                            add_unit<Form>(v, u, gain, squares, product);
                            continue;
                        }
                        finish_unit<Form>(v, u, gain, r, along, terms);
                        Raw::store(to + channel, apart, turns, u);
#pragma unroll
                        for (int k = 0; k < Form::kPacks; ++k) {
                            float term[2][2];
                            unpack2(terms.one[k], term[0][0], term[0][1]);
                            unpack2(terms.two[k], term[1][0], term[1][1]);
#pragma unroll
                            for (int second = 0; second < 2; ++second)
#pragma unroll
                                for (int half = 0; half < 2; ++half)
                                    if ((!second || !Form::kTwo || turns) && (V > 1 || half == 0)) sums[channel + (second && Form::kTwo ? apart : 0) + Form::place(k, half, second != 0)] += term[second][half];
                        }
                    }
                    if (pass == 0) {
                        r = inverse_root<T>(__fmaf_rn(sum_over(sum2(squares), 32), a.inverse_d, a.epsilon));
                        along = r * r * (sum_over(sum2(product), 32) * a.inverse_d);
                    }
                }
            }
            if (s.per_head && sums_wanted) {
                __syncwarp();
                for (int c = lane; c < a.d; c += 32) {
                    s.partial[(static_cast<int64_t>(tile) * s.heads + head0 + head) * a.d + c] = sums[c];
                    sums[c] = 0.0f;
                }
                __syncwarp();
            }
        }
        if (s.per_head || !sums_wanted) continue;
        __syncthreads();
        const int64_t sum_row = static_cast<int64_t>(tile) * s.runs + (static_cast<int>(blockIdx.y) - s.first_run);
        for (int c = threadIdx.x; c < a.d; c += kNormThreads) {
            float sum = meeting[c];
#pragma unroll
            for (int w = 1; w < kNormWarps; ++w) sum += meeting[w * a.d + c];
            s.partial[sum_row * a.d + c] = sum;
        }
        __syncthreads();
    }
}

// ---- dgain: the sums of all CTAs, column by column in 64 bits ------------------------------------------------------
struct GainSide {
    const float* partial;
    void* out;
    int64_t rows, columns, out_head;
    int32_t type, d;
};
struct GainArgs {
    GainSide side[2];
    int32_t first_blocks, cluster;   // cluster: CTAs that share a block's rows
};
// 16 columns a CTA, 64 rows at a time: what bounds it is the latency of a thread's loads, which are few and all on their way at once. Many rows are shared out
// over a cluster, whose sums meet in order (3518 + 3518 rows of 128 columns: 15 us by one CTA each).
constexpr int kGainColumns = 16, kGainCluster = 8;
__global__ void __launch_bounds__(1024)
gain_sums_kernel(const __grid_constant__ GainArgs a) {
    __shared__ double sums[32][kGainColumns];
    __shared__ double whole[kGainColumns];
    const int block = static_cast<int>(blockIdx.x) / a.cluster, rank = static_cast<int>(blockIdx.x) - block * a.cluster;
    const int which = block >= a.first_blocks;
    const GainSide& s = a.side[which];
    const int tx = threadIdx.x % kGainColumns, ty = threadIdx.x / kGainColumns;
    const int64_t column = (static_cast<int64_t>(block) - (which ? a.first_blocks : 0)) * kGainColumns + tx;
    chain_begin();
    double sum = 0.0;
    if (column < s.columns) {
        const float* from = s.partial + column;
        const int step = a.cluster * (1024 / kGainColumns);
#pragma unroll 8
        for (int64_t row = rank * (1024 / kGainColumns) + ty; row < s.rows; row += step) sum += static_cast<double>(from[row * s.columns]);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    if ((threadIdx.x & 16) == 0) sums[threadIdx.x >> 5][tx] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += sums[(threadIdx.x >> 4) * 16 + i][tx];
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (threadIdx.x < 16) whole[tx] = sum;
    }
    if (a.cluster > 1) {
        cluster_barrier();
        if (rank == 0 && threadIdx.x < 16) {
            for (int r = 1; r < a.cluster; ++r) {
                uint32_t remote;
                double other;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(&whole[tx])), "r"(r));
                asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(other) : "r"(remote) : "memory");
                sum += other;
            }
        }
        cluster_barrier();   // (no CTA leaves while its sums are read)
    }
    if (rank != 0 || threadIdx.x >= 16 || column >= s.columns) return;
    const int64_t head = column / s.d;
    store_from_f32(s.out, s.type, head * s.out_head + (column - head * s.d), static_cast<float>(sum));
}

// ---- host ---------------------------------------------------------------------------------------------------------

bool float_type(int dtype) { return dtype == DFGPU_F32 || dtype == DFGPU_F16 || dtype == DFGPU_BF16; }

// x and one tensor of its extents (Y, dY or dX).
int check_rows(const dfgpu_tensor& x, const dfgpu_tensor& t, const char* name, bool output) {
    if (!valid_tensor(t) || t.rank != 4) return fail(kInvalidShape, "HEAD_NORM: %s must have rank 4 and positive extents", name);
    for (int i = 0; i < 4; ++i)
        if (t.dim[i] != x.dim[i]) return fail(kInvalidShape, "HEAD_NORM: %s and its input differ in extent", name);
    if (t.dtype != x.dtype) return fail(kUnsupported, "HEAD_NORM: %s and its input differ in type", name);
    if (t.stride[3] != 1 && t.dim[3] != 1) return fail(kInvalidLayout, "HEAD_NORM: the head dimension of %s must have unit stride", name);
    if (output && overlaps_itself(t)) return fail(kInvalidLayout, "HEAD_NORM: %s overlaps itself", name);
    return kOk;
}
int check_gain(const dfgpu_tensor& x, const dfgpu_tensor& gain, const char* name, bool output) {
    if (gain.rank == 0) return kOk;
    if (!valid_tensor(gain) || gain.rank != 4 || gain.dim[0] != 1 || gain.dim[2] != 1 || gain.dim[3] != x.dim[3] || (gain.dim[1] != 1 && gain.dim[1] != x.dim[1]))
        return fail(kInvalidShape, "HEAD_NORM: %s must be [1, 1 or H, 1, D]", name);
    if (!float_type(gain.dtype)) return fail(kUnsupported, "HEAD_NORM: %s must be FLOAT, HALF or BFLOAT16", name);
    if (gain.stride[3] != 1 && gain.dim[3] != 1) return fail(kInvalidLayout, "HEAD_NORM: the channels of %s must have unit stride", name);
    if (output && overlaps_itself(gain)) return fail(kInvalidLayout, "HEAD_NORM: %s overlaps itself", name);
    return kOk;
}

// What both directions have in common. tensors: X and its like of each side (output flags alike), rank 0 where the second side is absent.
struct NormProblem {
    const dfgpu_tensor* row[2][3];    // X, then Y, or dY and dX
    const dfgpu_tensor* gain[2];
    const dfgpu_tensor* dgain[2];     // null: forward
    const dfgpu_tensor* positions;
    const dfgpu_tensor* frequencies;
    int count;                        // tensors of a side
    int interleaved, kernel;
    float scale, epsilon, gain_offset;
    bool two;
    int width;                        // values a vector
    // (where nothing turns pairs may be anywhere: side by side a unit is one vector, all of which counts)
    NormProblem without_pairs() {
        if (positions->rank == 0) interleaved = 1;
        return *this;
    }
};
NormProblem problem_of(const dfgpu_head_norm_params& p) {
    return NormProblem{{{&p.x, &p.y, nullptr}, {&p.x2, &p.y2, nullptr}}, {&p.gain, &p.gain2}, {nullptr, nullptr}, &p.positions, &p.frequencies, 2, p.interleaved, p.kernel, p.scale,
                       p.epsilon, p.gain_offset, p.x2.rank != 0 || p.y2.rank != 0, 1}.without_pairs();
}
NormProblem problem_of(const dfgpu_head_norm_grad_params& p) {
    return NormProblem{{{&p.x, &p.dy, &p.dx}, {&p.x2, &p.dy2, &p.dx2}}, {&p.gain, &p.gain2}, {&p.dgain, &p.dgain2}, &p.positions, &p.frequencies, 3, p.interleaved, p.kernel, p.scale,
                       p.epsilon, p.gain_offset, p.x2.rank != 0 || p.dy2.rank != 0 || p.dx2.rank != 0, 1}.without_pairs();
}
// Values to a vector by the descriptors alone: 16 bytes, 8 (of 16-bit types), or one value.
int norm_width(const NormProblem& p) {
    const int bytes = dtype_bytes(p.row[0][0]->dtype);
    const int64_t half = p.positions->rank ? p.frequencies->dim[3] : 0;
    for (int width = 16 / bytes; width >= 4; width /= 2) {
        bool fits = p.row[0][0]->dim[3] % width == 0 && (2 * half) % width == 0 && (p.interleaved || half % width == 0);
        for (int s = 0; s < (p.two ? 2 : 1); ++s)
            for (int t = 0; t < p.count; ++t)
                for (int i = 0; i < 3; ++i) fits = fits && (p.row[s][t]->dim[i] == 1 || p.row[s][t]->stride[i] % width == 0);
        if (fits) return width;
    }
    return 1;
}
int check_norm(NormProblem& p) {
    const dfgpu_tensor& x = *p.row[0][0];
    static const char* const names[2][2][3] = {{{"X", "Y", ""}, {"X2", "Y2", ""}}, {{"X", "dY", "dX"}, {"X2", "dY2", "dX2"}}};
    static const char* const gains[2][2] = {{"gain", "gain2"}, {"dgain", "dgain2"}};
    if (!valid_tensor(x) || x.rank != 4) return fail(kInvalidShape, "HEAD_NORM: X must have rank 4 and positive extents");
    if (!float_type(x.dtype)) return fail(kUnsupported, "HEAD_NORM: X must be FLOAT, HALF or BFLOAT16");
    for (int s = 0; s < (p.two ? 2 : 1); ++s) {
        const dfgpu_tensor& own = *p.row[s][0];
        if (s == 1) {
            if (!valid_tensor(own) || own.rank != 4 || own.dim[0] != x.dim[0] || own.dim[2] != x.dim[2] || own.dim[3] != x.dim[3])
                return fail(kInvalidShape, "HEAD_NORM: X and X2 differ in batch, length or head dimension");
            if (own.dtype != x.dtype) return fail(kUnsupported, "HEAD_NORM: X and X2 differ in type");
        }
        int status = kOk;
        for (int t = 0; t < p.count && !status; ++t) status = check_rows(own, *p.row[s][t], names[p.count == 3][s][t], t == p.count - 1);
        if (!status) status = check_gain(own, *p.gain[s], gains[0][s], false);
        if (!status && p.dgain[s]) status = check_gain(own, *p.dgain[s], gains[1][s], true);
        if (status) return status;
        if (p.dgain[s] && p.dgain[s]->rank && p.gain[s]->rank && p.dgain[s]->dim[1] != p.gain[s]->dim[1]) return fail(kInvalidShape, "HEAD_NORM: %s and its gradient differ in extent", gains[0][s]);
    }
    if (!p.two && (p.gain[1]->rank || (p.dgain[1] && p.dgain[1]->rank))) return fail(kInvalidArgument, "HEAD_NORM: a second gain without X2");
    if ((p.positions->rank == 0) != (p.frequencies->rank == 0)) return fail(kInvalidArgument, "HEAD_NORM: positions and frequencies go together");
    if (p.positions->rank) {
        const dfgpu_tensor &at = *p.positions, &f = *p.frequencies;
        if (!valid_tensor(at) || at.rank != 4 || (at.dim[0] != 1 && at.dim[0] != x.dim[0]) || at.dim[1] != 1 || at.dim[2] != x.dim[2] || at.dim[3] != 1)
            return fail(kInvalidShape, "HEAD_NORM: positions must be [B or 1, 1, S, 1]");
        if (at.dtype != DFGPU_I32 && at.dtype != DFGPU_I64) return fail(kUnsupported, "HEAD_NORM: positions must be INT32 or INT64");
        if (!valid_tensor(f) || f.rank != 4 || f.dim[0] != 1 || f.dim[1] != 1 || f.dim[2] != 1) return fail(kInvalidShape, "HEAD_NORM: frequencies must be [1, 1, 1, R/2]");
        if (f.dtype != DFGPU_F32) return fail(kUnsupported, "HEAD_NORM: frequencies must be FLOAT");
        if (f.dim[3] > x.dim[3] / 2) return fail(kInvalidShape, "HEAD_NORM: two channels for each frequency are more than the head dimension");
    }
    if (x.dim[3] > kNormMaxD) return fail(kUnsupported, "HEAD_NORM: head dimension above %lld", static_cast<long long>(kNormMaxD));
    const int64_t heads = x.dim[1] + (p.two ? p.row[1][0]->dim[1] : 0);
    if (heads > 65535 || x.dim[2] >= (1ll << 30) || x.dim[0] >= (1ll << 30) || x.dim[0] * x.dim[2] >= (1ll << 31) - 64) return fail(kUnsupported, "HEAD_NORM: too many heads or tokens");
    if (!(p.epsilon >= 0.0f) || !std::isfinite(p.epsilon)) return fail(kInvalidValue, "HEAD_NORM: epsilon must be finite and not negative");
    if (p.kernel < DFGPU_HEAD_NORM_AUTO || p.kernel > DFGPU_HEAD_NORM_SCALAR) return fail(kInvalidArgument, "HEAD_NORM: unknown kernel id %d", p.kernel);
    p.width = p.kernel == DFGPU_HEAD_NORM_SCALAR ? 1 : norm_width(p);
    if (p.kernel == DFGPU_HEAD_NORM_VECTOR && p.width == 1) return fail(kUnsupported, "HEAD_NORM: the vector kernel needs extents and strides of whole vectors of 8 bytes (FLOAT: 16)");
    return kOk;
}

// As few lanes as hold a row, 32 bytes each; single values (width 1) and rows beyond a warp: a warp a row, read twice (per_lane 0).
struct LaneForm {
    int turning, units, per_lane, group_shift;
};
LaneForm lane_form(const NormProblem& p, int width) {
    const int half = p.positions->rank ? static_cast<int>(p.frequencies->dim[3]) : 0, d = static_cast<int>(p.row[0][0]->dim[3]);
    const int pairs = p.interleaved && width > 1 ? width / 2 : width;   // of a unit
    LaneForm form{half / pairs, half / pairs + (d - 2 * half) / width, width == 1 ? 0 : 16 / dtype_bytes(p.row[0][0]->dtype) / pairs, 5};
    if (form.units > 32 * form.per_lane) form.per_lane = 0;
    if (form.per_lane)
        for (form.group_shift = 0; (form.per_lane << form.group_shift) < form.units;) ++form.group_shift;
    return form;
}

// The table, lanes and strides; `pointers`: of row[side][tensor], `positions` and `frequencies`.
int build_norm(NormProblem& p, void* const (&pointers)[2][3], const void* positions, const void* frequencies, const void* const (&gains)[2], NormArgs& a, int& per_lane) {
    const dfgpu_tensor& x = *p.row[0][0];
    const int bytes = dtype_bytes(x.dtype), sides = p.two ? 2 : 1;
    for (int s = 0; s < sides; ++s) {
        Region regions[3];
        for (int t = 0; t < p.count; ++t) {
            if (!pointers[s][t]) return fail(kInvalidArgument, "HEAD_NORM: a tensor of rows is null");
            if (!aligned(pointers[s][t], bytes)) return fail(kInvalidArgument, "HEAD_NORM: a tensor is not aligned to its type");
            while (p.width > 1 && !aligned(pointers[s][t], p.width * bytes)) {
                const int narrower = p.width * bytes > 8 && p.width / 2 >= 4 ? p.width / 2 : 1;
                if (p.kernel == DFGPU_HEAD_NORM_VECTOR && narrower == 1) return fail(kInvalidArgument, "HEAD_NORM: the vector kernel needs tensors on 8-byte boundaries (FLOAT: 16)");
                p.width = narrower;
            }
            regions[t] = region_of(pointers[s][t], *p.row[s][t]);
        }
        const int out = p.count - 1;
        for (int t = 0; t < out; ++t) {
            if (pointers[s][t] != pointers[s][out]) {
                if (overlaps(regions[t], regions[out])) return fail(kInvalidArgument, "HEAD_NORM: an output overlaps an input");
                continue;
            }
            for (int i = 0; i < 3; ++i)
                if (p.row[s][t]->dim[i] > 1 && p.row[s][t]->stride[i] != p.row[s][out]->stride[i]) return fail(kInvalidLayout, "HEAD_NORM: in place, input and output have the same strides");
        }
        if (p.gain[s]->rank) {
            if (!gains[s]) return fail(kInvalidArgument, "HEAD_NORM: a gain is declared but null");
            if (!aligned(gains[s], dtype_bytes(p.gain[s]->dtype))) return fail(kInvalidArgument, "HEAD_NORM: a gain is not aligned to its type");
            if (overlaps(region_of(gains[s], *p.gain[s]), regions[out])) return fail(kInvalidArgument, "HEAD_NORM: an output overlaps a gain");
        }
    }
    if (p.two)
        for (int s = 0; s < 2; ++s)
            for (int t = 0; t < p.count; ++t)
                if (overlaps(region_of(pointers[s][p.count - 1], *p.row[s][p.count - 1]), region_of(pointers[1 - s][t], *p.row[1 - s][t])))
                    return fail(kInvalidArgument, "HEAD_NORM: the output of one pair overlaps a tensor of the other");
    if (p.positions->rank) {
        if (!positions || !frequencies) return fail(kInvalidArgument, "HEAD_NORM: positions or frequencies are declared but null");
        if (!aligned(positions, p.positions->dtype == DFGPU_I64 ? 8 : 4) || !aligned(frequencies, 4)) return fail(kInvalidArgument, "HEAD_NORM: positions or frequencies are not aligned to their type");
        a.at = Positions{positions, static_cast<const float*>(frequencies), p.positions->dim[0] == 1 ? 0 : p.positions->stride[0], p.positions->stride[2], p.frequencies->stride[3],
                         p.positions->dtype == DFGPU_I64};
        a.half = static_cast<int>(p.frequencies->dim[3]);
    }
    for (int s = 0; s < sides; ++s) {
        NormSide& side = a.side[s];
        const int out = p.count - 1;
        side.x = pointers[s][0];
        side.dy = p.count == 3 ? pointers[s][1] : nullptr;
        side.out = pointers[s][out];
        for (int i = 0; i < 3; ++i) {
            const bool one = p.row[s][0]->dim[i] == 1;
            side.x_stride[i] = one ? 0 : p.row[s][0]->stride[i];
            side.dy_stride[i] = one ? 0 : p.row[s][1]->stride[i];
            side.out_stride[i] = one ? 0 : p.row[s][out]->stride[i];
        }
        side.heads = static_cast<int>(p.row[s][0]->dim[1]);
        side.gain = p.gain[s]->rank ? gains[s] : nullptr;
        side.gain_type = p.gain[s]->dtype;
        side.gain_head = p.gain[s]->rank && p.gain[s]->dim[1] > 1 ? p.gain[s]->stride[1] : 0;
    }
    const int64_t d = x.dim[3];
    const LaneForm form = lane_form(p, p.width);
    a.d = static_cast<int>(d);
    a.by_d = make_fast_divisor(static_cast<uint32_t>(d));
    a.turning = form.turning;
    a.units = form.units;
    a.group_shift = form.group_shift;
    per_lane = form.per_lane;
    a.seq = static_cast<int>(x.dim[2]);
    a.tokens = static_cast<int>(x.dim[0] * x.dim[2]);
    a.by_seq = make_fast_divisor(static_cast<uint32_t>(a.seq));
    a.scale = p.scale;
    a.epsilon = p.epsilon;
    a.gain_offset = p.gain_offset;
    a.inverse_d = static_cast<float>(1.0 / static_cast<double>(d));
    return kOk;
}

// Ring::kBytes
constexpr size_t ring_bytes(int stages, int tensors) { return static_cast<size_t>(32) * stages * tensors * kNormThreads; }

enum NormKernel { kForward, kForwardOfHeads, kForwardLong, kGradient, kGradientOfHeads, kGradientLong };
template <typename T, int V, bool INTERLEAVED>
void launch_norm(NormKernel kernel, const NormArgs& a, dim3 grid, size_t shared, cudaStream_t stream) {
    void (*function)(const NormArgs) = head_norm_long_kernel<T, V, INTERLEAVED>;
    if (kernel == kGradientLong) function = head_norm_grad_long_kernel<T, V, INTERLEAVED>;
    if constexpr (V > 1) {
        if (kernel == kForward) function = head_norm_kernel<T, V, INTERLEAVED, false>;
        if (kernel == kForwardOfHeads) function = head_norm_kernel<T, V, INTERLEAVED, true>;
        if (kernel == kGradient) function = head_norm_grad_kernel<T, V, INTERLEAVED, false>;
        if (kernel == kGradientOfHeads) function = head_norm_grad_kernel<T, V, INTERLEAVED, true>;
    }
    launch_chained(function, grid, dim3(kNormThreads), shared, stream, a);
}
template <typename T, int V>
void launch_norm(NormKernel kernel, const NormArgs& a, bool interleaved, dim3 grid, size_t shared, cudaStream_t stream) {
    interleaved ? launch_norm<T, V, true>(kernel, a, grid, shared, stream) : launch_norm<T, V, false>(kernel, a, grid, shared, stream);
}
void launch_norm(NormKernel kernel, const NormArgs& a, int dtype, int width, bool interleaved, dim3 grid, size_t shared, cudaStream_t stream) {
    if (dtype == DFGPU_F32) {
        if (width == 4) launch_norm<float, 4>(kernel, a, interleaved, grid, shared, stream);
        else launch_norm<float, 1>(kernel, a, interleaved, grid, shared, stream);
    } else if (dtype == DFGPU_F16) {
        if (width == 8) launch_norm<__half, 8>(kernel, a, interleaved, grid, shared, stream);
        else if (width == 4) launch_norm<__half, 4>(kernel, a, interleaved, grid, shared, stream);
        else launch_norm<__half, 1>(kernel, a, interleaved, grid, shared, stream);
    } else {
        if (width == 8) launch_norm<__nv_bfloat16, 8>(kernel, a, interleaved, grid, shared, stream);
        else if (width == 4) launch_norm<__nv_bfloat16, 4>(kernel, a, interleaved, grid, shared, stream);
        else launch_norm<__nv_bfloat16, 1>(kernel, a, interleaved, grid, shared, stream);
    }
}

// The gradient's cut: tokens a CTA (1 << shift) and heads a run. A function of the descriptors alone: the scratch depends on it.
struct GradCut {
    int shift, heads_per_cta;
    int64_t tiles, runs, of_side[2], first_of_second;   // runs of heads: all, and those that hold some of a side's
};
bool sums_of_heads(const dfgpu_tensor& dgain) { return dgain.rank && dgain.dim[1] > 1; }
bool any_sums_of_heads(const NormProblem& p) { return sums_of_heads(*p.dgain[0]) || (p.two && sums_of_heads(*p.dgain[1])); }
GradCut grad_cut(const NormProblem& p) {
    const dfgpu_tensor& x = *p.row[0][0];
    const int64_t half = p.positions->rank ? p.frequencies->dim[3] : 0;
    const int64_t tokens = x.dim[0] * x.dim[2], heads[2] = {x.dim[1], p.two ? p.row[1][0]->dim[1] : 0};
    GradCut cut{};
    // With sums for each head 16 tokens and few heads (3 x 1001 f32 tokens of 32 heads: four or eight heads 37.5 us, 16 61.8; eight tokens 43.9, 41.4 and 41.3); otherwise
    // as many tokens as there are groups of lanes and many heads (4 x 2048 bf16 tokens of 32 + 8 heads: 40 heads 50.5 us, 32 50.4, 20 56.2, 10 61.0; eight tokens 51.4, 51.9, 58.3, 72.7).
    const bool of_heads = any_sums_of_heads(p);
    cut.shift = 4;
    if (!of_heads) {
        const LaneForm form = lane_form(p, p.width);
        cut.shift = std::min(7 - form.group_shift, 5);
    }
    while (cut.shift > 0 && 8 * (half << cut.shift) > kNormShared) --cut.shift;
    cut.heads_per_cta = static_cast<int>(std::min<int64_t>(heads[0] + heads[1], 40));
    auto ctas = [&] {
        cut.tiles = (tokens + (1ll << cut.shift) - 1) >> cut.shift;
        cut.runs = (heads[0] + heads[1] + cut.heads_per_cta - 1) / cut.heads_per_cta;
        cut.of_side[0] = (heads[0] + cut.heads_per_cta - 1) / cut.heads_per_cta;
        cut.first_of_second = heads[0] / cut.heads_per_cta;
        cut.of_side[1] = cut.runs - cut.first_of_second;
        return cut.tiles * cut.runs;
    };
    // Few tokens: runs of heads that fill the SMs once, since a CTA's own chain (places, angles, first rows, sums) is most of what it takes, fewer tokens and heads only where half the SMs would be left
    // (3 x 2167 tokens of 1 + 1 heads of 80: 17.3 us by three CTAs an SM and any rest, 12.5 so; 4 x 67 of 2 + 2 of 64 13.3, 8.6; 1 x 411 of 56 + 8 of 128 19.8, 17.2; 8 x 26 of 47 + 8 of 96 15.1, 11.9).
    const int64_t all = heads[0] + heads[1], slots = (x.dtype == DFGPU_F32 ? 6 : 4) * 148;   // CTAs that run at once
    auto spread = [&] {
        if (!of_heads) {   // runs that fill the slots once
            ctas();
            const int64_t runs = std::max<int64_t>(1, std::min(all, slots / cut.tiles));
            cut.heads_per_cta = static_cast<int>(std::min<int64_t>(40, (all + runs - 1) / runs));
        }
        return ctas();
    };
    if (of_heads)
        while (ctas() < 10 * 148 && cut.heads_per_cta > 4) cut.heads_per_cta = (cut.heads_per_cta + 1) / 2;
    while (2 * spread() <= slots && cut.shift > 2) --cut.shift;
    while (2 * ctas() <= slots && cut.heads_per_cta > 1) cut.heads_per_cta = (cut.heads_per_cta + 1) / 2;
    ctas();
    return cut;
}
// Floats of partial sums of a side, none where no dgain is wanted.
int64_t grad_partials(const NormProblem& p, const GradCut& cut, int s) {
    if ((s == 1 && !p.two) || p.dgain[s]->rank == 0) return 0;
    return cut.tiles * p.row[s][0]->dim[3] * (any_sums_of_heads(p) ? p.row[s][0]->dim[1] : cut.of_side[s]);
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_head_norm(const dfgpu_head_norm_params* params, dfgpu_plan_info* info) {
    if (!params || !info) return fail(kInvalidArgument, "HEAD_NORM: null params");
    NormProblem p = problem_of(*params);
    const int status = check_norm(p);
    if (status) return status;
    info->kernel = p.width > 1 ? DFGPU_HEAD_NORM_VECTOR : DFGPU_HEAD_NORM_SCALAR;
    info->launches = 1;
    info->scratch_bytes = 0;
    return kOk;
}

extern "C" int dfgpu_head_norm(const dfgpu_head_norm_params* params, void* const* tensors, void* scratch, void* stream) {
    (void)scratch;
    if (!params || !tensors) return fail(kInvalidArgument, "HEAD_NORM: null params");
    NormProblem p = problem_of(*params);
    int status = check_norm(p);
    if (status) return status;
    NormArgs a{};
    int per_lane;
    void* const rows[2][3] = {{tensors[0], tensors[1], nullptr}, {p.two ? tensors[5] : nullptr, p.two ? tensors[6] : nullptr, nullptr}};
    const void* const gains[2] = {p.gain[0]->rank ? tensors[2] : nullptr, p.gain[1]->rank ? tensors[7] : nullptr};
    status = build_norm(p, rows, p.positions->rank ? tensors[3] : nullptr, p.positions->rank ? tensors[4] : nullptr, gains, a, per_lane);
    if (status) return status;
    // Up to eight tokens a CTA and all heads, which share the tokens' angles; fewer heads where the CTAs would be few. (2 x 8192 tokens of 40 heads of 128 bf16 channels: 60.7 us;
    // sixteen tokens 66.7, four 64.2; the heads in two runs 61.9, in four 76.9.)
    const int heads = a.side[0].heads + a.side[1].heads, groups = kNormThreads >> a.group_shift;
    while (a.token_shift < 3 && (2 << a.token_shift) <= groups && (1 << a.token_shift) < a.seq && (a.half << (a.token_shift + 1)) <= kNormTable) ++a.token_shift;
    a.tiles = (a.seq + (1 << a.token_shift) - 1) >> a.token_shift;
    a.by_tiles = make_fast_divisor(static_cast<uint32_t>(a.tiles));
    const int64_t tiles = p.row[0][0]->dim[0] * a.tiles;
    // (gains of each head take 4 KiB of shared memory for eight heads of 128 channels)
    const bool gains_of_heads = a.side[0].gain_head || a.side[1].gain_head;
    a.heads_per_cta = gains_of_heads && per_lane ? std::min(heads, std::max(kNormGains / (4 * a.d), 1)) : heads;
    auto runs = [&] { return (heads + a.heads_per_cta - 1) / a.heads_per_cta; };
    // Runs of heads by what they would take: as many rounds as the CTAs need of the six an SM holds, three quarters of one lost beyond the first, each six steps of a CTA's own chain and its rows' (4 x 2048 tokens of 32 + 8 heads 31.3 us in
    // two runs, 34.7 in one; 1 x 1024 9.6 in four, 12.0 in more; 1 x 411 of 56 + 8 7.2 in 16, 9.6 in 32). f32 rows take more runs (7 x 281 tokens of 10 + 8 heads 14.6 in six, 15.8 in two).
    if (p.row[0][0]->dtype == DFGPU_F32) {
        while (tiles * runs() < 8 * 148 && (a.heads_per_cta << a.token_shift) > groups && a.heads_per_cta > 1) a.heads_per_cta = (a.heads_per_cta + 1) / 2;
    } else {
        auto cost = [&] {
            const double rounds = static_cast<double>(tiles * runs()) / (6 * 148);
            return (rounds <= 1.0 ? 1.0 : rounds + 0.75) * (6 + ((a.heads_per_cta << a.token_shift) + groups - 1) / groups);
        };
        int best = a.heads_per_cta;
        double least = cost();
        while ((a.heads_per_cta << a.token_shift) > groups && a.heads_per_cta > 1) {
            a.heads_per_cta = (a.heads_per_cta + 1) / 2;
            if (cost() < least) {
                least = cost();
                best = a.heads_per_cta;
            }
        }
        a.heads_per_cta = best;
    }
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(runs()));
    a.gain_floats = a.d * (gains_of_heads ? a.heads_per_cta + 1 : 2);
    const size_t shared = sizeof(float) * static_cast<size_t>((2 * a.half) << a.token_shift) + (per_lane ? 4 * static_cast<size_t>(a.gain_floats) + ring_bytes(kForwardStages, 1) : 0);
    launch_norm(!per_lane ? kForwardLong : gains_of_heads ? kForwardOfHeads : kForward, a, p.row[0][0]->dtype, p.width, p.interleaved != 0, grid, shared, as_stream(stream));
    return check_launch("HEAD_NORM");
}

extern "C" int dfgpu_query_head_norm_grad(const dfgpu_head_norm_grad_params* params, dfgpu_plan_info* info) {
    if (!params || !info) return fail(kInvalidArgument, "HEAD_NORM gradient: null params");
    NormProblem p = problem_of(*params);
    const int status = check_norm(p);
    if (status) return status;
    const GradCut cut = grad_cut(p);
    const int64_t partials = grad_partials(p, cut, 0) + grad_partials(p, cut, 1);
    info->kernel = p.width > 1 ? DFGPU_HEAD_NORM_VECTOR : DFGPU_HEAD_NORM_SCALAR;
    info->launches = partials ? 2 : 1;
    info->scratch_bytes = 4 * partials;
    return kOk;
}

extern "C" int dfgpu_head_norm_grad(const dfgpu_head_norm_grad_params* params, void* const* tensors, void* scratch, void* stream) {
    if (!params || !tensors) return fail(kInvalidArgument, "HEAD_NORM gradient: null params");
    NormProblem p = problem_of(*params);
    int status = check_norm(p);
    if (status) return status;
    const GradCut cut = grad_cut(p);   // (by the descriptors, as the query has it: places off the vectors' boundaries change the width below)
    NormArgs a{};
    int per_lane;
    void* const rows[2][3] = {{tensors[0], tensors[1], tensors[2]}, {p.two ? tensors[7] : nullptr, p.two ? tensors[8] : nullptr, p.two ? tensors[9] : nullptr}};
    const void* const gains[2] = {p.gain[0]->rank ? tensors[3] : nullptr, p.gain[1]->rank ? tensors[10] : nullptr};
    status = build_norm(p, rows, p.positions->rank ? tensors[5] : nullptr, p.positions->rank ? tensors[6] : nullptr, gains, a, per_lane);
    if (status) return status;
    const int64_t first_partials = grad_partials(p, cut, 0), partials = first_partials + grad_partials(p, cut, 1);
    if (partials && (!scratch || !aligned(scratch, 4))) return fail(kInvalidArgument, "HEAD_NORM gradient: %s", scratch ? "the scratch is not aligned" : "scratch is needed for the sums of dgain");
    GainArgs g{};
    int blocks = 0;
    for (int s = 0; s < (p.two ? 2 : 1); ++s) {
        const dfgpu_tensor& dgain = *p.dgain[s];
        if (dgain.rank == 0) continue;
        void* out = tensors[s ? 11 : 4];
        if (!out) return fail(kInvalidArgument, "HEAD_NORM gradient: a dgain is declared but null");
        if (!aligned(out, dtype_bytes(dgain.dtype))) return fail(kInvalidArgument, "HEAD_NORM gradient: a dgain is not aligned to its type");
        const Region region = region_of(out, dgain);
        for (int o = 0; o < (p.two ? 2 : 1); ++o) {
            for (int t = 0; t < 3; ++t)
                if (overlaps(region, region_of(rows[o][t], *p.row[o][t]))) return fail(kInvalidArgument, "HEAD_NORM gradient: a dgain overlaps another tensor");
            if (overlaps(region, region_of(gains[o], *p.gain[o])) || (o != s && p.dgain[o]->rank && overlaps(region, region_of(tensors[o ? 11 : 4], *p.dgain[o]))))
                return fail(kInvalidArgument, "HEAD_NORM gradient: a dgain overlaps another gain");
        }
        NormSide& side = a.side[s];
        side.partial = static_cast<float*>(scratch) + (s ? first_partials : 0);
        side.per_head = any_sums_of_heads(p);
        const bool apart = sums_of_heads(dgain);   // (where only the other side's are, a side's heads meet in the second kernel)
        GainSide& sums = g.side[s];
        sums.partial = side.partial;
        sums.out = out;
        sums.d = a.d;
        sums.rows = cut.tiles * (apart ? 1 : side.per_head ? side.heads : cut.of_side[s]);
        sums.columns = apart ? static_cast<int64_t>(side.heads) * a.d : a.d;
        sums.out_head = apart ? dgain.stride[1] : 0;
        sums.type = dgain.dtype;
        const int more = static_cast<int>((sums.columns + kGainColumns - 1) / kGainColumns);
        if (s == 0) g.first_blocks = more;
        blocks += more;
    }
    a.token_shift = cut.shift;
    a.heads_per_cta = cut.heads_per_cta;
    for (int s = 0; s < 2; ++s) {
        a.side[s].runs = static_cast<int>(cut.of_side[s]);
        a.side[s].first_run = s ? static_cast<int>(cut.first_of_second) : 0;
    }
    const dim3 grid(static_cast<unsigned>(cut.tiles), static_cast<unsigned>(cut.runs));
    const size_t table = sizeof(float) * static_cast<size_t>((2 * a.half) << a.token_shift), meeting = sizeof(float) * kNormWarps * static_cast<size_t>(a.d);
    // (The form for tokens a group needs as many groups as tokens, and has them where the vectors are narrower than the cut had in mind too: a row of half as long vectors has twice the units, of
    // which a lane has twice as many; single values are a warp's.)
    const bool of_heads = any_sums_of_heads(p);
    launch_norm(!per_lane ? kGradientLong : of_heads ? kGradientOfHeads : kGradient, a, p.row[0][0]->dtype, p.width, p.interleaved != 0, grid,
                table + (per_lane ? 8 * static_cast<size_t>(a.d) + std::max(ring_bytes(kGradientStages, 2), meeting) : meeting),
                                as_stream(stream));
    status = check_launch("HEAD_NORM gradient");
    if (status || !blocks) return status;
    g.cluster = std::max(g.side[0].rows, g.side[1].rows) > 1024 ? kGainCluster : 1;
    launch_chained_cluster(gain_sums_kernel, dim3(static_cast<unsigned>(blocks * g.cluster)), dim3(1024), g.cluster > 1 ? kGainCluster : 0u, 0, as_stream(stream), g);
    return check_launch("HEAD_NORM gradient, dgain");
}
