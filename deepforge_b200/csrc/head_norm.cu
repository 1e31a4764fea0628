// RMS norms of query and key heads with their gains and rotary positions in one pass, and the gradients of all three.
//
// A row is one token's head, D channels. It is taken by a group of lanes that hold it in registers between its sum of squares and its result
// (pairs that turn together lie in one lane), so that it is read once and written once: HBM is what bounds both kernels.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"

namespace dfgpu {
namespace {

constexpr int kNormThreads = 128, kNormWarps = kNormThreads / 32;
constexpr int kNormTable = 2048;      // (cosine, sine) pairs of a CTA, forward: 16 KiB
constexpr int kNormShared = 47 * 1024;   // gradient: the table and each warp's sums, in bytes
constexpr int64_t kNormMaxD = 1024;

struct NormSide {
    const void* x;
    const void* dy;                   // (gradient)
    void* out;                        // Y or dX
    const void* gain;                 // null: ones
    float* partial;                   // (gradient: sums of dgain, null where it is not wanted)
    int64_t x_stride[3], dy_stride[3], out_stride[3];   // batch, head, token
    int64_t gain_head;
    int32_t gain_type, heads, per_head;   // per_head: sums of dgain for each head
};
struct NormArgs {
    NormSide side[2];
    Positions at;
    int32_t seq, tokens, tiles, token_shift;   // tokens: of all sequences; a CTA's: 1 << token_shift
    int32_t first_side, heads_per_cta;         // first_side: runs of heads of the first pair of tensors
    int32_t d, half, turning, units, pitch;    // units of V pairs (half) or V channels (interleaved, or not turned) a row; pitch: of a token in the table
    int32_t group_shift;                       // lanes of a row: 1 << group_shift
    FastDivisor by_tiles, by_seq;
    float scale, epsilon, gain_offset, inverse_d;
};

__device__ __forceinline__ float gain_at(const NormSide& s, float offset, int64_t at) {
    if (!s.gain) return 1.0f;
    if (s.gain_type == DFGPU_F32) return static_cast<const float*>(s.gain)[at] + offset;
    if (s.gain_type == DFGPU_F16) return __half2float(static_cast<const __half*>(s.gain)[at]) + offset;
    return bf16_bits_to_f32(static_cast<const uint16_t*>(s.gain)[at]) + offset;
}

// One unit of a row in registers: V pairs as two vectors (i and i + half), or with INTERLEAVED V channels as one (V = 1: one pair as two values);
// of channels that do not turn, V as one.
template <typename T, int V, bool INTERLEAVED>
struct NormUnit {
    static constexpr bool kTwo = !INTERLEAVED || V == 1;
    static constexpr int kPairs = kTwo ? V : V / 2, kValues = kTwo ? 2 * V : V;
    // places of pair p
    static constexpr __device__ int one(int p) { return kTwo ? p : 2 * p; }
    static constexpr __device__ int two(int p) { return kTwo ? V + p : 2 * p + 1; }
    static __device__ __forceinline__ int channel(const NormArgs& a, int unit) {
        return unit < a.turning ? (INTERLEAVED ? unit * (V == 1 ? 2 : V) : unit * V) : 2 * a.half + (unit - a.turning) * V;
    }
    static __device__ __forceinline__ int apart(const NormArgs& a) { return INTERLEAVED ? 1 : a.half; }
};
template <typename T, int V, bool INTERLEAVED>
struct RawUnit {
    using Form = NormUnit<T, V, INTERLEAVED>;
    Pack<T, V> first, second;
    __device__ __forceinline__ void load(const T* from, int apart, bool live, bool turns) {
#pragma unroll
        for (int i = 0; i < V; ++i) first.v[i] = second.v[i] = narrow<T>(0.0f);
        if (live) first = *reinterpret_cast<const Pack<T, V>*>(from);
        if (Form::kTwo && live && turns) second = *reinterpret_cast<const Pack<T, V>*>(from + apart);
    }
    __device__ __forceinline__ void values(float (&v)[Form::kValues]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = widen(first.v[i]);
            if constexpr (Form::kTwo) v[V + i] = widen(second.v[i]);
        }
    }
    static __device__ __forceinline__ void store(T* to, int apart, bool turns, const float (&v)[Form::kValues]) {
        Pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out.v[i] = narrow<T>(v[i]);
        *reinterpret_cast<Pack<T, V>*>(to) = out;
        if constexpr (Form::kTwo) {
            if (turns) {
#pragma unroll
                for (int i = 0; i < V; ++i) out.v[i] = narrow<T>(v[V + i]);
                *reinterpret_cast<Pack<T, V>*>(to + apart) = out;
            }
        }
    }
};
template <typename Form>
__device__ __forceinline__ void load_gains(const NormArgs& a, const NormSide& s, int head, int channel, bool live, bool turns, int apart, int v, float (&gain)[Form::kValues]) {
#pragma unroll
    for (int i = 0; i < Form::kValues; ++i) {
        const bool second = Form::kTwo && i >= v;
        gain[i] = live && (!second || turns) ? gain_at(s, a.gain_offset, head * s.gain_head + channel + (second ? apart + i - v : i)) : 0.0f;
    }
}
// The pairs of a unit by the angles at `table` (pair p of neighbouring units side by side); BACK: the other way.
template <typename Form, bool BACK>
__device__ __forceinline__ void turn_unit(const NormArgs& a, const float2* angles, int table, float (&v)[Form::kValues]) {
#pragma unroll
    for (int p = 0; p < Form::kPairs; ++p) {
        const float2 cs = angles[table + p * a.turning];
        const float x1 = v[Form::one(p)], x2 = v[Form::two(p)];
        if (BACK) {
            v[Form::one(p)] = __fmaf_rn(x1, cs.x, x2 * cs.y);
            v[Form::two(p)] = __fmaf_rn(x2, cs.x, -(x1 * cs.y));
        } else {
            v[Form::one(p)] = __fmaf_rn(x1, cs.x, -(x2 * cs.y));
            v[Form::two(p)] = __fmaf_rn(x2, cs.x, x1 * cs.y);
        }
    }
}
template <typename Form>
__device__ __forceinline__ void put_angle(const NormArgs& a, float2* angles, int local, int pair, float2 turn) {
    const int unit = pair / Form::kPairs;
    angles[local * a.pitch + (pair - unit * Form::kPairs) * a.turning + unit] = make_float2(turn.x * a.scale, turn.y * a.scale);
}
__device__ __forceinline__ float sum_over(float v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---- forward: a CTA takes a few tokens of one sequence and a run of heads --------------------------------------
// U units a lane (1 or 2), or 0: a row is a whole warp's and read a second time (from the cache).
template <typename T, int V, bool INTERLEAVED, int U>
__global__ void __launch_bounds__(kNormThreads)
head_norm_kernel(const NormArgs a) {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Raw = RawUnit<T, V, INTERLEAVED>;
    extern __shared__ float2 angles[];
    const int tile = static_cast<int>(blockIdx.x);
    const int batch_index = static_cast<int>(fast_divide(static_cast<uint32_t>(tile), a.by_tiles));
    const int token0 = (tile - batch_index * a.tiles) << a.token_shift;
    const bool second_side = static_cast<int>(blockIdx.y) >= a.first_side;
    const NormSide& s = second_side ? a.side[1] : a.side[0];
    const int head0 = (static_cast<int>(blockIdx.y) - (second_side ? a.first_side : 0)) * a.heads_per_cta;
    const int rows = min(a.heads_per_cta, s.heads - head0) << a.token_shift, tokens = a.seq - token0, mask = (1 << a.token_shift) - 1;
    const T* x = static_cast<const T*>(s.x) + batch_index * s.x_stride[0] + head0 * s.x_stride[1] + token0 * s.x_stride[2];
    T* y = static_cast<T*>(s.out) + batch_index * s.out_stride[0] + head0 * s.out_stride[1] + token0 * s.out_stride[2];
    const int lanes = 1 << a.group_shift, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> a.group_shift, groups = kNormThreads >> a.group_shift;
    const int apart = Form::apart(a);
    auto fill_angles = [&] {
        for (int i = threadIdx.x; i < a.half << a.token_shift; i += kNormThreads) {
            const int local = i & mask, pair = i >> a.token_shift;
            if (local < tokens) put_angle<Form>(a, angles, local, pair, turn_of(a.at, batch_index, token0 + local, pair));
        }
        __syncthreads();
    };
    chain_begin();
    if constexpr (U > 0) {
        int channel[U];
        bool there[U], turns[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int unit = lane + j * lanes;
            there[j] = unit < a.units;
            turns[j] = unit < a.turning;
            channel[j] = Form::channel(a, unit);
        }
        Raw now[U], next[U];
        auto load = [&](Raw (&raw)[U], int row) {
            const int local = row & mask, head = row >> a.token_shift;
            const bool live = row < rows && local < tokens;
            const T* from = x + head * s.x_stride[1] + local * s.x_stride[2];
#pragma unroll
            for (int j = 0; j < U; ++j) raw[j].load(from + channel[j], apart, live && there[j], turns[j]);
        };
        load(now, group);   // (on its way while the angles are worked out)
        fill_angles();
        float gain[U][Form::kValues];
        int held = -1;      // the head whose gains these are
        for (int base = 0; base < rows; base += groups) {   // (whole warps stay together)
            const int row = base + group, local = row & mask, head = row >> a.token_shift;
            load(next, row + groups);
            const int wanted = s.gain_head ? head0 + min(head, s.heads - head0 - 1) : 0;
            if (wanted != held) {
#pragma unroll
                for (int j = 0; j < U; ++j) load_gains<Form>(a, s, wanted, channel[j], there[j], turns[j], apart, V, gain[j]);
                held = wanted;
            }
            float v[U][Form::kValues], squares = 0.0f;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                now[j].values(v[j]);
#pragma unroll
                for (int i = 0; i < Form::kValues; ++i) squares = __fmaf_rn(v[j][i], v[j][i], squares);
            }
            const float r = rsqrtf(__fmaf_rn(sum_over(squares, lanes), a.inverse_d, a.epsilon));
            if (row < rows && local < tokens) {
                T* to = y + head * s.out_stride[1] + local * s.out_stride[2];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    if (!there[j]) continue;
#pragma unroll
                    for (int i = 0; i < Form::kValues; ++i) v[j][i] = v[j][i] * r * gain[j][i];
                    if (turns[j]) turn_unit<Form, false>(a, angles, local * a.pitch + lane + j * lanes, v[j]);
                    Raw::store(to + channel[j], apart, turns[j], v[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < U; ++j) now[j] = next[j];
        }
    } else {
        fill_angles();
        for (int row = group; row < rows; row += groups) {
            const int local = row & mask, head = row >> a.token_shift;
            if (local >= tokens) continue;   // (a whole warp's row)
            const T* from = x + head * s.x_stride[1] + local * s.x_stride[2];
            T* to = y + head * s.out_stride[1] + local * s.out_stride[2];
            float squares = 0.0f;
            for (int unit = lane; unit < a.units; unit += 32) {
                Raw raw;
                float v[Form::kValues];
                raw.load(from + Form::channel(a, unit), apart, true, unit < a.turning);
                raw.values(v);
#pragma unroll
                for (int i = 0; i < Form::kValues; ++i) squares = __fmaf_rn(v[i], v[i], squares);
            }
            const float r = rsqrtf(__fmaf_rn(sum_over(squares, 32), a.inverse_d, a.epsilon));
            for (int unit = lane; unit < a.units; unit += 32) {
                const bool turns = unit < a.turning;
                const int channel = Form::channel(a, unit);
                Raw raw;
                float v[Form::kValues], gain[Form::kValues];
                raw.load(from + channel, apart, true, turns);
                raw.values(v);
                load_gains<Form>(a, s, s.gain_head ? head0 + head : 0, channel, true, turns, apart, V, gain);
#pragma unroll
                for (int i = 0; i < Form::kValues; ++i) v[i] = v[i] * r * gain[i];
                if (turns) turn_unit<Form, false>(a, angles, local * a.pitch + unit, v);
                Raw::store(to + channel, apart, turns, v);
            }
        }
    }
}

// ---- gradients: a CTA takes tokens of all sequences in a row and a run of heads; each warp has heads of its own, whose sums of dgain it keeps ----
template <typename T, int V, bool INTERLEAVED, int U>
__global__ void __launch_bounds__(kNormThreads)
head_norm_grad_kernel(const NormArgs a) {
    using Form = NormUnit<T, V, INTERLEAVED>;
    using Raw = RawUnit<T, V, INTERLEAVED>;
    extern __shared__ float2 angles[];                                // the table; where a lane keeps no sums, those of each warp behind it
    __shared__ int64_t places[3][32];                                 // of the tokens in X, dY, dX
    const int tile = static_cast<int>(blockIdx.x), token0 = tile << a.token_shift, tokens = min(a.tokens - token0, 1 << a.token_shift);
    const bool second_side = static_cast<int>(blockIdx.y) >= a.first_side;
    const NormSide& s = second_side ? a.side[1] : a.side[0];
    const int run = static_cast<int>(blockIdx.y) - (second_side ? a.first_side : 0), runs = second_side ? static_cast<int>(gridDim.y) - a.first_side : a.first_side;
    const int head0 = run * a.heads_per_cta, heads = min(a.heads_per_cta, s.heads - head0);
    const int warp = threadIdx.x >> 5, lanes = 1 << a.group_shift, lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) >> a.group_shift, groups = 32 >> a.group_shift;
    const int apart = Form::apart(a);
    const bool sums_wanted = s.partial != nullptr;
    if (threadIdx.x < tokens) {
        const int token = token0 + threadIdx.x, b = static_cast<int>(fast_divide(static_cast<uint32_t>(token), a.by_seq)), t = token - b * a.seq;
        places[0][threadIdx.x] = b * s.x_stride[0] + t * s.x_stride[2];
        places[1][threadIdx.x] = b * s.dy_stride[0] + t * s.dy_stride[2];
        places[2][threadIdx.x] = b * s.out_stride[0] + t * s.out_stride[2];
    }
    chain_begin();
    for (int i = threadIdx.x; i < a.half << a.token_shift; i += kNormThreads) {
        const int local = i & ((1 << a.token_shift) - 1), pair = i >> a.token_shift;
        if (local >= tokens) continue;
        const int token = token0 + local, b = static_cast<int>(fast_divide(static_cast<uint32_t>(token), a.by_seq));
        put_angle<Form>(a, angles, local, pair, turn_of(a.at, b, token - b * a.seq, pair));
    }
    __syncthreads();
    const T* x = static_cast<const T*>(s.x);
    const T* dy = static_cast<const T*>(s.dy);
    T* dx = static_cast<T*>(s.out);
    float* of_tile = s.partial + (s.per_head ? (static_cast<int64_t>(tile) * s.heads) * a.d : (static_cast<int64_t>(tile) * runs + run) * a.d);
    if constexpr (U > 0) {
        int channel[U];
        bool there[U], turns[U];
        float gain[U][Form::kValues], sums[U][Form::kValues];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int unit = lane + j * lanes;
            there[j] = unit < a.units;
            turns[j] = unit < a.turning;
            channel[j] = Form::channel(a, unit);
#pragma unroll
            for (int i = 0; i < Form::kValues; ++i) sums[j][i] = 0.0f;
        }
        // The groups' sums, met in one group's lanes, to channels at `to`.
        auto put_sums = [&](float* to) {
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int i = 0; i < Form::kValues; ++i) {
                    float v = sums[j][i];
                    for (int o = lanes; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    const bool second = Form::kTwo && i >= V;
                    if (group == 0 && there[j] && (!second || turns[j])) to[channel[j] + (second ? apart + i - V : i)] = v;
                    sums[j][i] = 0.0f;
                }
        };
        Raw x_now[U], dy_now[U], x_next[U], dy_next[U];
        auto load = [&](Raw (&raw_x)[U], Raw (&raw_dy)[U], int head, int local) {
            const bool live = head < heads && local < tokens;
            const int at = live ? local : 0;
            const T* from_x = x + (head0 + head) * s.x_stride[1] + places[0][at];
            const T* from_dy = dy + (head0 + head) * s.dy_stride[1] + places[1][at];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                raw_x[j].load(from_x + channel[j], apart, live && there[j], turns[j]);
                raw_dy[j].load(from_dy + channel[j], apart, live && there[j], turns[j]);
            }
        };
        int head = warp, base = 0;
        load(x_now, dy_now, head, group);
        bool fresh = true;
        while (head < heads) {
            const int local = base + group;
            const bool last = base + groups >= tokens;
            const int next_head = last ? head + kNormWarps : head, next_base = last ? 0 : base + groups;
            load(x_next, dy_next, next_head, next_base + group);
            if (fresh) {
#pragma unroll
                for (int j = 0; j < U; ++j) load_gains<Form>(a, s, s.gain_head ? head0 + head : 0, channel[j], there[j], turns[j], apart, V, gain[j]);
                fresh = false;
            }
            const bool live = local < tokens;
            float v[U][Form::kValues], u[U][Form::kValues], squares = 0.0f, product = 0.0f;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                x_now[j].values(v[j]);
                dy_now[j].values(u[j]);
                if (turns[j] && live) turn_unit<Form, true>(a, angles, local * a.pitch + lane + j * lanes, u[j]);
#pragma unroll
                for (int i = 0; i < Form::kValues; ++i) {
                    squares = __fmaf_rn(v[j][i], v[j][i], squares);
                    product = __fmaf_rn(u[j][i] * gain[j][i], v[j][i], product);
                }
            }
            for (int o = 1; o < lanes; o <<= 1) {
                squares += __shfl_xor_sync(0xffffffffu, squares, o);
                product += __shfl_xor_sync(0xffffffffu, product, o);
            }
            const float r = live ? rsqrtf(__fmaf_rn(squares, a.inverse_d, a.epsilon)) : 0.0f;
            const float along = r * r * (product * a.inverse_d);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                float out[Form::kValues];
#pragma unroll
                for (int i = 0; i < Form::kValues; ++i) {
                    sums[j][i] = __fmaf_rn(u[j][i], v[j][i] * r, sums[j][i]);
                    out[i] = r * __fmaf_rn(-v[j][i], along, u[j][i] * gain[j][i]);
                }
                if (live && there[j]) Raw::store(dx + (head0 + head) * s.out_stride[1] + places[2][local] + channel[j], apart, turns[j], out);
                x_now[j] = x_next[j];
                dy_now[j] = dy_next[j];
            }
            if (last && s.per_head && sums_wanted) put_sums(of_tile + (head0 + head) * a.d);
            if (last && s.gain_head) fresh = true;
            head = next_head;
            base = next_base;
        }
        if (s.per_head || !sums_wanted) return;
        __syncthreads();   // (the angles are not needed any more)
        float* meeting = reinterpret_cast<float*>(angles);
        put_sums(meeting + warp * a.d);
        __syncthreads();
        for (int c = threadIdx.x; c < a.d; c += kNormThreads) {
            float sum = meeting[c];
#pragma unroll
            for (int w = 1; w < kNormWarps; ++w) sum += meeting[w * a.d + c];
            of_tile[c] = sum;
        }
    } else {
        float* meeting = reinterpret_cast<float*>(angles + (a.pitch << a.token_shift));
        float* sums = meeting + warp * a.d;   // (a lane's channels are its own)
        for (int c = threadIdx.x & 31; c < a.d; c += 32) sums[c] = 0.0f;
        __syncwarp();
        for (int head = warp; head < heads; head += kNormWarps) {
            for (int local = 0; local < tokens; ++local) {
                const T* from_x = x + (head0 + head) * s.x_stride[1] + places[0][local];
                const T* from_dy = dy + (head0 + head) * s.dy_stride[1] + places[1][local];
                T* to = dx + (head0 + head) * s.out_stride[1] + places[2][local];
                float r = 0.0f, along = 0.0f, squares = 0.0f, product = 0.0f;
                for (int pass = 0; pass < 2; ++pass) {
                    for (int unit = lane; unit < a.units; unit += 32) {
                        const bool turns = unit < a.turning;
                        const int channel = Form::channel(a, unit);
                        Raw raw_x, raw_dy;
                        float v[Form::kValues], u[Form::kValues], gain[Form::kValues];
                        raw_x.load(from_x + channel, apart, true, turns);
                        raw_dy.load(from_dy + channel, apart, true, turns);
                        raw_x.values(v);
                        raw_dy.values(u);
                        load_gains<Form>(a, s, s.gain_head ? head0 + head : 0, channel, true, turns, apart, V, gain);
                        if (turns) turn_unit<Form, true>(a, angles, local * a.pitch + unit, u);
                        if (pass == 0) {
#pragma unroll
                            for (int i = 0; i < Form::kValues; ++i) {
                                squares = __fmaf_rn(v[i], v[i], squares);
                                product = __fmaf_rn(u[i] * gain[i], v[i], product);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < Form::kValues; ++i) {
                                const bool second = Form::kTwo && i >= V;
                                if (!second || turns) {
                                    float& sum = sums[channel + (second ? apart + i - V : i)];
                                    sum = __fmaf_rn(u[i], v[i] * r, sum);
                                }
                                u[i] = r * __fmaf_rn(-v[i], along, u[i] * gain[i]);
                            }
                            Raw::store(to + channel, apart, turns, u);
                        }
                    }
                    if (pass == 0) {
                        r = rsqrtf(__fmaf_rn(sum_over(squares, 32), a.inverse_d, a.epsilon));
                        along = r * r * (sum_over(product, 32) * a.inverse_d);
                    }
                }
            }
            if (s.per_head && sums_wanted) {
                __syncwarp();
                for (int c = threadIdx.x & 31; c < a.d; c += 32) {
                    of_tile[(head0 + head) * static_cast<int64_t>(a.d) + c] = sums[c];
                    sums[c] = 0.0f;
                }
                __syncwarp();
            }
        }
        if (s.per_head || !sums_wanted) return;
        __syncthreads();
        for (int c = threadIdx.x; c < a.d; c += kNormThreads) {
            float sum = meeting[c];
#pragma unroll
            for (int w = 1; w < kNormWarps; ++w) sum += meeting[w * a.d + c];
            of_tile[c] = sum;
        }
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
    int32_t first_blocks;
};
__global__ void __launch_bounds__(1024)
gain_sums_kernel(const GainArgs a) {
    chain_begin();
    __shared__ double sums[32][33];
    const bool second = static_cast<int>(blockIdx.x) >= a.first_blocks;
    const GainSide& s = second ? a.side[1] : a.side[0];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t column = (static_cast<int64_t>(blockIdx.x) - (second ? a.first_blocks : 0)) * 32 + tx;
    double sum = 0.0;
    if (column < s.columns) {
        const float* from = s.partial + column;
#pragma unroll 8
        for (int64_t row = ty; row < s.rows; row += 32) sum += static_cast<double>(from[row * s.columns]);
    }
    sums[ty][tx] = sum;
    __syncthreads();
    if (ty != 0 || column >= s.columns) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += sums[i][tx];
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
};
NormProblem problem_of(const dfgpu_head_norm_params& p) {
    return NormProblem{{{&p.x, &p.y, nullptr}, {&p.x2, &p.y2, nullptr}}, {&p.gain, &p.gain2}, {nullptr, nullptr}, &p.positions, &p.frequencies, 2, p.interleaved, p.kernel, p.scale,
                       p.epsilon, p.gain_offset, p.x2.rank != 0 || p.y2.rank != 0, 1};
}
NormProblem problem_of(const dfgpu_head_norm_grad_params& p) {
    return NormProblem{{{&p.x, &p.dy, &p.dx}, {&p.x2, &p.dy2, &p.dx2}}, {&p.gain, &p.gain2}, {&p.dgain, &p.dgain2}, &p.positions, &p.frequencies, 3, p.interleaved, p.kernel, p.scale,
                       p.epsilon, p.gain_offset, p.x2.rank != 0 || p.dy2.rank != 0 || p.dx2.rank != 0, 1};
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

// Units a lane and lanes a row, the table, and the strides; `pointers`: of row[side][tensor], `positions` and `frequencies`.
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
    const int pairs = p.interleaved && p.width > 1 ? p.width / 2 : p.width;   // of a unit
    a.d = static_cast<int>(d);
    a.turning = a.half / pairs;
    a.units = a.turning + (a.d - 2 * a.half) / p.width;
    a.pitch = a.half + a.turning;   // (eight units of a token and the next token's do not meet in the same banks)
    a.seq = static_cast<int>(x.dim[2]);
    a.tokens = static_cast<int>(x.dim[0] * x.dim[2]);
    a.by_seq = make_fast_divisor(static_cast<uint32_t>(a.seq));
    a.scale = p.scale;
    a.epsilon = p.epsilon;
    a.gain_offset = p.gain_offset;
    a.inverse_d = static_cast<float>(1.0 / static_cast<double>(d));
    // One unit a lane up to a warp's 32, two beyond; single values (V = 1) and longer rows: a warp a row, read twice.
    per_lane = p.width == 1 || a.units > 64 ? 0 : (a.units > 32 ? 2 : 1);
    a.group_shift = 5;
    if (per_lane == 1)
        for (a.group_shift = 0; (1 << a.group_shift) < a.units;) ++a.group_shift;
    return kOk;
}

template <bool GRAD, typename T, int V, bool INTERLEAVED, int U>
void launch_norm(const NormArgs& a, dim3 grid, size_t shared, cudaStream_t stream) {
    if constexpr (GRAD) {
        launch_chained(head_norm_grad_kernel<T, V, INTERLEAVED, U>, grid, dim3(kNormThreads), shared, stream, a);
    } else {
        launch_chained(head_norm_kernel<T, V, INTERLEAVED, U>, grid, dim3(kNormThreads), shared, stream, a);
    }
}
template <bool GRAD, typename T, int V>
void launch_norm(const NormArgs& a, bool interleaved, int per_lane, dim3 grid, size_t shared, cudaStream_t stream) {
    if constexpr (V > 1) {
        if (per_lane == 1) return interleaved ? launch_norm<GRAD, T, V, true, 1>(a, grid, shared, stream) : launch_norm<GRAD, T, V, false, 1>(a, grid, shared, stream);
        if (per_lane == 2) return interleaved ? launch_norm<GRAD, T, V, true, 2>(a, grid, shared, stream) : launch_norm<GRAD, T, V, false, 2>(a, grid, shared, stream);
    }
    interleaved ? launch_norm<GRAD, T, V, true, 0>(a, grid, shared, stream) : launch_norm<GRAD, T, V, false, 0>(a, grid, shared, stream);
}
template <bool GRAD>
void launch_norm(const NormArgs& a, int dtype, int width, bool interleaved, int per_lane, dim3 grid, size_t shared, cudaStream_t stream) {
    if (dtype == DFGPU_F32) {
        if (width == 4) launch_norm<GRAD, float, 4>(a, interleaved, per_lane, grid, shared, stream);
        else launch_norm<GRAD, float, 1>(a, interleaved, per_lane, grid, shared, stream);
    } else if (dtype == DFGPU_F16) {
        if (width == 8) launch_norm<GRAD, __half, 8>(a, interleaved, per_lane, grid, shared, stream);
        else if (width == 4) launch_norm<GRAD, __half, 4>(a, interleaved, per_lane, grid, shared, stream);
        else launch_norm<GRAD, __half, 1>(a, interleaved, per_lane, grid, shared, stream);
    } else {
        if (width == 8) launch_norm<GRAD, __nv_bfloat16, 8>(a, interleaved, per_lane, grid, shared, stream);
        else if (width == 4) launch_norm<GRAD, __nv_bfloat16, 4>(a, interleaved, per_lane, grid, shared, stream);
        else launch_norm<GRAD, __nv_bfloat16, 1>(a, interleaved, per_lane, grid, shared, stream);
    }
}

// The gradient's cut: tokens a CTA (1 << shift) and heads a run. A function of the descriptors alone (the scratch depends on it): of the pitch of the widest
// and of the scalar form alike, whichever the pointers allow.
struct GradCut {
    int shift, heads_per_cta;
    int64_t tiles, runs[2];
};
GradCut grad_cut(const NormProblem& p) {
    const dfgpu_tensor& x = *p.row[0][0];
    const int64_t half = p.positions->rank ? p.frequencies->dim[3] : 0, pitch = 2 * half;   // (the largest: V = 1)
    const int64_t tokens = x.dim[0] * x.dim[2], heads[2] = {x.dim[1], p.two ? p.row[1][0]->dim[1] : 0};
    GradCut cut{};
    cut.shift = 5;
    while (cut.shift > 0 && (8 * (pitch << cut.shift) + 16 * x.dim[3] > kNormShared)) --cut.shift;
    cut.heads_per_cta = 16;
    auto ctas = [&] {
        cut.tiles = (tokens + (1ll << cut.shift) - 1) >> cut.shift;
        for (int s = 0; s < 2; ++s) cut.runs[s] = (heads[s] + cut.heads_per_cta - 1) / cut.heads_per_cta;
        return cut.tiles * (cut.runs[0] + cut.runs[1]);
    };
    while (ctas() < 4 * 148 && cut.heads_per_cta > 4) cut.heads_per_cta /= 2;
    while (ctas() < 4 * 148 && cut.shift > 2) --cut.shift;
    ctas();
    return cut;
}
bool sums_of_heads(const dfgpu_tensor& dgain) { return dgain.dim[1] > 1; }
// Floats of partial sums of a side, none where no dgain is wanted.
int64_t grad_partials(const NormProblem& p, const GradCut& cut, int s) {
    if ((s == 1 && !p.two) || p.dgain[s]->rank == 0) return 0;
    return cut.tiles * p.row[s][0]->dim[3] * (sums_of_heads(*p.dgain[s]) ? p.row[s][0]->dim[1] : cut.runs[s]);
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
    // Up to eight tokens a CTA, so that a long run of heads shares each token's sines; then as few heads as give each thread eight units.
    while (a.token_shift < 3 && (1 << a.token_shift) < a.seq && (a.pitch << (a.token_shift + 1)) <= kNormTable) ++a.token_shift;
    a.tiles = (a.seq + (1 << a.token_shift) - 1) >> a.token_shift;
    a.by_tiles = make_fast_divisor(static_cast<uint32_t>(a.tiles));
    const int64_t tiles = p.row[0][0]->dim[0] * a.tiles;
    a.heads_per_cta = std::min(std::max(a.side[0].heads, a.side[1].heads), (8 * kNormThreads - 1) / (a.units << a.token_shift) + 1);
    a.first_side = (a.side[0].heads + a.heads_per_cta - 1) / a.heads_per_cta;
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(a.first_side + (a.side[1].heads + a.heads_per_cta - 1) / a.heads_per_cta));
    const size_t shared = sizeof(float2) * static_cast<size_t>(a.pitch << a.token_shift);
    launch_norm<false>(a, p.row[0][0]->dtype, p.width, p.interleaved != 0, per_lane, grid, shared, as_stream(stream));
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
    NormArgs a{};
    int per_lane;
    void* const rows[2][3] = {{tensors[0], tensors[1], tensors[2]}, {p.two ? tensors[7] : nullptr, p.two ? tensors[8] : nullptr, p.two ? tensors[9] : nullptr}};
    const void* const gains[2] = {p.gain[0]->rank ? tensors[3] : nullptr, p.gain[1]->rank ? tensors[10] : nullptr};
    status = build_norm(p, rows, p.positions->rank ? tensors[5] : nullptr, p.positions->rank ? tensors[6] : nullptr, gains, a, per_lane);
    if (status) return status;
    const GradCut cut = grad_cut(p);
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
            if (overlaps(region, region_of(gains[o], *p.gain[o])) || (o != s && overlaps(region, region_of(tensors[o ? 11 : 4], *p.dgain[o]))))
                return fail(kInvalidArgument, "HEAD_NORM gradient: a dgain overlaps another gain");
        }
        NormSide& side = a.side[s];
        side.partial = static_cast<float*>(scratch) + (s ? first_partials : 0);
        side.per_head = sums_of_heads(dgain);
        GainSide& sums = g.side[s];
        sums.partial = side.partial;
        sums.out = out;
        sums.d = a.d;
        sums.rows = cut.tiles * (side.per_head ? 1 : cut.runs[s]);
        sums.columns = side.per_head ? static_cast<int64_t>(side.heads) * a.d : a.d;
        sums.out_head = side.per_head ? dgain.stride[1] : 0;
        sums.type = dgain.dtype;
        const int more = static_cast<int>((sums.columns + 31) / 32);
        if (s == 0) g.first_blocks = more;
        blocks += more;
    }
    a.token_shift = cut.shift;
    a.heads_per_cta = cut.heads_per_cta;
    a.first_side = static_cast<int>(cut.runs[0]);
    const dim3 grid(static_cast<unsigned>(cut.tiles), static_cast<unsigned>(cut.runs[0] + cut.runs[1]));
    const size_t table = sizeof(float2) * static_cast<size_t>(a.pitch << a.token_shift), meeting = sizeof(float) * kNormWarps * static_cast<size_t>(a.d);
    launch_norm<true>(a, p.row[0][0]->dtype, p.width, p.interleaved != 0, per_lane, grid, per_lane ? std::max(table, meeting) : table + meeting, as_stream(stream));
    status = check_launch("HEAD_NORM gradient");
    if (status || !blocks) return status;
    launch_chained(gain_sums_kernel, dim3(static_cast<unsigned>(blocks)), dim3(1024), 0, as_stream(stream), g);
    return check_launch("HEAD_NORM gradient, dgain");
}
