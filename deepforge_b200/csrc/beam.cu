// Beam search: the W best continuations of each batch entry over its beams and the vocabulary, and the states of the beams that go on.
//
// Selection, first kernel: the logits are read once. A CTA takes a part of a row, each warp some blocks of 32 R vectors in a row with the next block on its way, and
// sums exponentials against the largest value so far, which counts as 1 exactly: the log-probability of a token that has nearly all of it is no rounding's
// leftover. Of the largest values of the CTA's lanes (32 of them, each over all warps) the W-th largest is a bound that W values reach at least, and hardly more than W lanes
// of some warp: their vectors are looked through again (from the caches), and what reaches the bound is sorted, a lane an entry.
// Second kernel: a CTA an entry, a warp a beam, which merges its parts' lists; scores are added in 64 bits, beams merged pair by pair.
// What bounds it are the two kernels' chains, not the bytes: 16 x 8 beams over 128000 bf16 tokens 17.8 us (bytes 5.0, exponentials 3.6), of which the second look and the sorts
// take 3 to 4 and the second kernel 4; one user's four beams over 32000 tokens 7.5; 7 x 5 over 50001 f32 tokens 10.1.
//
// Reordering: a copy, by the widest vectors that divide all of a state's places and its rows' bytes. HBM bounds it from 8-byte vectors up: 2 x 8 layers of 8 x 4 rows of 131072 bf16 values 36 us (134 MB
// each way; a part of it stays in the L2 cache), of 131076 36. Below that the loads' number does: of 131074 (4 bytes) 45, 131071 (2) 77, 262143 single bytes 153; 2 x 32 layers of 33333 f32 values 89,
// 33332 67. A token history of 1000 2.5.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"
#include "umma_ptx.cuh"
#include "unaligned.cuh"

namespace dfgpu {
namespace {

constexpr int kCandidates = 256;  // of a CTA, that are sorted at once (32 beams leave some 130)
constexpr int kMaxBeams = 32;
constexpr float kMaxPenalty = 28.0f;
constexpr float kLog2e = 1.44269504088896341f;

struct alignas(16) PartSum {
    double sum;                // of exp(x - most)
    double divisor;            // of the row's worths; of its first part only
    float most;
};
struct Logits {
    const void* data;
    int64_t batch_stride, beam_stride;
    int32_t beams, vocabulary, parts, blocks;   // parts of a row, blocks of a warp
    PartSum* sums;                              // of a part
    uint64_t* keys;                             // of a part: W, falling; 0: none
};
struct Ints {
    int32_t* data;              // null: absent
    int64_t batch, beam;
    __device__ __forceinline__ int32_t& at(int b, int w) const { return data[b * batch + w * beam]; }
};
struct ScanArgs {
    Logits logits;
    Ints finished, lengths;
    float length_penalty;
    FastDivisor by_parts, by_beams;
};

// What a row's scores are divided by; n counts the token to come.
__device__ __noinline__ double divisor_of(int length, bool done, float penalty) {
    return pow(static_cast<double>(min(max(static_cast<int64_t>(length) + (done ? 0 : 1), static_cast<int64_t>(1)), static_cast<int64_t>(0x7fffffff))), static_cast<double>(penalty));
}

// Floats as whole numbers in the same order (0 is below all of them).
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);   // (one zero)
    return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return bits ^ ((bits >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double double_from_ordered(uint64_t o) { return __longlong_as_double(static_cast<long long>(o ^ ((o >> 63) ? 1ull << 63 : ~0ull))); }

// An entry of a list: greater keys first, then lower places.
struct Key {
    uint64_t key;
    __device__ __forceinline__ Key from(int lane) const { return Key{__shfl_sync(0xffffffffu, key, lane)}; }
    __device__ __forceinline__ Key across(int mask) const { return Key{__shfl_xor_sync(0xffffffffu, key, mask)}; }
    __device__ __forceinline__ bool before(const Key& o) const { return key > o.key; }
};
struct Place {
    uint64_t key;
    uint32_t place;
    __device__ __forceinline__ Place from(int lane) const { return Place{__shfl_sync(0xffffffffu, key, lane), __shfl_sync(0xffffffffu, place, lane)}; }
    __device__ __forceinline__ Place across(int mask) const { return Place{__shfl_xor_sync(0xffffffffu, key, mask), __shfl_xor_sync(0xffffffffu, place, mask)}; }
    __device__ __forceinline__ bool before(const Place& o) const { return key > o.key || (key == o.key && place < o.place); }
};
// One lane an entry, in order.
template <typename Entry>
__device__ __forceinline__ void exchange(Entry& mine, int mask, bool want_first) {
    const Entry other = mine.across(mask);
    if (mine.before(other) != want_first) mine = other;   // (equal entries are the same)
}
template <typename Entry>
__device__ __forceinline__ void sort_lanes(Entry& mine, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int mask = size >> 1; mask > 0; mask >>= 1) exchange(mine, mask, ((lane & size) == 0) == ((lane & mask) == 0));
}
// The first 32 of two lists in order.
template <typename Entry>
__device__ __forceinline__ void merge_lanes(Entry& mine, const Entry& theirs, int lane) {
    const Entry turned = theirs.from(31 - lane);
    if (turned.before(mine)) mine = turned;
#pragma unroll
    for (int mask = 16; mask > 0; mask >>= 1) exchange(mine, mask, (lane & mask) == 0);
}

__device__ __forceinline__ float power_of_two(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Vectors first, first + 32, ... of a row that starts `before` elements behind a 16-byte boundary; what lies past its end is -inf.
// Nothing outside the row is read (`first` is not negative): vectors whose aligned halves are not all the row's come element by element.
template <typename T, int R>
__device__ __forceinline__ void load_vectors(Pack<T, 16 / sizeof(T)> (&held)[R], const T* row, int first, int before, int length) {
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
    const int64_t last = static_cast<int64_t>(first + (R - 1) * 32 + 1) * VE;   // behind this lane's last vector
    if (before == 0 && last <= length) {
#pragma unroll
        for (int j = 0; j < R; ++j) held[j] = *reinterpret_cast<const Pack<T, VE>*>(row + static_cast<int64_t>(first + j * 32) * VE);
        return;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int64_t at = static_cast<int64_t>(first + j * 32) * VE;
        if (before != 0 && at > 0 && at + 2 * VE - before <= length) {
            const uint4* halves = reinterpret_cast<const uint4*>(row + at - before);
            *reinterpret_cast<uint4*>(&held[j]) = shifted(halves[0], halves[1], before * static_cast<int>(sizeof(T)));
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) held[j].v[i] = at + i < length ? row[at + i] : narrow<T>(-INFINITY);
        }
    }
}

// (One copy: instructions that a warp runs once are waited for. 7 x 5 beams over 50001 f32 tokens 10.1 us, with a copy in each place 10.6.)
template <typename T>
__device__ __noinline__ uint4 one_vector(const T* row, int vector, int before, int length) {
    Pack<T, 16 / sizeof(T)> own[1];
    load_vectors<T, 1>(own, row, vector, before, length);
    return *reinterpret_cast<const uint4*>(&own[0]);
}

// A key into a list in order, where it belongs; the last of 32 falls out.
__device__ __forceinline__ void insert(Key& list, uint64_t key, int lane) {
    const int place = __popc(__ballot_sync(0xffffffffu, list.key > key));
    const uint64_t above = __shfl_up_sync(0xffffffffu, list.key, 1);
    list.key = lane < place ? list.key : lane == place ? key : above;
}

// The largest of R vectors' values; a NaN is left out (the sum has it).
template <typename T, int R>
__device__ __forceinline__ float largest_of(const Pack<T, 16 / sizeof(T)> (&v)[R]) {
    if constexpr (sizeof(T) == 4) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, v[j].v[i]);
        return most;
    } else {
        using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        Two most = reinterpret_cast<const Two*>(&v[0])[0];
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = __hmax2(most, reinterpret_cast<const Two*>(&v[j])[i]);
        return fmaxf(fmaxf(widen(most.x), widen(most.y)), -INFINITY);
    }
}

constexpr int kScanVectors = 4;   // of a lane and block
template <typename T> constexpr int kVector = 16 / static_cast<int>(sizeof(T));
// Vector `number` of a lane, counted from the row's beginning; `first`: the part's first.
__device__ __forceinline__ int vector_at(int first, int number, int lane) { return first + (number / kScanVectors) * (32 * kScanVectors) + (number % kScanVectors) * 32 + lane; }

// The lanes' values in falling order.
__device__ __forceinline__ float in_order(float v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int mask = size >> 1; mask > 0; mask >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, v, mask);
            v = ((lane & size) == 0) == ((lane & mask) == 0) ? fmaxf(v, other) : fminf(v, other);
        }
    return v;
}

// A lane's vector of the row, and what it may add to a list: values above `least`, or equal to it and below `last_token`.
template <typename T>
struct Look {
    static constexpr int kValues = kVector<T>;
    uint4 words;
    int vector;
    __device__ __forceinline__ float value(int i) const {   // (`i` the same in all lanes, or known)
        const int place = i * static_cast<int>(sizeof(T)) / 4;
        const uint32_t word = place < 2 ? (place == 0 ? words.x : words.y) : (place == 2 ? words.z : words.w);
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(word);
        } else {
            const uint16_t half = static_cast<uint16_t>(i & 1 ? word >> 16 : word);
            return widen(*reinterpret_cast<const T*>(&half));
        }
    }
};

// A CTA's candidates.
template <int WARPS>
struct Found {
    uint64_t candidates[kCandidates];
    uint32_t first_equals[WARPS][kMaxBeams];
    int equals[WARPS], count;
    uint8_t lanes[WARPS][32];
    __device__ __forceinline__ void add(float value, uint32_t token) {
        const int at = atomicAdd(&count, 1);   // (in any order: they are sorted)
        if (at < kCandidates) candidates[at] = static_cast<uint64_t>(ordered(value)) << 32 | ~token;
    }
    template <typename L>
    __device__ __forceinline__ void take(const L& own, float bound, int vocabulary) {
        if (own.vector < 0) return;
        const uint32_t token = static_cast<uint32_t>(own.vector) * L::kValues;
#pragma unroll
        for (int i = 0; i < L::kValues; ++i) {
            const float x = own.value(i);
            if (x >= bound && token + i < static_cast<uint32_t>(vocabulary)) add(x, token + i);
        }
    }
};
// Where too many values equal the bound (masks, equal logits) for the candidates' room: what passes it, and of the equals each warp's first W, of which the first W of all are taken.
// By all threads; the candidates are complete when it returns. (16 x 8 beams over 128000 tokens, all but five masked: 20 us; value by value through the list 48.)
template <typename T, int WARPS>
__device__ __noinline__ void collect_again(Found<WARPS>& found, const T* logits, int first_vector, int of_lane, int before, int vocabulary, int beams, float largest, float least) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto look = [&](int whose, int number) {
        const bool there = number < of_lane;
        const int vector = vector_at(first_vector, there ? number : 0, whose);
        return Look<T>{one_vector(logits, vector, before, there ? vocabulary : 0), there ? vector : -1};
    };
    __syncthreads();   // (all have seen the count)
    if (threadIdx.x == 0) found.count = 0;
    int equal = 0;
#pragma unroll 1
    for (int number = 0; number < of_lane && equal < beams; ++number) {   // (a warp's tokens in their order)
        const Look<T> own = look(lane, number);
        const uint32_t token = static_cast<uint32_t>(own.vector) * Look<T>::kValues;
        uint32_t equals = 0;
#pragma unroll
        for (int i = 0; i < Look<T>::kValues; ++i) equals |= static_cast<uint32_t>(own.value(i) == least && token + i < static_cast<uint32_t>(vocabulary)) << i;
        int upto = __popc(equals);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += below;
        }
        for (int at = equal + upto - __popc(equals); equals != 0 && at < beams; ++at, equals &= equals - 1) found.first_equals[warp][at] = token + __ffs(static_cast<int>(equals)) - 1;
        equal += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) found.equals[warp] = min(equal, beams);
    __syncthreads();
    const int before_own = __reduce_add_sync(0xffffffffu, lane < warp ? found.equals[lane] : 0);
    if (lane < min(beams - before_own, found.equals[warp])) found.add(least, found.first_equals[warp][lane]);
    const float bound = from_ordered(ordered(least) + 1);   // (the next value; a NaN behind infinity, which none reaches)
    for (uint32_t lanes = __ballot_sync(0xffffffffu, largest >= bound); lanes != 0; lanes &= lanes - 1) {
#pragma unroll 1
        for (int from = 0; from < of_lane; from += 32) found.take(look(__ffs(static_cast<int>(lanes)) - 1, from + lane), bound, vocabulary);
        if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&found.count) > kCandidates)) break;   // (all lanes or none)
    }
    __syncthreads();
}

template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 32 / WARPS)
beam_scan_kernel(const ScanArgs a) {
    constexpr int VE = kVector<T>, R = kScanVectors;
    __shared__ float largest_of_warp[WARPS][32];
    __shared__ double whole_of_warp[WARPS];
    __shared__ float reference_of_warp[WARPS];
    __shared__ Found<WARPS> found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Logits& l = a.logits;
    const int row = static_cast<int>(fast_divide(blockIdx.x, a.by_parts)), part = static_cast<int>(blockIdx.x) - row * l.parts;
    const int entry = static_cast<int>(fast_divide(static_cast<uint32_t>(row), a.by_beams)), beam = row - entry * l.beams;
    if (threadIdx.x == 0) found.count = 0;
    chain_begin();
    const bool done = a.finished.data && a.finished.at(entry, beam) != 0;   // (on its way with the first logits)
    const bool divides = part == 0 && a.lengths.data && a.length_penalty != 0.0f;
    const T* logits = static_cast<const T*>(l.data) + entry * l.batch_stride + beam * l.beam_stride;
    // A lane's logits depend on their numbers alone, wherever the row starts, so that equal rows have equal sums.
    const int before = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
    const int of_lane = l.blocks * R, first_vector = (part * WARPS + warp) * of_lane * 32;
    Pack<T, VE> held[R], next[R];
    load_vectors<T, R>(held, logits, first_vector + lane, before, l.vocabulary);
    if (done) {
        if (divides && threadIdx.x == 0) l.sums[blockIdx.x].divisor = divisor_of(a.lengths.at(entry, beam), true, a.length_penalty);
        return;
    }
    float reference = 0.0f, largest = -INFINITY;   // reference: what exponentials are taken against, once there is `some` value
    bool some = false;
    uint64_t sums = 0;                             // of two halves, at most 64 terms each, before they go into `whole`
    double whole = 0.0;
    auto add_up = [&] {
        float one, two;
        unpack2(sums, one, two);
        whole += static_cast<double>(one) + static_cast<double>(two);
        sums = 0;
    };
#pragma unroll 1
    for (int block = 0; block < l.blocks; ++block) {
        if (block + 1 < l.blocks) load_vectors<T, R>(next, logits, first_vector + (block + 1) * (32 * R) + lane, before, l.vocabulary);
        largest = fmaxf(largest, largest_of<T, R>(held));
        if (__any_sync(0xffffffffu, largest > (some ? reference : -INFINITY))) {
            const float top = from_ordered(__reduce_max_sync(0xffffffffu, ordered(largest)));
            if (some) {
                add_up();
                whole *= static_cast<double>(power_of_two((reference - top) * kLog2e));
            }
            reference = top;
            some = true;
        }
        const uint64_t away = pack2(-reference, -reference), by = pack2(kLog2e, kLog2e);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < VE; i += 2) {
                float lo, hi;
                unpack2(mul2(add2(pack2(widen(held[j].v[i]), widen(held[j].v[i + 1])), away), by), lo, hi);
                sums = add2(sums, pack2(power_of_two(lo), power_of_two(hi)));
            }
        if ((block & 3) == 3) add_up();
#pragma unroll
        for (int j = 0; j < R; ++j) held[j] = next[j];
    }
    add_up();
    for (int o = 16; o > 0; o >>= 1) whole += __shfl_xor_sync(0xffffffffu, whole, o);
    largest_of_warp[warp][lane] = largest;
    if (lane == 0) {
        whole_of_warp[warp] = whole;
        reference_of_warp[warp] = some ? reference : -INFINITY;
    }
    __syncthreads();
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) most = fmaxf(most, largest_of_warp[w][lane]);
    most = in_order(most, lane);
    float least = __shfl_sync(0xffffffffu, most, l.beams - 1);
    auto look = [&](int of_warp, int whose, int number) {
        const bool there = number < of_lane;
        const int vector = vector_at((part * WARPS + of_warp) * of_lane * 32, there ? number : 0, whose);
        return Look<T>{one_vector(logits, vector, before, there ? l.vocabulary : 0), there ? vector : -1};
    };
    // (Loops that are not unrolled: a warp comes by here once, and instructions that are run once are waited for.)
    // The lanes that reach the bound have their vectors looked through side by side, 32 at a time.
    const uint32_t lanes = __ballot_sync(0xffffffffu, largest >= least);
    if (largest >= least) found.lanes[warp][__popc(lanes & ((1u << lane) - 1))] = static_cast<uint8_t>(lane);
    __syncwarp();
    int vectors = __popc(lanes) * of_lane;
    if (lanes == 0xffffffffu) {   // (masks, equal logits: the second turn's)
        vectors = 0;
        if (lane == 0) atomicAdd(&found.count, kCandidates + 1);
    }
#pragma unroll 1
    for (int from = 0; from < vectors; from += 32) {
        const int place = (from + lane) / of_lane;
        const bool there = from + lane < vectors;
        found.take(look(warp, there ? found.lanes[warp][place] : 0, there ? from + lane - place * of_lane : of_lane), least, l.vocabulary);
        if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&found.count) > kCandidates)) break;   // (all lanes or none)
    }
    __syncthreads();
    if (__builtin_expect(found.count > kCandidates, 0)) collect_again<T, WARPS>(found, logits, first_vector, of_lane, before, l.vocabulary, l.beams, largest, least);
    if (warp == 1) {
        // the warps' sums against the CTA's largest value (a warp of -inf alone has no reference that means anything)
        const float own_reference = lane < WARPS ? reference_of_warp[lane] : -INFINITY;
        const float top = __shfl_sync(0xffffffffu, most, 0);
        const double own_whole = lane < WARPS ? whole_of_warp[lane] : 0.0;
        double sum = own_whole == 0.0 ? 0.0 : own_whole * (own_reference == top || own_reference == -INFINITY ? 1.0 : exp(static_cast<double>(own_reference) - static_cast<double>(top)));
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            l.sums[blockIdx.x].sum = sum;
            l.sums[blockIdx.x].most = top;
        }
    }
    if (warp == 2 && lane == 0 && divides) l.sums[blockIdx.x].divisor = divisor_of(a.lengths.at(entry, beam), false, a.length_penalty);   // (a power takes as long as the sort)
    if (warp != 0) return;
    Key list{0};
    if (found.count <= kCandidates) {
#pragma unroll 1
        for (int from = 0; from < found.count; from += 32) {
            Key more{from + lane < found.count ? found.candidates[from + lane] : 0};
            sort_lanes(more, lane);
            if (from == 0) list = more;
            else merge_lanes(list, more, lane);
        }
    } else {
        // Many that pass the bound, all in few lanes: one after another. The list fills up with the lowest tokens, and vectors behind them are no candidates any more.
        uint32_t last_token = 0xffffffffu;
        uint64_t bound = static_cast<uint64_t>(ordered(least)) << 32;
#pragma unroll 1
        for (int w = 0; w < WARPS; ++w) {
            const float value = largest_of_warp[w][lane];
            const uint32_t first_token = static_cast<uint32_t>((part * WARPS + w) * of_lane * 32 + lane) * VE;
#pragma unroll 1
            for (uint32_t lanes = __ballot_sync(0xffffffffu, value > least || (value == least && first_token < last_token)); lanes != 0; lanes &= lanes - 1) {
#pragma unroll 1
                for (int from = 0; from < of_lane; from += 32) {
                    const Look<T> own = look(w, __ffs(static_cast<int>(lanes)) - 1, from + lane);
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < VE; ++i) top = fmaxf(top, own.value(i));
                    const bool reaches = own.vector >= 0 && (top > least || (top == least && static_cast<uint32_t>(own.vector) * VE < last_token));
#pragma unroll 1
                    for (uint32_t reaching = __ballot_sync(0xffffffffu, reaches); reaching != 0; reaching &= reaching - 1) {
                        const int source = __ffs(static_cast<int>(reaching)) - 1;
                        const uint32_t token = static_cast<uint32_t>(__shfl_sync(0xffffffffu, own.vector, source)) * VE;
#pragma unroll 1
                        for (int i = 0; i < VE; ++i) {
                            const float x = __shfl_sync(0xffffffffu, own.value(i), source);
                            const uint64_t key = static_cast<uint64_t>(ordered(x)) << 32 | ~(token + i);
                            if (!(x >= least) || key <= bound || token + i >= static_cast<uint32_t>(l.vocabulary)) continue;
                            insert(list, key, lane);
                            const uint64_t last = list.from(l.beams - 1).key;
                            if (last > bound) {
                                bound = last;
                                least = from_ordered(static_cast<uint32_t>(bound >> 32));
                                last_token = ~static_cast<uint32_t>(bound);
                            }
                        }
                    }
                }
            }
        }
    }
    if (lane < l.beams) l.keys[static_cast<int64_t>(blockIdx.x) * l.beams + lane] = list.key;
}

struct MergeArgs {
    Logits logits;
    const float* scores;
    float* scores_out;
    int64_t scores_batch, scores_beam, out_batch, out_beam;
    Ints finished, lengths, tokens, parents, finished_out, lengths_out;
    int32_t* forks;
    int32_t end, pad, source_base, target_base;
    float length_penalty;
};

__global__ void __launch_bounds__(32 * kMaxBeams)
beam_merge_kernel(const MergeArgs a) {
    __shared__ uint64_t keys[kMaxBeams][32];
    __shared__ uint32_t places[kMaxBeams][32];
    __shared__ double divisors[kMaxBeams];
    __shared__ int32_t finished[kMaxBeams], lengths[kMaxBeams];
    const int entry = static_cast<int>(blockIdx.x), beam = threadIdx.x >> 5, lane = threadIdx.x & 31;   // (as many warps as beams)
    const Logits& l = a.logits;
    const int64_t first = (static_cast<int64_t>(entry) * l.beams + beam) * l.parts;
    chain_begin();
    // All that most rows need is on its way at once. (Of a finished beam it is whatever the scratch held.)
    const float score = a.scores[entry * a.scores_batch + beam * a.scores_beam];
    const bool done = a.finished.data && a.finished.at(entry, beam) != 0;
    int64_t length = a.lengths.data ? static_cast<int64_t>(a.lengths.at(entry, beam)) + (done ? 0 : 1) : 1;
    constexpr int kAhead = 8;
    uint64_t ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = i < l.parts && lane < l.beams ? l.keys[(first + i) * l.beams + lane] : 0;
    PartSum sums = lane < l.parts ? l.sums[first + lane] : PartSum{0.0, 1.0, 0.0f};
    const bool divides = a.lengths.data && a.length_penalty != 0.0f;
    const double divisor = divides ? __shfl_sync(0xffffffffu, sums.divisor, 0) : 1.0;
    Key list{ahead[0]};
    if (!done) {
#pragma unroll 1
        for (int from = 0; from < l.parts; from += kAhead) {
            if (from > 0) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) ahead[i] = from + i < l.parts && lane < l.beams ? l.keys[(first + from + i) * l.beams + lane] : 0;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (from + i > 0 && from + i < l.parts && __shfl_sync(0xffffffffu, ahead[i], 0) > list.from(l.beams - 1).key) merge_lanes(list, Key{ahead[i]}, lane);
        }
    }
    Place mine{0, 0xffffffffu};
    {
        length = min(max(length, static_cast<int64_t>(1)), static_cast<int64_t>(0x7fffffff));
        const bool alive = isfinite(score);
        const uint32_t row = static_cast<uint32_t>(beam) * static_cast<uint32_t>(l.vocabulary);
        if (done) {
            if (lane == 0) mine = Place{ordered(!alive ? -static_cast<double>(INFINITY) : divides ? static_cast<double>(score) / divisor : static_cast<double>(score)), row + static_cast<uint32_t>(a.pad)};
        } else {
            for (int from = 32; from < l.parts; from += 32) {   // a lane's parts against the largest of them
                const PartSum more = from + lane < l.parts ? l.sums[first + from + lane] : PartSum{0.0, 1.0, 0.0f};
                if (more.sum == 0.0) continue;   // (of -inf alone: its reference means nothing)
                const float top = sums.sum != 0.0 ? fmaxf(sums.most, more.most) : more.most;
                sums.sum = (sums.sum != 0.0 ? sums.sum * exp(static_cast<double>(sums.most) - static_cast<double>(top)) : 0.0) + more.sum * exp(static_cast<double>(more.most) - static_cast<double>(top));
                sums.most = top;
            }
            float most = sums.sum != 0.0 ? sums.most : -INFINITY;
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            double sum = sums.sum != 0.0 ? sums.sum * (sums.most == most ? 1.0 : exp(static_cast<double>(sums.most) - static_cast<double>(most))) : 0.0;
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const double normaliser = static_cast<double>(most) + log(sum);
            if (!alive || !isfinite(normaliser)) {   // all continuations at -inf
                if (lane < l.vocabulary) mine = Place{ordered(-static_cast<double>(INFINITY)), row + static_cast<uint32_t>(lane)};
            } else if (list.key != 0) {
                const double logit = static_cast<double>(from_ordered(static_cast<uint32_t>(list.key >> 32)));
                const double worth = static_cast<double>(score) + (logit - normaliser);
                mine = Place{ordered(divides ? worth / divisor : worth), row + ~static_cast<uint32_t>(list.key)};
            }
            if (lane >= l.beams) mine = Place{0, 0xffffffffu};
            // (equal worths of different logits, where 64 bits do not tell them apart, may be out of order)
            const Place above{__shfl_up_sync(0xffffffffu, mine.key, 1), __shfl_up_sync(0xffffffffu, mine.place, 1)};
            if (__any_sync(0xffffffffu, lane > 0 && mine.before(above))) sort_lanes(mine, lane);
        }
        keys[beam][lane] = mine.key;
        places[beam][lane] = mine.place;
        if (lane == 0) {
            divisors[beam] = divisor;
            finished[beam] = done;
            lengths[beam] = static_cast<int32_t>(length);
        }
    }
    __syncthreads();
    for (int step = 1; step < l.beams; step <<= 1) {
        if ((beam & (2 * step - 1)) == 0 && beam + step < l.beams) {
            merge_lanes(mine, Place{keys[beam + step][lane], places[beam + step][lane]}, lane);
            keys[beam][lane] = mine.key;
            places[beam][lane] = mine.place;
        }
        __syncthreads();
    }
    if (beam != 0 || lane >= l.beams) return;
    const int parent = static_cast<int>(mine.place / static_cast<uint32_t>(l.vocabulary)), token = static_cast<int>(mine.place - static_cast<uint32_t>(parent) * static_cast<uint32_t>(l.vocabulary));
    a.scores_out[entry * a.out_batch + lane * a.out_beam] = static_cast<float>(double_from_ordered(mine.key) * divisors[parent]);
    a.tokens.at(entry, lane) = token;
    a.parents.at(entry, lane) = parent;
    if (a.finished_out.data) a.finished_out.at(entry, lane) = finished[parent] || (a.end >= 0 && token == a.end) ? 1 : 0;
    if (a.lengths_out.data) a.lengths_out.at(entry, lane) = lengths[parent];
    if (a.forks) {
        int32_t* pair = a.forks + 2 * (static_cast<int64_t>(entry) * l.beams + lane);
        pair[0] = a.source_base + entry * l.beams + parent;
        pair[1] = a.target_base + entry * l.beams + lane;
    }
}

// ---- states ------------------------------------------------------------------------------------

constexpr int kSegmentVectors = 8;   // of a lane: a warp moves 32 x 8 vectors of a row
struct StateSide {
    const uint8_t* source;
    uint8_t* target;
    int64_t source_stride[3], target_stride[3];   // layer, entry, beam, in bytes
    int64_t row_bytes;
    int32_t width, first_unit;                    // bytes of a vector; the state's first unit
    FastDivisor by_segments;
};
struct ReorderArgs {
    const int32_t* parents;
    int64_t parent_batch, parent_beam;
    int32_t beams, count;
    int64_t units;
    FastDivisor by_beams, by_entries;
    StateSide state[DFGPU_BEAM_MAX_STATES];
};

template <typename V>
__device__ __forceinline__ void copy_segment(const uint8_t* from, uint8_t* to, int64_t first, int64_t vectors, int lane) {
    const V* source = reinterpret_cast<const V*>(from);
    V* target = reinterpret_cast<V*>(to);
    V held[kSegmentVectors];
#pragma unroll
    for (int j = 0; j < kSegmentVectors; ++j)
        if (first + lane + 32 * j < vectors) held[j] = source[first + lane + 32 * j];
#pragma unroll
    for (int j = 0; j < kSegmentVectors; ++j)
        if (first + lane + 32 * j < vectors) target[first + lane + 32 * j] = held[j];
}

__global__ void __launch_bounds__(256)
beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    chain_begin();
    if (unit >= a.units) return;
    int which = 0;
    while (which + 1 < a.count && unit >= a.state[which + 1].first_unit) ++which;
    const StateSide& s = a.state[which];
    const uint32_t local = static_cast<uint32_t>(unit - s.first_unit);
    const uint32_t row = fast_divide(local, s.by_segments), segment = local - row * s.by_segments.divisor;
    const uint32_t rest = fast_divide(row, a.by_beams), beam = row - rest * a.by_beams.divisor;
    const uint32_t layer = fast_divide(rest, a.by_entries), entry = rest - layer * a.by_entries.divisor;
    const int parent = a.parents[entry * a.parent_batch + beam * a.parent_beam];
    if (parent < 0 || parent >= a.beams) return;
    const uint8_t* from = s.source + layer * s.source_stride[0] + entry * s.source_stride[1] + parent * s.source_stride[2];
    uint8_t* to = s.target + layer * s.target_stride[0] + entry * s.target_stride[1] + beam * s.target_stride[2];
    const int64_t first = static_cast<int64_t>(segment) * (32 * kSegmentVectors), vectors = s.row_bytes / s.width;
    if (s.width == 16) copy_segment<uint4>(from, to, first, vectors, lane);
    else if (s.width == 8) copy_segment<uint2>(from, to, first, vectors, lane);
    else if (s.width == 4) copy_segment<uint32_t>(from, to, first, vectors, lane);
    else if (s.width == 2) copy_segment<uint16_t>(from, to, first, vectors, lane);
    else copy_segment<uint8_t>(from, to, first, vectors, lane);
}

// ---- host -----------------------------------------------------------------------------------------

int check_beams(const dfgpu_tensor& t, const dfgpu_beam_select_params& p, int dtype, const char* name, bool output) {
    if (!valid_tensor(t) || t.rank != 2 || t.dim[0] != p.logits.dim[0] || t.dim[1] != p.logits.dim[1]) return fail(kInvalidShape, "BEAM_SELECT: %s must be [B, W]", name);
    if (t.dtype != dtype) return fail(kUnsupported, "BEAM_SELECT: %s must be %s", name, dtype == DFGPU_F32 ? "FLOAT" : "INT32");
    if (output && overlaps_itself(t)) return fail(kInvalidLayout, "BEAM_SELECT: %s overlaps itself", name);
    return kOk;
}

struct SelectCut {
    int64_t parts, blocks;   // of a row; of a part
    int warps;               // of a CTA
};
int check_select(const dfgpu_beam_select_params& p, SelectCut& cut) {
    if (!valid_tensor(p.logits) || p.logits.rank != 3) return fail(kInvalidShape, "BEAM_SELECT: logits must be [B, W, V] with positive extents");
    if (p.logits.dtype != DFGPU_F32 && p.logits.dtype != DFGPU_F16 && p.logits.dtype != DFGPU_BF16) return fail(kUnsupported, "BEAM_SELECT: logits must be FLOAT, HALF or BFLOAT16");
    if (p.logits.dim[2] > 1 && p.logits.stride[2] != 1) return fail(kInvalidLayout, "BEAM_SELECT: the vocabulary must have unit stride");
    if (p.logits.dim[1] > kMaxBeams) return fail(kUnsupported, "BEAM_SELECT: more than %d beams", kMaxBeams);
    if (p.logits.dim[2] >= (1ll << 26) || p.logits.dim[0] >= (1ll << 24)) return fail(kUnsupported, "BEAM_SELECT: too many tokens or entries");
    int status = check_beams(p.scores, p, DFGPU_F32, "scores", false);
    if (!status) status = check_beams(p.scores_out, p, DFGPU_F32, "scores_out", true);
    if (!status) status = check_beams(p.tokens, p, DFGPU_I32, "tokens", true);
    if (!status) status = check_beams(p.parents, p, DFGPU_I32, "parents", true);
    if (!status && p.finished.rank) status = check_beams(p.finished, p, DFGPU_I32, "finished", false);
    if (!status && p.lengths.rank) status = check_beams(p.lengths, p, DFGPU_I32, "lengths", false);
    if (!status && p.finished_out.rank) status = check_beams(p.finished_out, p, DFGPU_I32, "finished_out", true);
    if (!status && p.lengths_out.rank) status = check_beams(p.lengths_out, p, DFGPU_I32, "lengths_out", true);
    if (status) return status;
    if (p.lengths_out.rank && !p.lengths.rank) return fail(kInvalidArgument, "BEAM_SELECT: lengths_out without lengths");
    // (n^28 is at most 2^868: what f32 scores are over it and times it stays within 64 bits, where worths are compared and scores come back from them)
    if (p.lengths.rank && !(std::fabs(p.length_penalty) <= kMaxPenalty)) return fail(kInvalidValue, "BEAM_SELECT: the length penalty must be within -28 and 28");
    if (p.finished.rank && (p.pad < 0 || p.pad >= p.logits.dim[2])) return fail(kInvalidValue, "BEAM_SELECT: pad is no token");
    const int64_t rows = p.logits.dim[0] * p.logits.dim[1];
    if (p.forks.rank) {
        if (!valid_tensor(p.forks) || p.forks.rank != 2 || p.forks.dim[0] != rows || p.forks.dim[1] != 2 || p.forks.dtype != DFGPU_I32) return fail(kInvalidShape, "BEAM_SELECT: forks must be INT32 [B * W, 2]");
        if (!is_packed_row_major(p.forks)) return fail(kInvalidLayout, "BEAM_SELECT: forks must be packed");
        if (p.source_base < 0 || p.target_base < 0 || p.source_base + rows > 0x7fffffff || p.target_base + rows > 0x7fffffff) return fail(kInvalidValue, "BEAM_SELECT: sequence numbers out of range");
    }
    // A block a warp, up to 32 warps for every SM, which run at once; then more blocks (16 x 8 beams, 128000 bf16 logits: 19.0 us; up to four CTAs of 16 warps 21.5, eight 28.8).
    const int64_t values = 32 * kScanVectors * (16 / dtype_bytes(p.logits.dtype)), blocks = (p.logits.dim[2] + values - 1) / values;
    // Sixteen warps a CTA; four where the rows are more than two CTAs an SM, whose second look and sorts then run under the others' loads (45 x 8 beams, 20001 bf16 logits: 22.9 us and 16.6;
    // 26 x 12, 306 f32 ones 13.8 and 9.0), or short (2 x 15, 2024 f16 ones 10.1 and 9.4). With 256 rows of 32000 sixteen are the quicker, 13.5 and 15.3, with 7 x 5 of 50001 11.1 and 14.0.
    cut.warps = rows > 2 * 148 || blocks <= 4 ? 4 : 16;
    cut.blocks = 1;
    while (cut.parts = (blocks + cut.warps * cut.blocks - 1) / (cut.warps * cut.blocks), cut.parts > 1 && rows * cut.parts > 32 / cut.warps * 148) ++cut.blocks;
    if (rows * cut.parts >= (1ll << 31)) return fail(kUnsupported, "BEAM_SELECT: too many tokens or entries");
    return kOk;
}
int64_t select_scratch(const dfgpu_beam_select_params& p, const SelectCut& cut) { return p.logits.dim[0] * p.logits.dim[1] * cut.parts * (static_cast<int64_t>(sizeof(PartSum)) + 8 * p.logits.dim[1]); }

int check_reorder(const dfgpu_beam_reorder_params& p) {
    if (!valid_tensor(p.parents) || p.parents.rank != 2) return fail(kInvalidShape, "BEAM_REORDER: parents must be [B, W] with positive extents");
    if (p.parents.dtype != DFGPU_I32) return fail(kUnsupported, "BEAM_REORDER: parents must be INT32");
    if (p.count < 1 || p.count > DFGPU_BEAM_MAX_STATES) return fail(kInvalidArgument, "BEAM_REORDER: 1 to %d states", DFGPU_BEAM_MAX_STATES);
    if (p.parents.dim[0] >= (1ll << 31) || p.parents.dim[1] >= (1ll << 31)) return fail(kUnsupported, "BEAM_REORDER: too many beams");
    int64_t units = 0;
    for (int i = 0; i < p.count; ++i) {
        const dfgpu_tensor &s = p.source[i], &t = p.target[i];
        if (!valid_tensor(s) || !valid_tensor(t) || s.rank != 4 || t.rank != 4 || s.dim[1] != p.parents.dim[0] || s.dim[2] != p.parents.dim[1])
            return fail(kInvalidShape, "BEAM_REORDER: state %d must be [layers, B, W, n]", i);
        for (int d = 0; d < 4; ++d)
            if (s.dim[d] != t.dim[d]) return fail(kInvalidShape, "BEAM_REORDER: source and target %d differ in extent", i);
        if (s.dtype != t.dtype) return fail(kUnsupported, "BEAM_REORDER: source and target %d differ in type", i);
        if (s.dtype == DFGPU_FP4 || s.dtype == DFGPU_I4 || s.dtype < 0 || s.dtype > DFGPU_I8) return fail(kUnsupported, "BEAM_REORDER: state %d must be of whole bytes", i);
        if (s.dim[3] > 1 && (s.stride[3] != 1 || t.stride[3] != 1)) return fail(kInvalidLayout, "BEAM_REORDER: the rows of state %d must be contiguous", i);
        if (overlaps_itself(t)) return fail(kInvalidLayout, "BEAM_REORDER: target %d overlaps itself", i);
        if (s.dim[0] >= (1ll << 31) || s.dim[3] >= (1ll << 40)) return fail(kUnsupported, "BEAM_REORDER: state %d is too large", i);
        const double rows = static_cast<double>(s.dim[0]) * static_cast<double>(s.dim[1]) * static_cast<double>(s.dim[2]);
        if (rows * (static_cast<double>(s.dim[3]) * dtype_bytes(s.dtype) / 256.0 + 1.0) >= 2147483647.0) return fail(kUnsupported, "BEAM_REORDER: state %d is too large", i);   // (bytes one by one)
        units += static_cast<int64_t>(rows * (static_cast<double>(s.dim[3]) * dtype_bytes(s.dtype) / 256.0 + 1.0)) + 1;
    }
    if (units >= (1ll << 31)) return fail(kUnsupported, "BEAM_REORDER: the states are too large");
    return kOk;
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_beam_select(const dfgpu_beam_select_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "BEAM_SELECT: null params");
    SelectCut cut;
    const int status = check_select(*p, cut);
    if (status) return status;
    info->kernel = 0;
    info->launches = 2;
    info->scratch_bytes = select_scratch(*p, cut);
    return kOk;
}

extern "C" int dfgpu_beam_select(const dfgpu_beam_select_params* p, void* const* tensors, void* scratch, void* stream) {
    if (!p || !tensors) return fail(kInvalidArgument, "BEAM_SELECT: null params");
    SelectCut cut;
    int status = check_select(*p, cut);
    if (status) return status;
    const dfgpu_tensor* described[10] = {&p->logits, &p->scores, &p->finished, &p->lengths, &p->scores_out, &p->tokens, &p->parents, &p->finished_out, &p->lengths_out, &p->forks};
    void* port[10];
    Region regions[10];
    for (int i = 0; i < 10; ++i) {
        port[i] = described[i]->rank ? tensors[i] : nullptr;
        if (described[i]->rank && !port[i]) return fail(kInvalidArgument, "BEAM_SELECT: port %d is null", i);
        if (!aligned(port[i], i == 0 ? dtype_bytes(p->logits.dtype) : 4)) return fail(kInvalidArgument, "BEAM_SELECT: port %d is not aligned to its type", i);
        regions[i] = region_of(port[i], *described[i]);
    }
    if (!scratch || !aligned(scratch, 16)) return fail(kInvalidArgument, "BEAM_SELECT: scratch is needed, on a 16-byte boundary");
    for (int o = 4; o < 10; ++o) {
        if (!port[o]) continue;
        for (int i = 0; i < 10; ++i) {
            if (i == o) continue;
            const bool own = (o == 4 && i == 1) || (o == 7 && i == 2) || (o == 8 && i == 3);   // (may be its input)
            if (own && port[i] == port[o]) {
                for (int d = 0; d < 2; ++d)
                    if (described[i]->dim[d] > 1 && described[i]->stride[d] != described[o]->stride[d]) return fail(kInvalidLayout, "BEAM_SELECT: in place, input and output have the same strides");
            } else if (overlaps(regions[o], regions[i])) {
                return fail(kInvalidArgument, "BEAM_SELECT: port %d overlaps port %d", o, i);
            }
        }
    }
    const int64_t entries = p->logits.dim[0], beams = p->logits.dim[1], units = entries * beams * cut.parts;
    ScanArgs s{};
    s.logits.data = port[0];
    s.logits.batch_stride = p->logits.stride[0];
    s.logits.beam_stride = p->logits.stride[1];
    s.logits.beams = static_cast<int>(beams);
    s.logits.vocabulary = static_cast<int>(p->logits.dim[2]);
    s.logits.parts = static_cast<int>(cut.parts);
    s.logits.blocks = static_cast<int>(cut.blocks);
    s.logits.sums = static_cast<PartSum*>(scratch);
    s.logits.keys = reinterpret_cast<uint64_t*>(s.logits.sums + units);
    auto ints = [&](int i) {
        return Ints{static_cast<int32_t*>(port[i]), port[i] ? described[i]->stride[0] : 0, port[i] ? described[i]->stride[1] : 0};
    };
    s.finished = ints(2);
    s.lengths = ints(3);
    s.length_penalty = p->length_penalty;
    s.by_parts = make_fast_divisor(static_cast<uint32_t>(cut.parts));
    s.by_beams = make_fast_divisor(static_cast<uint32_t>(beams));
    cudaStream_t on = as_stream(stream);
    const dim3 grid(static_cast<unsigned>(units)), block(static_cast<unsigned>(32 * cut.warps));
    void (*scan)(const ScanArgs) = beam_scan_kernel<__nv_bfloat16, 16>;
    if (p->logits.dtype == DFGPU_F32) scan = cut.warps == 4 ? beam_scan_kernel<float, 4> : beam_scan_kernel<float, 16>;
    else if (p->logits.dtype == DFGPU_F16) scan = cut.warps == 4 ? beam_scan_kernel<__half, 4> : beam_scan_kernel<__half, 16>;
    else if (cut.warps == 4) scan = beam_scan_kernel<__nv_bfloat16, 4>;
    launch_chained(scan, grid, block, 0, on, s);
    status = check_launch("BEAM_SELECT");
    if (status) return status;
    MergeArgs m{};
    m.logits = s.logits;
    m.scores = static_cast<const float*>(port[1]);
    m.scores_batch = p->scores.stride[0];
    m.scores_beam = p->scores.stride[1];
    m.scores_out = static_cast<float*>(port[4]);
    m.out_batch = p->scores_out.stride[0];
    m.out_beam = p->scores_out.stride[1];
    m.finished = ints(2);
    m.lengths = ints(3);
    m.tokens = ints(5);
    m.parents = ints(6);
    m.finished_out = ints(7);
    m.lengths_out = ints(8);
    m.forks = static_cast<int32_t*>(port[9]);
    m.end = p->end;
    m.pad = p->pad;
    m.source_base = p->source_base;
    m.target_base = p->target_base;
    m.length_penalty = p->length_penalty;
    launch_chained(beam_merge_kernel, dim3(static_cast<unsigned>(entries)), dim3(static_cast<unsigned>(32 * beams)), 0, on, m);
    return check_launch("BEAM_SELECT, join");
}

extern "C" int dfgpu_query_beam_reorder(const dfgpu_beam_reorder_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "BEAM_REORDER: null params");
    const int status = check_reorder(*p);
    if (status) return status;
    info->kernel = 0;
    info->launches = 1;
    info->scratch_bytes = 0;
    return kOk;
}

extern "C" int dfgpu_beam_reorder(const dfgpu_beam_reorder_params* p, void* const* tensors, void* scratch, void* stream) {
    (void)scratch;
    if (!p || !tensors) return fail(kInvalidArgument, "BEAM_REORDER: null params");
    const int status = check_reorder(*p);
    if (status) return status;
    if (!tensors[0] || !aligned(tensors[0], 4)) return fail(kInvalidArgument, "BEAM_REORDER: parents are null or not aligned to their type");
    ReorderArgs a{};
    a.parents = static_cast<const int32_t*>(tensors[0]);
    a.parent_batch = p->parents.stride[0];
    a.parent_beam = p->parents.stride[1];
    a.beams = static_cast<int>(p->parents.dim[1]);
    a.count = p->count;
    a.by_beams = make_fast_divisor(static_cast<uint32_t>(p->parents.dim[1]));
    a.by_entries = make_fast_divisor(static_cast<uint32_t>(p->parents.dim[0]));
    for (int i = 0; i < p->count; ++i) {
        const dfgpu_tensor &s = p->source[i], &t = p->target[i];
        if (!tensors[1 + 2 * i] || !tensors[2 + 2 * i]) return fail(kInvalidArgument, "BEAM_REORDER: a tensor of state %d is null", i);
        const int bytes = dtype_bytes(s.dtype);
        StateSide& side = a.state[i];
        side.source = static_cast<const uint8_t*>(tensors[1 + 2 * i]);
        side.target = static_cast<uint8_t*>(tensors[2 + 2 * i]);
        side.row_bytes = s.dim[3] * bytes;
        side.width = 16;
        uint64_t places = reinterpret_cast<uintptr_t>(side.source) | reinterpret_cast<uintptr_t>(side.target) | static_cast<uint64_t>(side.row_bytes);
        for (int d = 0; d < 3; ++d) {
            side.source_stride[d] = s.dim[d] == 1 ? 0 : s.stride[d] * bytes;
            side.target_stride[d] = t.dim[d] == 1 ? 0 : t.stride[d] * bytes;
            places |= static_cast<uint64_t>(side.source_stride[d]) | static_cast<uint64_t>(side.target_stride[d]);
        }
        while (places & static_cast<uint64_t>(side.width - 1)) side.width /= 2;
        const int64_t segments = (side.row_bytes / side.width + 32 * kSegmentVectors - 1) / (32 * kSegmentVectors);
        side.by_segments = make_fast_divisor(static_cast<uint32_t>(segments));
        side.first_unit = static_cast<int32_t>(a.units);
        a.units += segments * s.dim[0] * s.dim[1] * s.dim[2];
    }
    for (int i = 0; i < p->count; ++i) {
        const Region target = region_of(tensors[2 + 2 * i], p->target[i]);
        if (overlaps(target, region_of(tensors[0], p->parents))) return fail(kInvalidArgument, "BEAM_REORDER: target %d overlaps the parents", i);
        for (int o = 0; o < p->count; ++o)
            if (overlaps(target, region_of(tensors[1 + 2 * o], p->source[o])) || (o != i && overlaps(target, region_of(tensors[2 + 2 * o], p->target[o]))))
                return fail(kInvalidArgument, "BEAM_REORDER: target %d overlaps another state", i);
    }
    launch_chained(beam_reorder_kernel, dim3(static_cast<unsigned>((a.units + 7) / 8)), dim3(256), 0, as_stream(stream), a);
    return check_launch("BEAM_REORDER");
}
