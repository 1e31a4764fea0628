// Beam search: the W best continuations of each batch entry over its beams and the vocabulary, and the states of the beams that go on.
//
// Selection, first kernel: the logits are read once, in chunks that a CTA holds in registers. Of 256 threads' largest values the W-th largest is a bound that W values
// reach at least, and no more than W threads hold values that reach it: those few are sorted. (Equals are told apart by the number of
// their 16-byte vector, so that this holds for constant rows too.) The exponentials are summed against the chunk's largest value, which is
// known by then and counts as 1 exactly: the log-probability of a token that has nearly all of it is no rounding's leftover.
// Second kernel: a CTA an entry. Each warp merges the lists of its beams' chunks, 32 lanes a list, and adds scores in 64 bits; one warp merges the beams.
//
// Reordering: a copy; HBM bounds it.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"

namespace dfgpu {
namespace {

constexpr int kScanThreads = 256, kScanWarps = kScanThreads / 32;
constexpr int kMaxBeams = 32;
constexpr float kLog2e = 1.44269504088896341f;

struct alignas(16) ChunkSum {
    double sum;                // of exp(x - most)
    float most, unused;
};
struct ScanArgs {
    const void* logits;
    const int32_t* finished;
    ChunkSum* sums;            // of a chunk
    uint64_t* keys;            // of a chunk: W, falling; 0: none
    int64_t batch_stride, beam_stride, finished_batch, finished_beam;
    int32_t beams, vocabulary, chunks;
    FastDivisor by_chunks, by_beams;
};

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

// The 16 bytes that start `shift` bytes (a multiple of 2 or 4) into two aligned vectors.
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, int shift) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int k = 0; k < 6; ++k) w[k] = shift & 8 ? w[k + 2] : w[k];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = shift & 4 ? w[k + 1] : w[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], (shift & 2) * 8);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Vectors first, first + kScanThreads, ... of a row that starts `before` elements behind a 16-byte boundary; what lies past its end is -inf.
// Nothing outside the row is read: vectors whose aligned halves are not all the row's come element by element.
template <typename T, int R>
__device__ __forceinline__ void load_vectors(Pack<T, 16 / sizeof(T)> (&held)[R], const T* row, int first, int before, int length) {
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int64_t at = static_cast<int64_t>(first + j * kScanThreads) * VE;
        if (before == 0 && at + VE <= length) {
            held[j] = *reinterpret_cast<const Pack<T, VE>*>(row + at);
        } else if (before != 0 && at > 0 && at + 2 * VE - before <= length) {
            const uint4* halves = reinterpret_cast<const uint4*>(row + at - before);
            *reinterpret_cast<uint4*>(&held[j]) = shifted(halves[0], halves[1], before * static_cast<int>(sizeof(T)));
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) held[j].v[i] = at + i < length ? row[at + i] : narrow<T>(-INFINITY);
        }
    }
}

// R vectors of 16 bytes a thread.
template <typename T, int R>
__global__ void __launch_bounds__(kScanThreads)
beam_scan_kernel(const ScanArgs a) {
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
    extern __shared__ uint64_t candidates[];            // W * R * VE
    __shared__ uint64_t best[kScanWarps * kMaxBeams];   // the largest of each warp's threads
    __shared__ uint64_t bound, top;
    __shared__ double partial[kScanWarps];
    __shared__ int count;
    const int row = static_cast<int>(fast_divide(blockIdx.x, a.by_chunks)), chunk = static_cast<int>(blockIdx.x) - row * a.chunks;
    const int entry = static_cast<int>(fast_divide(static_cast<uint32_t>(row), a.by_beams)), beam = row - entry * a.beams;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) count = 0;
    chain_begin();
    if (a.finished && a.finished[entry * a.finished_batch + beam * a.finished_beam] != 0) return;
    const T* logits = static_cast<const T*>(a.logits) + entry * a.batch_stride + beam * a.beam_stride;
    // A thread's logits depend on their numbers alone, wherever the row starts, so that equal rows have equal sums.
    const int before = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
    const int first_vector = chunk * (kScanThreads * R) + threadIdx.x;
    Pack<T, VE> held[R];
    float most[R], largest = -INFINITY;
    load_vectors<T, R>(held, logits, first_vector, before, a.vocabulary);
#pragma unroll
    for (int j = 0; j < R; ++j) {
        most[j] = -INFINITY;
#pragma unroll
        for (int i = 0; i < VE; ++i) most[j] = fmaxf(most[j], widen(held[j].v[i]));   // (a NaN is left out here; the sum has it)
        largest = fmaxf(largest, most[j]);
    }
    int vector = 0;
#pragma unroll
    for (int j = R - 1; j >= 0; --j)
        if (most[j] == largest) vector = first_vector + j * kScanThreads;
    Key mine{static_cast<uint64_t>(ordered(largest)) << 32 | ~static_cast<uint32_t>(vector)};
    sort_lanes(mine, lane);
    if (lane < a.beams) best[warp * a.beams + lane] = mine.key;
    __syncthreads();
    for (int i = threadIdx.x; i < kScanWarps * a.beams; i += kScanThreads) {
        const uint64_t own = best[i];
        int rank = 0;
        for (int o = 0; o < kScanWarps * a.beams; ++o) rank += best[o] > own ? 1 : 0;
        if (rank == 0) top = own;
        if (rank == a.beams - 1) bound = own;
    }
    __syncthreads();
    const float least = from_ordered(static_cast<uint32_t>(bound >> 32)), most_of_all = from_ordered(static_cast<uint32_t>(top >> 32));
    const uint32_t last_vector = ~static_cast<uint32_t>(bound);
    const float reference = most_of_all == -INFINITY ? 0.0f : most_of_all;
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < R; ++j) {
#pragma unroll
        for (int i = 0; i < VE; ++i) sum[i & 1] += power_of_two((widen(held[j].v[i]) - reference) * kLog2e);
        if (most[j] >= least) {
            const uint32_t number = static_cast<uint32_t>(first_vector + j * kScanThreads);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float x = widen(held[j].v[i]);
                const int64_t token = static_cast<int64_t>(number) * VE + i;
                if ((x > least || (x == least && number <= last_vector)) && token < a.vocabulary)
                    candidates[atomicAdd(&count, 1)] = static_cast<uint64_t>(ordered(x)) << 32 | ~static_cast<uint32_t>(token);   // (in any order: they are sorted)
            }
        }
    }
    double whole = static_cast<double>(sum[0]) + static_cast<double>(sum[1]);
    for (int o = 16; o > 0; o >>= 1) whole += __shfl_xor_sync(0xffffffffu, whole, o);
    if (lane == 0) partial[warp] = whole;
    __syncthreads();
    if (warp != 0) return;
    const int found = count;
    Key list{0};
    for (int from = 0; from < found; from += 32) {
        Key more{from + lane < found ? candidates[from + lane] : 0};
        sort_lanes(more, lane);
        merge_lanes(list, more, lane);
    }
    const int64_t at = blockIdx.x;
    if (lane < a.beams) a.keys[at * a.beams + lane] = list.key;
    if (lane == 0) {
        for (int w = 1; w < kScanWarps; ++w) whole += partial[w];
        a.sums[at] = ChunkSum{whole, reference, 0.0f};
    }
}

struct Ints {
    int32_t* data;              // null: absent
    int64_t batch, beam;
    __device__ __forceinline__ int32_t& at(int b, int w) const { return data[b * batch + w * beam]; }
};
struct MergeArgs {
    const void* logits;
    const ChunkSum* sums;
    const uint64_t* keys;
    int64_t batch_stride, beam_stride;
    const float* scores;
    float* scores_out;
    int64_t scores_batch, scores_beam, out_batch, out_beam;
    Ints finished, lengths, tokens, parents, finished_out, lengths_out;
    int32_t* forks;
    int32_t beams, vocabulary, chunks, logits_type, end, pad, source_base, target_base;
    float length_penalty;
};

__global__ void __launch_bounds__(kScanThreads)
beam_merge_kernel(const MergeArgs a) {
    __shared__ uint64_t keys[kMaxBeams][32];
    __shared__ uint32_t places[kMaxBeams][32];
    __shared__ double normalisers[kMaxBeams];   // ln sum exp; NaN: all continuations at -inf
    __shared__ float scores[kMaxBeams];
    __shared__ int32_t finished[kMaxBeams], lengths[kMaxBeams];
    const int entry = static_cast<int>(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    chain_begin();
    for (int beam = warp; beam < a.beams; beam += kScanWarps) {
        const float score = a.scores[entry * a.scores_batch + beam * a.scores_beam];
        const bool done = a.finished.data && a.finished.at(entry, beam) != 0;
        int64_t length = a.lengths.data ? static_cast<int64_t>(a.lengths.at(entry, beam)) + (done ? 0 : 1) : 1;
        length = min(max(length, static_cast<int64_t>(1)), static_cast<int64_t>(0x7fffffff));
        const double divisor = a.lengths.data && a.length_penalty != 0.0f ? pow(static_cast<double>(length), static_cast<double>(a.length_penalty)) : 1.0;
        const bool alive = isfinite(score);
        double normaliser = 0.0;
        Place mine{0, 0xffffffffu};
        const uint32_t row = static_cast<uint32_t>(beam) * static_cast<uint32_t>(a.vocabulary);
        if (done) {
            if (lane == 0) mine = Place{ordered(alive ? static_cast<double>(score) / divisor : -INFINITY), row + static_cast<uint32_t>(a.pad)};
        } else {
            const int64_t first = (static_cast<int64_t>(entry) * a.beams + beam) * a.chunks;
            float most = -INFINITY;
            for (int i = lane; i < a.chunks; i += 32) {   // (a chunk of -inf alone has no largest value that means anything)
                const ChunkSum part = a.sums[first + i];
                if (part.sum != 0.0) most = fmaxf(most, part.most);
            }
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            double sum = 0.0;
            for (int i = lane; i < a.chunks; i += 32) {
                const ChunkSum part = a.sums[first + i];
                if (part.sum != 0.0) sum += part.sum * exp(static_cast<double>(part.most) - static_cast<double>(most));
            }
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            normaliser = static_cast<double>(most) + log(sum);
            if (!alive || !isfinite(normaliser)) normaliser = nan("");
            Key list{0};
            for (int i = 0; i < a.chunks; ++i) {
                const Key more{lane < a.beams ? a.keys[(first + i) * a.beams + lane] : 0};
                merge_lanes(list, more, lane);
            }
            if (normaliser != normaliser) {
                if (lane < a.vocabulary) mine = Place{ordered(-static_cast<double>(INFINITY)), row + static_cast<uint32_t>(lane)};
            } else if (list.key != 0) {
                const double logit = static_cast<double>(from_ordered(static_cast<uint32_t>(list.key >> 32)));
                mine = Place{ordered((static_cast<double>(score) + (logit - normaliser)) / divisor), row + ~static_cast<uint32_t>(list.key)};
            }
            if (lane >= a.beams) mine = Place{0, 0xffffffffu};
            sort_lanes(mine, lane);   // (equal worths of different logits, where 64 bits do not tell them apart: by place)
        }
        keys[beam][lane] = mine.key;
        places[beam][lane] = mine.place;
        if (lane == 0) {
            normalisers[beam] = normaliser;
            scores[beam] = alive ? score : -INFINITY;
            finished[beam] = done;
            lengths[beam] = static_cast<int32_t>(length);
        }
    }
    __syncthreads();
    if (warp != 0) return;
    Place mine{keys[0][lane], places[0][lane]};
    for (int beam = 1; beam < a.beams; ++beam) merge_lanes(mine, Place{keys[beam][lane], places[beam][lane]}, lane);
    if (lane >= a.beams) return;
    const int parent = static_cast<int>(mine.place / static_cast<uint32_t>(a.vocabulary)), token = static_cast<int>(mine.place - static_cast<uint32_t>(parent) * static_cast<uint32_t>(a.vocabulary));
    float score = scores[parent];
    if (!finished[parent]) {
        const double normaliser = normalisers[parent];
        const double logit = static_cast<double>(load_as_f32(a.logits, a.logits_type, entry * a.batch_stride + parent * a.beam_stride + token));
        score = normaliser == normaliser ? static_cast<float>(static_cast<double>(score) + (logit - normaliser)) : -INFINITY;
    }
    a.scores_out[entry * a.out_batch + lane * a.out_beam] = score;
    a.tokens.at(entry, lane) = token;
    a.parents.at(entry, lane) = parent;
    if (a.finished_out.data) a.finished_out.at(entry, lane) = finished[parent] || (a.end >= 0 && token == a.end) ? 1 : 0;
    if (a.lengths_out.data) a.lengths_out.at(entry, lane) = lengths[parent];
    if (a.forks) {
        int32_t* pair = a.forks + 2 * (static_cast<int64_t>(entry) * a.beams + lane);
        pair[0] = a.source_base + entry * a.beams + parent;
        pair[1] = a.target_base + entry * a.beams + lane;
    }
}

// ---- states ------------------------------------------------------------------------------------

constexpr int kSegmentVectors = 8;   // of a lane: a warp moves 32 x 8 vectors of a row
struct StateSide {
    const uint8_t* source;
    uint8_t* target;
    int64_t source_stride[3], target_stride[3];   // layer, entry, beam, in bytes
    int64_t row_bytes;
    int32_t width, layers, first_unit;            // bytes of a vector; the state's first unit
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
    int vectors;      // a thread
    int64_t chunks;   // a row
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
    if (p.lengths.rank && !std::isfinite(p.length_penalty)) return fail(kInvalidValue, "BEAM_SELECT: the length penalty must be finite");
    if (p.finished.rank && (p.pad < 0 || p.pad >= p.logits.dim[2])) return fail(kInvalidValue, "BEAM_SELECT: pad is no token");
    const int64_t rows = p.logits.dim[0] * p.logits.dim[1];
    if (p.forks.rank) {
        if (!valid_tensor(p.forks) || p.forks.rank != 2 || p.forks.dim[0] != rows || p.forks.dim[1] != 2 || p.forks.dtype != DFGPU_I32) return fail(kInvalidShape, "BEAM_SELECT: forks must be INT32 [B * W, 2]");
        if (!is_packed_row_major(p.forks)) return fail(kInvalidLayout, "BEAM_SELECT: forks must be packed");
        if (p.source_base < 0 || p.target_base < 0 || p.source_base + rows > 0x7fffffff || p.target_base + rows > 0x7fffffff) return fail(kInvalidValue, "BEAM_SELECT: sequence numbers out of range");
    }
    // As many vectors a thread as still give every SM two chunks.
    const int width = 16 / dtype_bytes(p.logits.dtype);
    const int64_t vectors = (p.logits.dim[2] + width - 1) / width;
    for (cut.vectors = 8;; cut.vectors /= 2) {
        cut.chunks = (vectors + kScanThreads * cut.vectors - 1) / (kScanThreads * cut.vectors);
        if (cut.vectors == 1 || rows * cut.chunks >= 2 * 148) break;
    }
    if (rows * cut.chunks >= (1ll << 31)) return fail(kUnsupported, "BEAM_SELECT: too many tokens or entries");
    return kOk;
}
int64_t select_scratch(const dfgpu_beam_select_params& p, const SelectCut& cut) { return p.logits.dim[0] * p.logits.dim[1] * cut.chunks * (static_cast<int64_t>(sizeof(ChunkSum)) + 8 * p.logits.dim[1]); }

template <typename T>
void launch_scan(const ScanArgs& a, int vectors, int64_t chunks, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(chunks));
    const size_t shared = static_cast<size_t>(a.beams) * vectors * (16 / sizeof(T)) * sizeof(uint64_t);
    if (vectors == 8) launch_chained(beam_scan_kernel<T, 8>, grid, dim3(kScanThreads), shared, stream, a);
    else if (vectors == 4) launch_chained(beam_scan_kernel<T, 4>, grid, dim3(kScanThreads), shared, stream, a);
    else if (vectors == 2) launch_chained(beam_scan_kernel<T, 2>, grid, dim3(kScanThreads), shared, stream, a);
    else launch_chained(beam_scan_kernel<T, 1>, grid, dim3(kScanThreads), shared, stream, a);
}

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
    const int64_t entries = p->logits.dim[0], beams = p->logits.dim[1], chunks = entries * beams * cut.chunks;
    ScanArgs s{};
    s.logits = port[0];
    s.finished = static_cast<const int32_t*>(port[2]);
    s.sums = static_cast<ChunkSum*>(scratch);
    s.keys = reinterpret_cast<uint64_t*>(s.sums + chunks);
    s.batch_stride = p->logits.stride[0];
    s.beam_stride = p->logits.stride[1];
    s.finished_batch = p->finished.rank ? p->finished.stride[0] : 0;
    s.finished_beam = p->finished.rank ? p->finished.stride[1] : 0;
    s.beams = static_cast<int>(beams);
    s.vocabulary = static_cast<int>(p->logits.dim[2]);
    s.chunks = static_cast<int>(cut.chunks);
    s.by_chunks = make_fast_divisor(static_cast<uint32_t>(cut.chunks));
    s.by_beams = make_fast_divisor(static_cast<uint32_t>(beams));
    cudaStream_t on = as_stream(stream);
    if (p->logits.dtype == DFGPU_F32) launch_scan<float>(s, cut.vectors, chunks, on);
    else if (p->logits.dtype == DFGPU_F16) launch_scan<__half>(s, cut.vectors, chunks, on);
    else launch_scan<__nv_bfloat16>(s, cut.vectors, chunks, on);
    status = check_launch("BEAM_SELECT");
    if (status) return status;
    MergeArgs m{};
    auto ints = [&](int i) {
        return Ints{static_cast<int32_t*>(port[i]), port[i] ? described[i]->stride[0] : 0, port[i] ? described[i]->stride[1] : 0};
    };
    m.logits = s.logits;
    m.sums = s.sums;
    m.keys = s.keys;
    m.batch_stride = s.batch_stride;
    m.beam_stride = s.beam_stride;
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
    m.beams = s.beams;
    m.vocabulary = s.vocabulary;
    m.chunks = s.chunks;
    m.logits_type = p->logits.dtype;
    m.end = p->end;
    m.pad = p->pad;
    m.source_base = p->source_base;
    m.target_base = p->target_base;
    m.length_penalty = p->length_penalty;
    launch_chained(beam_merge_kernel, dim3(static_cast<unsigned>(entries)), dim3(kScanThreads), 0, on, m);
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
        side.layers = static_cast<int>(s.dim[0]);
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
