// Attention over a paged cache of E4M3 codes with E8M0 scales: the streaming form, for few query rows a KV head (single tokens,
// drafted tokens) and for every type and head dimension.
//
// Bound by HBM: each held code is read once for all query heads of its KV head. A row of the products is a (token, head) pair.
// Codes are exact in f16 (448 to 2^-9), so K and V go from shared memory through one convert for two codes straight into the
// register operands of mma.sync.m16n8k16: a tcgen05 product wants its operands in shared memory, and writing the converted tile there
// and reading it back is 144 bytes of shared-memory traffic a clock at HBM speed, where the port moves 128. Both products are taken
// transposed, S^T = K Q^T and O^T = V^T P^T, so that rows come in eights (most groups of query heads are no larger) and 16 keys or
// channels share an instruction; P^T turns from the first one's result into the second one's operand by movmatrix.
//   * Q is not rounded: each row is scaled by a power of two that puts its largest magnitude at 2^14, and is exact in f16 down to
//     2^-38 of that (below, within 2^-39 of it).
//   * 16 consecutive keys share a page and a scale (both are multiples of 16 tokens). The K scale multiplies their scores. O is
//     held in units of a power of two, 2^unit: the V scale of 16 keys goes into their probabilities, as 2^(scale - unit), where that is from 2^-10
//     to 1, and else the unit moves and O with it (exactly, as far as scales within 2^80 of one another go).
//   * Probabilities are rounded to f16 as p * 2^15: 11 bits down to 2^-29 (2^-19 beside a V scale of 2^-10 units), where p is measured
//     against the largest score so far.
// Channels and keys may go to any index of a product as long as both operands agree; the ones taken here give each thread 16-byte
// reads without bank conflicts: of K 32 consecutive channels of a key, of V 16 consecutive channels of four keys, and of O 16
// consecutive channels of a row.
// The work is one row of units of 32 keys, list by list (a sequence's block of rows, a KV head), cut into equal parts for the CTAs that are on
// the chip together (three an SM for single tokens): lengths differ, and a grid of lists or of pieces of them pays for it with idle SMs
// at the end and with a prologue for each piece. A fifth warp brings a CTA's units by TMA into a ring, across lists, so that the
// next list's codes are on their way while O of the last one is written; four take them in turn, or in pairs or all of them with rows
// of their own where there are more than 16. Lists that were cut leave partial results, which a second kernel merges.
#include <algorithm>
#include <cmath>

#include "cache_sdpa.cuh"
#include "dfgpu_cache.h"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

constexpr int kWarps = 4, kThreads = 160;
constexpr int kUnit = 32;          // keys that a warp takes at a time
constexpr int kBatch = 4;          // units that the loader looks up at a time
constexpr int kLeastUnits = 8;     // of a CTA: fewer cost more in prologues and partial results than they gain
constexpr int kSms = 148;          // (the cut is a function of the shape and the lengths alone, as the scratch is of the shape)
constexpr float kUp = 15.0f;       // probabilities are held as p * 2^15
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kNoUnit = -100000;   // O is zero and has no unit yet
constexpr int kNaN = 0x7fc00000;

// EIGHTS: eights of rows that a warp takes.
template <int D, int EIGHTS>
struct Shape {
    static constexpr int kCtas = D == 256 ? (EIGHTS == 1 ? 2 : 1) : EIGHTS == 1 ? 3 : 2;   // on an SM
    static constexpr int kSide = kUnit * D;                                                // bytes of a unit's K or V
    // A multiple of the warps, so that a slot's units are always the same warp's: it then knows one phase of the slot's barrier from the
    // next. (With six slots a warp that was ahead took the phase before last, of another warp's unit, for its own.)
    static constexpr int kSlots = (kCtas == 3 ? 64 : D == 256 ? (EIGHTS == 1 ? 64 : 192) : 96) * 1024 / (2 * kSide);
    static_assert(kSlots % kWarps == 0, "a slot belongs to one warp");
    static constexpr int kRing = kSlots * 2 * kSide;
    static constexpr int kFragments = kRing;                                  // [warp][pairs of O][32] float2, of one row of two of an eight
    static constexpr int kMeeting = kFragments + kWarps * (D / 16) * 32 * 8;  // [warp][eight][row of two][quad] float2
    static constexpr int kScales = kMeeting + kWarps * EIGHTS * 2 * 4 * 8;    // [slot] K scales of its two runs of 16 keys as f32 (-1: the page's rows read as zeros), V's as codes (-1 likewise)
    static constexpr int kBarriers = kScales + kSlots * 16;                   // full[slots], empty[slots]
    static constexpr int kScan = kBarriers + 2 * kSlots * 8;                  // [warps] int64, then where the CTA begins
    static constexpr int kTotal = kScan + 64 + 32;
    static constexpr int kDynamic = kTotal + 1024;
};

// Byte offset of a 16-byte chunk of a unit's row, as TMA lays rows of 128 or 64 bytes out (a D of 256: two halves): the reads above meet each bank once.
template <int D>
__device__ __forceinline__ uint32_t at_chunk(int row, int chunk) {
    return D == 64 ? row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4) : (chunk >> 3) * (kUnit * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

__device__ __forceinline__ void four_codes(uint32_t codes, uint32_t& low, uint32_t& high) {   // as f16
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(low), "=r"(high) : "r"(codes));
}
__device__ __forceinline__ uint32_t two_halves(float lo, float hi) {
    uint32_t v;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void multiply(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void multiply_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t pair) {   // of an 8 x 8 matrix of f16 over the warp
    uint32_t v;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(v) : "r"(pair));
    return v;
}
__device__ __forceinline__ uint32_t times(uint32_t pair, uint32_t factor) {
    uint32_t v;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"(pair), "r"(factor));
    return v;
}
__device__ __forceinline__ uint4 read_16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }   // -126 to 127

__device__ __forceinline__ float value_of(__half v) { return __half2float(v); }
__device__ __forceinline__ float value_of(__nv_bfloat16 v) { return __bfloat162float(v); }

// Two neighbouring values of a row of O.
__device__ __forceinline__ void store_pair(const CacheSdpaArgs& a, int64_t at, float first, float second) {
    if (a.o_vector) {
        if (a.o_type == DFGPU_F32) *reinterpret_cast<float2*>(static_cast<float*>(a.o) + at) = make_float2(first, second);
        else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + at) =
                 a.o_type == DFGPU_F16 ? two_halves(first, second) : static_cast<uint32_t>(f32_to_bf16_bits(first)) | static_cast<uint32_t>(f32_to_bf16_bits(second)) << 16;
        return;
    }
    store_from_f32(a.o, a.o_type, at, first);
    store_from_f32(a.o, a.o_type, at + 1, second);
}

// The page of a slot in a side's table, -1 where there is none.
__device__ __forceinline__ int page_of(const CacheSdpaArgs& a, const CacheSide& s, int64_t batch, int slot) {
    if (slot >= s.table_len) return -1;
    const int page = s.table[batch * s.table_batch + slot * s.table_slot];
    return page >= 0 && page < s.pages ? page : -1;
}

// EIGHTS * 8 rows against the codes of K and V that their warp takes. Thread (eighth, quad) = (lane / 4, lane % 4) has scores of keys
// eighth and eighth + 8 of each 16, and O's channels channel_of(j) and the next one, both for rows 2 quad and 2 quad + 1 of each eight.
template <int D, int EIGHTS>
struct RowTile {
    static constexpr int kDeep = D / 16;                     // products along the channels of K
    static constexpr int kWide = D / 16;                     // pairs of channels of V
    uint32_t q[kDeep][EIGHTS][2];
    float factor[EIGHTS][2];            // of a score: 1 / the row's power of two, attention scale, log2(e)
    int row_lo[EIGHTS][2], row_hi[EIGHTS][2];   // keys that a row sees
    float largest[EIGHTS][2], sum[EIGHTS][2];
    float o[kWide][EIGHTS][4];          // (channel, row), (channel, next row), (next channel, row), (next channel, next row)
    int unit;

    __device__ static __forceinline__ int channel_of(int j, int eighth) { return D == 64 ? eighth * 8 + 2 * j : (j >> 3) * 128 + eighth * 16 + 2 * (j & 7); }

    // A unit of keys from key0 of the sequence on. SPECIAL: some row does not see all of them, or a page or scale is none.
    template <bool SPECIAL>
    __device__ __forceinline__ void step(const uint8_t* k_unit, const uint8_t* v_unit, const float* k_scales, const int* v_scales, int key0, int lo, int hi, bool mixed) {
        const int lane = threadIdx.x & 31, quad = lane & 3, eighth = lane >> 2;
        float s[2][EIGHTS][4];   // neighbouring products add to different ones
#pragma unroll
        for (int u = 0; u < kDeep / 4; ++u) {
            uint32_t w[4][4];    // of keys eighth, + 8, + 16, + 24
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint4 raw = read_16(k_unit + at_chunk<D>(r * 8 + eighth, D == 64 ? quad : quad * 2 + (u & 1) + (u >> 1) * 8));
                w[r][0] = raw.x, w[r][1] = raw.y, w[r][2] = raw.z, w[r][3] = raw.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    uint32_t a0, a1, a2, a3;
                    four_codes(w[2 * r][i], a0, a2);
                    four_codes(w[2 * r + 1][i], a1, a3);
#pragma unroll
                    for (int n = 0; n < EIGHTS; ++n) {
                        if (u + i == 0) multiply_first(s[r][n], a0, a1, a2, a3, q[0][n]);
                        else multiply(s[r][n], a0, a1, a2, a3, q[u * 4 + i][n]);
                    }
                }
        }
        bool above = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float k_scale = k_scales[r];
#pragma unroll
            for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float& x = s[r][n][c];
                    x *= factor[n][c & 1] * k_scale;
                    if (SPECIAL) {
                        const int key = key0 + r * 16 + eighth + (c >> 1) * 8;
                        if (k_scale < 0.0f) x = 0.0f;
                        if (static_cast<uint32_t>(key - row_lo[n][c & 1]) >= static_cast<uint32_t>(row_hi[n][c & 1] - row_lo[n][c & 1])) x = -INFINITY;
                    }
                    above = above || x > largest[n][c & 1];
                }
        }
        if (__any_sync(0xffffffffu, above)) {   // a new largest score in some row (rare after the first units)
#pragma unroll
            for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2])), largest[n][c]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float down = top == -INFINITY ? 1.0f : exp2_of(largest[n][c] - top);
                    largest[n][c] = top;
                    sum[n][c] *= down;
#pragma unroll
                    for (int j = 0; j < kWide; ++j) o[j][n][c] *= down, o[j][n][c + 2] *= down;
                }
        }
        uint32_t p[2][EIGHTS][2];
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) {
            const float from0 = largest[n][0] == -INFINITY ? 0.0f : kUp - largest[n][0], from1 = largest[n][1] == -INFINITY ? 0.0f : kUp - largest[n][1];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float p0 = exp2_of(s[r][n][0] + from0), p1 = exp2_of(s[r][n][1] + from1), p2 = exp2_of(s[r][n][2] + from0), p3 = exp2_of(s[r][n][3] + from1);
                sum[n][0] += p0 + p2;
                sum[n][1] += p1 + p3;
                p[r][n][0] = transposed(two_halves(p0, p1));
                p[r][n][1] = transposed(two_halves(p2, p3));
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int code = v_scales[r], apart = code - unit;   // (the same in all threads)
            if ((!SPECIAL || (code >= 0 && code != 255)) && apart != 0) {
                if (apart < 0 && (apart >= -10 || apart < -80)) {
                    const uint32_t less = apart < -80 ? 0u : static_cast<uint32_t>(15 + apart) << 10, both = less | less << 16;
#pragma unroll
                    for (int n = 0; n < EIGHTS; ++n) p[r][n][0] = times(p[r][n][0], both), p[r][n][1] = times(p[r][n][1], both);
                } else {
                    const float to = unit == kNoUnit ? 1.0f : power_of_two(max(-apart, -126));
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
#pragma unroll
                        for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[j][n][c] *= to;
                    unit = code;
                }
            }
            // V: channels from 16 * eighth on (8 * eighth for a D of 64) of keys 2 quad, 2 quad + 1 and those plus 8
            uint32_t w[4][kWide / 2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = r * 16 + quad * 2 + (k & 1) + (k >> 1) * 8;
                if constexpr (D == 64) {
                    const uint2 raw = *reinterpret_cast<const uint2*>(v_unit + at_chunk<D>(at, eighth >> 1) + (eighth & 1) * 8);
                    w[k][0] = raw.x, w[k][1] = raw.y;
                } else {
#pragma unroll
                    for (int u = 0; u < kWide / 8; ++u) {
                        const uint4 raw = read_16(v_unit + at_chunk<D>(at, eighth + u * 8));
                        w[k][u * 4] = raw.x, w[k][u * 4 + 1] = raw.y, w[k][u * 4 + 2] = raw.z, w[k][u * 4 + 3] = raw.w;
                    }
                }
                if (SPECIAL) {   // rows that nothing was brought to, or that no query sees: anything may lie there, NaN codes too
                    const int key = key0 + at;
                    if (code < 0 || key < lo || key >= hi) {
#pragma unroll
                        for (int i = 0; i < kWide / 2; ++i) w[k][i] = 0;
                    }
                }
            }
            if (SPECIAL) {
                const int run0 = key0 + r * 16;
                if (code == 255) {   // a scale that is a NaN: for the rows that see one of its keys
#pragma unroll
                    for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (run0 < row_hi[n][c & 1] && run0 + 16 > row_lo[n][c & 1]) {
#pragma unroll
                                for (int j = 0; j < kWide; ++j) o[j][n][c] = __int_as_float(kNaN);
                            }
                }
                if (mixed) {
                    // A NaN code must reach the rows that see its key and no others, whose probability for it is 0: such codes become zeros in the
                    // products, and NaNs in the sums of the rows that they belong to.
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < kWide / 2; ++i) {
                            const uint32_t found = ((w[k][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                            w[k][i] &= ~((found >> 7) * 0xffu);
                            nan |= found;
                        }
                    if (__any_sync(0xffffffffu, nan != 0)) {
#pragma unroll 1
                        for (int k = 0; k < 16; ++k)
#pragma unroll
                            for (int j = 0; j < kWide; ++j)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int channel = channel_of(j, eighth) + e;
                                    const uint8_t found = v_unit[at_chunk<D>(r * 16 + k, channel >> 4) + (channel & 15)];
                                    if ((found & 0x7fu) != 0x7fu) continue;
#pragma unroll
                                    for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                                        for (int c = 0; c < 2; ++c)
                                            if (run0 + k >= row_lo[n][c] && run0 + k < row_hi[n][c]) o[j][n][e * 2 + c] = __int_as_float(kNaN);
                                }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kWide / 2; ++i) {   // four channels: two products
                uint32_t near[4], far[4];
                four_codes(__byte_perm(w[0][i], w[1][i], 0x5140), near[0], near[1]);
                four_codes(__byte_perm(w[0][i], w[1][i], 0x7362), near[2], near[3]);
                four_codes(__byte_perm(w[2][i], w[3][i], 0x5140), far[0], far[1]);
                four_codes(__byte_perm(w[2][i], w[3][i], 0x7362), far[2], far[3]);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int n = 0; n < EIGHTS; ++n) multiply(o[i * 2 + e][n], near[2 * e], near[2 * e + 1], far[2 * e], far[2 * e + 1], p[r][n]);
            }
        }
    }
};

// Units of keys of an entry (a sequence's block of rows), the same for each of its KV heads.
__device__ __forceinline__ int units_of(const CacheSdpaArgs& a, int entry, int& lo, int& hi) {
    const int sequence = entry / a.row_blocks, row_first = (entry - sequence * a.row_blocks) * a.block_rows;
    window_of_tokens(a, sequence_window(a, sequence), row_first / a.group, (min(row_first + a.block_rows, a.rows) - 1) / a.group, lo, hi);
    return hi > lo ? (hi + kUnit - 1) / kUnit - lo / kUnit : 0;
}

// A CTA's way through the lists: entry, KV head, the next unit of the list and how many of the CTA's are left.
struct Walk {
    int entry, head, offset, left;
    int lo, hi, units;      // of the entry
    bool first;             // nothing has been taken yet

    // The next piece of a list, `take` units from unit `offset` on; false after the last. Every lane of a warp walks alike. Entries without
    // keys are passed over 32 at a time.
    __device__ __forceinline__ bool next(const CacheSdpaArgs& a, int& take) {
        if (left <= 0) return false;
        while (units == 0) {
            const int lane = threadIdx.x & 31;
            int from = 0, until = 0;
            const int n = entry + lane < a.entries ? units_of(a, entry + lane, from, until) : 0;
            const uint32_t some = __ballot_sync(0xffffffffu, n > 0);
            if (some == 0) {
                entry += 32;
                if (entry >= a.entries) return false;
                continue;
            }
            const int found = __ffs(some) - 1;
            entry += found;
            lo = __shfl_sync(0xffffffffu, from, found), hi = __shfl_sync(0xffffffffu, until, found), units = __shfl_sync(0xffffffffu, n, found);
        }
        take = min(units - offset, left);
        return true;
    }
    __device__ __forceinline__ void taken(const CacheSdpaArgs& a, int take) {
        left -= take;
        offset = 0;
        first = false;
        if (++head == a.heads_kv) head = 0, ++entry, units = 0;
    }
};

// ROW_WARPS: warps with rows of their own.
template <typename T, int D, int EIGHTS, int ROW_WARPS>
__global__ void __launch_bounds__(kThreads, Shape<D, EIGHTS>::kCtas)
cache_sdpa_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CacheSdpaArgs a) {
    using S = Shape<D, EIGHTS>;
    using Rows = RowTile<D, EIGHTS>;
    constexpr int kGroups = kWarps / ROW_WARPS;       // warps that take units in turn
    constexpr int kWide = Rows::kWide, kRows = EIGHTS * 8;
    extern __shared__ uint8_t raw_smem[];
    const uint32_t ring = (smem_u32(raw_smem) + 1023u) & ~1023u;
    uint8_t* smem = raw_smem + (ring - smem_u32(raw_smem));
    auto full = [&](int s) { return ring + S::kBarriers + 8u * s; };
    auto empty = [&](int s) { return ring + S::kBarriers + 8u * (S::kSlots + s); };
    const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
        for (int s = 0; s < S::kSlots; ++s) {
            mbar_init(full(s), 5);            // the loader's bytes, four scales
            mbar_init(empty(s), ROW_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_begin();

    // All units before those of this thread's entries, and their number: where this CTA's part begins.
    Walk walk{};
    int per;
    {
        int64_t* sums = reinterpret_cast<int64_t*>(smem + S::kScan);
        int* begin = reinterpret_cast<int*>(smem + S::kScan + 64);
        const int each = (a.entries + kThreads - 1) / kThreads, from = min(static_cast<int>(threadIdx.x) * each, a.entries), until = min(from + each, a.entries);
        int64_t own = 0;
        int lo, hi;
        for (int e = from; e < until; ++e) own += units_of(a, e, lo, hi);
        own *= a.heads_kv;
        int64_t up_to = own;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int64_t other = __shfl_up_sync(0xffffffffu, up_to, x);
            if (lane >= x) up_to += other;
        }
        if (lane == 31) sums[warp] = up_to;
        __syncthreads();
        int64_t all = 0, before = up_to - own;
#pragma unroll
        for (int w = 0; w <= kWarps; ++w) {
            if (w < warp) before += sums[w];
            all += sums[w];
        }
        per = max(static_cast<int>((all + gridDim.x - 1) / gridDim.x), kLeastUnits);
        if (blockIdx.x == 0 && threadIdx.x == 0) a.starts[0] = per;
        int64_t start = static_cast<int64_t>(blockIdx.x) * per;
        walk.left = static_cast<int>(max(min(static_cast<int64_t>(per), all - start), static_cast<int64_t>(0)));
        if (walk.left > 0 && start >= before && start < before + own) {
            start -= before;
            for (int e = from; e < until; ++e) {
                const int n = units_of(a, e, lo, hi);
                if (start < static_cast<int64_t>(n) * a.heads_kv) {
                    begin[0] = e, begin[1] = static_cast<int>(start / n), begin[2] = static_cast<int>(start % n);
                    break;
                }
                start -= static_cast<int64_t>(n) * a.heads_kv;
            }
        }
        __syncthreads();
        if (walk.left <= 0) return;
        walk.entry = begin[0], walk.head = begin[1], walk.offset = begin[2];
        walk.first = true;
    }

    if (warp == kWarps) {
        // The loader looks up four units at a time: lane l has one box of one of them, `box` rows (16 or 32 of a page) of K or V by 128 or 64 bytes, and
        // the first sixteen lanes one of their scales each. Page ids are read two batches ahead of their use, scales one.
        constexpr int kHalves = D == 256 ? 2 : 1;
        const int boxes = kUnit / a.box * kHalves, box = lane % boxes, side = lane / boxes & 1, own_unit = lane / boxes >> 1;
        const int box_row = box / kHalves * a.box, half = box % kHalves;
        const uint32_t box_bytes = static_cast<uint32_t>(a.box) * (D == 64 ? 64u : 128u);
        const uint32_t to = side * S::kSide + half * (kUnit * 128) + box_row * (D == 64 ? 64 : 128);
        const int scale_unit = lane >> 2 & 3, scale_side = lane >> 1 & 1, scale_run = lane & 1;
        const int scale_from = (scale_unit * 2 + scale_side) * boxes + scale_run * 16 / a.box * kHalves;   // the lane that has the scale's page
        struct Batch {
            int entry, head, unit, count, lo, hi;   // count: 0 after the last
            int page, token;                        // of this lane's box
        };
        int u = 0, take = 0;
        auto following = [&](Batch& b) {   // the next four units, or what is left of their list
            if (u >= take) {
                if (take > 0) walk.taken(a, take);
                u = 0;
                if (!walk.next(a, take)) take = 0;
            }
            b.count = min(kBatch, take - u);
            b.entry = walk.entry, b.head = walk.head, b.lo = walk.lo, b.hi = walk.hi;
            b.unit = walk.lo / kUnit + walk.offset + u;
            b.page = -1, b.token = 0;
            if (own_unit < b.count) {
                const int key = (b.unit + own_unit) * kUnit + box_row, at = static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page));
                b.token = key - at * a.page;
                if (key < b.hi && key + a.box > b.lo) b.page = page_of(a, a.side[side], b.entry / a.row_blocks, at);
            }
            u += kBatch;
        };
        auto scale_of = [&](const Batch& b) {
            const int page = __shfl_sync(0xffffffffu, b.page, scale_from), token = __shfl_sync(0xffffffffu, b.token, scale_from) + scale_run * 16 % a.box;
            const int key = (b.unit + scale_unit) * kUnit + scale_run * 16;
            if (lane >= 16 || page < 0 || key >= b.hi || key + 16 <= b.lo) return -1;
            const CacheSide& s = a.side[scale_side];
            return static_cast<int>(s.scales[page * s.scale_stride[0] + b.head * s.scale_stride[1] + fast_divide(static_cast<uint32_t>(token >> 4), a.by_tokens) * s.scale_stride[2]]);
        };
        Batch now, next, later;
        following(now);
        following(next);
        int code = scale_of(now);
        int slot = 0;
        uint32_t turn = 1;
        const uint32_t of_unit = own_unit < kBatch ? ((1u << (2 * boxes)) - 1u) << (2 * boxes * own_unit) : 0u;   // the lanes with this unit's boxes (2, 4 or 8)
        const bool first_of_unit = own_unit < kBatch && lane % (2 * boxes) == 0;
        while (now.count > 0) {
            following(later);
            const int next_code = scale_of(next);
            // the slots of this lane's box and of its scale, free when all four units' are
            const int box_slot = slot + own_unit < S::kSlots ? slot + own_unit : slot + own_unit - S::kSlots, scale_slot = slot + scale_unit < S::kSlots ? slot + scale_unit : slot + scale_unit - S::kSlots;
            const bool mine = own_unit < now.count;
            const uint32_t bar = full(mine ? box_slot : slot), living = __ballot_sync(0xffffffffu, now.page >= 0);
            if (!mbar_wait_warp(mine ? empty(box_slot) : empty(slot), mine && slot + own_unit >= S::kSlots ? turn ^ 1 : turn, 701)) break;
            if (first_of_unit && mine) mbar_expect_tx(bar, __popc(living & of_unit) * box_bytes);   // (also the first arrival; no byte where no page is)
            __syncwarp();
            if (now.page >= 0) tma_load_4d(ring + box_slot * (2 * S::kSide) + to, side ? &map_v : &map_k, half * 128, now.token, now.head, now.page, bar);
            if (lane < 16 && scale_unit < now.count) {   // the other arrivals, behind the scales
                reinterpret_cast<float*>(smem + S::kScales + scale_slot * 16)[lane & 3] = scale_side ? __int_as_float(code) : code < 0 ? -1.0f : decode_e8m0(static_cast<uint32_t>(code));
                mbar_arrive(full(scale_slot));
            }
            __syncwarp();
            slot += now.count;
            if (slot >= S::kSlots) slot -= S::kSlots, turn ^= 1;
            now = next, next = later, code = next_code;
        }
        return;
    }

    const int quad = lane & 3, eighth = lane >> 2, row_warp = warp % ROW_WARPS, group = warp / ROW_WARPS;
    bool ok = true;
    int behind = 0, take;      // units of the lists before
    for (; walk.next(a, take); behind += take, walk.taken(a, take)) {
        const int64_t batch = walk.entry / a.row_blocks;
        const int row_first = (walk.entry - static_cast<int>(batch) * a.row_blocks) * a.block_rows, lo = walk.lo, hi = walk.hi, head = walk.head;
        const SequenceWindow window = sequence_window(a, batch);
        const bool whole = walk.offset == 0 && take == walk.units;
        if (threadIdx.x == 0 && walk.offset == 0) a.starts[1 + static_cast<int64_t>(walk.entry) * a.heads_kv + head] = whole ? -1 : static_cast<int64_t>(blockIdx.x) * per + behind;
        Rows rows;
        const int own_row = row_first + row_warp * kRows;
        auto place_of = [&](int row, int& token, int& head_q) {   // of a row that there is
            token = row / a.group;
            head_q = head * a.group + (row - token * a.group);
        };
        int common_lo = lo, common_hi = hi, any_lo = hi, any_hi = lo;   // what the warp's rows see in common, and what any of them sees
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) {
            // Q of row `eighth`: this quarter of its channels
            const int row = own_row + n * 8 + eighth;
            int token = 0, head_q = 0;
            if (row < a.rows) place_of(row, token, head_q);
            const T* from = static_cast<const T*>(a.q) + batch * a.q_stride[0] + head_q * a.q_stride[1] + token * a.q_stride[2];
            float v[Rows::kDeep][4];
            float largest = 0.0f;
#pragma unroll
            for (int i = 0; i < Rows::kDeep; ++i) {
                const int channel = D == 64 ? quad * 16 + i * 4 : (quad * 2 + ((i >> 2) & 1) + (i >> 3) * 8) * 16 + (i & 3) * 4;
                struct alignas(8) Four { T v[4]; } four{};
                if (row < a.rows) {
                    if (a.q_vector) four = *reinterpret_cast<const Four*>(from + channel);
                    else four = Four{{from[channel], from[channel + 1], from[channel + 2], from[channel + 3]}};
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[i][e] = value_of(four.v[e]);
                    largest = fmaxf(largest, fabsf(v[i][e]));
                }
            }
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            int up = 14 - (static_cast<int>(__float_as_uint(largest) >> 23) - 127);
            up = largest == 0.0f ? 0 : min(max(up, -126), 126);
            const float power = power_of_two(up), factor = power_of_two(-up) * a.scale_log2;
#pragma unroll
            for (int i = 0; i < Rows::kDeep; ++i) {
                rows.q[i][n][0] = two_halves(v[i][0] * power, v[i][1] * power);
                rows.q[i][n][1] = two_halves(v[i][2] * power, v[i][3] * power);
            }
            // rows 2 quad and 2 quad + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                rows.factor[n][c] = __shfl_sync(0xffffffffu, factor, (quad * 2 + c) * 4);
                const int column = own_row + n * 8 + quad * 2 + c;
                const bool there = column < a.rows && column / a.group < window.len_q;
                rows.row_lo[n][c] = lo, rows.row_hi[n][c] = hi;      // (rows without a part see what the others see; their results go nowhere)
                if (there) {
                    window_of_tokens(a, window, column / a.group, column / a.group, rows.row_lo[n][c], rows.row_hi[n][c]);
                    any_lo = min(any_lo, rows.row_lo[n][c]);
                    any_hi = max(any_hi, rows.row_hi[n][c]);
                }
                rows.row_hi[n][c] = max(rows.row_hi[n][c], rows.row_lo[n][c]);
                common_lo = max(common_lo, rows.row_lo[n][c]);
                common_hi = min(common_hi, rows.row_hi[n][c]);
                rows.largest[n][c] = -INFINITY;
                rows.sum[n][c] = 0.0f;
            }
        }
        rows.unit = kNoUnit;
#pragma unroll
        for (int j = 0; j < kWide; ++j)
#pragma unroll
            for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) rows.o[j][n][c] = 0.0f;
        common_lo = __reduce_max_sync(0xffffffffu, common_lo), common_hi = __reduce_min_sync(0xffffffffu, common_hi);
        any_lo = __reduce_min_sync(0xffffffffu, any_lo), any_hi = __reduce_max_sync(0xffffffffu, any_hi);

        // (on a wait that gave up, walk on without units: the warps meet at their barriers)
        for (int u = (group - behind) & (kGroups - 1); u < take; u += kGroups) {
            const int nth = behind + u, slot = nth % S::kSlots;
            if (ok) ok = mbar_wait_warp(full(slot), (nth / S::kSlots) & 1, 702);
            if (!ok) continue;
            const uint8_t* k_unit = smem + slot * (2 * S::kSide);
            const float* k_scale = reinterpret_cast<const float*>(smem + S::kScales + slot * 16);
            const int* v_scale = reinterpret_cast<const int*>(k_scale + 2);
            const int key0 = (lo / kUnit + walk.offset + u) * kUnit;
            if (key0 < any_hi && key0 + kUnit > any_lo) {
                const bool special = key0 < common_lo || key0 + kUnit > common_hi || fminf(k_scale[0], k_scale[1]) < 0.0f ||
                                     max(static_cast<uint32_t>(v_scale[0]), static_cast<uint32_t>(v_scale[1])) > 254u;
                if (special) rows.template step<true>(k_unit, k_unit + S::kSide, k_scale, v_scale, key0, lo, hi, a.seq_q > 1);
                else rows.template step<false>(k_unit, k_unit + S::kSide, k_scale, v_scale, key0, lo, hi, false);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(slot));
        }

        // The warps with the same rows meet: (largest score, sum, O) triples by shared memory, one row of two of an eight at a time, in the
        // order of the fragments, so that each bank is met once. Each warp then has pairs of channels of its own: j * groups / pairs == group.
        const float absolute = rows.unit == kNoUnit ? 1.0f : decode_e8m0(static_cast<uint32_t>(rows.unit));
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) {
#pragma unroll
            for (int j = 0; j < kWide; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) rows.o[j][n][c] *= absolute;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) rows.sum[n][c] += __shfl_xor_sync(0xffffffffu, rows.sum[n][c], x);
        }
        if constexpr (kGroups > 1) {
            float2* fragments = reinterpret_cast<float2*>(smem + S::kFragments);
            float2* meeting = reinterpret_cast<float2*>(smem + S::kMeeting);
#pragma unroll
            for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    asm volatile("bar.sync 1, 128;" ::: "memory");   // (what was there before has been read)
                    if (eighth == 0) meeting[((warp * EIGHTS + n) * 2 + c) * 4 + quad] = make_float2(rows.largest[n][c], rows.sum[n][c]);
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        if (j * kGroups / kWide != group) fragments[(warp * kWide + j) * 32 + lane] = make_float2(rows.o[j][n][c], rows.o[j][n][c + 2]);
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    float2 other[kGroups];
                    float top = -INFINITY, total = 0.0f, own_weight = 0.0f;
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        other[g] = meeting[(((g * ROW_WARPS + row_warp) * EIGHTS + n) * 2 + c) * 4 + quad];
                        top = fmaxf(top, other[g].x);
                    }
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        other[g].x = other[g].x == -INFINITY ? 1.0f : exp2_of(other[g].x - top);   // (a group without keys has zeros)
                        total = fmaf(other[g].y, other[g].x, total);
                        if (g == group) own_weight = other[g].x;
                    }
                    rows.largest[n][c] = top, rows.sum[n][c] = total;
#pragma unroll
                    for (int j = 0; j < kWide; ++j) {
                        if (j * kGroups / kWide != group) continue;
                        float2 v = make_float2(rows.o[j][n][c] * own_weight, rows.o[j][n][c + 2] * own_weight);
#pragma unroll
                        for (int g = 0; g < kGroups; ++g) {
                            if (g == group) continue;
                            const float2 part = fragments[((g * ROW_WARPS + row_warp) * kWide + j) * 32 + lane];
                            v.x = fmaf(part.x, other[g].x, v.x);
                            v.y = fmaf(part.y, other[g].x, v.y);
                        }
                        rows.o[j][n][c] = v.x, rows.o[j][n][c + 2] = v.y;
                    }
                }
        }
        if (!ok || g_device_status != 0) continue;
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = own_row + n * 8 + quad * 2 + c;
                if (row >= a.rows) continue;
                const float top = rows.largest[n][c], total = rows.sum[n][c];
                if (!whole) {
                    float* partial = a.partial + ((static_cast<int64_t>(blockIdx.x) * 2 + (walk.first ? 0 : 1)) * a.block_rows + (row - row_first)) * (D + 2);
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        if (j * kGroups / kWide == group)
                            *reinterpret_cast<float2*>(partial + Rows::channel_of(j, eighth)) = make_float2(rows.o[j][n][c], rows.o[j][n][c + 2]);
                    if (eighth == 0 && group == 0) *reinterpret_cast<float2*>(partial + D) = make_float2(top, total);
                } else {
                    int token, head_q;
                    place_of(row, token, head_q);
                    const bool none = token >= window.len_q || total == 0.0f;   // (a NaN sum is a NaN result)
                    const float inverse = 1.0f / total;
                    const int64_t at = batch * a.o_stride[0] + head_q * a.o_stride[1] + token * a.o_stride[2];
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        if (j * kGroups / kWide == group)
                            store_pair(a, at + Rows::channel_of(j, eighth), none ? 0.0f : rows.o[j][n][c] * inverse, none ? 0.0f : rows.o[j][n][c + 2] * inverse);
                    if (eighth == 0 && group == 0 && a.stats)
                        a.stats[batch * a.stats_stride[0] + head_q * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : top * kLn2 + logf(total * 0x1p-15f);
                }
            }
    }
}

// A CTA a row, a thread a channel: the rows of lists that were cut, and of those without keys. Latency-bound: the maxima and sums of 32 parts come at
// once, a part a lane in every warp, together with their values.
template <int D>
__global__ void __launch_bounds__(D)
cache_sdpa_merge_kernel(const __grid_constant__ CacheSdpaArgs a) {
    const int lane = threadIdx.x & 31;
    const int in_rows = static_cast<int>(blockIdx.x % a.rows), token = in_rows / a.group;
    const int64_t list = blockIdx.x / a.rows, batch = list / a.heads_kv;
    const int head_kv = static_cast<int>(list - batch * a.heads_kv), head = head_kv * a.group + (in_rows - token * a.group);
    const int block = in_rows / a.block_rows, row = in_rows - block * a.block_rows, entry = static_cast<int>(batch) * a.row_blocks + block;
    chain_begin();
    const int64_t per = a.starts[0], start = a.starts[1 + static_cast<int64_t>(entry) * a.heads_kv + head_kv];   // (written where the list has keys)
    int lo, hi;
    const int units = units_of(a, entry, lo, hi);
    const bool takes_part = token < sequence_window(a, batch).len_q;
    float top = -INFINITY, total = 0.0f, value = 0.0f;
    if (units > 0) {
        if (start < 0) return;   // not cut: its CTA has written O
        const int64_t first = start / per;
        const int parts = static_cast<int>((start + units - 1) / per - first) + 1;
        const bool second_place = start != first * per;   // of the first part in its CTA
        auto part_of = [&](int i) { return a.partial + (((first + i) * 2 + (i == 0 && second_place ? 1 : 0)) * a.block_rows + row) * (D + 2); };
        for (int i0 = 0; i0 < parts; i0 += 32) {
            float ahead[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) ahead[k] = i0 + k < parts ? part_of(i0 + k)[threadIdx.x] : 0.0f;
            float2 pair = make_float2(-INFINITY, 0.0f);
            if (i0 + lane < parts) pair = *reinterpret_cast<const float2*>(part_of(i0 + lane) + D);
            float largest = fmaxf(top, pair.x);
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, s));
            const float down = top == -INFINITY ? 1.0f : exp2_of(top - largest);   // (no score above -inf: zeros, or NaNs that are to be seen)
            const float weight = pair.x == -INFINITY ? 1.0f : exp2_of(pair.x - largest);
            top = largest;
            float part = pair.y * weight;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) part += __shfl_xor_sync(0xffffffffu, part, s);
            total = fmaf(total, down, part);
            value *= down;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const float w = __shfl_sync(0xffffffffu, weight, k);
                if (i0 + k < parts) value = fmaf(ahead[k], w, value);
            }
        }
    }
    const bool none = !takes_part || total == 0.0f;
    store_from_f32(a.o, a.o_type, batch * a.o_stride[0] + head * a.o_stride[1] + token * a.o_stride[2] + threadIdx.x, none ? 0.0f : value / total);
    if (threadIdx.x == 0 && a.stats) a.stats[batch * a.stats_stride[0] + head * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : top * kLn2 + logf(total * 0x1p-15f);
}

struct StreamPlan {
    int eights, row_warps, block_rows, row_blocks;
    int64_t rows, grid, starts, scratch;   // starts: integers before the partial results
};

StreamPlan plan_stream(const dfgpu_cache_sdpa_params& p) {
    StreamPlan plan{};
    const int64_t d = p.q.dim[3], group = p.q.dim[1] / p.k.dim[1];
    plan.rows = group * p.q.dim[2];
    plan.eights = plan.rows <= 8 ? 1 : 2;
    plan.row_warps = plan.rows <= 16 ? 1 : plan.rows <= 32 ? 2 : 4;
    plan.block_rows = plan.eights * 8 * plan.row_warps;
    plan.row_blocks = static_cast<int>((plan.rows + plan.block_rows - 1) / plan.block_rows);
    const int64_t lists = p.q.dim[0] * p.k.dim[1] * plan.row_blocks, units = (p.s_kv + kUnit - 1) / kUnit;
    const int64_t ctas = kSms * (d == 256 ? (plan.eights == 1 ? 2 : 1) : plan.eights == 1 ? 3 : 2);   // (Shape::kCtas)
    plan.grid = std::min(ctas, (lists * units + kLeastUnits - 1) / kLeastUnits);
    plan.starts = (1 + lists + 1) / 2 * 2;
    plan.scratch = plan.starts * 8 + plan.grid * 2 * plan.block_rows * (d + 2) * 4;
    return plan;
}

bool on_16(const void* pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 15u) == 0; }

int check_side(const dfgpu_cache_sdpa_params& p, const dfgpu_tensor& cache, const dfgpu_tensor& scale, const dfgpu_tensor& table, const char* name) {
    if (!valid_tensor(cache) || cache.rank != 4 || cache.dtype != DFGPU_E4M3 || cache.dim[3] != p.q.dim[3]) return fail(kInvalidShape, "CACHE_SDPA: the container of %s must be FP8_E4M3 [pages, Hk, T, D]", name);
    if (cache.dim[1] != p.k.dim[1] || cache.dim[2] != p.k.dim[2]) return fail(kInvalidShape, "CACHE_SDPA: the containers differ in heads or tokens a page");
    if (cache.stride[3] != 1) return fail(kInvalidLayout, "CACHE_SDPA: the head dimension of a container must have unit stride");
    for (int i = 0; i < 3; ++i)
        if (cache.dim[i] > 1 && (cache.stride[i] % 16 != 0 || cache.stride[i] >= (1ll << 40))) return fail(kInvalidLayout, "CACHE_SDPA: the strides of the container of %s must be multiples of 16", name);
    if (!valid_tensor(scale) || scale.rank != 4 || scale.dtype != DFGPU_E8M0 || scale.reorder != DFGPU_REORDER_NONE || scale.dim[0] != cache.dim[0] || scale.dim[1] != cache.dim[1] ||
        scale.dim[3] != 1 || cache.dim[2] % scale.dim[2] != 0 || scale.dim[2] != p.k_scale.dim[2])
        return fail(kInvalidShape, "CACHE_SDPA: the scales of %s must be FP8_E8M0 [pages, Hk, T / t, 1], t a divisor of T and one for K and V", name);
    if ((cache.dim[2] / scale.dim[2]) % 16 != 0) return fail(kUnsupported, "CACHE_SDPA: a scale must stand for a multiple of 16 tokens");
    if (!valid_tensor(table) || table.rank != 4 || table.dtype != DFGPU_I32 || table.dim[0] != p.q.dim[0] || table.dim[1] != 1 || table.dim[3] != 1)
        return fail(kInvalidShape, "CACHE_SDPA: page tables must be INT32 [B,1,P,1]");
    if (table.dim[2] * cache.dim[2] < p.s_kv) return fail(kInvalidShape, "CACHE_SDPA: page table capacity is below the key/value length");
    return kOk;
}

int check_cache_sdpa(const dfgpu_cache_sdpa_params& p, int& kernel) {
    if (!valid_tensor(p.q) || !valid_tensor(p.o) || p.q.rank != 4 || p.o.rank != 4) return fail(kInvalidShape, "CACHE_SDPA: Q and O must have rank 4 and positive extents");
    if (p.q.dtype != DFGPU_F16 && p.q.dtype != DFGPU_BF16) return fail(kUnsupported, "CACHE_SDPA: Q must be HALF or BFLOAT16");
    if (p.o.dtype != p.q.dtype && p.o.dtype != DFGPU_F32) return fail(kUnsupported, "CACHE_SDPA: O must be of Q's type or FLOAT");
    for (int i = 0; i < 4; ++i)
        if (p.o.dim[i] != p.q.dim[i]) return fail(kInvalidShape, "CACHE_SDPA: O must be [B, Hq, Sq, D] as Q is");
    if (p.q.stride[3] != 1 || p.o.stride[3] != 1) return fail(kInvalidLayout, "CACHE_SDPA: the head dimension must have unit stride");
    for (int i = 0; i < 3; ++i)
        if (p.o.dim[i] > 1 && p.o.stride[i] == 0) return fail(kInvalidLayout, "CACHE_SDPA: O overlaps itself");
    if (p.q.dim[3] != 64 && p.q.dim[3] != 128 && p.q.dim[3] != 256) return fail(kUnsupported, "CACHE_SDPA: head dimension %lld (64, 128 or 256)", static_cast<long long>(p.q.dim[3]));
    if (p.s_kv <= 0) return fail(kInvalidShape, "CACHE_SDPA: key/value length must be positive");
    if (p.s_kv >= (1ll << 30)) return fail(kUnsupported, "CACHE_SDPA: 2^30 keys or more");
    int status = check_side(p, p.k, p.k_scale, p.page_table_k, "K");
    if (!status) status = check_side(p, p.v, p.v_scale, p.page_table_v, "V");
    if (status) return status;
    if (p.q.dim[1] % p.k.dim[1] != 0) return fail(kInvalidShape, "CACHE_SDPA: query heads must be a multiple of K and V heads");
    for (const dfgpu_tensor* t : {&p.seq_kv, &p.seq_q}) {
        if (t == &p.seq_q && t->rank == 0) continue;
        if (!valid_tensor(*t) || t->rank != 4 || t->dtype != DFGPU_I32 || t->dim[0] != p.q.dim[0] || t->dim[1] != 1 || t->dim[2] != 1 || t->dim[3] != 1)
            return fail(kInvalidShape, "CACHE_SDPA: sequence length tensors must be INT32 [B,1,1,1]");
    }
    if (p.stats.rank && (!valid_tensor(p.stats) || p.stats.rank != 4 || p.stats.dtype != DFGPU_F32 || p.stats.dim[0] != p.q.dim[0] || p.stats.dim[1] != p.q.dim[1] ||
                         p.stats.dim[2] != p.q.dim[2] || p.stats.dim[3] != 1))
        return fail(kInvalidShape, "CACHE_SDPA: Stats must be FLOAT [B, Hq, Sq, 1]");
    if (!std::isfinite(p.attn_scale)) return fail(kInvalidValue, "CACHE_SDPA: the attention scale must be finite");
    const StreamPlan plan = plan_stream(p);
    if (p.q.dim[2] >= (1ll << 30) || p.q.dim[0] * p.k.dim[1] * plan.rows >= (1ll << 31)) return fail(kUnsupported, "CACHE_SDPA: too many sequences, heads or query rows");
    if (p.kernel < DFGPU_CACHE_SDPA_AUTO || p.kernel > DFGPU_CACHE_SDPA_STREAM) return fail(kInvalidArgument, "CACHE_SDPA: unknown kernel id %d", p.kernel);
    kernel = DFGPU_CACHE_SDPA_STREAM;
    return kOk;
}

// Codes as [pages, Hk, T, D] boxes of `box` tokens by 128 or 64 bytes.
int make_side_map(CUtensorMap* map, const dfgpu_tensor& cache, const void* base, int box_rows) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return fail(kExecutionFailed, "CACHE_SDPA: cuTensorMapEncodeTiled is unavailable");
    const bool narrow = cache.dim[3] == 64;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(cache.dim[3]), static_cast<cuuint64_t>(cache.dim[2]), static_cast<cuuint64_t>(cache.dim[1]), static_cast<cuuint64_t>(cache.dim[0])};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; ++i) strides[i] = static_cast<cuuint64_t>(cache.dim[2 - i] > 1 ? cache.stride[2 - i] : cache.dim[3]);
    const cuuint32_t box[4] = {narrow ? 64u : 128u, static_cast<cuuint32_t>(box_rows), 1, 1}, steps[4] = {1, 1, 1, 1};
    const CUresult result = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS) return fail(kExecutionFailed, "CACHE_SDPA: tensor map encode failed (CUresult %d)", static_cast<int>(result));
    return kOk;
}

template <typename T, int D, int EIGHTS, int ROW_WARPS>
int launch_rows(const CUtensorMap& map_k, const CUtensorMap& map_v, const CacheSdpaArgs& a, dim3 grid, cudaStream_t stream) {
    constexpr int kBytes = Shape<D, EIGHTS>::kDynamic;
    const auto kernel = cache_sdpa_stream_kernel<T, D, EIGHTS, ROW_WARPS>;
    const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (error != cudaSuccess) return fail(kExecutionFailed, "CACHE_SDPA: cannot reserve %d bytes of shared memory: %s", kBytes, cudaGetErrorString(error));
    launch_chained(kernel, grid, dim3(kThreads), kBytes, stream, map_k, map_v, a);
    return check_launch("CACHE_SDPA");
}

template <typename T, int D>
int launch_stream(const CUtensorMap& map_k, const CUtensorMap& map_v, const CacheSdpaArgs& a, const StreamPlan& plan, dim3 grid, cudaStream_t stream) {
    const int status = plan.eights == 1      ? launch_rows<T, D, 1, 1>(map_k, map_v, a, grid, stream)
                       : plan.row_warps == 1 ? launch_rows<T, D, 2, 1>(map_k, map_v, a, grid, stream)
                       : plan.row_warps == 2 ? launch_rows<T, D, 2, 2>(map_k, map_v, a, grid, stream)
                                             : launch_rows<T, D, 2, 4>(map_k, map_v, a, grid, stream);
    if (status) return status;
    launch_chained(cache_sdpa_merge_kernel<D>, dim3(static_cast<unsigned>(static_cast<int64_t>(a.entries / a.row_blocks) * a.heads_kv * a.rows)), dim3(D), 0, stream, a);
    return check_launch("CACHE_SDPA merge");
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_cache_sdpa(const dfgpu_cache_sdpa_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "CACHE_SDPA: null params");
    int kernel;
    const int status = check_cache_sdpa(*p, kernel);
    if (status) return status;
    const StreamPlan plan = plan_stream(*p);
    info->kernel = kernel;
    info->launches = 2;
    info->scratch_bytes = plan.scratch;
    return kOk;
}

extern "C" int dfgpu_cache_sdpa(const dfgpu_cache_sdpa_params* p, void* const* tensors, void* scratch, void* stream) {
    if (!p || !tensors) return fail(kInvalidArgument, "CACHE_SDPA: null params");
    int kernel;
    const int status = check_cache_sdpa(*p, kernel);
    if (status) return status;
    const StreamPlan plan = plan_stream(*p);
    for (int i = 0; i < 11; ++i) {
        const bool needed = i == 4 ? p->stats.rank != 0 : i == 7 ? p->seq_q.rank != 0 : true;
        if (needed && !tensors[i]) return fail(kInvalidArgument, "CACHE_SDPA: port %d is null", i);
    }
    if (!on_16(tensors[1]) || !on_16(tensors[2])) return fail(kInvalidArgument, "CACHE_SDPA: the containers must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(tensors[0]) & 1u) != 0 || (reinterpret_cast<uintptr_t>(tensors[3]) & static_cast<uintptr_t>(dtype_bytes(p->o.dtype) - 1)) != 0)
        return fail(kInvalidArgument, "CACHE_SDPA: Q or O is not aligned to its type");
    for (int i : {4, 7, 8, 9, 10})
        if ((reinterpret_cast<uintptr_t>(tensors[i]) & 3u) != 0) return fail(kInvalidArgument, "CACHE_SDPA: port %d is not aligned to its type", i);
    if (!scratch || !on_16(scratch)) return fail(kInvalidArgument, "CACHE_SDPA: needs the 16-byte aligned scratch dfgpu_query_cache_sdpa reports");
    CacheSdpaArgs a{};
    a.q = tensors[0];
    a.o = tensors[3];
    a.stats = p->stats.rank ? static_cast<float*>(tensors[4]) : nullptr;
    for (int s = 0; s < 2; ++s) {
        const dfgpu_tensor &cache = s ? p->v : p->k, &scale = s ? p->v_scale : p->k_scale, &table = s ? p->page_table_v : p->page_table_k;
        CacheSide& side = a.side[s];
        side.codes = static_cast<const uint8_t*>(tensors[1 + s]);
        side.scales = static_cast<const uint8_t*>(tensors[5 + s]);
        side.table = static_cast<const int32_t*>(tensors[9 + s]);
        for (int i = 0; i < 3; ++i) {
            side.stride[i] = cache.dim[i] > 1 ? cache.stride[i] : 0;
            side.scale_stride[i] = scale.dim[i] > 1 ? scale.stride[i] : 0;
        }
        side.table_batch = table.stride[0];
        side.table_slot = table.stride[2];
        side.table_len = static_cast<int>(std::min<int64_t>(table.dim[2], 1 << 30));
        side.pages = cache.dim[0];
    }
    for (int i = 0; i < 3; ++i) {
        a.q_stride[i] = p->q.stride[i];
        a.o_stride[i] = p->o.stride[i];
        a.stats_stride[i] = p->stats.rank ? p->stats.stride[i] : 0;
    }
    a.o_type = p->o.dtype;
    a.o_vector = (reinterpret_cast<uintptr_t>(a.o) & static_cast<uintptr_t>(2 * dtype_bytes(p->o.dtype) - 1)) == 0;   // pairs of O, fours of Q
    a.q_vector = (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0;
    for (int i = 0; i < 3; ++i) {
        a.o_vector = a.o_vector && (p->o.dim[i] == 1 || p->o.stride[i] % 2 == 0);
        a.q_vector = a.q_vector && (p->q.dim[i] == 1 || p->q.stride[i] % 4 == 0);
    }
    a.seq_q_data = p->seq_q.rank ? static_cast<const int32_t*>(tensors[7]) : nullptr;
    a.seq_kv_data = static_cast<const int32_t*>(tensors[8]);
    a.seq_q_stride = p->seq_q.rank ? p->seq_q.stride[0] : 0;
    a.seq_kv_stride = p->seq_kv.stride[0];
    a.heads_kv = static_cast<int>(p->k.dim[1]);
    a.group = static_cast<int>(p->q.dim[1] / p->k.dim[1]);
    a.rows = static_cast<int>(plan.rows);
    a.seq_q = static_cast<int>(p->q.dim[2]);
    a.s_kv = static_cast<int>(p->s_kv);
    a.page = static_cast<int>(p->k.dim[2]);
    a.by_page = make_fast_divisor(static_cast<uint32_t>(a.page / 16));
    a.by_tokens = make_fast_divisor(static_cast<uint32_t>(p->k.dim[2] / p->k_scale.dim[2] / 16));
    a.has_left = p->has_left_bound;
    a.has_right = p->has_right_bound;
    a.bottom_right = p->bottom_right;
    const int64_t far = 1ll << 40;   // (as good as none, and sums with it stay in range)
    a.left = std::min(std::max(p->left_bound, -far), far);
    a.right = std::min(std::max(p->right_bound, -far), far);
    a.scale_log2 = p->attn_scale * 1.4426950408889634f;
    a.row_blocks = plan.row_blocks;
    a.block_rows = plan.block_rows;
    a.entries = static_cast<int>(p->q.dim[0] * plan.row_blocks);
    a.starts = static_cast<int64_t*>(scratch);
    a.partial = reinterpret_cast<float*>(a.starts + plan.starts);
    a.box = a.page % 32 == 0 ? 32 : 16;
    CUtensorMap map_k, map_v;
    int made = make_side_map(&map_k, p->k, tensors[1], a.box);
    if (!made) made = make_side_map(&map_v, p->v, tensors[2], a.box);
    if (made) return made;
    const dim3 grid(static_cast<unsigned>(plan.grid));
    cudaStream_t on = as_stream(stream);
    const bool half = p->q.dtype == DFGPU_F16;
    switch (p->q.dim[3]) {
        case 64: return half ? launch_stream<__half, 64>(map_k, map_v, a, plan, grid, on) : launch_stream<__nv_bfloat16, 64>(map_k, map_v, a, plan, grid, on);
        case 128: return half ? launch_stream<__half, 128>(map_k, map_v, a, plan, grid, on) : launch_stream<__nv_bfloat16, 128>(map_k, map_v, a, plan, grid, on);
        default: return half ? launch_stream<__half, 256>(map_k, map_v, a, plan, grid, on) : launch_stream<__nv_bfloat16, 256>(map_k, map_v, a, plan, grid, on);
    }
}

namespace dfgpu {
int cache_sdpa_device_status(int* status) { return read_and_clear_device_status(status); }
}  // namespace dfgpu
