// Attention over a paged cache of E4M3 codes with E8M0 scales: the streaming form, for few query rows a KV head (single tokens, a few
// drafted ones) and for every type and head dimension.
//
// Bound by HBM: each held code is read once for all query heads of its KV head. A row of the products is a (token, head) pair.
// Codes are exact in f16 (448 to 2^-9), so K and V go from shared memory through one convert for two codes straight into the
// register operands of mma.sync.m16n8k16: a tcgen05 product wants its operands in shared memory, and writing the converted tile there
// and reading it back is 144 bytes of shared-memory traffic a clock at HBM speed, where the port moves 128. Both products are taken
// transposed, S^T = K Q^T and O^T = V^T P^T, so that rows come in eights (most groups of query heads are no larger) and 16 keys or
// channels share an instruction; P^T turns from the first one's result into the second one's operand by movmatrix.
//   * Q is scaled row by row by a power of two that puts its largest magnitude at 2^14: f16 holds it exactly down to 2^-28 of that (bf16:
//     2^-31), and to within 2^-39 of that below.
//   * 16 consecutive keys share a page and a scale (both are multiples of 16 tokens). The K scale multiplies their scores. O is
//     held in units of a power of two, 2^unit: the V scale of 16 keys goes into their probabilities, as 2^(scale - unit), where that is from 2^-10
//     to 1, and else the unit moves and O with it (exactly, as far as scales within 2^80 of one another go: what lies further below the largest so far counts as zeros).
//   * Probabilities are rounded to f16 as p * 2^15: 11 bits down to 2^-29 (2^-19 beside a V scale of 2^-10 units), where p is measured
//     against the largest score so far.
// Channels and keys may go to any index of a product as long as both operands agree; the ones taken here give each thread 16-byte
// reads without bank conflicts: of K 32 consecutive channels of a key, of V 16 consecutive channels of four keys, and of O 16
// consecutive channels of a row.
// The work is one row of units of 32 keys, list by list (a sequence, a KV head, a block of 8 or 16 rows), cut into equal parts for the WARPS that
// are on the chip together, sixteen an SM for single tokens. A warp is on its own: it brings its units by TMA into a private ring of K and V
// tiles, computes on them and refills each as soon as it has read it, so that nothing is shared and nobody waits for another warp. (CTAs
// whose warps shared each list's units spent a third of their time on meeting and on beginning lists; a loading warp for four
// others was what they waited for.) Lists that were cut leave partial results, which a second kernel merges. Rows beyond 16 (8) are
// lists of their own, whose keys come from L2.
// 64 sequences of 512 to 8192 keys, 8 KV heads of 128 channels, 4 query heads each: 122 us, 4.7 TB/s, 71 % of the copy rate (110 without the arithmetic; as long
// with the pages in order as with pages anywhere); two such sequences: 19 us, of which 15 are look-ups, launches and the merge. More rows: at the choice of a form below.
#include <algorithm>
#include <cmath>

#include "cache_sdpa.cuh"
#include "dfgpu_cache.h"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

constexpr int kWarps = 4, kThreads = 128;
constexpr int kUnit = 32;          // keys that a warp takes at a time
constexpr int kLeastUnits = 4;     // of a part: fewer cost more in prologues and partial results than they gain
constexpr int kSms = 148;          // (the cut is a function of the shape and the lengths alone, as the scratch is of the shape)
constexpr float kUp = 15.0f;       // probabilities are held as p * 2^15
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kNoUnit = -100000;   // O is zero and has no unit yet
constexpr int kMostDown = 80;      // O's unit goes down no further below its largest: n keys make at most 2^(15 + 9 + 80) n of it, below f32's range up to 2^24 keys of a warp's part
constexpr int kNaN = 0x7fc00000;

// EIGHTS: eights of rows that a warp takes.
template <int D, int EIGHTS>
struct Shape {
    static_assert(EIGHTS == 1 || D == 64, "see plan_stream");
    static constexpr int kCtas = D == 256 ? 2 : EIGHTS == 1 ? 4 : 3;          // on an SM, by registers
    static constexpr int kSide = kUnit * D;                                   // bytes of a unit's K or V
    static constexpr int kSlots = D == 64 ? (EIGHTS == 1 ? 6 : 8) : 3;   // K and V tiles of a warp's ring
    static constexpr int kRing = kWarps * kSlots * kSide;
    static constexpr int kBarriers = kRing;                                   // [warp][slot]
    static constexpr int kTotal = kBarriers + kWarps * kSlots * 8;
    static constexpr int kDynamic = kTotal + 1024;
    static_assert(kCtas * (kDynamic + 1024) <= 228 * 1024, "CTAs an SM");
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
    int unit, most;                     // most: the largest unit that O has had, over which its values may stand at most 2^80 up (kNoUnit: none)

    __device__ static __forceinline__ int channel_of(int j, int eighth) { return D == 64 ? eighth * 8 + 2 * j : (j >> 3) * 128 + eighth * 16 + 2 * (j & 7); }

    // Probabilities of a unit of keys, from key0 of the sequence on. SPECIAL: some row does not see all of them, or a page or scale is none (k_scales of
    // 16 keys each, -1 where the page's rows read as zeros).
    template <bool SPECIAL>
    __device__ __forceinline__ void scores(const uint8_t* k_unit, const float (&k_scales)[2], int key0, uint32_t (&p)[2][EIGHTS][2]) {
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
    }

    // Their values to O (v_scales: codes, -1 likewise). [lo, hi): the keys that any row sees.
    template <bool SPECIAL>
    __device__ __forceinline__ void values(const uint8_t* v_unit, const int (&v_scales)[2], int key0, int lo, int hi, bool mixed, uint32_t (&p)[2][EIGHTS][2]) {
        const int lane = threadIdx.x & 31, quad = lane & 3, eighth = lane >> 2;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int code = v_scales[r], apart = code - unit;   // (the same in all threads)
            if ((!SPECIAL || (code >= 0 && code != 255)) && apart != 0) {
                const bool least = code < most - kMostDown;   // (against all that O holds, not against the last unit: steps down add up)
                if (apart < 0 && (apart >= -10 || least)) {
                    const uint32_t less = least ? 0u : static_cast<uint32_t>(15 + apart) << 10, both = less | less << 16;
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
                    unit = code, most = max(most, code);
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

__device__ __forceinline__ int divided(int n, const FastDivisor& by) { return static_cast<int>(fast_divide(static_cast<uint32_t>(n), by)); }

// Units of keys of an entry (a sequence's block of rows), the same for each of its KV heads.
__device__ __forceinline__ int units_of(const CacheSdpaArgs& a, int entry, int& lo, int& hi) {
    const int sequence = divided(entry, a.by_row_blocks), row_first = (entry - sequence * a.row_blocks) * a.block_rows;
    window_of_tokens(a, sequence_window(a, sequence), divided(row_first, a.by_group), divided(min(row_first + a.block_rows, a.rows) - 1, a.by_group), lo, hi);
    return hi > lo ? (hi + kUnit - 1) / kUnit - lo / kUnit : 0;
}

// Whether the kernel has anything to do (whole warps).
__device__ __forceinline__ bool wanted(const CacheSdpaArgs& a) {
    if (__builtin_expect(a.only_if == nullptr, 1)) return true;
    bool some = false;
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < a.only_if_count; i += 32) some = some || a.only_if[i] != 0;
    return __any_sync(0xffffffffu, some);
}

template <typename T, int D, int EIGHTS>
__global__ void __launch_bounds__(kThreads, Shape<D, EIGHTS>::kCtas)
cache_sdpa_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CacheSdpaArgs a) {
    using S = Shape<D, EIGHTS>;
    using Rows = RowTile<D, EIGHTS>;
    constexpr int kWide = Rows::kWide, kRows = EIGHTS * 8;
    extern __shared__ uint8_t raw_smem[];
    const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
    uint8_t* smem = raw_smem + (base - smem_u32(raw_smem));
    const int warp = uniform_warp_index(), lane = threadIdx.x & 31, quad = lane & 3, eighth = lane >> 2;
    const uint32_t bars = base + S::kBarriers + warp * (S::kSlots * 8), ring = base + warp * (S::kSlots * S::kSide);
    const uint8_t* ring_data = smem + warp * (S::kSlots * S::kSide);
    if (lane == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
        for (int s = 0; s < S::kSlots; ++s) mbar_init(bars + 8u * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_begin();
    if (!wanted(a)) return;

    // The units before each lane's entries, and all of them (fewer than 2^30): where the warp's part begins. (Every warp for itself: the lengths come
    // from L1 for the later ones, and a pass over a few of them is shorter than a barrier of the CTA.)
    const int each = (a.entries + 31) / 32, from = min(lane * each, a.entries), until = min(from + each, a.entries);
    int own = 0, lo = 0, hi = 0;
    for (int e = from; e < until; ++e) own += units_of(a, e, lo, hi);
    own *= a.heads_kv;
    int up_to = own;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, up_to, x);
        if (lane >= x) up_to += other;
    }
    const int all = __shfl_sync(0xffffffffu, up_to, 31);
    const int warps = static_cast<int>(gridDim.x) * kWarps, per = max((all + warps - 1) / warps, kLeastUnits);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.starts[0] = per;
    // Neighbouring parts go to different SMs: with fewer parts than warps all SMs have some.
    const int part = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
    if (part >= (all + per - 1) / per) return;
    int left = min(per, all - part * per), entry, head, offset, units = 0;
    bool first_piece = true;
    {
        const int start = part * per, found = __ffs(__ballot_sync(0xffffffffu, up_to > start)) - 1;   // the lane with the part's first entry
        int rest = start - (up_to - own);
        entry = from;
        if (lane == found)
            for (;; ++entry) {
                units = units_of(a, entry, lo, hi);
                if (rest < units * a.heads_kv) break;
                rest -= units * a.heads_kv;
            }
        entry = __shfl_sync(0xffffffffu, entry, found), units = __shfl_sync(0xffffffffu, units, found), rest = __shfl_sync(0xffffffffu, rest, found);
        lo = __shfl_sync(0xffffffffu, lo, found), hi = __shfl_sync(0xffffffffu, hi, found);
        head = rest / units;
        offset = rest - head * units;
    }

    constexpr int kHalves = D == 256 ? 2 : 1, kAhead = 16;   // units a look-up
    const int boxes = kUnit / a.box;                         // of `box` keys, 16 or 32 of a page
    const uint32_t box_bytes = static_cast<uint32_t>(a.box) * (D == 64 ? 64u : 128u);
    int tiles = 0;   // K and V tiles of the pieces before: tile t is in slot t % kSlots, in phase t / kSlots of its barrier
    for (;;) {
        while (units == 0) {   // entries without keys, 32 at a time
            int from = 0, until = 0;
            const int n = entry + lane < a.entries ? units_of(a, entry + lane, from, until) : 0;
            const uint32_t some = __ballot_sync(0xffffffffu, n > 0);
            const int which = some ? __ffs(some) - 1 : 32;
            entry += which;
            if (some) units = __shfl_sync(0xffffffffu, n, which), lo = __shfl_sync(0xffffffffu, from, which), hi = __shfl_sync(0xffffffffu, until, which);
        }
        const int take = min(units - offset, left), unit0 = lo / kUnit + offset;
        const int64_t batch = divided(entry, a.by_row_blocks);
        const int row_first = (entry - static_cast<int>(batch) * a.row_blocks) * a.block_rows;
        const bool whole = offset == 0 && take == units;
        if (lane == 0 && offset == 0) a.starts[1 + static_cast<int64_t>(entry) * a.heads_kv + head] = whole ? -1 : min((part + 1) * per, all) - left;

        // Of sixteen units, lane l has the table's entries of box l and the scales of the l-th 16 keys. Whether an entry is a page is asked when
        // it is used: a comparison here would wait for it.
        int page[2], page_next[2] = {-1, -1}, code[2] = {-1, -1}, code_next[2];   // K, V
        auto look_up = [&](int from, int (&to)[2]) {
            const int key = (unit0 + from) * kUnit + lane * a.box, slot = static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page));
            const bool in = lane < kAhead * boxes && from + lane / boxes < take && key < hi && key + a.box > lo;
#pragma unroll
            for (int w = 0; w < 2; ++w) to[w] = in && slot < a.side[w].table_len ? a.side[w].table[batch * a.side[w].table_batch + slot * a.side[w].table_slot] : -1;
        };
        auto is_page = [&](int id, int w) { return id >= 0 && id < a.side[w].pages; };
        auto look_up_scales = [&](int from) {
            const int key = (unit0 + from) * kUnit + lane * 16, token = key - static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page)) * a.page;
            const int64_t block = fast_divide(static_cast<uint32_t>(token >> 4), a.by_tokens);
            const bool in = from + (lane >> 1) < take && key < hi && key + 16 > lo;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const CacheSide& s = a.side[w];
                const int id = __shfl_sync(0xffffffffu, page[w], lane * 16 / a.box);
                code_next[w] = in && is_page(id, w) ? s.scales[id * s.scale_stride[0] + head * s.scale_stride[1] + block * s.scale_stride[2]] : -1;
            }
        };
        // Brings tile t of the piece, K (t even) or V of unit t / 2: in order, each as soon as its slot has been read.
        auto fetch = [&](int t) {
            if (t >= 2 * take) return;
            const int u = t >> 1, w = t & 1, slot = (tiles + t) % S::kSlots;
            if (w == 0 && u > 0 && u % kAhead == 0) {
                page[0] = page_next[0], page[1] = page_next[1];
                look_up(u + kAhead, page_next);
                look_up_scales(u);
            }
            const int box = lane / kHalves, half = lane % kHalves, key = (unit0 + u) * kUnit + box * a.box;
            const int id = __shfl_sync(0xffffffffu, page[w], (u % kAhead) * boxes + (box & 1));
            const bool live = box < boxes && is_page(id, w);
            const uint32_t count = __popc(__ballot_sync(0xffffffffu, live)), bar = bars + 8u * slot;
            if (lane == 0) mbar_expect_tx(bar, count * box_bytes);   // (also the arrival; no byte where no page is)
            __syncwarp();
            if (live) {
                const int token = key - static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page)) * a.page;
                tma_load_4d(ring + slot * S::kSide + half * (kUnit * 128) + box * a.box * (D == 64 ? 64 : 128), w ? &map_v : &map_k, half * 128, token, head, id, bar);
            }
            __syncwarp();
        };
        look_up(0, page);
        look_up(kAhead, page_next);
        look_up_scales(0);
#pragma unroll 1
        for (int t = 0; t < S::kSlots; ++t) fetch(t);

        Rows rows;
        const SequenceWindow window = sequence_window(a, batch);
        auto place_of = [&](int row, int& token, int& head_q) {   // of a row that there is
            token = static_cast<int>(fast_divide(static_cast<uint32_t>(row), a.by_group));
            head_q = head * a.group + (row - token * a.group);
        };
        int common_lo = lo, common_hi = hi, any_lo = hi, any_hi = lo;   // what the rows see in common, and what any of them sees
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n) {
            // Q of row `eighth`: this quarter of its channels
            const int row = row_first + n * 8 + eighth;
            int token = 0, head_q = 0;
            if (row < a.rows) place_of(row, token, head_q);
            const T* from = static_cast<const T*>(a.q) + batch * a.q_stride[0] + head_q * a.q_stride[1] + token * a.q_stride[2];
            struct alignas(8) Four { T v[4]; } v[Rows::kDeep];
#pragma unroll
            for (int i = 0; i < Rows::kDeep; ++i) {
                const int channel = D == 64 ? quad * 16 + i * 4 : (quad * 2 + ((i >> 2) & 1) + (i >> 3) * 8) * 16 + (i & 3) * 4;
                v[i] = Four{};
                if (row < a.rows) {
                    if (a.q_vector) v[i] = *reinterpret_cast<const Four*>(from + channel);
                    else v[i] = Four{{from[channel], from[channel + 1], from[channel + 2], from[channel + 3]}};
                }
            }
            float largest = 0.0f;
#pragma unroll
            for (int i = 0; i < Rows::kDeep; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(value_of(v[i].v[e])));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            int up = 14 - (static_cast<int>(__float_as_uint(largest) >> 23) - 127);
            up = largest == 0.0f ? 0 : min(max(up, -126), 126);
            const float power = power_of_two(up), factor = power_of_two(-up) * a.scale_log2;
#pragma unroll
            for (int i = 0; i < Rows::kDeep; ++i) {
                rows.q[i][n][0] = two_halves(value_of(v[i].v[0]) * power, value_of(v[i].v[1]) * power);
                rows.q[i][n][1] = two_halves(value_of(v[i].v[2]) * power, value_of(v[i].v[3]) * power);
            }
            // rows 2 quad and 2 quad + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                rows.factor[n][c] = __shfl_sync(0xffffffffu, factor, (quad * 2 + c) * 4);
                const int column = row_first + n * 8 + quad * 2 + c;
                rows.row_lo[n][c] = lo, rows.row_hi[n][c] = hi;      // (rows without a part see what the others see; their results go nowhere)
                if (a.seq_q > 1) {
                    int of, head_of;
                    place_of(column, of, head_of);
                    if (column < a.rows && of < window.len_q) {
                        window_of_tokens(a, window, of, of, rows.row_lo[n][c], rows.row_hi[n][c]);
                        any_lo = min(any_lo, rows.row_lo[n][c]);
                        any_hi = max(any_hi, rows.row_hi[n][c]);
                    }
                    rows.row_hi[n][c] = max(rows.row_hi[n][c], rows.row_lo[n][c]);
                    common_lo = max(common_lo, rows.row_lo[n][c]);
                    common_hi = min(common_hi, rows.row_hi[n][c]);
                }
                rows.largest[n][c] = -INFINITY;
                rows.sum[n][c] = 0.0f;
            }
        }
        if (a.seq_q > 1) {
            common_lo = __reduce_max_sync(0xffffffffu, common_lo), common_hi = __reduce_min_sync(0xffffffffu, common_hi);
            any_lo = __reduce_min_sync(0xffffffffu, any_lo), any_hi = __reduce_max_sync(0xffffffffu, any_hi);
        } else {
            any_lo = lo, any_hi = hi;
        }
        rows.unit = rows.most = kNoUnit;
#pragma unroll
        for (int j = 0; j < kWide; ++j)
#pragma unroll
            for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) rows.o[j][n][c] = 0.0f;

        bool ok = true;
#pragma unroll 1
        for (int u = 0; u < take; ++u) {
            if (u % kAhead == 0) code[0] = code_next[0], code[1] = code_next[1];
            float k_scale[2];
            int v_scale[2];
            const int key0 = (unit0 + u) * kUnit;
            bool special = key0 < common_lo || key0 + kUnit > common_hi;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int k_code = __shfl_sync(0xffffffffu, code[0], (u % kAhead) * 2 + r);
                v_scale[r] = __shfl_sync(0xffffffffu, code[1], (u % kAhead) * 2 + r);
                k_scale[r] = k_code < 0 ? -1.0f : decode_e8m0(static_cast<uint32_t>(k_code));
                special = special || k_code < 0 || static_cast<uint32_t>(v_scale[r]) > 254u;
            }
            const bool seen = key0 < any_hi && key0 + kUnit > any_lo;
            uint32_t p[2][EIGHTS][2];
            const int k_slot = (tiles + 2 * u) % S::kSlots, v_slot = (tiles + 2 * u + 1) % S::kSlots;
            ok = mbar_wait_warp(bars + 8u * k_slot, ((tiles + 2 * u) / S::kSlots) & 1, 702);
            if (!ok) break;
            if (seen) {
                if (special) rows.template scores<true>(ring_data + k_slot * S::kSide, k_scale, key0, p);
                else rows.template scores<false>(ring_data + k_slot * S::kSide, k_scale, key0, p);
            }
            __syncwarp();
            fetch(2 * u + S::kSlots);
            ok = mbar_wait_warp(bars + 8u * v_slot, ((tiles + 2 * u + 1) / S::kSlots) & 1, 703);
            if (!ok) break;
            if (seen) {
                if (special) rows.template values<true>(ring_data + v_slot * S::kSide, v_scale, key0, lo, hi, a.seq_q > 1, p);
                else rows.template values<false>(ring_data + v_slot * S::kSide, v_scale, key0, lo, hi, false, p);
            }
            __syncwarp();
            fetch(2 * u + 1 + S::kSlots);
        }
        if (!ok || g_device_status != 0) {
            // A wait gave up, here or elsewhere: what is on its way comes first, so that nothing lands in another CTA's shared memory (each of these waits is
            // bounded too).
            for (int s = 0; s < S::kSlots && !ok; ++s) {
                mbar_wait_warp(bars + 8u * s, 0, 704);
                mbar_wait_warp(bars + 8u * s, 1, 704);
            }
            return;
        }

        const float absolute = rows.unit == kNoUnit ? 1.0f : decode_e8m0(static_cast<uint32_t>(rows.unit));
#pragma unroll
        for (int n = 0; n < EIGHTS; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) rows.sum[n][c] += __shfl_xor_sync(0xffffffffu, rows.sum[n][c], x);
                const int row = row_first + n * 8 + quad * 2 + c;
                if (row >= a.rows) continue;
                // The sum goes first: O alone carries the probabilities' 2^15 and as many values as there are keys, which V far above one takes past f32's range.
                const float top = rows.largest[n][c], total = rows.sum[n][c], inverse = total == 0.0f ? 1.0f : 1.0f / total;
                if (!whole) {
                    float* partial = a.partial + (static_cast<int64_t>(part * 2 + (first_piece ? 0 : 1)) * a.block_rows + (row - row_first)) * (D + 2);
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        *reinterpret_cast<float2*>(partial + Rows::channel_of(j, eighth)) = make_float2(rows.o[j][n][c] * inverse * absolute, rows.o[j][n][c + 2] * inverse * absolute);
                    if (eighth == 0) *reinterpret_cast<float2*>(partial + D) = make_float2(top, total);
                } else {
                    int token, head_q;
                    place_of(row, token, head_q);
                    const bool none = token >= window.len_q || total == 0.0f;   // (a NaN sum is a NaN result)
                    const int64_t at = batch * a.o_stride[0] + head_q * a.o_stride[1] + token * a.o_stride[2];
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
                        store_pair(a, at + Rows::channel_of(j, eighth), none ? 0.0f : rows.o[j][n][c] * inverse * absolute, none ? 0.0f : rows.o[j][n][c + 2] * inverse * absolute);
                    if (eighth == 0 && a.stats)
                        a.stats[batch * a.stats_stride[0] + head_q * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : top * kLn2 + logf(total * 0x1p-15f);
                }
            }
        tiles += 2 * take;
        left -= take;
        if (left == 0) return;
        offset = 0;
        first_piece = false;
        if (++head == a.heads_kv) head = 0, ++entry, units = 0;
    }
}

// Loads where it stands: left to itself, the compiler moves each load of a run of them down to its use, and they come one after the other.
__device__ __forceinline__ float2 load_now(const float* p) {
    float2 v;
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(__cvta_generic_to_global(p)) : "memory");
    return v;
}

// A CTA a row: the rows of lists that were cut, and of those without keys. Latency-bound, so each warp has eight parts on their way at a time.
template <int D>
__global__ void __launch_bounds__(D)
cache_sdpa_merge_kernel(const __grid_constant__ CacheSdpaArgs a) {
    constexpr int kWarpsHere = D / 32, kOwn = D / 32, kAhead = D == 256 ? 4 : 8;   // channels a lane, parts on their way a warp
    __shared__ float2 meeting[kWarpsHere];
    __shared__ __align__(16) float values[kWarpsHere][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int list = divided(static_cast<int>(blockIdx.x), a.by_rows), in_rows = static_cast<int>(blockIdx.x) - list * a.rows, token = divided(in_rows, a.by_group);
    const int64_t batch = divided(list, a.by_heads);
    const int head_kv = list - static_cast<int>(batch) * a.heads_kv, head = head_kv * a.group + (in_rows - token * a.group);
    const int block = in_rows >> (a.block_rows == 8 ? 3 : 4), row = in_rows - block * a.block_rows, entry = static_cast<int>(batch) * a.row_blocks + block;
    chain_begin();
    if (!wanted(a)) return;
    const int per = a.starts[0], start = a.starts[1 + static_cast<int64_t>(entry) * a.heads_kv + head_kv];   // (written where the list has keys)
    int lo, hi;
    const int units = units_of(a, entry, lo, hi);
    const bool takes_part = token < sequence_window(a, batch).len_q;
    // A part has its own O, which counts by its sum. Sums are at most 2^15 for each key: taken by a power of two above them all, no sum of values passes the largest of V.
    const int keys_log2 = 32 - __clz(units * kUnit);
    const float share = power_of_two(-15 - keys_log2);
    float top = -INFINITY, total = 0.0f, value[kOwn];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) value[e] = 0.0f;
    if (units > 0) {
        if (start < 0) return;   // not cut: its CTA has written O
        const int first = start / per, parts = (start + units - 1) / per - first + 1;
        const bool second_place = start != first * per;   // of the first part in its CTA
        // Each warp takes every fourth (eighth) part, with all channels; they meet below.
        for (int i0 = warp; i0 < parts; i0 += kWarpsHere * kAhead) {
            float2 pair[kAhead];
            float ahead[kAhead][kOwn];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = min(i0 + k * kWarpsHere, parts - 1);
                const float* part = a.partial + (static_cast<int64_t>((first + i) * 2 + (i == 0 && second_place ? 1 : 0)) * a.block_rows + row) * (D + 2);
                pair[k] = load_now(part + D);
#pragma unroll
                for (int e = 0; e < kOwn; e += 2) {
                    const float2 v = load_now(part + lane * kOwn + e);
                    ahead[k][e] = v.x, ahead[k][e + 1] = v.y;
                }
            }
            float largest = top;
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (i0 + k * kWarpsHere < parts) largest = fmaxf(largest, pair[k].x);
            const float down = top == -INFINITY ? 1.0f : exp2_of(top - largest);   // (no score above -inf: zeros, or NaNs that are to be seen)
            total *= down;
#pragma unroll
            for (int e = 0; e < kOwn; ++e) value[e] *= down;
            top = largest;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (i0 + k * kWarpsHere >= parts) continue;
                const float weight = pair[k].y * share * (pair[k].x == -INFINITY ? 1.0f : exp2_of(pair[k].x - largest));
                total += weight;
#pragma unroll
                for (int e = 0; e < kOwn; ++e) value[e] = fmaf(ahead[k][e], weight, value[e]);
            }
        }
    }
    if (lane == 0) meeting[warp] = make_float2(top, total);
#pragma unroll
    for (int e = 0; e < kOwn; e += 2) *reinterpret_cast<float2*>(&values[warp][lane * kOwn + e]) = make_float2(value[e], value[e + 1]);
    __syncthreads();
    float result = 0.0f;
    top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarpsHere; ++w) top = fmaxf(top, meeting[w].x);
#pragma unroll
    for (int w = 0; w < kWarpsHere; ++w) {
        const float weight = meeting[w].x == -INFINITY ? 1.0f : exp2_of(meeting[w].x - top);
        total = fmaf(meeting[w].y, weight, total);
        result = fmaf(values[w][threadIdx.x], weight, result);
    }
    const bool none = !takes_part || total == 0.0f;
    store_from_f32(a.o, a.o_type, batch * a.o_stride[0] + head * a.o_stride[1] + token * a.o_stride[2] + threadIdx.x, none ? 0.0f : result / total);
    if (threadIdx.x == 0 && a.stats) a.stats[batch * a.stats_stride[0] + head * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : top * kLn2 + logf(total * power_of_two(keys_log2));
}

struct StreamPlan {
    int eights, block_rows, row_blocks;
    int64_t rows, units, grid, starts, scratch;   // units: the most there can be; starts: integers before the partial results
};

StreamPlan plan_stream(const dfgpu_cache_sdpa_params& p) {
    StreamPlan plan{};
    const int64_t d = p.q.dim[3], group = p.q.dim[1] / p.k.dim[1];
    plan.rows = group * p.q.dim[2];
    // With 64 channels two eights of rows share the conversions of a unit (16 rows, 64 sequences, 8 KV heads, 2000 keys: 54 us, 65 in eights; 40 rows: 33 and 32);
    // with more their registers cost what that gains (128 channels, 16 rows, 24 sequences, 4000 keys: 73 and 70 us, 40 rows: 66 and 60, 64 rows: 81 and 83;
    // 256 channels, 2000 rows: 831 and 773).
    plan.eights = plan.rows > 8 && d == 64 ? 2 : 1;
    plan.block_rows = plan.eights * 8;
    plan.row_blocks = static_cast<int>((plan.rows + plan.block_rows - 1) / plan.block_rows);
    const int64_t lists = p.q.dim[0] * p.k.dim[1] * plan.row_blocks, units = (p.s_kv + kUnit - 1) / kUnit;
    plan.units = lists * units;
    const int64_t ctas = kSms * (d == 256 ? 2 : plan.eights == 1 ? 4 : 3);   // (Shape::kCtas)
    plan.grid = std::min(ctas, (plan.units + kLeastUnits - 1) / kLeastUnits);
    plan.starts = (1 + lists + 3) / 4 * 4;
    plan.scratch = plan.starts * 4 + plan.grid * kWarps * 2 * plan.block_rows * (d + 2) * 4;
    return plan;
}

// The tcgen05 form has blocks of 256 rows, an SM for each piece of their keys; the streaming form cuts any shape evenly but runs at a fourth to a seventh of
// its rate. Streaming and tcgen05: 1000 tokens of 4 query heads, 8 KV heads, 2000 keys, 128 pieces: 283 and 102 us; 40 of 8, 8 heads, 2000 keys, 32 pieces: 46 and 40;
// 64 of 4, 2 heads, 4000 keys, 14 pieces: 34 and 38; 32 of 4, one head, 1100 keys, 2 pieces: 22 and 28.
// Of 256 rows few may be there: 16 rows, 24 sequences, 8 heads, 4000 keys: 70 and 121 us; 32 rows, 16 sequences: 84 and 82; 40 rows, 16 sequences, 4 heads: 60 and 53; 64 rows: 83 and
// 57; 96 rows, 4 sequences, 8 heads, 8000 keys: 104 and 56.
bool umma_pays(const dfgpu_cache_sdpa_params& p, const StreamPlan& plan) { return plan.rows >= 32 && 7 * cache_sdpa_umma_items(p) * cache_sdpa_umma_pieces(p) >= kSms; }
int64_t flag_count(const dfgpu_cache_sdpa_params& p) { return cache_sdpa_umma_items(p) * cache_sdpa_umma_pieces(p); }
int64_t flag_bytes(const dfgpu_cache_sdpa_params& p, int kernel) { return kernel == DFGPU_CACHE_SDPA_UMMA ? (flag_count(p) + 3) / 4 * 16 : 0; }

bool on_16(const void* pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 15u) == 0; }

int check_side(const dfgpu_cache_sdpa_params& p, const dfgpu_tensor& cache, const dfgpu_tensor& scale, const dfgpu_tensor& table, const char* name) {
    if (!valid_tensor(cache) || cache.rank != 4 || cache.dtype != DFGPU_E4M3 || cache.dim[3] != p.q.dim[3]) return fail(kInvalidShape, "CACHE_SDPA: the container of %s must be FP8_E4M3 [pages, Hk, T, D]", name);
    if (cache.dim[1] != p.k.dim[1] || cache.dim[2] != p.k.dim[2]) return fail(kInvalidShape, "CACHE_SDPA: the containers differ in heads or tokens a page");
    if (cache.stride[3] != 1) return fail(kInvalidLayout, "CACHE_SDPA: the head dimension of a container must have unit stride");
    for (int i = 0; i < 3; ++i)
        if (cache.dim[i] > 1 && (cache.stride[i] <= 0 || cache.stride[i] % 16 != 0 || cache.stride[i] >= (1ll << 40)))
            return fail(kInvalidLayout, "CACHE_SDPA: the strides of the container of %s must be positive multiples of 16", name);
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
    for (int i = 0; i < 3 && p.stats.rank; ++i)
        if (p.stats.dim[i] > 1 && p.stats.stride[i] == 0) return fail(kInvalidLayout, "CACHE_SDPA: Stats overlaps itself");
    if (!std::isfinite(p.attn_scale)) return fail(kInvalidValue, "CACHE_SDPA: the attention scale must be finite");
    const StreamPlan plan = plan_stream(p);
    if (p.q.dim[2] >= (1ll << 30) || p.q.dim[0] * p.k.dim[1] * plan.rows >= (1ll << 31) || plan.units >= (1ll << 30)) return fail(kUnsupported, "CACHE_SDPA: too many sequences, heads or query rows");
    if (p.kernel < DFGPU_CACHE_SDPA_AUTO || p.kernel > DFGPU_CACHE_SDPA_UMMA) return fail(kInvalidArgument, "CACHE_SDPA: unknown kernel id %d", p.kernel);
    const bool umma = cache_sdpa_umma_supported(p);
    if (p.kernel == DFGPU_CACHE_SDPA_UMMA && !umma) return fail(kUnsupported, "CACHE_SDPA: the tcgen05 kernel needs a head dimension of 64 or 128 and at most 128 query heads a KV head");
    kernel = p.kernel != DFGPU_CACHE_SDPA_AUTO ? p.kernel : umma && umma_pays(p, plan) ? DFGPU_CACHE_SDPA_UMMA : DFGPU_CACHE_SDPA_STREAM;
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

template <typename T, int D, int EIGHTS>
int launch_rows(const CUtensorMap& map_k, const CUtensorMap& map_v, const CacheSdpaArgs& a, dim3 grid, cudaStream_t stream) {
    constexpr int kBytes = Shape<D, EIGHTS>::kDynamic;
    const auto kernel = cache_sdpa_stream_kernel<T, D, EIGHTS>;
    const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (error != cudaSuccess) return fail(kExecutionFailed, "CACHE_SDPA: cannot reserve %d bytes of shared memory: %s", kBytes, cudaGetErrorString(error));
    launch_chained(kernel, grid, dim3(kThreads), kBytes, stream, map_k, map_v, a);
    return check_launch("CACHE_SDPA");
}

template <typename T, int D>
int launch_stream(const CUtensorMap& map_k, const CUtensorMap& map_v, const CacheSdpaArgs& a, const StreamPlan& plan, dim3 grid, cudaStream_t stream) {
    int status;
    if constexpr (D == 64) status = plan.eights == 1 ? launch_rows<T, D, 1>(map_k, map_v, a, grid, stream) : launch_rows<T, D, 2>(map_k, map_v, a, grid, stream);
    else status = launch_rows<T, D, 1>(map_k, map_v, a, grid, stream);
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
    info->launches = kernel != DFGPU_CACHE_SDPA_UMMA ? 2 : cache_sdpa_umma_pieces(*p) == 1 ? 3 : 4;
    // (the two forms' partial results take turns)
    info->scratch_bytes = flag_bytes(*p, kernel) + std::max(plan.scratch, kernel == DFGPU_CACHE_SDPA_UMMA ? cache_sdpa_umma_partial_bytes(*p) : 0);
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
    // (what the tcgen05 form leaves to the streaming form reads Q again after O has been written)
    if (tensors[0] == tensors[3]) return fail(kInvalidArgument, "CACHE_SDPA: O is Q");
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
    a.by_group = make_fast_divisor(static_cast<uint32_t>(a.group));
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
    a.by_rows = make_fast_divisor(static_cast<uint32_t>(a.rows));
    a.by_heads = make_fast_divisor(static_cast<uint32_t>(a.heads_kv));
    a.by_row_blocks = make_fast_divisor(static_cast<uint32_t>(a.row_blocks));
    const int64_t flags = flag_bytes(*p, kernel);
    a.starts = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(scratch) + flags);
    a.partial = reinterpret_cast<float*>(a.starts + plan.starts);
    a.box = a.page % 32 == 0 ? 32 : 16;
    CUtensorMap map_k, map_v;
    int made = make_side_map(&map_k, p->k, tensors[1], a.box);
    if (!made) made = make_side_map(&map_v, p->v, tensors[2], a.box);
    if (made) return made;
    const dim3 grid(static_cast<unsigned>(plan.grid));
    cudaStream_t on = as_stream(stream);
    if (kernel == DFGPU_CACHE_SDPA_UMMA) {
        const int launched = launch_cache_sdpa_umma(*p, a, static_cast<int32_t*>(scratch), reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + flags), on);
        if (launched) return launched;
        a.only_if = static_cast<const int32_t*>(scratch);
        a.only_if_count = static_cast<int>(flag_count(*p));
    }
    const bool half = p->q.dtype == DFGPU_F16;
    switch (p->q.dim[3]) {
        case 64: return half ? launch_stream<__half, 64>(map_k, map_v, a, plan, grid, on) : launch_stream<__nv_bfloat16, 64>(map_k, map_v, a, plan, grid, on);
        case 128: return half ? launch_stream<__half, 128>(map_k, map_v, a, plan, grid, on) : launch_stream<__nv_bfloat16, 128>(map_k, map_v, a, plan, grid, on);
        default: return half ? launch_stream<__half, 256>(map_k, map_v, a, plan, grid, on) : launch_stream<__nv_bfloat16, 256>(map_k, map_v, a, plan, grid, on);
    }
}

namespace dfgpu {
int cache_sdpa_device_status(int* status) {
    int own = 0, umma = 0;
    int code = read_and_clear_device_status(&own);
    if (!code) code = cache_sdpa_umma_device_status(&umma);
    *status = own ? own : umma;
    return code;
}
}  // namespace dfgpu
