// Attention over a paged cache of E4M3 codes with E8M0 scales: the streaming form, for few query rows a KV head (single tokens,
// drafted tokens) and for every type and head dimension.
//
// Bound by HBM: each held code is read once for all query heads of its KV head. A row of the products is a (token, head) pair,
// 16 rows an M tile. Codes are exact in f16 (448 to 2^-9), so K and V go from shared memory through one convert for two codes
// straight into the register operands of mma.sync.m16n8k16: a tcgen05 product wants its operands in shared memory, and writing the
// converted tile there and reading it back is 144 bytes of shared-memory traffic a clock at HBM speed, where the port moves 128.
// With 16 rows the tensor cores have 16 multiply-adds for each code, 384 a clock and SM at HBM speed.
//   * Q is not rounded: each row is scaled by a power of two that puts its largest magnitude at 2^14, and is exact in f16 down to
//     2^-38 of that (below, within 2^-39 of it).
//   * 16 consecutive keys share a page and a scale (both are multiples of 16 tokens). The K scale multiplies their scores. O is
//     held in units of a power of two, 2^unit: the V scale of 16 keys goes into their probabilities, as 2^(scale - unit), where that is from 2^-10
//     to 1, and else the unit moves and O with it (exactly, as far as scales within 2^80 of one another go).
//   * Probabilities are rounded to f16 as p * 2^15: 11 bits down to 2^-29 (2^-19 beside a V scale of 2^-10 units), where p is measured
//     against the largest score so far.
// Channels and keys may go to any k index of a product as long as both operands agree; the ones taken here give each thread 16-byte
// reads without bank conflicts: of K 32 consecutive channels of a key, of V 16 consecutive channels of four keys, and of O 32
// consecutive channels of a row.
// CTA: one (sequence, KV head, block of rows), a run of key tiles; a fifth warp brings the tiles by TMA (whole pages or runs of them,
// swizzled) into a ring, four share each tile's keys out between them, or its rows where there are more than 16, or
// both. Two CTAs fit on an SM. More than one run of key tiles a sequence leaves partial results that a second kernel merges.
#include <algorithm>
#include <cmath>

#include "cache_sdpa.cuh"
#include "dfgpu_cache.h"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

constexpr int kWarps = 4, kConsumers = 128, kThreads = 160;
constexpr int kMostTiles = 32;     // key tiles a CTA
constexpr float kUp = 15.0f;       // probabilities are held as p * 2^15
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kNoUnit = -100000;   // O is zero and has no unit yet
constexpr int kNaN = 0x7fc00000;

template <int D>
struct Shape {
    static constexpr int kKeys = D == 256 ? 64 : 128;     // keys a tile
    static constexpr int kRuns = kKeys / 16;
    static constexpr int kTile = kKeys * D;               // bytes of a K or V tile
    static constexpr int kCtas = D == 256 ? 1 : 2;        // on an SM: a D of 256 takes 255 registers a thread
    static constexpr int kStages = D == 64 ? 4 : 3 * (3 - kCtas);
    static constexpr int kRing = kStages * 2 * kTile;
    static constexpr int kKScales = kRing;                                    // [runs] f32, -1: the page's rows read as zeros
    static constexpr int kVScales = kKScales + kMostTiles * kRuns * 4;        // [runs] the code, -1 likewise
    static constexpr int kBarriers = kVScales + kMostTiles * kRuns * 4;       // full[stages], empty[stages]
    static constexpr int kTotal = kBarriers + 2 * kStages * 8;
    static constexpr int kDynamic = kTotal + 1024;
};

// Byte offset of a 16-byte chunk of a tile's row, as TMA lays rows of 128 or 64 bytes out (a D of 256: two halves): the reads above meet each bank once.
template <int D>
__device__ __forceinline__ uint32_t at_chunk(int row, int chunk) {
    return D == 64 ? row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4) : (chunk >> 3) * (Shape<D>::kKeys * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
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
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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

// `count` (8 or 16) neighbouring values of a row of O.
template <int COUNT>
__device__ __forceinline__ void store_values(const CacheSdpaArgs& a, int64_t at, const float (&v)[COUNT]) {
    if (a.o_vector) {
        if (a.o_type == DFGPU_F32) {
#pragma unroll
            for (int i = 0; i < COUNT; i += 4) *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
            uint32_t words[COUNT / 2];
#pragma unroll
            for (int i = 0; i < COUNT; i += 2)
                words[i / 2] = a.o_type == DFGPU_F16 ? two_halves(v[i], v[i + 1]) : static_cast<uint32_t>(f32_to_bf16_bits(v[i])) | static_cast<uint32_t>(f32_to_bf16_bits(v[i + 1])) << 16;
#pragma unroll
            for (int i = 0; i < COUNT / 2; i += 4)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + at + 2 * i) = make_uint4(words[i], words[i + 1], words[i + 2], words[i + 3]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < COUNT; ++i) store_from_f32(a.o, a.o_type, at + i, v[i]);
}

// The page of a tile's key in a side's table, -1 where there is none.
__device__ __forceinline__ int page_of(const CacheSdpaArgs& a, const CacheSide& s, int64_t batch, int slot) {
    if (slot >= s.table_len) return -1;
    const int page = s.table[batch * s.table_batch + slot * s.table_slot];
    return page >= 0 && page < s.pages ? page : -1;
}

// 16 rows of one M tile against the codes of K and V that its warp takes.
template <int D>
struct RowTile {
    static constexpr int kDeep = D / 16;                     // products along the channels
    static constexpr int kWide = D / 8;                      // products along the channels of V: thread value j
    static constexpr int kReach = D == 64 ? 8 : 16;          // consecutive channels that a thread reads of a V row
    uint32_t q[kDeep][4];
    float factor[2];            // of a score: 1 / the row's power of two, attention scale, log2(e)
    int row_lo[2], row_hi[2];   // keys that the thread's two rows see
    float largest[2], sum[2];
    float o[kWide][4];
    int unit;

    // KEYS keys from row `row` of a tile, key0 of the sequence. SPECIAL: some row does not see all of them, or a page or scale is none.
    template <bool SPECIAL, int KEYS>
    __device__ __forceinline__ void step(const uint8_t* k_tile, const uint8_t* v_tile, const float* k_scales, const int* v_scales, int row, int key0, int lo, int hi, bool mixed) {
        const int lane = threadIdx.x & 31, quad = lane & 3, eighth = lane >> 2;
        constexpr int kRuns = KEYS / 16;
        float s[KEYS / 8][4];   // scores: 8 keys a product, keys along its columns
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
            for (int u = 0; u < kDeep / 4; ++u) {
                const uint4 raw = read_16(k_tile + at_chunk<D>(row + n * 8 + eighth, D == 64 ? quad : quad * 2 + (u & 1) + (u >> 1) * 8));
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t b0, b1;
                    four_codes(w[i], b0, b1);
                    if (u + i == 0) multiply_first(s[n], q[0], b0, b1);
                    else multiply(s[n], q[u * 4 + i], b0, b1);
                }
            }
        }
        bool above = false;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) {
            const float k_scale = k_scales[n >> 1];
            const float f0 = factor[0] * k_scale, f1 = factor[1] * k_scale;
            s[n][0] *= f0, s[n][1] *= f0, s[n][2] *= f1, s[n][3] *= f1;
            if (SPECIAL) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = key0 + n * 8 + quad * 2 + (c & 1);
                    if (k_scale < 0.0f) s[n][c] = 0.0f;
                    if (static_cast<uint32_t>(key - row_lo[c >> 1]) >= static_cast<uint32_t>(row_hi[c >> 1] - row_lo[c >> 1])) s[n][c] = -INFINITY;
                }
            }
            above = above || fmaxf(s[n][0], s[n][1]) > largest[0] || fmaxf(s[n][2], s[n][3]) > largest[1];
        }
        if (__any_sync(0xffffffffu, above)) {   // a new largest score in some row (rare after the first tiles)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float top = largest[half];
#pragma unroll
                for (int n = 0; n < KEYS / 8; ++n) top = fmaxf(top, fmaxf(s[n][2 * half], s[n][2 * half + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float down = top == -INFINITY ? 1.0f : exp2_of(largest[half] - top);
                largest[half] = top;
                sum[half] *= down;
#pragma unroll
                for (int j = 0; j < kWide; ++j) o[j][2 * half] *= down, o[j][2 * half + 1] *= down;
            }
        }
        const float from0 = largest[0] == -INFINITY ? 0.0f : kUp - largest[0], from1 = largest[1] == -INFINITY ? 0.0f : kUp - largest[1];
        uint32_t p[kRuns][4];
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) {
            const float p0 = exp2_of(s[n][0] + from0), p1 = exp2_of(s[n][1] + from0), p2 = exp2_of(s[n][2] + from1), p3 = exp2_of(s[n][3] + from1);
            sum[0] += p0 + p1;
            sum[1] += p2 + p3;
            p[n >> 1][(n & 1) * 2] = two_halves(p0, p1);
            p[n >> 1][(n & 1) * 2 + 1] = two_halves(p2, p3);
        }
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
            const int code = v_scales[r], apart = code - unit;   // (the same in all threads)
            if ((!SPECIAL || (code >= 0 && code != 255)) && apart != 0) {
                if (apart < 0 && (apart >= -10 || apart < -80)) {
                    const uint32_t less = apart < -80 ? 0u : static_cast<uint32_t>(15 + apart) << 10, both = less | less << 16;
#pragma unroll
                    for (int c = 0; c < 4; ++c) p[r][c] = times(p[r][c], both);
                } else {
                    const float to = unit == kNoUnit ? 1.0f : power_of_two(max(-apart, -126));
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[j][c] *= to;
                    unit = code;
                }
            }
            // V: thread value j of a run is channel 16 * eighth + j of keys 2 quad, 2 quad + 1 and those plus 8
            uint32_t w[4][kWide / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = row + r * 16 + quad * 2 + (k & 1) + (k >> 1) * 8;
                if constexpr (D == 64) {
                    const uint2 raw = *reinterpret_cast<const uint2*>(v_tile + at_chunk<D>(at, eighth >> 1) + (eighth & 1) * 8);
                    w[k][0] = raw.x, w[k][1] = raw.y;
                } else {
#pragma unroll
                    for (int u = 0; u < kWide / 16; ++u) {
                        const uint4 raw = read_16(v_tile + at_chunk<D>(at, eighth + u * 8));
                        w[k][u * 4] = raw.x, w[k][u * 4 + 1] = raw.y, w[k][u * 4 + 2] = raw.z, w[k][u * 4 + 3] = raw.w;
                    }
                }
                if (SPECIAL) {   // rows that nothing was brought to, or that no row sees: anything may lie there, NaN codes too
                    const int key = key0 + r * 16 + quad * 2 + (k & 1) + (k >> 1) * 8;
                    if (code < 0 || key < lo || key >= hi) {
#pragma unroll
                        for (int i = 0; i < kWide / 4; ++i) w[k][i] = 0;
                    }
                }
            }
            if (SPECIAL) {
                const int run0 = key0 + r * 16;
                const bool sees[2] = {run0 < row_hi[0] && run0 + 16 > row_lo[0], run0 < row_hi[1] && run0 + 16 > row_lo[1]};
                if (code == 255) {   // a scale that is a NaN: for the rows that see one of its keys
#pragma unroll
                    for (int j = 0; j < kWide; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (sees[c >> 1]) o[j][c] = __int_as_float(kNaN);
                }
                if (mixed) {
                    // A NaN code must reach the rows that see its key and no others, whose probability for it is 0: such codes become zeros in the
                    // products, and NaNs in the sums of the rows that they belong to.
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < kWide / 4; ++i) {
                            const uint32_t found = ((w[k][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                            w[k][i] &= ~((found >> 7) * 0xffu);
                            nan |= found;
                        }
                    if (__any_sync(0xffffffffu, nan != 0)) {
#pragma unroll 1
                        for (int k = 0; k < 16; ++k) {
                            const bool in0 = run0 + k >= row_lo[0] && run0 + k < row_hi[0], in1 = run0 + k >= row_lo[1] && run0 + k < row_hi[1];
#pragma unroll
                            for (int j = 0; j < kWide; ++j)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    const int channel = (quad * 2 + c) * kReach + (j & (kReach - 1)) + (j / kReach) * 128;
                                    const uint8_t found = v_tile[at_chunk<D>(row + r * 16 + k, channel >> 4) + (channel & 15)];
                                    if ((found & 0x7fu) == 0x7fu) {
                                        if (in0) o[j][c] = __int_as_float(kNaN);
                                        if (in1) o[j][2 + c] = __int_as_float(kNaN);
                                    }
                                }
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kWide / 4; ++i) {
                uint32_t first[4], second[4];
                four_codes(__byte_perm(w[0][i], w[1][i], 0x5140), first[0], first[1]);
                four_codes(__byte_perm(w[0][i], w[1][i], 0x7362), first[2], first[3]);
                four_codes(__byte_perm(w[2][i], w[3][i], 0x5140), second[0], second[1]);
                four_codes(__byte_perm(w[2][i], w[3][i], 0x7362), second[2], second[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) multiply(o[i * 4 + e], p[r], first[e], second[e]);
            }
        }
    }
};

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kThreads, Shape<D>::kCtas)
cache_sdpa_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CacheSdpaArgs a) {
    using S = Shape<D>;
    using Rows = RowTile<D>;
    constexpr int kGroups = kWarps / MT;              // warps that share an M tile's keys
    constexpr int kOwn = S::kKeys / kGroups;          // keys a warp and tile
    constexpr int kStep = kOwn < 32 ? kOwn : 32;      // keys at a time
    constexpr int kWide = Rows::kWide, kReach = Rows::kReach;
    extern __shared__ uint8_t raw_smem[];
    const uint32_t ring = (smem_u32(raw_smem) + 1023u) & ~1023u;
    uint8_t* smem = raw_smem + (ring - smem_u32(raw_smem));
    float* k_scales = reinterpret_cast<float*>(smem + S::kKScales);
    int* v_scales = reinterpret_cast<int*>(smem + S::kVScales);
    auto full = [&](int s) { return ring + S::kBarriers + 8u * s; };
    auto empty = [&](int s) { return ring + S::kBarriers + 8u * (S::kStages + s); };
    const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
    const int head = blockIdx.y % a.heads_kv, row_block = blockIdx.y / a.heads_kv;
    const int64_t batch = blockIdx.z;
    const int row_first = row_block * (MT * 16);
    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    chain_begin();

    const int chunk_first = static_cast<int>(blockIdx.x) * a.tiles_per_cta;
    if (warp == kWarps) {
        // The loader: lane l brings one box of a tile, `box` rows (a page or a part of one) of K or V by 128 or 64 bytes. Page ids are read a tile ahead of
        // their use, and the first ones before the lengths are known.
        constexpr int kHalves = D == 256 ? 2 : 1;
        const int boxes = S::kKeys / a.box, side = lane / (boxes * kHalves), within = lane % (boxes * kHalves);
        const bool has_box = side < 2;
        const CacheSide& s = a.side[has_box ? side : 0];
        const int box_row = (within / kHalves) * a.box, half = within % kHalves;
        const uint32_t box_bytes = static_cast<uint32_t>(a.box) * (D == 64 ? 64u : 128u);
        const uint32_t to = side * S::kTile + half * (S::kKeys * 128) + box_row * (D == 64 ? 64 : 128);
        auto locate = [&](int tile, int& page, int& token) {
            const int key = tile * S::kKeys + box_row, slot = static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page));
            token = key - slot * a.page;
            page = has_box ? page_of(a, s, batch, slot) : -1;
        };
        int page, token;
        locate(chunk_first, page, token);
        const SequenceWindow window = sequence_window(a, batch);
        int lo, hi;
        window_of_tokens(a, window, row_first / a.group, (min(row_first + MT * 16, a.rows) - 1) / a.group, lo, hi);
        const int tile_first = max(chunk_first, lo / S::kKeys), tile_end = hi > lo ? min(chunk_first + a.tiles_per_cta, (hi + S::kKeys - 1) / S::kKeys) : 0;
        if (tile_first != chunk_first && tile_first < tile_end) locate(tile_first, page, token);
        for (int t = 0; t < tile_end - tile_first; ++t) {
            const int key = (tile_first + t) * S::kKeys + box_row;
            const bool live = page >= 0 && key < hi && key + a.box > lo;
            const int now_page = page, now_token = token;
            if (tile_first + t + 1 < tile_end) locate(tile_first + t + 1, page, token);
            const int slot = t % S::kStages;
            if (!mbar_wait_warp(empty(slot), ((t / S::kStages) & 1) ^ 1, 701)) break;
            const uint32_t count = __popc(__ballot_sync(0xffffffffu, live));
            if (lane == 0) mbar_expect_tx(full(slot), count * box_bytes);   // (also the arrival; no byte where no page is)
            __syncwarp();
            if (live) tma_load_4d(ring + slot * (2 * S::kTile) + to, side ? &map_v : &map_k, half * 128, now_token, head, now_page, full(slot));
        }
        return;
    }

    const int quad = lane & 3, eighth = lane >> 2, mt = warp % MT, group = warp / MT;
    const SequenceWindow window = sequence_window(a, batch);
    // The keys that any row of the CTA sees, and this CTA's tiles among them.
    int lo, hi;
    window_of_tokens(a, window, row_first / a.group, (min(row_first + MT * 16, a.rows) - 1) / a.group, lo, hi);
    const int tile_first = max(chunk_first, lo / S::kKeys), tile_end = hi > lo ? min(chunk_first + a.tiles_per_cta, (hi + S::kKeys - 1) / S::kKeys) : 0;
    const int tiles = tile_end - tile_first;
    if (tiles <= 0 && a.chunks > 1) return;   // (the merge knows which chunks a row has)

    // The scales of the runs of 16 keys.
    for (int i = threadIdx.x; i < 2 * tiles * S::kRuns; i += kConsumers) {
        const bool is_v = i >= tiles * S::kRuns;
        const CacheSide& s = a.side[is_v ? 1 : 0];
        const int run = is_v ? i - tiles * S::kRuns : i, key = tile_first * S::kKeys + run * 16;
        const int slot = static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page)), block = static_cast<int>(fast_divide(static_cast<uint32_t>((key - slot * a.page) >> 4), a.by_tokens));
        const int page = key < hi && key + 16 > lo ? page_of(a, s, batch, slot) : -1;
        const int code = page >= 0 ? s.scales[page * s.scale_stride[0] + head * s.scale_stride[1] + block * s.scale_stride[2]] : -1;
        if (is_v) v_scales[run] = code;
        else k_scales[run] = page >= 0 ? decode_e8m0(static_cast<uint32_t>(code)) : -1.0f;
    }

    Rows rows;
    int64_t token_of[2];
    int head_of[2];
    bool live_row[2];           // has a place in O
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int row = row_first + mt * 16 + half * 8 + eighth;
        live_row[half] = row < a.rows;
        const int token = live_row[half] ? row / a.group : 0;
        token_of[half] = token;
        head_of[half] = head * a.group + (live_row[half] ? row - token * a.group : 0);
        const bool takes_part = live_row[half] && token < window.len_q;
        rows.row_lo[half] = lo, rows.row_hi[half] = hi;      // (rows without a part see what the others see; their results go nowhere)
        if (takes_part) window_of_tokens(a, window, token, token, rows.row_lo[half], rows.row_hi[half]);
        rows.row_hi[half] = max(rows.row_hi[half], rows.row_lo[half]);
        const T* from = static_cast<const T*>(a.q) + batch * a.q_stride[0] + head_of[half] * a.q_stride[1] + token * a.q_stride[2];
        float v[Rows::kDeep][4];
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < Rows::kDeep; ++i) {
            const int channel = D == 64 ? quad * 16 + i * 4 : (quad * 2 + ((i >> 2) & 1) + (i >> 3) * 8) * 16 + (i & 3) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[i][e] = live_row[half] ? value_of(from[channel + e]) : 0.0f;
                largest = fmaxf(largest, fabsf(v[i][e]));
            }
        }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        int up = 14 - (static_cast<int>(__float_as_uint(largest) >> 23) - 127);
        up = largest == 0.0f ? 0 : min(max(up, -126), 126);
        const float power = power_of_two(up);
        rows.factor[half] = power_of_two(-up) * a.scale_log2;
#pragma unroll
        for (int i = 0; i < Rows::kDeep; ++i) {
            rows.q[i][half] = two_halves(v[i][0] * power, v[i][1] * power);
            rows.q[i][2 + half] = two_halves(v[i][2] * power, v[i][3] * power);
        }
        rows.largest[half] = -INFINITY;
        rows.sum[half] = 0.0f;
    }
    rows.unit = kNoUnit;
#pragma unroll
    for (int j = 0; j < kWide; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) rows.o[j][c] = 0.0f;
    // What the warp's rows see in common, and what any of them sees.
    const int common_lo = __reduce_max_sync(0xffffffffu, max(rows.row_lo[0], rows.row_lo[1])), common_hi = __reduce_min_sync(0xffffffffu, min(rows.row_hi[0], rows.row_hi[1]));
    const int any_lo = __reduce_min_sync(0xffffffffu, min(rows.row_lo[0], rows.row_lo[1])), any_hi = __reduce_max_sync(0xffffffffu, max(rows.row_hi[0], rows.row_hi[1]));
    asm volatile("bar.sync 1, 128;" ::: "memory");   // the scales are there

    bool ok = true;
    for (int t = 0; t < tiles; ++t) {
        const int slot = t % S::kStages;
        if (ok) ok = mbar_wait_warp(full(slot), (t / S::kStages) & 1, 702);
        if (!ok) break;
        const uint8_t* k_tile = smem + slot * (2 * S::kTile);
        const uint8_t* v_tile = k_tile + S::kTile;
#pragma unroll 1
        for (int at = group * kOwn; at < (group + 1) * kOwn; at += kStep) {
            const int key0 = (tile_first + t) * S::kKeys + at, run = t * S::kRuns + (at >> 4);
            if (key0 >= any_hi || key0 + kStep <= any_lo) continue;
            bool special = key0 < common_lo || key0 + kStep > common_hi;
#pragma unroll
            for (int r = 0; r < kStep / 16; ++r) special = special || k_scales[run + r] < 0.0f || static_cast<uint32_t>(v_scales[run + r]) > 254u;
            if (special) rows.template step<true, kStep>(k_tile, v_tile, k_scales + run, v_scales + run, at, key0, lo, hi, a.seq_q > 1);
            else rows.template step<false, kStep>(k_tile, v_tile, k_scales + run, v_scales + run, at, key0, lo, hi, false);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(slot));
    }
    ok = ok && g_device_status == 0;

    // The warps of an M tile meet: (largest score, sum, O) triples by shared memory, in the order of the fragments, so that each bank
    // is met once. Warp g then has rows and columns of its own: fragment values c with c * groups / 4 == g.
    const float absolute = rows.unit == kNoUnit ? 1.0f : decode_e8m0(static_cast<uint32_t>(rows.unit));
#pragma unroll
    for (int j = 0; j < kWide; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) rows.o[j][c] *= absolute;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        rows.sum[half] += __shfl_xor_sync(0xffffffffu, rows.sum[half], 1);
        rows.sum[half] += __shfl_xor_sync(0xffffffffu, rows.sum[half], 2);
    }
    float top[2] = {rows.largest[0], rows.largest[1]}, total[2] = {rows.sum[0], rows.sum[1]};
    if constexpr (kGroups > 1) {
        asm volatile("bar.sync 1, 128;" ::: "memory");   // (every tile has come and been read)
        float* fragments = reinterpret_cast<float*>(smem);                 // [warp][4 * kWide][32]
        float* meeting = reinterpret_cast<float*>(smem + S::kKScales);     // [warp][half][32][2]
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            meeting[((warp * 2 + half) * 32 + lane) * 2] = rows.largest[half];
            meeting[((warp * 2 + half) * 32 + lane) * 2 + 1] = rows.sum[half];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < kWide; ++j) fragments[((warp * 4 + c) * kWide + j) * 32 + lane] = rows.o[j][c];
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float weight[kGroups][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            top[half] = -INFINITY, total[half] = 0.0f;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) top[half] = fmaxf(top[half], meeting[(((g * MT + mt) * 2 + half) * 32 + lane) * 2]);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const float* other = meeting + (((g * MT + mt) * 2 + half) * 32 + lane) * 2;
                weight[g][half] = other[0] == -INFINITY ? 1.0f : exp2_of(other[0] - top[half]);   // (a group without keys has zeros)
                total[half] = fmaf(other[1], weight[g][half], total[half]);
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (c * kGroups / 4 != group) continue;
#pragma unroll
            for (int j = 0; j < kWide; ++j) {
                float v = 0.0f;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) v = fmaf(fragments[(((g * MT + mt) * 4 + c) * kWide + j) * 32 + lane], weight[g][c >> 1], v);
                rows.o[j][c] = v;
            }
        }
    }
    if (!ok) return;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c * kGroups / 4 != group) continue;
        const int half = c >> 1, column = quad * 2 + (c & 1);
        if (!live_row[half]) continue;
        const bool first_of_row = column == 0;
        const bool takes_part = token_of[half] < window.len_q;
        if (a.chunks > 1) {
            const int64_t row = (batch * a.heads_kv + head) * a.rows + row_first + mt * 16 + half * 8 + eighth;
            float* partial = a.partial + (row * a.chunks + blockIdx.x) * (D + 2);
#pragma unroll
            for (int j = 0; j < kWide; j += 2) {
                const int channel = column * kReach + (j & (kReach - 1)) + (j / kReach) * 128;
                *reinterpret_cast<float2*>(partial + channel) = make_float2(rows.o[j][c], rows.o[j + 1][c]);
            }
            if (first_of_row) *reinterpret_cast<float2*>(partial + D) = make_float2(top[half], total[half]);
        } else {
            const bool none = !takes_part || total[half] == 0.0f;   // (a NaN sum is a NaN result)
            const float inverse = 1.0f / total[half];
#pragma unroll
            for (int j0 = 0; j0 < kWide; j0 += kReach) {
                float v[kReach];
#pragma unroll
                for (int j = 0; j < kReach; ++j) v[j] = none ? 0.0f : rows.o[j0 + j][c] * inverse;
                store_values(a, batch * a.o_stride[0] + head_of[half] * a.o_stride[1] + token_of[half] * a.o_stride[2] + column * kReach + (j0 / kReach) * 128, v);
            }
            if (first_of_row && a.stats)
                a.stats[batch * a.stats_stride[0] + head_of[half] * a.stats_stride[1] + token_of[half] * a.stats_stride[2]] =
                    none ? -INFINITY : top[half] * kLn2 + logf(total[half] * 0x1p-15f);
        }
    }
}

// A CTA a row, a thread a channel. Latency-bound: maxima and sums of the first 32 chunks, a chunk a lane in every warp, and the values of
// the first eight are on their way before the lengths say which of them the row has.
template <int D>
__global__ void __launch_bounds__(D)
cache_sdpa_merge_kernel(const __grid_constant__ CacheSdpaArgs a) {
    constexpr int kAhead = 8;
    const int lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x, list = row / a.rows, batch = list / a.heads_kv;
    const int in_list = static_cast<int>(row - list * a.rows), token = in_list / a.group;
    const int head = static_cast<int>(list - batch * a.heads_kv) * a.group + (in_list - token * a.group);
    const float* base = a.partial + row * a.chunks * (D + 2);
    chain_begin();
    float ahead[kAhead];
#pragma unroll
    for (int c = 0; c < kAhead; ++c) ahead[c] = c < a.chunks ? base[c * (D + 2) + threadIdx.x] : 0.0f;
    float2 first_pair = lane < a.chunks ? *reinterpret_cast<const float2*>(base + lane * (D + 2) + D) : make_float2(-INFINITY, 0.0f);
    const SequenceWindow window = sequence_window(a, batch);
    int lo = 0, hi = 0;
    if (token < window.len_q) window_of_tokens(a, window, token, token, lo, hi);
    const int keys = a.tiles_per_cta * a.tile_keys;
    const int first = lo / keys, end = hi > lo ? (hi + keys - 1) / keys : first;
    auto pair_of = [&](int c) {   // (largest score, sum); a chunk without keys of the row was perhaps not written
        if (c < first || c >= end) return make_float2(-INFINITY, 0.0f);
        return c == lane ? first_pair : *reinterpret_cast<const float2*>(base + c * (D + 2) + D);
    };
    float top = -INFINITY;
    for (int c = lane; c < end; c += 32) top = fmaxf(top, pair_of(c).x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    float total = 0.0f, value = 0.0f;
    for (int c0 = 0; c0 < end; c0 += 32) {
        const float2 pair = pair_of(c0 + lane);
        const float weight = pair.x == -INFINITY ? 1.0f : exp2_of(pair.x - top);   // (no score above -inf: its values are zeros, or NaNs that are to be seen)
        float part = pair.y * weight;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) part += __shfl_xor_sync(0xffffffffu, part, s);
        total += part;
#pragma unroll
        for (int c = 0; c < 32; c += kAhead) {
            if (c0 + c >= end) break;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const float w = __shfl_sync(0xffffffffu, weight, c + k);
                if (c0 + c + k >= first && c0 + c + k < end) value = fmaf(ahead[k], w, value);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int next = c0 + c + kAhead + k;
                if (next >= first && next < end) ahead[k] = base[next * (D + 2) + threadIdx.x];
            }
        }
    }
    const bool none = total == 0.0f;
    store_from_f32(a.o, a.o_type, batch * a.o_stride[0] + head * a.o_stride[1] + token * a.o_stride[2] + threadIdx.x, none ? 0.0f : value / total);
    if (threadIdx.x == 0 && a.stats) a.stats[batch * a.stats_stride[0] + head * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : top * kLn2 + logf(total * 0x1p-15f);
}

struct StreamPlan {
    int row_tiles, row_blocks, tile_keys, tiles_per_cta, chunks;
    int64_t rows, scratch;
};

StreamPlan plan_stream(const dfgpu_cache_sdpa_params& p) {
    StreamPlan plan{};
    const int64_t d = p.q.dim[3], group = p.q.dim[1] / p.k.dim[1];
    plan.rows = group * p.q.dim[2];
    plan.row_tiles = plan.rows <= 16 ? 1 : plan.rows <= 32 ? 2 : 4;
    plan.row_blocks = static_cast<int>((plan.rows + plan.row_tiles * 16 - 1) / (plan.row_tiles * 16));
    plan.tile_keys = d == 256 ? 64 : 128;
    const int64_t tiles = (p.s_kv + plan.tile_keys - 1) / plan.tile_keys, lists = p.q.dim[0] * p.k.dim[1] * plan.row_blocks;
    // Long runs of tiles save prologues and partial results (the more the more rows there are), short ones give a small batch more
    // CTAs: as long as there are three for every two SMs (148: a function of the shape alone, as the scratch is).
    int per_cta = 8 * plan.row_tiles;
    while (per_cta > 1 && 2 * lists * ((tiles + per_cta - 1) / per_cta) < 3 * 148) per_cta /= 2;
    plan.tiles_per_cta = per_cta;
    plan.chunks = static_cast<int>((tiles + per_cta - 1) / per_cta);
    plan.scratch = plan.chunks > 1 ? p.q.dim[0] * p.k.dim[1] * plan.rows * plan.chunks * (d + 2) * 4 : 0;
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
    if (p.q.dim[0] > 65535 || p.k.dim[1] * plan.row_blocks > 65535 || p.q.dim[2] >= (1ll << 30) || p.q.dim[0] * p.k.dim[1] * plan.rows >= (1ll << 31)) return fail(kUnsupported, "CACHE_SDPA: too many sequences, heads or query rows");
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

template <typename T, int D>
int launch_stream(const CUtensorMap& map_k, const CUtensorMap& map_v, const CacheSdpaArgs& a, const StreamPlan& plan, dim3 grid, cudaStream_t stream) {
    auto run = [&](auto kernel) -> int {
        const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kDynamic);
        if (error != cudaSuccess) return fail(kExecutionFailed, "CACHE_SDPA: cannot reserve %d bytes of shared memory: %s", Shape<D>::kDynamic, cudaGetErrorString(error));
        launch_chained(kernel, grid, dim3(kThreads), Shape<D>::kDynamic, stream, map_k, map_v, a);
        return check_launch("CACHE_SDPA");
    };
    const int status = plan.row_tiles == 1 ? run(cache_sdpa_stream_kernel<T, D, 1>) : plan.row_tiles == 2 ? run(cache_sdpa_stream_kernel<T, D, 2>) : run(cache_sdpa_stream_kernel<T, D, 4>);
    if (status || plan.chunks == 1) return status;
    launch_chained(cache_sdpa_merge_kernel<D>, dim3(static_cast<unsigned>(static_cast<int64_t>(grid.z) * a.heads_kv * a.rows)), dim3(D), 0, stream, a);
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
    info->launches = plan.chunks > 1 ? 2 : 1;
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
    if (plan.scratch && (!scratch || !on_16(scratch))) return fail(kInvalidArgument, "CACHE_SDPA: needs the 16-byte aligned scratch dfgpu_query_cache_sdpa reports");
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
    const int64_t o_row = 16 / dtype_bytes(p->o.dtype);
    a.o_vector = on_16(a.o);
    for (int i = 0; i < 3; ++i) a.o_vector = a.o_vector && (p->o.dim[i] == 1 || p->o.stride[i] % o_row == 0);
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
    a.chunks = plan.chunks;
    a.tiles_per_cta = plan.tiles_per_cta;
    a.tile_keys = plan.tile_keys;
    a.partial = static_cast<float*>(scratch);
    // TMA boxes: the most tokens up to 64 that divide a page's
    a.box = a.page % 64 == 0 ? 64 : a.page % 32 == 0 ? 32 : 16;
    CUtensorMap map_k, map_v;
    int made = make_side_map(&map_k, p->k, tensors[1], a.box);
    if (!made) made = make_side_map(&map_v, p->v, tensors[2], a.box);
    if (made) return made;
    const dim3 grid(static_cast<unsigned>(plan.chunks), static_cast<unsigned>(a.heads_kv * plan.row_blocks), static_cast<unsigned>(p->q.dim[0]));
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
