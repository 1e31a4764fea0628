// Attention over the 8-bit paged cache for many query rows a KV head (chunks of prompts, drafted tokens of large groups), on tcgen05.
//
// Bound by the tensor pipe and the exponentials, about 1024 clocks each for 128 rows x 128 keys of 128 channels. The codes have to become f16
// (exactly) before the tensor core can take them, and that is paid once for 256 rows: a CTA has two query tiles of 128 rows, (token, head of the
// group) pairs of one KV head, and both read the same converted K and V tiles.
//   warps 0-3, 4-7   softmax of query tile 0 and 1, a thread a row; Q to f16 at the start, O out of tensor memory at the end
//   warps 8-11, 12-15  codes of K and of V from global memory (looked up and loaded a tile ahead, in registers) to f16 tiles in shared memory, two of each
//   warp 16, 17      issue the products, S = Q K^T and O += P V with P from tensor memory, the two query tiles in turn
// (With four converting warps for both, these set the pace: 6500 clocks a pair of score tiles; with one issuing warp, it did: 75 clocks a product, 3600.)
// Tensor memory: S (then P, in its place) of the query tiles at 0 and 128, O at 256 and 384. S comes in halves of 64 keys, two a query
// tile: the next half's scores are made while a half's softmax is under way, so that no softmax waits for a product (with whole tiles each waited
// 1250 of 4900 clocks), and a half of a row fits a thread's registers, so that scores are read once.
// Q is exact as in the streaming form (a power of two a row). The K scale of 16 keys is a factor of their scores. The V scale is
// part of the exponent: with t = score + log2(V scale), a row's reference r follows the largest t, P = 2^(t - r + 11) in f16 multiplies codes, and the
// row's sum adds up P / (V scale), so nothing but the final division knows of either. r is raised when t passes it by 2^4 (O
// is rescaled in tensor memory then, which is rare).
// What this cannot do exactly it says in a flag of the item, and the streaming form then computes the whole call again (its kernels return at
// once otherwise): a NaN among V codes of a tile that some rows do not see all of (their zero probability times it is NaN), a V
// scale of 2^126 or more, a scale that is a NaN, V scales more than 2^16
// apart or below 2^-80 over codes that are not zero, V scales above 2^16 beside zeros under the least one or pages that are none, scores beyond 2^10.
// 1000 tokens behind 3000 and 16000 keys, 8 KV heads of 128 channels, 4 query heads each: 438 us, 674 TFLOP/s, 41 % of the bf16 rate. Under the profiler this
// kernel takes 393, its tensor pipe busy 38 % of that, and the streaming form's two kernels, which find nothing to do, 7 and 72 (the merge has a CTA a row; for one
// sequence of 2000 tokens with 128 query heads over 8 KV heads 332, 14 and 397). A pair of score tiles every 5000 clocks, where the products take 2048. Without the exponentials 443 of 457 us then: the chain of a half's scores, maxima,
// exponentials and store, on two warps a scheduler, and the last items' end (148 of 128 tiles' time on 148 SMs).
// Polynomial exponentials on the FMA pipe, one in two to one in four: 463 to 479 us for 457.
#include <algorithm>
#include <type_traits>

#include "cache_sdpa.cuh"
#include "dfgpu_cache.h"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

constexpr int kRows = 128, kKeys = 128, kHalfKeys = 64, kRuns = kKeys / 16;
constexpr int kThreads = 18 * 32, kConverters = 128, kIssuer = 16;   // (the first of the issuing warps has the tensor memory)
constexpr int kScaleStages = 4;      // (K's converters write tile j's with K of j - 3 used up: its last scores came behind the products with V of j - 4, and those behind all softmax of j - 4, as the second query tile, which comes last, sees as many halves as the first or none)
constexpr float kUp = 11.0f;         // P = 2^(t - r + 11): at most 2^15 while t is within 4 of r
constexpr float kRaise = 4.0f;
constexpr int kLeastCode = 47;       // V scales below 2^-80 count as that (over zeros; else a flag)
constexpr int kMostApart = 16;
constexpr int kMostAboveLeast = 96;  // beside zeros under the least scale: P of these, 2^(-80 - r + 11) where r is up to 96 - 80, has to stay in f32's range for the sum, down to 2^-30 of the row's largest weight, where the sum made so far is taken down to a new r
constexpr float kLeastFactor = 1.17549435e-38f;   // (of a score: not zero, so that -inf stays -inf)
constexpr float kMostReference = 1024.0f;   // |r|: the exponent's one rounding, of score * factor + (scale - r), is below 2^-14 up to there
constexpr int kSms = 148, kLeastTiles = 4;   // of key tiles that a piece has
constexpr int kMostRanked = 128;     // sequences that are put in order of length
constexpr float kLn2 = 0.6931471805599453f;

struct CachePrefillArgs {
    CacheSdpaArgs a;
    int32_t* flags;       // by CTA
    float* partial;       // [item in the order of O][piece][row]{O, not divided by its sum; its reference, its sum}, where there are pieces
    int32_t tokens;       // of a query tile: 128 / group
    int32_t blocks;       // of two query tiles
    int32_t batches;
    int32_t pieces;       // of an item's keys
    int32_t rows;         // of O
};

template <int D>
struct Smem {
    static constexpr int kHalves = D / 64, kHalf = kRows * 128;
    static constexpr int kTile = kHalves * kHalf;              // of f16: 128 rows by 64 channels, swizzled, once or twice
    static constexpr int kQ = 0, kK = 2 * kTile, kV = 4 * kTile;
    static constexpr int kScales = 6 * kTile;                  // [stage][run]{K factor, -, log2 of V's, 1 / V's}
    static constexpr int kBarriers = kScales + kScaleStages * kRuns * 16;
    // q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], o_full[2], pv_done[tile][half], s_full[tile][half], p_full[tile][half], scale_full[4]
    static constexpr int kBarrierCount = 1 + 22 + kScaleStages;
    static constexpr int kMisc = kBarriers + kBarrierCount * 8;    // tensor memory's address, flag, {least, largest} V scale by converter warp
    static constexpr int kTotal = kMisc + 64;
    static constexpr int kDynamic = kTotal + 1024;
};

__device__ __forceinline__ void tmem_load_32_now(uint32_t taddr, uint32_t (&r)[32]) {
    tmem_load_32(taddr, r);
    tmem_load_wait();
}
__device__ __forceinline__ void tmem_store_16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_load_16_now(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
// Waits for the loads in flight; their registers pass through, so that nothing that reads them stands above the wait.
__device__ __forceinline__ void tmem_load_wait_both(uint32_t (&a)[32], uint32_t (&b)[32]) {
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(a[i]), "+r"(b[i])::"memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem]: A are pairs of f16, one row per lane.
__device__ __forceinline__ void umma_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t two_halves(float lo, float hi) {
    uint32_t v;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ void four_codes(uint32_t codes, uint32_t& low, uint32_t& high) {   // as f16
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(low), "=r"(high) : "r"(codes));
}
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }   // -126 to 127
// ln(2^reference * sum). The V scales stand in both, against each other: the powers of two meet first, as exact differences.
__device__ __forceinline__ float log_of_sum(float reference, float sum) {
    const uint32_t bits = __float_as_uint(sum);
    if (bits - 0x00800000u >= 0x7f000000u) return kLn2 * reference + logf(sum);   // (not a normal number above zero)
    return fmaf(kLn2, reference + static_cast<float>(static_cast<int>(bits >> 23) - 127), logf(__uint_as_float((bits & 0x007fffffu) | 0x3f800000u)));
}
__device__ __forceinline__ float value_of(__half v) { return __half2float(v); }
__device__ __forceinline__ float value_of(__nv_bfloat16 v) { return __bfloat162float(v); }

// PIECES: an item's keys are cut (3 % slower where they are not).
template <typename T, int D, bool PIECES>
__global__ void __launch_bounds__(kThreads, 1)
cache_sdpa_umma_kernel(const __grid_constant__ CachePrefillArgs args) {
    using S = Smem<D>;
    constexpr int kChunks = D / 16, kAtOnce = kConverters / kChunks, kPasses = kKeys / kAtOnce;   // a converter's 16 codes at a time
    const CacheSdpaArgs& a = args.a;
    extern __shared__ uint8_t raw_smem[];
    const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
    uint8_t* smem = raw_smem + (base - smem_u32(raw_smem));
    const uint32_t bars = base + S::kBarriers;
    const uint32_t q_full = bars;
    auto k_full = [&](int s) { return bars + 8u * (1 + s); };
    auto k_empty = [&](int s) { return bars + 8u * (3 + s); };
    auto v_full = [&](int s) { return bars + 8u * (5 + s); };
    auto v_empty = [&](int s) { return bars + 8u * (7 + s); };
    auto o_full = [&](int i) { return bars + 8u * (9 + i); };
    auto pv_done = [&](int i, int h) { return bars + 8u * (11 + 2 * i + (h & 1)); };   // (by half: a late look at one barrier for both could find half h - 1 done and take it for h - 3)
    auto s_full = [&](int i, int h) { return bars + 8u * (15 + 2 * i + (h & 1)); };
    auto p_full = [&](int i, int h) { return bars + 8u * (19 + 2 * i + (h & 1)); };
    auto scale_full = [&](int s) { return bars + 8u * (23 + s); };
    int* misc = reinterpret_cast<int*>(smem + S::kMisc);
    const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 8);
        for (int s = 0; s < 2; ++s) {
            mbar_init(k_full(s), 4), mbar_init(k_empty(s), 1);
            mbar_init(v_full(s), 4), mbar_init(v_empty(s), 1);
            mbar_init(o_full(s), 1);
            for (int h = 0; h < 2; ++h) mbar_init(s_full(s, h), 1), mbar_init(p_full(s, h), 4), mbar_init(pv_done(s, h), 1);
        }
        for (int s = 0; s < kScaleStages; ++s) mbar_init(scale_full(s), 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        misc[1] = 0;
    }
    if (warp == kIssuer) {
        tmem_alloc(base + S::kMisc, 512);
        tmem_relinquish();
        tc_fence_before();
    }
    chain_wait();

    // The piece of an item: sequences by falling length (those beyond the first 128 as they are stored), their last query blocks first, a block's heads side by side.
    const int per_batch = a.heads_kv * args.blocks;
    const int item = PIECES ? static_cast<int>(blockIdx.x) / args.pieces : static_cast<int>(blockIdx.x), piece = PIECES ? static_cast<int>(blockIdx.x) - item * args.pieces : 0;
    int nth = item / per_batch;
    if (args.batches <= kMostRanked) {
        if (static_cast<int>(threadIdx.x) < args.batches) {
            const int own = a.seq_kv_data[threadIdx.x * a.seq_kv_stride];
            int rank = 0;
            for (int b = 0; b < args.batches; ++b) {
                const int other = a.seq_kv_data[b * a.seq_kv_stride];
                rank += other > own || (other == own && b < static_cast<int>(threadIdx.x));
            }
            if (rank == nth) misc[2] = threadIdx.x;
        }
    } else if (threadIdx.x == 0) {
        misc[2] = nth;
    }
    __syncthreads();
    tc_fence_after();
    chain_release();
    const uint32_t tmem = static_cast<uint32_t>(misc[0]);
    const int64_t batch = misc[2];
    const int in_batch = item % per_batch, head = in_batch % a.heads_kv, block = args.blocks - 1 - in_batch / a.heads_kv;
    const SequenceWindow window = sequence_window(a, batch);
    const int token0 = block * 2 * args.tokens;
    // Keys that the query tiles see; the first key tile is common.
    int lo[2], hi[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) window_of_tokens(a, window, token0 + i * args.tokens, min(token0 + (i + 1) * args.tokens, a.seq_q) - 1, lo[i], hi[i]);
    const bool some[2] = {hi[0] > lo[0], hi[1] > lo[1]};
    const int all_lo = some[0] && some[1] ? min(lo[0], lo[1]) : some[0] ? lo[0] : lo[1];
    int all_hi = max(hi[0], hi[1]), first = all_lo / kKeys;
    if constexpr (PIECES) {
        const int each = ((all_hi + kKeys - 1) / kKeys - first + args.pieces - 1) / args.pieces;   // key tiles of a piece
        first += piece * each;
        all_hi = min(all_hi, (first + each) * kKeys);
    }
    // halves of key tiles that a query tile walks
    auto halves_to = [&](bool any, int until) { return any ? max(min(until, all_hi) - first * kKeys + kHalfKeys - 1, 0) / kHalfKeys : 0; };
    const int n[2] = {halves_to(some[0], hi[0]), halves_to(some[1], hi[1])};
    const int halves = max(n[0], n[1]), tiles = (halves + 1) / 2;
    bool ok = true;

    if (warp >= kIssuer) {
        // ---- the products
        const bool leader = elect_one();
        constexpr uint32_t idesc_s = (1u << 4) | (static_cast<uint32_t>(kHalfKeys >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);   // f16 operands, f32 sums
        constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);   // V read MN-major
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        if (warp == kIssuer) {
            if (tiles > 0) ok = mbar_wait_warp(q_full, 0, 721);
            for (int h = 0; h < halves && ok; ++h) {
                const int j = h >> 1;
                if (ok) ok = mbar_wait_warp(k_full(j & 1), (j >> 1) & 1, 722);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (h >= n[i]) continue;
                    if (ok && h >= 2) ok = mbar_wait_warp(pv_done(i, h), ((h >> 1) & 1) ^ 1, 731);   // S goes over P of half h - 2
                    tc_fence_after();
                    if (leader && ok) {
                        const uint32_t q_lo = smem_desc_lo(base + S::kQ + i * S::kTile, 16), k_lo = smem_desc_lo(base + S::kK + (j & 1) * S::kTile + (h & 1) * (kHalfKeys * 128), 16);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint32_t at = ((k >> 2) * S::kHalf + (k & 3) * 32) >> 4;
                            umma_bf16(tmem_u + i * 128 + (h & 1) * kHalfKeys, desc_words(q_lo + at, smem_desc_hi(1024)), desc_words(k_lo + at, smem_desc_hi(1024)), idesc_s, k != 0 ? 1u : 0u);
                        }
                        umma_commit(s_full(i, h));
                    }
                    __syncwarp();
                }
                // K of a tile is free behind its last scores, of the second half, or of the first where that is the last there is.
                if (leader && ok && ((h & 1) != 0 || h + 1 == halves)) umma_commit(k_empty(j & 1));
                __syncwarp();
            }
        } else {
            for (int h = 0; h < halves && ok; ++h) {
                const int j = h >> 1;
                if (ok) ok = mbar_wait_warp(v_full(j & 1), (j >> 1) & 1, 724);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (h >= n[i]) continue;
                    if (ok) ok = mbar_wait_warp(p_full(i, h), (h >> 1) & 1, 723);
                    tc_fence_after();
                    if (leader && ok) {
                        const uint32_t v_lo = smem_desc_lo(base + S::kV + (j & 1) * S::kTile + (h & 1) * (kHalfKeys * 128), S::kHalf);
#pragma unroll
                        for (int k = 0; k < kHalfKeys / 16; ++k)
                            umma_a_tmem(tmem_u + 256 + i * 128, tmem_u + i * 128 + (h & 1) * kHalfKeys + k * 8, desc_words(v_lo + ((k * 2048) >> 4), smem_desc_hi(1024)), idesc_o, (h | k) != 0 ? 1u : 0u);
                        umma_commit(pv_done(i, h));
                        if (h + 1 == n[i]) umma_commit(o_full(i));
                    }
                    __syncwarp();
                }
                if (leader && ok && ((h & 1) != 0 || h + 1 == halves)) umma_commit(v_empty(j & 1));
                __syncwarp();
            }
        }
    } else if (warp >= 8) {
        // ---- codes to f16
        const int which = warp >= 12 ? 1 : 0, thread = threadIdx.x - 256 - which * kConverters, chunk = thread % kChunks, row0 = thread / kChunks;
        const bool writer = (warp & 3) == 0;   // of the scales
        const CacheSide& side = a.side[which];
        int common_lo, common_hi;   // what all rows see
        {
            int l0, h0, l1, h1;
            window_of_tokens(a, window, token0, token0, l0, h0);
            const int last = min(min(token0 + 2 * args.tokens, a.seq_q), window.len_q) - 1;
            window_of_tokens(a, window, last, last, l1, h1);
            common_lo = max(l0, l1), common_hi = min(h0, h1);
        }
        int v_least = 1 << 20, v_most = -1;
        bool flag = false, least = false;   // least: some key that is seen has the least V scale, or no page
        // Lane l has run l % 8: its page (as the table has it), where it begins in it, and its scale.
        const int run = lane & 7;
        auto look_up = [&](int j, int& page, int& token) {
            const int key = (first + j) * kKeys + run * 16, slot = static_cast<int>(fast_divide(static_cast<uint32_t>(key >> 4), a.by_page));
            token = key - slot * a.page;
            page = j < tiles && key < all_hi && key + 16 > all_lo && slot < side.table_len ? side.table[batch * side.table_batch + slot * side.table_slot] : -1;
        };
        auto checked = [&](int page) { return page >= 0 && page < side.pages ? page : -1; };
        auto look_up_scale = [&](int page, int token) {
            return page >= 0 ? static_cast<int>(side.scales[page * side.scale_stride[0] + head * side.scale_stride[1] + fast_divide(static_cast<uint32_t>(token >> 4), a.by_tokens) * side.scale_stride[2]]) : -1;
        };
        // Where a lane's run begins, -1 where there is no page.
        auto offset_of = [&](int page, int token) { return page >= 0 ? page * side.stride[0] + head * side.stride[1] + token * side.stride[2] : -1ll; };
        // A tile's codes, 16 of a row at a time; zeros where there is no page and where no row sees the key.
        const uint8_t* own = side.codes + (row0 & 15) * side.stride[2] + chunk * 16;
        uint4 raw[kPasses];
        auto load = [&](int j, int64_t offset) {
            const int key0 = (first + j) * kKeys;
            const bool edge = key0 < all_lo || key0 + kKeys > all_hi;
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                const int row = i * kAtOnce + row0;
                const int64_t at = __shfl_sync(0xffffffffu, offset, row >> 4);
                raw[i] = make_uint4(0, 0, 0, 0);
                if (at >= 0 && (!edge || (key0 + row >= all_lo && key0 + row < all_hi))) raw[i] = __ldcg(reinterpret_cast<const uint4*>(own + at));
            }
        };
        const uint32_t tile_at = base + (which ? S::kV : S::kK), row_at = (chunk >> 2) * S::kHalf + row0 * 128, place = chunk * 2 & 7;
        const bool odd = (chunk >> 2) != 0;   // (the halves lie in the same banks: their chunks go in opposite order)
        const uint32_t first_at = row_at + (((place + (odd ? 1 : 0)) ^ (row0 & 7)) << 4), second_at = row_at + (((place + (odd ? 0 : 1)) ^ (row0 & 7)) << 4);   // (rows of later passes are 16 or 32 on: the same swizzle)
        int page, token, page_next, token_next, code;
        look_up(0, page, token);
        look_up(1, page_next, token_next);
        page = checked(page);
        code = look_up_scale(page, token);
        load(0, offset_of(page, token));
        for (int j = 0; j < tiles; ++j) {
            const int now = j & 1;
            page = checked(page_next), token = token_next;   // of tile j + 1
            look_up(j + 2, page_next, token_next);
            const int code_next = look_up_scale(page, token);
            const int64_t offset = offset_of(page, token);
            if (writer) {
                if (lane < 8) {
                    // (a V scale that the exponent does not take counts as the least)
                    float* scale = reinterpret_cast<float*>(smem + S::kScales + ((j & (kScaleStages - 1)) * kRuns + run) * 16);
                    if (which == 0) {
                        scale[0] = code < 0 ? 1.0f : decode_e8m0(static_cast<uint32_t>(code));
                        flag = flag || code == 255;
                    } else {
                        const int exponent = max(code, kLeastCode) - 127;   // (the least where there is no page: its zeros must not lift the reference above the scales beside them)
                        *reinterpret_cast<float2*>(scale + 2) = make_float2(static_cast<float>(exponent), power_of_two(max(-exponent, -126)));
                        const int key = (first + j) * kKeys + run * 16;
                        if (code >= kLeastCode) v_least = min(v_least, code), v_most = max(v_most, code);
                        else least = least || (key < all_hi && key + 16 > all_lo);
                        flag = flag || code >= 253;   // (a NaN among them)
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_full(j & (kScaleStages - 1)));
            }
            if (which == 1) {
                const int key0 = (first + j) * kKeys;
                const bool mixed = key0 < common_lo || key0 + kKeys > common_hi;
                if (mixed || __any_sync(0xffffffffu, code >= 0 && code < kLeastCode)) {
#pragma unroll
                    for (int i = 0; i < kPasses; ++i) {
                        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                        const int run_code = __shfl_sync(0xffffffffu, code, (i * kAtOnce + row0) >> 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            flag = flag || (mixed && (((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0) || (run_code >= 0 && run_code < kLeastCode && (w[e] & 0x7f7f7f7fu) != 0);
                    }
                }
            }
            if (ok) ok = mbar_wait_warp(which ? v_empty(now) : k_empty(now), ((j >> 1) & 1) ^ 1, 725 + which);
            if (!ok) break;
            const uint32_t to = tile_at + now * S::kTile;
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                uint32_t h[8];
                four_codes(odd ? raw[i].z : raw[i].x, h[0], h[1]), four_codes(odd ? raw[i].w : raw[i].y, h[2], h[3]);
                four_codes(odd ? raw[i].x : raw[i].z, h[4], h[5]), four_codes(odd ? raw[i].y : raw[i].w, h[6], h[7]);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + first_at + i * (kAtOnce * 128)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + second_at + i * (kAtOnce * 128)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(which ? v_full(now) : k_full(now));
            load(j + 1, offset);
            code = code_next;
        }
        v_least = __reduce_min_sync(0xffffffffu, v_least), v_most = __reduce_max_sync(0xffffffffu, v_most);
        if (flag || v_most - v_least > kMostApart || (least && v_most > kLeastCode + kMostAboveLeast)) misc[1] = 1;
    } else {
        // ---- a row a thread
        const int i = warp >> 2, row = threadIdx.x & 127, quarter = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16, s_tmem = tmem + lanes + i * 128, o_tmem = tmem + lanes + 256 + i * 128;
        const int in_group = row / args.tokens, token = token0 + i * args.tokens + (row - in_group * args.tokens);
        const bool there = in_group < a.group && token < a.seq_q;   // has a place in O
        const int head_q = head * a.group + (there ? in_group : 0);
        int row_lo = 0, row_hi = 0;
        if (there && token < window.len_q) window_of_tokens(a, window, token, token, row_lo, row_hi);
        float factor;
        {
            const T* from = static_cast<const T*>(a.q) + batch * a.q_stride[0] + head_q * a.q_stride[1] + (there ? token : 0) * a.q_stride[2];
            struct alignas(8) Four { T v[4]; };
            auto four_of = [&](int c) {
                if (!there) return Four{};
                if (a.q_vector) return *reinterpret_cast<const Four*>(from + c);
                return Four{{from[c], from[c + 1], from[c + 2], from[c + 3]}};
            };
            float largest = 0.0f;
#pragma unroll 8
            for (int c = 0; c < D; c += 4) {
                const Four v = four_of(c);
#pragma unroll
                for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(value_of(v.v[e])));
            }
            int up = 14 - (static_cast<int>(__float_as_uint(largest) >> 23) - 127);
            up = largest == 0.0f ? 0 : min(max(up, -126), 126);
            const float power = a.scale_log2 < 0.0f ? -power_of_two(up) : power_of_two(up);   // (a negative scale turns Q about: larger products are larger scores)
            factor = power_of_two(-up) * fabsf(a.scale_log2);
#pragma unroll 4
            for (int c = 0; c < D; c += 8) {
                const Four v = four_of(c), w = four_of(c + 4);
                const uint32_t at = base + S::kQ + i * S::kTile + (c >> 6) * S::kHalf + row * 128 + ((((c >> 3) & 7) ^ (row & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(two_halves(value_of(v.v[0]) * power, value_of(v.v[1]) * power)),
                             "r"(two_halves(value_of(v.v[2]) * power, value_of(v.v[3]) * power)), "r"(two_halves(value_of(w.v[0]) * power, value_of(w.v[1]) * power)),
                             "r"(two_halves(value_of(w.v[2]) * power, value_of(w.v[3]) * power))
                             : "memory");
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const int common_lo = __reduce_max_sync(0xffffffffu, there ? row_lo : 0), common_hi = __reduce_min_sync(0xffffffffu, there ? row_hi : 0x7fffffff);
        float r = -INFINITY, sum = 0.0f;
        for (int h = 0; h < n[i]; ++h) {
            const int j = h >> 1;
            const float4* scale = reinterpret_cast<const float4*>(smem + S::kScales + ((j & (kScaleStages - 1)) * kRuns + (h & 1) * (kRuns / 2)) * 16);
            if (ok) ok = mbar_wait_warp(scale_full(j & (kScaleStages - 1)), (j / kScaleStages) & 1, 727);
            if (ok) ok = mbar_wait_warp(s_full(i, h), (h >> 1) & 1, 728);
            if (!ok) break;
            tc_fence_after();
            const int key0 = first * kKeys + h * kHalfKeys;
            const bool masked = key0 < common_lo || key0 + kHalfKeys > common_hi;
            const uint32_t own_s = s_tmem + (h & 1) * kHalfKeys;
            uint32_t raw[2][32];
            tmem_load_32(own_s, raw[0]);
            tmem_load_32(own_s + 32, raw[1]);
            tmem_load_wait_both(raw[0], raw[1]);
            if (masked) {
                const uint32_t from = static_cast<uint32_t>(row_lo - key0), span = static_cast<uint32_t>(row_hi - row_lo);   // column c is seen where c - from < span
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (static_cast<uint32_t>(c) - from >= span) raw[c >> 5][c & 31] = 0xff800000u;
            }
            // the largest t, by runs of 16 keys
            float top = -INFINITY;
#pragma unroll
            for (int run = 0; run < 4; ++run) {
                float part[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 16; e += 2)
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(part[(e >> 1) & 1]) : "f"(__uint_as_float(raw[run >> 1][(run & 1) * 16 + e])), "f"(__uint_as_float(raw[run >> 1][(run & 1) * 16 + e + 1])));
                const float4 of = scale[run];
                top = fmaxf(top, fmaf(fmaxf(part[0], part[1]), fmaxf(factor * of.x, kLeastFactor), of.z));
            }
            const bool raise = top > r + kRaise || (r == -INFINITY && top > -INFINITY);
            if (__any_sync(0xffffffffu, raise)) {
                // (To 2^-13: r - kUp and the difference of two are exact up to kMostReference, and the largest weight's f16 is off by 2^-14, as next to exact as before. Of
                // whole numbers it was off by up to 2^-12: errors of 2.9e-4 instead of 2.5e-4 with HALF outputs.)
                const float next = raise ? rintf(top * 0x1p13f) * 0x1p-13f : r, down = raise ? exp2_of(r - next) : 1.0f;
                r = next;
                sum *= down;
                if (h > 0) {   // (S of this half came behind the products with V of all halves but the last)
                    if (ok) ok = mbar_wait_warp(pv_done(i, h - 1), ((h - 1) >> 1) & 1, 730);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t acc[16];
                        tmem_load_16_now(o_tmem + c, acc);
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[e] = __float_as_uint(__uint_as_float(acc[e]) * down);
                        tmem_store_16(o_tmem + c, acc);
                    }
                }
            }
            const float reference = r == -INFINITY ? 0.0f : r - kUp;
#pragma unroll
            for (int run = 0; run < 4; ++run) {
                const float4 of = scale[run];
                const float f = fmaxf(factor * of.x, kLeastFactor), bias = of.z - reference;
                const uint64_t f2 = pack2(f, f), bias2 = pack2(bias, bias);
                uint64_t sums = pack2(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = (run & 1) * 16 + 2 * e;
                    float x0, x1;
                    unpack2(fma2(pack2(__uint_as_float(raw[run >> 1][at]), __uint_as_float(raw[run >> 1][at + 1])), f2, bias2), x0, x1);
                    const float p0 = exp2_of(x0), p1 = exp2_of(x1);
                    sums = add2(sums, pack2(p0, p1));
                    raw[run >> 1][(run & 1) * 8 + e] = two_halves(p0, p1);   // (the first halves of the array take the pairs: what lay there has been read)
                }
                float sum0, sum1;
                unpack2(sums, sum0, sum1);
                sum = fmaf(sum0 + sum1, of.w, sum);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = raw[c][e];
                tmem_store_16(own_s + c * 16, p);
            }
            tmem_store_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(i, h));
        }
        if (fabsf(r) > kMostReference && r != -INFINITY) misc[1] = 1;
        // O, normalised
        if (ok && n[i] > 0) ok = mbar_wait_warp(o_full(i), 0, 729);
        tc_fence_after();
        if constexpr (PIECES) {
            float* to = args.partial + ((static_cast<int64_t>((batch * a.heads_kv + head) * args.blocks + block) * args.pieces + piece) * (2 * kRows) + i * kRows + row) * (D + 4);
            if (ok) {
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t acc[16];
                    __syncwarp();
                    if (n[i] > 0) tmem_load_16_now(o_tmem + c, acc);
                    if (!there) continue;
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        uint4 v = make_uint4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                        if (n[i] == 0) v = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(to + c + e) = v;
                    }
                }
                if (there) *reinterpret_cast<float4*>(to + D) = make_float4(r, sum, 0.0f, 0.0f);
            }
            ok = false;   // (nothing more to do)
        }
        const bool healthy = ok && g_device_status == 0, none = !(sum != 0.0f);   // (a NaN sum is a NaN result)
        const float inverse = 1.0f / sum;
        const int64_t at = batch * a.o_stride[0] + head_q * a.o_stride[1] + token * a.o_stride[2];
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t acc[32];
                __syncwarp();
                if (n[i] > 0) tmem_load_32_now(o_tmem + c, acc);
                if (!there || !healthy) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[e] = n[i] == 0 || none ? 0u : __float_as_uint(__uint_as_float(acc[e]) * inverse);
                if (a.o_vector && a.o_type != DFGPU_F32) {
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float v0 = __uint_as_float(acc[e]), v1 = __uint_as_float(acc[e + 1]);
                        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + at + c + e) =
                            a.o_type == DFGPU_F16 ? two_halves(v0, v1) : static_cast<uint32_t>(f32_to_bf16_bits(v0)) | static_cast<uint32_t>(f32_to_bf16_bits(v1)) << 16;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) store_from_f32(a.o, a.o_type, at + c + e, __uint_as_float(acc[e]));
                }
            }
            if (there && healthy && a.stats)
                a.stats[batch * a.stats_stride[0] + head_q * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : log_of_sum(r - kUp, sum);
        }
        tc_fence_before();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) args.flags[blockIdx.x] = misc[1];
    if (warp == kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// A warp a row of O: its pieces.
template <int D>
__global__ void __launch_bounds__(128)
cache_sdpa_pieces_kernel(const __grid_constant__ CachePrefillArgs args) {
    constexpr int kOwn = D / 32;
    const CacheSdpaArgs& a = args.a;
    const int lane = threadIdx.x & 31;
    auto divided = [](int n, const FastDivisor& by) { return static_cast<int>(fast_divide(static_cast<uint32_t>(n), by)); };
    const int nth = static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 5);   // (sequence, KV head, token, head of the group)
    const int list = divided(nth, a.by_rows), in_list = nth - list * a.rows, token = divided(in_list, a.by_group), in_group = in_list - token * a.group;
    const int64_t batch = divided(list, a.by_heads);
    const int head = (list - static_cast<int>(batch) * a.heads_kv) * a.group + in_group;
    const int tile = token / args.tokens, row = (tile & 1) * kRows + in_group * args.tokens + (token - tile * args.tokens);
    const int64_t item = static_cast<int64_t>(list) * args.blocks + (tile >> 1);
    chain_begin();
    if (nth >= args.rows || g_device_status != 0) return;
    const float* from = args.partial + (item * args.pieces * (2 * kRows) + row) * (D + 4);
    constexpr int64_t kNext = 2 * kRows * (D + 4);
    float top = -INFINITY, total = 0.0f, value[kOwn] = {};
    for (int i = 0; i < args.pieces; ++i) top = fmaxf(top, from[i * kNext + D]);
#pragma unroll 4
    for (int i = 0; i < args.pieces; ++i) {
        const float2 of = *reinterpret_cast<const float2*>(from + i * kNext + D);
        // In two halves: under V scales far apart the references are so too, by up to 2^205, and a small weight may meet a large sum.
        const float root = of.x == -INFINITY ? 1.0f : exp2_of(0.5f * (of.x - top));   // (no score above -inf: zeros, or NaNs that are to be seen)
        total = fmaf(of.y * root, root, total);
#pragma unroll
        for (int e = 0; e < kOwn; ++e) value[e] = fmaf(from[i * kNext + lane * kOwn + e] * root, root, value[e]);
    }
    const bool none = total == 0.0f;
    const int64_t at = batch * a.o_stride[0] + head * a.o_stride[1] + token * a.o_stride[2] + lane * kOwn;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) store_from_f32(a.o, a.o_type, at + e, none ? 0.0f : value[e] / total);
    if (lane == 0 && a.stats) a.stats[batch * a.stats_stride[0] + head * a.stats_stride[1] + token * a.stats_stride[2]] = none ? -INFINITY : log_of_sum(top - kUp, total);
}

}  // namespace

bool cache_sdpa_umma_supported(const dfgpu_cache_sdpa_params& p) {
    return (p.q.dim[3] == 64 || p.q.dim[3] == 128) && p.q.dim[1] / p.k.dim[1] <= kRows && cache_sdpa_umma_items(p) < (1ll << 30);
}
int64_t cache_sdpa_umma_items(const dfgpu_cache_sdpa_params& p) {
    const int64_t tokens = kRows / (p.q.dim[1] / p.k.dim[1]);
    return p.q.dim[0] * p.k.dim[1] * ((p.q.dim[2] + 2 * tokens - 1) / (2 * tokens));
}

// Items that do not fill the SMs evenly have their keys cut into pieces. The time of a wave of CTAs is that of a piece's key tiles and about four more, for
// its beginning and its results (pieces of fewer than four tiles gain nothing, of eight and more they are up to a third slower), if all sequences
// are as long as they may be; it has to fall by 15 % at least, and the partial results are those of three waves at most, 60 MB.
// 256 tokens, 8 KV heads, 16000 keys (32 items): 123 us in four pieces, 329 in one.
int cache_sdpa_umma_pieces(const dfgpu_cache_sdpa_params& p) {
    const int64_t tiles = (p.s_kv + kKeys - 1) / kKeys, items = cache_sdpa_umma_items(p);
    auto cost = [&](int64_t pieces) { return (items * pieces + kSms - 1) / kSms * ((tiles + pieces - 1) / pieces + kLeastTiles); };
    int64_t best = 1;
    for (int64_t pieces = 2; pieces * kLeastTiles <= tiles && items * pieces <= 3 * kSms; ++pieces)
        if (cost(pieces) * 115 < cost(1) * 100 && cost(pieces) < cost(best)) best = pieces;
    return static_cast<int>(best);
}
int64_t cache_sdpa_umma_partial_bytes(const dfgpu_cache_sdpa_params& p) {
    const int pieces = cache_sdpa_umma_pieces(p);
    return pieces > 1 ? cache_sdpa_umma_items(p) * pieces * (2 * kRows) * (p.q.dim[3] + 4) * 4 : 0;
}

int launch_cache_sdpa_umma(const dfgpu_cache_sdpa_params& p, const CacheSdpaArgs& a, int32_t* flags, float* partial, cudaStream_t stream) {
    CachePrefillArgs args{};
    args.a = a;
    args.flags = flags;
    args.partial = partial;
    args.tokens = kRows / a.group;
    args.blocks = (a.seq_q + 2 * args.tokens - 1) / (2 * args.tokens);
    args.batches = static_cast<int>(p.q.dim[0]);
    args.pieces = cache_sdpa_umma_pieces(p);
    args.rows = static_cast<int>(p.q.dim[0] * p.q.dim[1] * p.q.dim[2]);   // (below 2^31, as the streaming form's merge needs)
    const int64_t items = cache_sdpa_umma_items(p);
    auto run = [&](auto kernel, int bytes) -> int {
        const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (error != cudaSuccess) return fail(kExecutionFailed, "CACHE_SDPA: cannot reserve %d bytes of shared memory: %s", bytes, cudaGetErrorString(error));
        launch_chained(kernel, dim3(static_cast<unsigned>(items * args.pieces)), dim3(kThreads), bytes, stream, args);
        return check_launch("CACHE_SDPA (tcgen05)");
    };
    auto run_type = [&](auto type, auto merge, auto d) -> int {
        using T = decltype(type);
        constexpr int D = decltype(d)::value;
        if (args.pieces == 1) return run(cache_sdpa_umma_kernel<T, D, false>, Smem<D>::kDynamic);
        const int status = run(cache_sdpa_umma_kernel<T, D, true>, Smem<D>::kDynamic);
        if (status) return status;
        launch_chained(merge, dim3(static_cast<unsigned>((args.rows + 3) / 4)), dim3(128), 0, stream, args);
        return check_launch("CACHE_SDPA pieces");
    };
    const bool half = p.q.dtype == DFGPU_F16;
    const std::integral_constant<int, 64> narrow;
    const std::integral_constant<int, 128> wide;
    if (p.q.dim[3] == 64) return half ? run_type(__half(), cache_sdpa_pieces_kernel<64>, narrow) : run_type(__nv_bfloat16(), cache_sdpa_pieces_kernel<64>, narrow);
    return half ? run_type(__half(), cache_sdpa_pieces_kernel<128>, wide) : run_type(__nv_bfloat16(), cache_sdpa_pieces_kernel<128>, wide);
}

int cache_sdpa_umma_device_status(int* status) { return read_and_clear_device_status(status); }

}  // namespace dfgpu
