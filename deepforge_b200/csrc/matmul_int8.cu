// C = (sum_k A B) a_scale b_scale + bias: 8-bit integers with a scale for each token (row of A) and each channel (column of B).
//
// The sums are exact in 32-bit integers, so every kernel gives the same bits; rows on 16-byte boundaries go to tcgen05 (umma_matmul.cu: 8192 x 4096 x 4096 86 us, 96 % of the rate)
// or, few of them, to the second kernel here, everything else to the CUDA cores: 64 x 64 outputs a CTA, operands as words of four neighbours along K in shared memory, four products
// an instruction (dp4a). That is a form for any layout, not a fast one: its operands come byte by byte. 512 x 4096 x 4096 with A's rows off the 16-byte boundaries 493 us (11 on tcgen05), 4 tokens 140 (5),
// a batch of 8 x 1024 tokens out of a padded buffer 6340 (86 where the rows lie evenly).
#include <algorithm>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"
#include "umma.cuh"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

constexpr int64_t kMaxDepth = 131071;   // 131071 * 2^14 < 2^31
constexpr int kTile = 64, kWords = 16, kPitch = kWords + 1;

struct Int8Args {
    const int8_t* a;
    const int8_t* b;
    void* c;
    const float* a_scale;
    const float* b_scale;
    const void* bias;
    int64_t a_stride[2], b_stride[2], c_stride[2];   // of the two trailing axes
    int64_t a_scale_stride, b_scale_stride, bias_stride;
    int64_t a_batch[DFGPU_MAX_RANK], b_batch[DFGPU_MAX_RANK], c_batch[DFGPU_MAX_RANK], a_scale_batch[DFGPU_MAX_RANK], batch[DFGPU_MAX_RANK];
    int64_t m, n;
    int32_t k, batch_axes, c_type, bias_type;
    int64_t m_tiles;
};

__global__ void __launch_bounds__(256)
matmul_int8_cores_kernel(const Int8Args g) {
    chain_begin();
    __shared__ uint32_t a_words[kTile * kPitch], b_words[kTile * kPitch];
    int64_t rest = blockIdx.z, a_at = 0, b_at = 0, c_at = 0, a_scale_at = 0;
    for (int i = g.batch_axes - 1; i >= 0; --i) {
        const int64_t position = rest % g.batch[i];
        rest /= g.batch[i];
        a_at += position * g.a_batch[i];
        b_at += position * g.b_batch[i];
        c_at += position * g.c_batch[i];
        a_scale_at += position * g.a_scale_batch[i];
    }
    const int64_t n_tile = blockIdx.x / g.m_tiles, m_tile = blockIdx.x - n_tile * g.m_tiles, m0 = m_tile * kTile, n0 = n_tile * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int sums[4][4] = {};
    // One operand's 64 rows (of A, or columns of B) x 64 of K: neighbouring threads walk the axis that is contiguous.
    auto fill = [&](uint32_t* words, const int8_t* from, int64_t row_stride, int64_t k_stride, int64_t row0, int64_t rows, int k0) {
        const bool k_first = k_stride <= row_stride;
#pragma unroll
        for (int i = 0; i < kTile * kWords / 256; ++i) {
            const int item = static_cast<int>(threadIdx.x) + 256 * i;
            const int row = k_first ? item / kWords : item % kTile, word = k_first ? item % kWords : item / kTile;
            uint32_t packed = 0;
            if (row0 + row < rows) {
                const int8_t* p = from + (row0 + row) * row_stride;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t k = k0 + word * 4 + j;
                    if (k < g.k) packed |= static_cast<uint32_t>(static_cast<uint8_t>(p[k * k_stride])) << (8 * j);
                }
            }
            words[row * kPitch + word] = packed;
        }
    };
    for (int k0 = 0; k0 < g.k; k0 += 4 * kWords) {
        fill(a_words, g.a + a_at, g.a_stride[0], g.a_stride[1], m0, g.m, k0);
        fill(b_words, g.b + b_at, g.b_stride[1], g.b_stride[0], n0, g.n, k0);
        __syncthreads();
#pragma unroll 4
        for (int word = 0; word < kWords; ++word) {
            uint32_t a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = a_words[(ty + 16 * i) * kPitch + word];
                b[i] = b_words[(tx + 16 * i) * kPitch + word];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sums[i][j] = __dp4a(static_cast<int>(a[i]), static_cast<int>(b[j]), sums[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= g.m) continue;
        const float a_scale = g.a_scale[a_scale_at + m * g.a_scale_stride];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= g.n) continue;
            float value = __fmul_rn(__fmul_rn(__int2float_rn(sums[i][j]), a_scale), g.b_scale[n * g.b_scale_stride]);
            if (g.bias) value = __fadd_rn(value, load_as_f32(g.bias, g.bias_type, n * g.bias_stride));
            store_from_f32(g.c, g.c_type, c_at + m * g.c_stride[0] + n * g.c_stride[1], value);
        }
    }
}

// ---- few tokens: bound by the weights, and by the latency of a launch ---------------------------------------------------------
// A warp's product takes 16 columns of B x 32 of K and 32 of K x 8 tokens. Neighbouring lanes copy 64 bytes of K of a column, 16 each; a sum of integers has no order, so these bytes
// stand for K in whichever order the instruction names it: two products. A CTA has 16 columns, its warps share K in blocks of 64, each with private copies on their way (no barrier until
// their sums meet). 1 x 4096 x 4096 4.9 us (16.8 MB of weights: 2.6), 8 x 4096 x 4096 5.4, 1 x 4096 x 32000 21.9 (20.1). Loads straight into registers came out in any order (4.8 to 13 us).
constexpr int kFewTokens = 16;

// 16 bytes of a row from k on; what lies past its end counts as zeros.
__device__ __noinline__ uint4 last_words(const int8_t* row, int k, int depth) {
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < depth) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void multiply(int (&sums)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(sums[0]), "+r"(sums[1]), "+r"(sums[2]), "+r"(sums[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int TILES, int ROWS, int STAGES, int WARPS>
struct Few {
    static constexpr int kColumns = 16 * ROWS, kPitchOf = kColumns + 4, kThreads = 32 * WARPS, kOutputs = (8 * TILES * kColumns + kThreads - 1) / kThreads, kOfStage = 2 * ROWS + TILES;
    static constexpr int kBytes = std::max(STAGES * kOfStage * 16 * kThreads, 4 * WARPS * 8 * TILES * kPitchOf);
};
template <int TILES, int ROWS, int STAGES, int WARPS>   // of 8 tokens; of 16 columns; blocks of a warp on their way
__global__ void __launch_bounds__(32 * WARPS)
matmul_int8_few_kernel(const __grid_constant__ Int8Args g) {
    using F = Few<TILES, ROWS, STAGES, WARPS>;
    extern __shared__ __align__(16) uint4 ring[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, eighth = lane >> 2, quarter = lane & 3;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * F::kColumns;
    // Columns and tokens behind the last one are zeros, and nothing is read for them (many lanes that read one line of the L2 cache wait for one another).
    const int8_t* from[F::kOfStage];
    int bytes[F::kOfStage];
#pragma unroll
    for (int i = 0; i < F::kOfStage; ++i) {
        const bool weights = i < 2 * ROWS;
        const int64_t row = weights ? n0 + eighth + 8 * i : eighth + 8 * (i - 2 * ROWS), rows = weights ? g.n : g.m;
        bytes[i] = row < rows ? 16 : 0;
        from[i] = (weights ? g.b : g.a) + min(row, rows - 1) * (weights ? g.b_stride[1] : g.a_stride[0]) + quarter * 16;
    }
    int sums[TILES][ROWS][4] = {};
    const int blocks = g.k / 64;
    // A thread's copies are its own: it waits for them, and nobody else does.
    auto fill = [&](int stage, int block) {
        if (block < blocks) {
#pragma unroll
            for (int i = 0; i < F::kOfStage; ++i) {
                const uint32_t to = smem_u32(ring + (stage * F::kOfStage + i) * F::kThreads + static_cast<int>(threadIdx.x));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(__cvta_generic_to_global(from[i] + block * 64)), "r"(bytes[i]) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto add_up = [&](const uint4 (&at)[F::kOfStage]) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const uint4 &one = at[2 * r], &two = at[2 * r + 1], &x = at[2 * ROWS + t];
                multiply(sums[t][r], one.x, two.x, one.y, two.y, x.x, x.y);
                multiply(sums[t][r], one.z, two.z, one.w, two.w, x.z, x.w);
            }
    };
    chain_begin();
#pragma unroll
    for (int s = 0; s < STAGES; ++s) fill(s, warp + s * WARPS);
    float a_scale[F::kOutputs], b_scale[F::kOutputs], bias[F::kOutputs];
#pragma unroll
    for (int o = 0; o < F::kOutputs; ++o) {
        const int at = static_cast<int>(threadIdx.x) + o * F::kThreads, token = at / F::kColumns;
        const int64_t n = n0 + at % F::kColumns;
        const bool live = token < g.m && n < g.n;
        a_scale[o] = live ? g.a_scale[token * g.a_scale_stride] : 0.0f;
        b_scale[o] = live ? g.b_scale[n * g.b_scale_stride] : 0.0f;
        bias[o] = live && g.bias ? load_as_f32(g.bias, g.bias_type, n * g.bias_stride) : 0.0f;
    }
    int stage = 0;
    for (int block = warp; block < blocks; block += WARPS) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        uint4 at[F::kOfStage];
#pragma unroll
        for (int i = 0; i < F::kOfStage; ++i) at[i] = ring[(stage * F::kOfStage + i) * F::kThreads + static_cast<int>(threadIdx.x)];
        add_up(at);
        fill(stage, block + STAGES * WARPS);   // (the products have what the stage held)
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    if (g.k % 64 != 0 && warp == blocks % WARPS) {
        uint4 at[F::kOfStage];
#pragma unroll
        for (int i = 0; i < F::kOfStage; ++i) at[i] = last_words(from[i], blocks * 64, g.k - quarter * 16);
        __syncwarp();
        add_up(at);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();   // (nothing is on its way into the ring any more)
    int32_t* partial = reinterpret_cast<int32_t*>(ring);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) partial[(warp * 8 * TILES + 8 * t + 2 * quarter + (i & 1)) * F::kPitchOf + 16 * r + eighth + 8 * (i >> 1)] = sums[t][r][i];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < F::kOutputs; ++o) {
        const int at = static_cast<int>(threadIdx.x) + o * F::kThreads, token = at / F::kColumns, column = at % F::kColumns;
        const int64_t n = n0 + column;
        if (token >= 8 * TILES || token >= g.m || n >= g.n) continue;
        int sum = 0;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) sum += partial[(i * 8 * TILES + token) * F::kPitchOf + column];
        float value = __fmul_rn(__fmul_rn(__int2float_rn(sum), a_scale[o]), b_scale[o]);
        if (g.bias) value = __fadd_rn(value, bias[o]);
        store_from_f32(g.c, g.c_type, token * g.c_stride[0] + n * g.c_stride[1], value);
    }
}

template <int TILES, int ROWS, int STAGES, int WARPS>
int launch_few(const Int8Args& g, cudaStream_t stream) {
    using F = Few<TILES, ROWS, STAGES, WARPS>;
    if (F::kBytes > 48 * 1024) {
        const cudaError_t error = cudaFuncSetAttribute(matmul_int8_few_kernel<TILES, ROWS, STAGES, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kBytes);
        if (error != cudaSuccess) return fail(kExecutionFailed, "MATMUL_INT8: cannot reserve %d bytes of shared memory: %s", F::kBytes, cudaGetErrorString(error));
    }
    launch_chained(matmul_int8_few_kernel<TILES, ROWS, STAGES, WARPS>, dim3(static_cast<unsigned>((g.n + F::kColumns - 1) / F::kColumns)), dim3(F::kThreads), F::kBytes, stream, g);
    return check_launch("MATMUL_INT8");
}
// Where the CTAs are few, twice the warps hide the latency (4096 x 4096 and 8 tokens 5.4 us, 7.3 with eight); where they are many, four CTAs of eight fit an SM (12288 columns of
// 4096: 10.7, 11.8 with sixteen).
int launch_few(const Int8Args& g, cudaStream_t stream) {
    if (g.m > 8) return launch_few<2, 1, 4, 8>(g, stream);
    return g.n <= 16 * 2 * 148 ? launch_few<1, 1, 4, 16>(g, stream) : launch_few<1, 1, 4, 8>(g, stream);
}

int check_int8(const dfgpu_matmul_int8_params& p) {
    const int rank = p.c.rank;
    if (!valid_tensor(p.a) || !valid_tensor(p.b) || !valid_tensor(p.c) || rank < 2 || p.a.rank != rank || p.b.rank != rank)
        return fail(kInvalidShape, "MATMUL_INT8: A, B and C have one rank of at least two and positive extents");
    if (p.a.dtype != DFGPU_I8 || p.b.dtype != DFGPU_I8) return fail(kUnsupported, "MATMUL_INT8: A and B must be INT8");
    if (p.c.dtype != DFGPU_F32 && p.c.dtype != DFGPU_F16 && p.c.dtype != DFGPU_BF16) return fail(kUnsupported, "MATMUL_INT8: C must be FLOAT, HALF or BFLOAT16");
    const int64_t m = p.c.dim[rank - 2], n = p.c.dim[rank - 1], k = p.a.dim[rank - 1];
    if (p.b.dim[rank - 2] != k || p.a.dim[rank - 2] != m || p.b.dim[rank - 1] != n) return fail(kInvalidShape, "MATMUL_INT8: matrix M, N and K dimensions are inconsistent");
    if (k > kMaxDepth) return fail(kUnsupported, "MATMUL_INT8: sums of more than %lld products do not fit 32 bits", static_cast<long long>(kMaxDepth));
    int64_t batches = 1;
    for (int i = 0; i < rank - 2; ++i) {
        if ((p.a.dim[i] != 1 && p.a.dim[i] != p.c.dim[i]) || (p.b.dim[i] != 1 && p.b.dim[i] != p.c.dim[i])) return fail(kInvalidShape, "MATMUL_INT8: batch dimensions are not broadcast-compatible");
        if (p.c.dim[i] > (1ll << 31)) return fail(kUnsupported, "MATMUL_INT8: too many matrices");
        batches = std::min<int64_t>(batches * p.c.dim[i], 1ll << 31);
    }
    if (m >= (1ll << 31) || n >= (1ll << 31)) return fail(kUnsupported, "MATMUL_INT8: 2^31 rows or columns or more");
    if (overlaps_itself(p.c)) return fail(kInvalidLayout, "MATMUL_INT8: C overlaps itself");
    auto scale_ok = [&](const dfgpu_tensor& t, int64_t rows, int64_t columns, const dfgpu_tensor& batch_of) {
        if (!valid_tensor(t) || t.rank != rank) return false;
        for (int i = 0; i < rank - 2; ++i)
            if (t.dim[i] != 1 && t.dim[i] != batch_of.dim[i]) return false;
        return (t.dim[rank - 2] == 1 || t.dim[rank - 2] == rows) && (t.dim[rank - 1] == 1 || t.dim[rank - 1] == columns);
    };
    dfgpu_tensor one{};
    one.rank = rank;
    for (int i = 0; i < rank; ++i) one.dim[i] = 1;
    if (!scale_ok(p.a_scale, m, 1, p.a)) return fail(kInvalidShape, "MATMUL_INT8: a_scale must be [..., M or 1, 1]");
    if (!scale_ok(p.b_scale, 1, n, one)) return fail(kInvalidShape, "MATMUL_INT8: b_scale must be [..., 1, N or 1]");
    if (p.a_scale.dtype != DFGPU_F32 || p.b_scale.dtype != DFGPU_F32) return fail(kUnsupported, "MATMUL_INT8: scales must be FLOAT");
    if (p.bias.rank) {
        if (!scale_ok(p.bias, 1, n, one) || p.bias.dim[rank - 1] != n) return fail(kInvalidShape, "MATMUL_INT8: the bias must be [..., 1, N]");
        if (p.bias.dtype != DFGPU_F32 && p.bias.dtype != DFGPU_F16 && p.bias.dtype != DFGPU_BF16) return fail(kUnsupported, "MATMUL_INT8: the bias must be FLOAT, HALF or BFLOAT16");
    }
    if (p.kernel < DFGPU_MATMUL_INT8_AUTO || p.kernel > DFGPU_MATMUL_INT8_FEW) return fail(kInvalidArgument, "MATMUL_INT8: unknown kernel id %d", p.kernel);
    return kOk;
}

// The product as one of matrices, its batch axes folded into M: where B, its scale and the bias have none, and rows of A, of C and of a_scale lie evenly
// through all of them.
bool fold_batch(const dfgpu_matmul_int8_params& p, dfgpu_matmul_int8_params& folded) {
    const int rank = p.c.rank;
    folded = p;
    for (int i = 0; i < rank - 2; ++i)
        if (p.b.dim[i] != 1) return false;
    int64_t rows = 1, a_stride = 0, c_stride = 0, scale_stride = 0;
    bool one_scale = true;
    for (int i = 0; i < rank - 1; ++i) one_scale = one_scale && p.a_scale.dim[i] == 1;
    for (int i = rank - 2; i >= 0; --i) {
        if (p.c.dim[i] == 1) continue;
        if (p.a.dim[i] != p.c.dim[i] || (!one_scale && p.a_scale.dim[i] != p.c.dim[i])) return false;
        if (rows == 1) {
            a_stride = p.a.stride[i];
            c_stride = p.c.stride[i];
            scale_stride = p.a_scale.stride[i];
        } else if (p.a.stride[i] != rows * a_stride || p.c.stride[i] != rows * c_stride || (!one_scale && p.a_scale.stride[i] != rows * scale_stride)) {
            return false;
        }
        rows *= p.c.dim[i];
        if (rows >= (1ll << 31)) return false;
    }
    auto matrix = [&](dfgpu_tensor& t, const dfgpu_tensor& from, int64_t m, int64_t stride, int64_t n, int64_t n_stride) {
        t.dtype = from.dtype;
        t.rank = 2;
        t.dim[0] = m;
        t.dim[1] = n;
        t.stride[0] = stride;
        t.stride[1] = n_stride;
    };
    matrix(folded.a, p.a, rows, rows == 1 ? p.a.stride[rank - 2] : a_stride, p.a.dim[rank - 1], p.a.stride[rank - 1]);
    matrix(folded.c, p.c, rows, rows == 1 ? p.c.stride[rank - 2] : c_stride, p.c.dim[rank - 1], p.c.stride[rank - 1]);
    matrix(folded.b, p.b, p.b.dim[rank - 2], p.b.stride[rank - 2], p.b.dim[rank - 1], p.b.stride[rank - 1]);
    matrix(folded.a_scale, p.a_scale, one_scale ? 1 : rows, scale_stride, 1, 1);
    matrix(folded.b_scale, p.b_scale, 1, 0, p.b_scale.dim[rank - 1], p.b_scale.stride[rank - 1]);
    if (p.bias.rank) matrix(folded.bias, p.bias, 1, 0, p.bias.dim[rank - 1], p.bias.stride[rank - 1]);
    return true;
}

// The kernel for few tokens takes any C and bias; rows of A and columns of B lie along K on 16-byte boundaries.
bool few_tokens(const dfgpu_matmul_int8_params& folded) {
    const dfgpu_tensor &a = folded.a, &b = folded.b;
    return a.dim[0] <= kFewTokens && (a.dim[1] == 1 || (a.stride[1] == 1 && b.stride[0] == 1)) && (a.dim[0] == 1 || a.stride[0] % 16 == 0) && (b.dim[1] == 1 || b.stride[1] % 16 == 0);
}
int check_cores(const dfgpu_matmul_int8_params& p) {
    int64_t batches = 1;
    for (int i = 0; i < p.c.rank - 2; ++i) batches = std::min<int64_t>(batches * p.c.dim[i], 1ll << 31);
    const int64_t tiles = ((p.c.dim[p.c.rank - 2] + kTile - 1) / kTile) * ((p.c.dim[p.c.rank - 1] + kTile - 1) / kTile);
    if (batches > 65535 || tiles >= (1ll << 31)) return fail(kUnsupported, "MATMUL_INT8: more than 65535 matrices or 2^31 tiles on the CUDA cores");
    return kOk;
}
int choose_int8(const dfgpu_matmul_int8_params& p, int& kernel, dfgpu_matmul_int8_params& folded) {
    const bool folds = fold_batch(p, folded), tiles = folds && matmul_int8_umma_supported(folded), few = folds && few_tokens(folded);
    // Up to eight tokens the kernel for few of them is the quicker (1 x 4096 x 4096 4.9 us, tcgen05 6.8; x 12288 columns 10.7 and 13.1; 12288 x 4096 10.4 and 11.4; 4 x 1000 x 1111 3.0 and
    // 4.2), up to sixteen where the weights are few (16 x 512 x 512 1.7 and 3.5, 16 x 1000 x 1111 3.7 and 4.2; 16 x 4096 x 4096 7.1 both, 16 x 12288 x 4096 15.7 and 11.7).
    const bool quicker = few && (folded.c.dim[0] <= 8 || folded.a.dim[1] * folded.c.dim[1] <= 1 << 22);
    kernel = p.kernel == DFGPU_MATMUL_INT8_AUTO ? (quicker ? DFGPU_MATMUL_INT8_FEW : tiles ? DFGPU_MATMUL_INT8_UMMA : DFGPU_MATMUL_INT8_CORES) : p.kernel;
    if (kernel == DFGPU_MATMUL_INT8_FEW && !few) return fail(kUnsupported, "MATMUL_INT8: the kernel for few tokens does not cover this shape or layout");
    if (kernel == DFGPU_MATMUL_INT8_UMMA && !tiles) return fail(kUnsupported, "MATMUL_INT8: the tcgen05 kernel does not cover this shape or layout");
    return kernel == DFGPU_MATMUL_INT8_CORES ? check_cores(p) : kOk;
}

Int8Args args_of(const dfgpu_matmul_int8_params& p, void* const* tensors) {
    const int rank = p.c.rank;
    Int8Args g{};
    g.a = static_cast<const int8_t*>(tensors[0]);
    g.b = static_cast<const int8_t*>(tensors[1]);
    g.c = tensors[2];
    g.a_scale = static_cast<const float*>(tensors[3]);
    g.b_scale = static_cast<const float*>(tensors[4]);
    g.bias = p.bias.rank ? tensors[5] : nullptr;
    g.bias_type = p.bias.dtype;
    g.c_type = p.c.dtype;
    for (int i = 0; i < 2; ++i) {
        g.a_stride[i] = p.a.stride[rank - 2 + i];
        g.b_stride[i] = p.b.stride[rank - 2 + i];
        g.c_stride[i] = p.c.stride[rank - 2 + i];
    }
    g.a_scale_stride = p.a_scale.dim[rank - 2] == 1 ? 0 : p.a_scale.stride[rank - 2];
    g.b_scale_stride = p.b_scale.dim[rank - 1] == 1 ? 0 : p.b_scale.stride[rank - 1];
    g.bias_stride = p.bias.rank ? p.bias.stride[rank - 1] : 0;
    g.m = p.c.dim[rank - 2];
    g.n = p.c.dim[rank - 1];
    g.k = static_cast<int>(p.a.dim[rank - 1]);
    g.batch_axes = rank - 2;
    for (int i = 0; i < rank - 2; ++i) {
        g.batch[i] = p.c.dim[i];
        g.a_batch[i] = p.a.dim[i] == 1 ? 0 : p.a.stride[i];
        g.b_batch[i] = p.b.dim[i] == 1 ? 0 : p.b.stride[i];
        g.c_batch[i] = p.c.dim[i] == 1 ? 0 : p.c.stride[i];
        g.a_scale_batch[i] = p.a_scale.dim[i] == 1 ? 0 : p.a_scale.stride[i];
    }
    return g;
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_matmul_int8(const dfgpu_matmul_int8_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "MATMUL_INT8: null params");
    int kernel, status = check_int8(*p);
    dfgpu_matmul_int8_params folded;
    if (!status) status = choose_int8(*p, kernel, folded);
    if (status) return status;
    info->kernel = kernel;
    info->launches = 1;
    info->scratch_bytes = 0;
    return kOk;
}

extern "C" int dfgpu_matmul_int8(const dfgpu_matmul_int8_params* p, void* const* tensors, void* scratch, void* stream) {
    (void)scratch;
    if (!p || !tensors) return fail(kInvalidArgument, "MATMUL_INT8: null params");
    int kernel, status = check_int8(*p);
    dfgpu_matmul_int8_params folded;
    if (!status) status = choose_int8(*p, kernel, folded);
    if (status) return status;
    const int ports = p->bias.rank ? 6 : 5;
    for (int i = 0; i < ports; ++i)
        if (!tensors[i]) return fail(kInvalidArgument, "MATMUL_INT8: port %d is null", i);
    if (!aligned(tensors[2], dtype_bytes(p->c.dtype)) || !aligned(tensors[3], 4) || !aligned(tensors[4], 4) || (p->bias.rank && !aligned(tensors[5], dtype_bytes(p->bias.dtype))))
        return fail(kInvalidArgument, "MATMUL_INT8: C, a scale or the bias is not aligned to its type");
    const dfgpu_tensor* described[6] = {&p->a, &p->b, &p->c, &p->a_scale, &p->b_scale, &p->bias};
    const Region out = region_of(tensors[2], p->c);
    for (int i = 0; i < ports; ++i)
        if (i != 2 && overlaps(out, region_of(tensors[i], *described[i]))) return fail(kInvalidArgument, "MATMUL_INT8: C overlaps port %d", i);
    if (kernel == DFGPU_MATMUL_INT8_UMMA) {
        if (aligned(tensors[0], 16) && aligned(tensors[1], 16)) return launch_matmul_int8_umma(folded, tensors, as_stream(stream));
        if (p->kernel == DFGPU_MATMUL_INT8_UMMA) return fail(kInvalidArgument, "MATMUL_INT8: the tcgen05 kernel needs A and B on 16-byte boundaries");
    }
    if (kernel == DFGPU_MATMUL_INT8_FEW) {
        if (aligned(tensors[0], 16) && aligned(tensors[1], 16)) {
            return launch_few(args_of(folded, tensors), as_stream(stream));
        }
        if (p->kernel == DFGPU_MATMUL_INT8_FEW) return fail(kInvalidArgument, "MATMUL_INT8: the kernel for few tokens needs A and B on 16-byte boundaries");
    }
    status = check_cores(*p);   // (another kernel's rows may be off their boundaries only now)
    if (status) return status;
    Int8Args g = args_of(*p, tensors);
    int64_t batches = 1;
    for (int i = 0; i < p->c.rank - 2; ++i) batches *= p->c.dim[i];
    g.m_tiles = (g.m + kTile - 1) / kTile;
    const int64_t tiles = g.m_tiles * ((g.n + kTile - 1) / kTile);
    launch_chained(matmul_int8_cores_kernel, dim3(static_cast<unsigned>(tiles), 1, static_cast<unsigned>(batches)), dim3(256), 0, as_stream(stream), g);
    return check_launch("MATMUL_INT8");
}

// 1: head norms and their gradients, 8-bit integers, beam search.
extern "C" int dfgpu_decoder_abi_version(void) { return 1; }
