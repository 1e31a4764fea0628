// C = (sum_k A B) a_scale b_scale + bias: 8-bit integers with a scale for each token (row of A) and each channel (column of B).
//
// The sums are exact in 32-bit integers, so every kernel gives the same bits; rows on 16-byte boundaries go to tcgen05 (umma_matmul.cu), everything else to the
// CUDA cores here: 64 x 64 outputs a CTA, operands as words of four neighbours along K in shared memory, four products an instruction (dp4a).
#include <algorithm>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"
#include "umma.cuh"

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
    if (p.kernel < DFGPU_MATMUL_INT8_AUTO || p.kernel > DFGPU_MATMUL_INT8_UMMA) return fail(kInvalidArgument, "MATMUL_INT8: unknown kernel id %d", p.kernel);
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

int choose_int8(const dfgpu_matmul_int8_params& p, int& kernel, dfgpu_matmul_int8_params& folded) {
    const bool tiles = fold_batch(p, folded) && matmul_int8_umma_supported(folded);
    kernel = p.kernel == DFGPU_MATMUL_INT8_AUTO ? (tiles ? DFGPU_MATMUL_INT8_UMMA : DFGPU_MATMUL_INT8_CORES) : p.kernel;
    if (kernel == DFGPU_MATMUL_INT8_UMMA && !tiles) return fail(kUnsupported, "MATMUL_INT8: the tcgen05 kernel does not cover this shape or layout");
    return kOk;
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
    const int rank = p->c.rank;
    Int8Args g{};
    g.a = static_cast<const int8_t*>(tensors[0]);
    g.b = static_cast<const int8_t*>(tensors[1]);
    g.c = tensors[2];
    g.a_scale = static_cast<const float*>(tensors[3]);
    g.b_scale = static_cast<const float*>(tensors[4]);
    g.bias = p->bias.rank ? tensors[5] : nullptr;
    g.bias_type = p->bias.dtype;
    g.c_type = p->c.dtype;
    for (int i = 0; i < 2; ++i) {
        g.a_stride[i] = p->a.stride[rank - 2 + i];
        g.b_stride[i] = p->b.stride[rank - 2 + i];
        g.c_stride[i] = p->c.stride[rank - 2 + i];
    }
    g.a_scale_stride = p->a_scale.dim[rank - 2] == 1 ? 0 : p->a_scale.stride[rank - 2];
    g.b_scale_stride = p->b_scale.dim[rank - 1] == 1 ? 0 : p->b_scale.stride[rank - 1];
    g.bias_stride = p->bias.rank ? p->bias.stride[rank - 1] : 0;
    g.m = p->c.dim[rank - 2];
    g.n = p->c.dim[rank - 1];
    g.k = static_cast<int>(p->a.dim[rank - 1]);
    g.batch_axes = rank - 2;
    int64_t batches = 1;
    for (int i = 0; i < rank - 2; ++i) {
        g.batch[i] = p->c.dim[i];
        g.a_batch[i] = p->a.dim[i] == 1 ? 0 : p->a.stride[i];
        g.b_batch[i] = p->b.dim[i] == 1 ? 0 : p->b.stride[i];
        g.c_batch[i] = p->c.dim[i] == 1 ? 0 : p->c.stride[i];
        g.a_scale_batch[i] = p->a_scale.dim[i] == 1 ? 0 : p->a_scale.stride[i];
        batches = std::min<int64_t>(batches * p->c.dim[i], 1ll << 31);
    }
    g.m_tiles = (g.m + kTile - 1) / kTile;
    const int64_t tiles = g.m_tiles * ((g.n + kTile - 1) / kTile);
    if (batches > 65535 || tiles >= (1ll << 31)) return fail(kUnsupported, "MATMUL_INT8: more than 65535 matrices or 2^31 tiles on the CUDA cores");
    launch_chained(matmul_int8_cores_kernel, dim3(static_cast<unsigned>(tiles), 1, static_cast<unsigned>(batches)), dim3(256), 0, as_stream(stream), g);
    return check_launch("MATMUL_INT8");
}

// 1: head norms and their gradients, 8-bit integers, beam search.
extern "C" int dfgpu_decoder_abi_version(void) { return 1; }
