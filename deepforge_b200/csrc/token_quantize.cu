// Rows to 8-bit integers with a scale each: scale = max |x| / 127, code = x / scale to the nearest whole number.
//
// HBM bounds it (2 or 4 bytes in, 1 out for a value); the scale has to be known before the first code, so a row's vectors stay in registers between the two
// (what a row has beyond them is read again, from the cache).
#include <algorithm>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"

namespace dfgpu {
namespace {

constexpr int kHeld = 8;          // vectors that a thread keeps

struct QuantizeArgs {
    const void* x;
    int8_t* y;
    float* scale;
    int64_t x_stride[3], y_stride[3], scale_stride[3];   // the axes before K, the last of them first
    int32_t k, vectors;                                  // of a row
    int64_t rows;
    FastDivisor by[2];                                   // extents of the last two axes before K
};

// The largest |x|, ordered like whole numbers: a NaN is above all.
template <typename T, int V>
__device__ __forceinline__ uint32_t magnitude_bits(const Pack<T, V>& x, uint32_t bits) {
#pragma unroll
    for (int i = 0; i < V; ++i) bits = max(bits, __float_as_uint(widen(x.v[i])) & 0x7fffffffu);
    return bits;
}
__device__ __forceinline__ int8_t exact_code(float x, float scale) {
    const float q = __fdiv_rn(x, scale);
    return q != q ? 0 : static_cast<int8_t>(__float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f)));
}
// The codes of a vector. A division a value would cost three times the memory's time, so x times 1 / scale (each rounded: within 2^-23 of the quotient, 1.5e-5 of 127 codes
// at most, and the f32 quotient 4e-6 more) is rounded by adding 1.5 * 2^23, whose low byte is the code; a vector with a product that close to a half, one in 1500 of
// eight values, is divided after all, and so the code is always that of the f32 quotient.
constexpr float kNear = 0.5f - 4e-5f;
template <typename T, int V>
struct alignas(V) Codes {
    int8_t v[V];
};
template <typename T, int V>
__device__ __forceinline__ Codes<T, V> encode(const Pack<T, V>& x, float scale, float inverse, bool plain) {
    Codes<T, V> codes;
    float farthest = 0.5f;
    if (plain) {
        farthest = 0.0f;
        uint32_t bits[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float q = widen(x.v[i]) * inverse, moved = q + 12582912.0f;
            bits[i] = __float_as_uint(moved);
            farthest = fmaxf(farthest, fabsf(q - (moved - 12582912.0f)));
        }
        if constexpr (V >= 4) {
            uint32_t* words = reinterpret_cast<uint32_t*>(&codes);
#pragma unroll
            for (int i = 0; i < V / 4; ++i) words[i] = __byte_perm(__byte_perm(bits[4 * i], bits[4 * i + 1], 0x0040), __byte_perm(bits[4 * i + 2], bits[4 * i + 3], 0x0040), 0x5410);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) codes.v[i] = static_cast<int8_t>(bits[i]);
        }
    }
    if (farthest >= kNear) {
#pragma unroll
        for (int i = 0; i < V; ++i) codes.v[i] = scale > 0.0f ? exact_code(widen(x.v[i]), scale) : 0;   // (0 for a NaN scale too)
    }
    return codes;
}

// A row is taken by `THREADS` threads: a warp (four rows a CTA) or a CTA.
template <typename T, int V, int THREADS>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS)
token_quantize_kernel(const QuantizeArgs a) {
    __shared__ uint32_t largest[THREADS / 32];
    const int thread = THREADS == 32 ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
    const int64_t row = THREADS == 32 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : static_cast<int64_t>(blockIdx.x);
    chain_begin();
    if (row >= a.rows) return;
    const uint32_t outer = fast_divide(static_cast<uint32_t>(row), a.by[0]), inner = static_cast<uint32_t>(row) - outer * a.by[0].divisor;
    const uint32_t first = fast_divide(outer, a.by[1]), middle = outer - first * a.by[1].divisor;
    const T* x = static_cast<const T*>(a.x) + inner * a.x_stride[0] + middle * a.x_stride[1] + first * a.x_stride[2];
    int8_t* y = a.y + inner * a.y_stride[0] + middle * a.y_stride[1] + first * a.y_stride[2];
    Pack<T, V> held[kHeld];
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int at = thread + j * THREADS;
        if (at < a.vectors) held[j] = *reinterpret_cast<const Pack<T, V>*>(x + static_cast<int64_t>(at) * V);
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (thread + j * THREADS < a.vectors) bits = magnitude_bits(held[j], bits);
    for (int at = thread + kHeld * THREADS; at < a.vectors; at += THREADS) bits = magnitude_bits(*reinterpret_cast<const Pack<T, V>*>(x + static_cast<int64_t>(at) * V), bits);
    bits = __reduce_max_sync(0xffffffffu, bits);
    if (THREADS > 32) {
        if ((thread & 31) == 0) largest[thread >> 5] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) bits = max(bits, largest[w]);
    }
    const float scale = __fdiv_rn(__uint_as_float(bits), 127.0f);
    if (thread == 0) a.scale[inner * a.scale_stride[0] + middle * a.scale_stride[1] + first * a.scale_stride[2]] = scale;
    // (products within 2^-23 of the quotients: a normal scale, whose inverse is one too)
    const bool plain = scale >= 1e-30f && scale <= 1e30f;
    const float inverse = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (thread + j * THREADS < a.vectors) *reinterpret_cast<Codes<T, V>*>(y + static_cast<int64_t>(thread + j * THREADS) * V) = encode<T, V>(held[j], scale, inverse, plain);
    for (int at = thread + kHeld * THREADS; at < a.vectors; at += THREADS)
        *reinterpret_cast<Codes<T, V>*>(y + static_cast<int64_t>(at) * V) = encode<T, V>(*reinterpret_cast<const Pack<T, V>*>(x + static_cast<int64_t>(at) * V), scale, inverse, plain);
}

int check_quantize(const dfgpu_token_quantize_params& p, int& width) {
    const int rank = p.x.rank;
    if (!valid_tensor(p.x) || !valid_tensor(p.y) || !valid_tensor(p.scale) || rank < 2 || rank > 4 || p.y.rank != rank || p.scale.rank != rank)
        return fail(kInvalidShape, "TOKEN_QUANTIZE: X, Y and the scale have one rank of 2 to 4 and positive extents");
    if (p.x.dtype != DFGPU_F32 && p.x.dtype != DFGPU_F16 && p.x.dtype != DFGPU_BF16) return fail(kUnsupported, "TOKEN_QUANTIZE: X must be FLOAT, HALF or BFLOAT16");
    if (p.y.dtype != DFGPU_I8 || p.scale.dtype != DFGPU_F32) return fail(kUnsupported, "TOKEN_QUANTIZE: Y must be INT8 and the scale FLOAT");
    int64_t rows = 1;
    for (int i = 0; i < rank; ++i) {
        if (p.y.dim[i] != p.x.dim[i] || p.scale.dim[i] != (i == rank - 1 ? 1 : p.x.dim[i])) return fail(kInvalidShape, "TOKEN_QUANTIZE: Y must have X's extents, the scale one value a row");
        if (i < rank - 1) {
            if (p.x.dim[i] >= (1ll << 31)) return fail(kUnsupported, "TOKEN_QUANTIZE: 2^31 rows or more");
            rows *= p.x.dim[i];
            if (rows >= (1ll << 31) - 4) return fail(kUnsupported, "TOKEN_QUANTIZE: 2^31 rows or more");
            if ((p.y.dim[i] > 1 && p.y.stride[i] == 0) || (p.scale.dim[i] > 1 && p.scale.stride[i] == 0)) return fail(kInvalidLayout, "TOKEN_QUANTIZE: an output overlaps itself");
        }
    }
    if (p.x.dim[rank - 1] >= (1ll << 30)) return fail(kUnsupported, "TOKEN_QUANTIZE: rows of 2^30 values or more");
    if (p.x.dim[rank - 1] > 1 && (p.x.stride[rank - 1] != 1 || p.y.stride[rank - 1] != 1)) return fail(kInvalidLayout, "TOKEN_QUANTIZE: rows must be contiguous");
    if (p.kernel < DFGPU_TOKEN_QUANTIZE_AUTO || p.kernel > DFGPU_TOKEN_QUANTIZE_SCALAR) return fail(kInvalidArgument, "TOKEN_QUANTIZE: unknown kernel id %d", p.kernel);
    width = p.kernel == DFGPU_TOKEN_QUANTIZE_SCALAR ? 1 : 16 / dtype_bytes(p.x.dtype);
    bool fits = p.x.dim[rank - 1] % width == 0;
    for (int i = 0; i < rank - 1; ++i)
        for (const dfgpu_tensor* t : {&p.x, &p.y}) fits = fits && (t->dim[i] == 1 || t->stride[i] % width == 0);
    if (!fits) width = 1;
    if (p.kernel == DFGPU_TOKEN_QUANTIZE_VECTOR && width == 1) return fail(kUnsupported, "TOKEN_QUANTIZE: the vector kernel needs rows of whole 16-byte vectors that start on their boundaries");
    return kOk;
}

template <typename T, int V>
void launch_quantize(const QuantizeArgs& a, cudaStream_t stream) {
    const unsigned rows = static_cast<unsigned>(a.rows);
    if (a.vectors <= 64) launch_chained(token_quantize_kernel<T, V, 32>, dim3((rows + 3) / 4), dim3(128), 0, stream, a);
    else if (a.vectors <= 128 * kHeld) launch_chained(token_quantize_kernel<T, V, 128>, dim3(rows), dim3(128), 0, stream, a);
    else launch_chained(token_quantize_kernel<T, V, 512>, dim3(rows), dim3(512), 0, stream, a);
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_token_quantize(const dfgpu_token_quantize_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "TOKEN_QUANTIZE: null params");
    int width;
    const int status = check_quantize(*p, width);
    if (status) return status;
    info->kernel = width > 1 ? DFGPU_TOKEN_QUANTIZE_VECTOR : DFGPU_TOKEN_QUANTIZE_SCALAR;
    info->launches = 1;
    info->scratch_bytes = 0;
    return kOk;
}

extern "C" int dfgpu_token_quantize(const dfgpu_token_quantize_params* p, void* const* tensors, void* scratch, void* stream) {
    (void)scratch;
    if (!p || !tensors) return fail(kInvalidArgument, "TOKEN_QUANTIZE: null params");
    int width;
    const int status = check_quantize(*p, width);
    if (status) return status;
    for (int i = 0; i < 3; ++i)
        if (!tensors[i]) return fail(kInvalidArgument, "TOKEN_QUANTIZE: port %d is null", i);
    if (!aligned(tensors[0], dtype_bytes(p->x.dtype)) || !aligned(tensors[2], 4)) return fail(kInvalidArgument, "TOKEN_QUANTIZE: X or the scale is not aligned to its type");
    if (width > 1 && !(aligned(tensors[0], 16) && aligned(tensors[1], width))) {
        if (p->kernel == DFGPU_TOKEN_QUANTIZE_VECTOR) return fail(kInvalidArgument, "TOKEN_QUANTIZE: the vector kernel needs X on a 16-byte boundary, Y on that of a vector's codes");
        width = 1;
    }
    const Region x = region_of(tensors[0], p->x), y = region_of(tensors[1], p->y), scale = region_of(tensors[2], p->scale);
    if (overlaps(x, y) || overlaps(x, scale) || overlaps(y, scale)) return fail(kInvalidArgument, "TOKEN_QUANTIZE: an output overlaps another tensor");
    QuantizeArgs a{};
    a.x = tensors[0];
    a.y = static_cast<int8_t*>(tensors[1]);
    a.scale = static_cast<float*>(tensors[2]);
    const int rank = p->x.rank;
    a.rows = 1;
    for (int i = 0; i < 2; ++i) a.by[i] = make_fast_divisor(1);
    for (int i = 0; i < rank - 1; ++i) {
        const int axis = rank - 2 - i;
        a.x_stride[i] = p->x.stride[axis];
        a.y_stride[i] = p->y.stride[axis];
        a.scale_stride[i] = p->scale.stride[axis];
        if (i < 2) a.by[i] = make_fast_divisor(static_cast<uint32_t>(p->x.dim[axis]));
        a.rows *= p->x.dim[axis];
    }
    a.k = static_cast<int>(p->x.dim[rank - 1]);
    a.vectors = a.k / width;
    cudaStream_t on = as_stream(stream);
    if (p->x.dtype == DFGPU_F32) width > 1 ? launch_quantize<float, 4>(a, on) : launch_quantize<float, 1>(a, on);
    else if (p->x.dtype == DFGPU_F16) width > 1 ? launch_quantize<__half, 8>(a, on) : launch_quantize<__half, 1>(a, on);
    else width > 1 ? launch_quantize<__nv_bfloat16, 8>(a, on) : launch_quantize<__nv_bfloat16, 1>(a, on);
    return check_launch("TOKEN_QUANTIZE");
}
