// Rows to 8-bit integers with a scale each: scale = max |x| / 127, code = x / scale to the nearest whole number.
//
// HBM bounds it (2 or 4 bytes in, 1 out for a value), and close behind it the instructions of each value; the scale has to be known before the first code, so a row's
// vectors stay in registers between the two (what a row has beyond them is read again, from the cache). Alone, with more data than the L2 holds, 8192 x 4096: 25 us from
// bf16 (the bytes alone 15.4), 29 from f32 (25.7); 32 x 4096 2.1 to 2.6. Rows that start anywhere come as aligned vectors shifted together: 3498 x 3451 bf16 20 (5.5; value by value 29), 20000 x 333 f16 13 (3.1; 21).
#include <algorithm>

#include "common.cuh"
#include "dfgpu_decoder.h"
#include "ports.cuh"
#include "rotary.cuh"
#include "umma_ptx.cuh"
#include "unaligned.cuh"

namespace dfgpu {
namespace {

struct QuantizeArgs {
    const void* x;
    int8_t* y;
    float* scale;
    int64_t x_stride[3], y_stride[3], scale_stride[3];   // the axes before K, the last of them first
    int32_t k, vectors, flat;                            // of a row; flat: one axis before K
    int64_t rows;
    FastDivisor by[2];                                   // extents of the last two axes before K
};

// The largest |x|: without their signs floats are ordered like whole numbers, a NaN above all; of 16-bit values two at a time.
template <typename T>
struct Largest {
    uint32_t bits = 0;
    template <int V>
    __device__ __forceinline__ void take(const Pack<T, V>& x) {
        if constexpr (sizeof(T) == 2 && V > 1) {
            const uint32_t* pairs = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) bits = __vmaxu2(bits, pairs[i] & 0x7fff7fffu);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) bits = max(bits, whole(x.v[i]));
        }
    }
    static __device__ __forceinline__ uint32_t whole(T v) {
        if constexpr (sizeof(T) == 2) return *reinterpret_cast<const uint16_t*>(&v) & 0x7fffu;
        else return __float_as_uint(v) & 0x7fffffffu;
    }
    __device__ __forceinline__ uint32_t as_f32() const {
        if constexpr (sizeof(T) == 4) return bits;
        const uint16_t top = static_cast<uint16_t>(max(bits & 0xffffu, bits >> 16));
        return __float_as_uint(widen(*reinterpret_cast<const T*>(&top))) & 0x7fffffffu;
    }
};
__device__ __forceinline__ int8_t exact_code(float x, float scale) {
    const float q = __fdiv_rn(x, scale);
    return q != q ? 0 : static_cast<int8_t>(__float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f)));
}
// The codes of a vector. A division a value would cost three times the memory's time, so x / scale is rounded as x times 1 / scale plus 1.5 * 2^23, one rounding whose low
// byte is the code: the product of the rounded inverse is within 2^-24 of the quotient, 7.6e-6 of 127 codes at most, and the f32 quotient 4e-6 more. Of a product that
// close to a half h (one in 500 normal bf16 values, most of them exact halves of what scale was rounded from) e = x - h scale is exact in f32, since so much cancels:
// below half a step of f32 at h (times scale) the f32 quotient is h and goes to the even code, above it the sign of e decides, and only in between it is divided after all.
// So the code is always that of the f32 quotient.
constexpr float kNear = 0.5f - 4e-5f, kMove = 12582912.0f;
template <typename T, int V>
struct alignas(V) Codes {
    int8_t v[V];
};
template <typename T, int V>
__device__ __forceinline__ Codes<T, V> encode(const Pack<T, V>& x, float scale, float inverse, bool plain) {
    Codes<T, V> codes;
    if (plain) {
        float farthest = 0.0f;
        if constexpr (V >= 4) {
            uint32_t bits[V];
            const uint64_t by = pack2(inverse, inverse), move = pack2(kMove, kMove), minus = pack2(-1.0f, -1.0f);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const uint64_t two = pack2(widen(x.v[i]), widen(x.v[i + 1])), moved = fma2(two, by, move);
                const uint64_t rest = fma2(two, by, fma2(moved, minus, move));
                float lo, hi;
                unpack2(moved, lo, hi);
                bits[i] = __float_as_uint(lo);
                bits[i + 1] = __float_as_uint(hi);
                unpack2(rest, lo, hi);
                asm("max.abs.f32 %0, %0, %1, %2;" : "+f"(farthest) : "f"(lo), "f"(hi));
            }
            uint32_t* words = reinterpret_cast<uint32_t*>(&codes);
#pragma unroll
            for (int i = 0; i < V / 4; ++i) words[i] = __byte_perm(__byte_perm(bits[4 * i], bits[4 * i + 1], 0x0040), __byte_perm(bits[4 * i + 2], bits[4 * i + 3], 0x0040), 0x5410);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float moved = __fmaf_rn(widen(x.v[i]), inverse, kMove);
                codes.v[i] = static_cast<int8_t>(__float_as_uint(moved));
                farthest = fmaxf(farthest, fabsf(__fmaf_rn(widen(x.v[i]), inverse, -(moved - kMove))));
            }
        }
        if (farthest >= kNear) {
            uint32_t near = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = widen(x.v[i]);
                if (fabsf(__fmaf_rn(v, inverse, kMove - __fmaf_rn(v, inverse, kMove))) >= kNear) near |= 1u << i;
            }
            for (; near != 0; near &= near - 1) {   // (hardly ever two)
                const int at = __ffs(static_cast<int>(near)) - 1;
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i == at) v = widen(x.v[i]);
                const float whole = __fmaf_rn(v, inverse, kMove) - kMove, rest = __fmaf_rn(v, inverse, -whole);
                const float half = whole + copysignf(0.5f, rest), e = __fmaf_rn(-half, scale, v);
                const float step = __uint_as_float((__float_as_uint(half) & 0x7f800000u) - (24u << 23)) * scale;
                const float decided = fabsf(e) < step ? half : e > 0.0f ? half + 0.5f : half - 0.5f;
                const int8_t code = fabsf(e) == step ? exact_code(v, scale) : static_cast<int8_t>(__float_as_uint(decided + kMove));
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i == at) codes.v[i] = code;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) codes.v[i] = scale > 0.0f ? exact_code(widen(x.v[i]), scale) : 0;   // (0 for a NaN scale too)
    }
    return codes;
}

// A row is taken by `THREADS` threads, a warp (four rows a CTA) or a CTA, which keep kHeld vectors each.
// ANYWHERE: rows that are no whole vectors, or do not start on their boundaries.
template <typename T, bool ANYWHERE, int THREADS, int kHeld>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS)
token_quantize_kernel(const QuantizeArgs a) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    __shared__ uint32_t largest[THREADS / 32];
    const int thread = THREADS == 32 ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
    const int64_t row = THREADS == 32 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : static_cast<int64_t>(blockIdx.x);
    chain_begin();
    if (row >= a.rows) return;
    int64_t axis[3] = {row, 0, 0};
    if (!a.flat) {
        const uint32_t outer = fast_divide(static_cast<uint32_t>(row), a.by[0]);
        axis[0] = static_cast<uint32_t>(row) - outer * a.by[0].divisor;
        axis[2] = fast_divide(outer, a.by[1]);
        axis[1] = outer - static_cast<uint32_t>(axis[2]) * a.by[1].divisor;
    }
    const T* x = static_cast<const T*>(a.x) + axis[0] * a.x_stride[0] + axis[1] * a.x_stride[1] + axis[2] * a.x_stride[2];
    int8_t* y = a.y + axis[0] * a.y_stride[0] + axis[1] * a.y_stride[1] + axis[2] * a.y_stride[2];
    const int before = ANYWHERE ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)) : 0;
    const bool whole_codes = !ANYWHERE || (reinterpret_cast<uintptr_t>(y) & (V - 1)) == 0;
    const T* own_x = x + static_cast<int64_t>(thread) * V;
    int8_t* own_y = y + static_cast<int64_t>(thread) * V;
    const int left = a.vectors - thread;   // vectors from this thread's first on
    auto load = [&](int v) { return ANYWHERE ? vector_of<T>(x, (thread + v) * V, before, a.k) : *reinterpret_cast<const Pack<T, V>*>(own_x + v * V); };
    auto store = [&](int from, const Codes<T, V>& codes) {
        const int v = thread + from;
        if (whole_codes && (!ANYWHERE || (v + 1) * V <= a.k)) {
            *reinterpret_cast<Codes<T, V>*>(own_y + from * V) = codes;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (v * V + i < a.k) y[v * V + i] = codes.v[i];
        }
    };
    Pack<T, V> held[kHeld];
    Largest<T> most;
    if constexpr (ANYWHERE) {   // (all loads before the first is shifted)
        uint4 halves[kHeld][2];
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int at = (thread + j * THREADS) * V;
            if (!halves_inside<T>(at, before, a.k)) continue;
            halves[j][0] = *reinterpret_cast<const uint4*>(x + at - before);
            halves[j][1] = *reinterpret_cast<const uint4*>(x + at - before + V);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int at = (thread + j * THREADS) * V;
            uint4 row = shifted(halves[j][0], halves[j][1], before * static_cast<int>(sizeof(T)));
            if (at < a.k && !halves_inside<T>(at, before, a.k)) row = edge_vector<T>(x, at, a.k);
            held[j] = *reinterpret_cast<const Pack<T, V>*>(&row);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (j * THREADS < left) held[j] = load(j * THREADS);
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (j * THREADS < left) most.take(held[j]);
    for (int v = kHeld * THREADS; v < left; v += THREADS) most.take(load(v));
    uint32_t bits = __reduce_max_sync(0xffffffffu, most.as_f32());
    if (THREADS > 32) {
        if ((thread & 31) == 0) largest[thread >> 5] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) bits = max(bits, largest[w]);
    }
    const float scale = __fdiv_rn(__uint_as_float(bits), 127.0f);
    if (thread == 0) a.scale[axis[0] * a.scale_stride[0] + axis[1] * a.scale_stride[1] + axis[2] * a.scale_stride[2]] = scale;
    // (products within 2^-24 of the quotients: a normal scale, whose inverse is one too)
    const bool plain = scale >= 1e-30f && scale <= 1e30f;
    const float inverse = __frcp_rn(scale);
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (j * THREADS < left) store(j * THREADS, encode<T, V>(held[j], scale, inverse, plain));
    for (int v = kHeld * THREADS; v < left; v += THREADS) store(v, encode<T, V>(load(v), scale, inverse, plain));
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

template <typename T, bool ANYWHERE>
void launch_quantize(const QuantizeArgs& a, cudaStream_t stream) {
    // Many rows: four vectors a thread, since eight cost registers and so warps (8192 x 4096 bf16 35 us, 25 with four) and a persistent grid whose warps load the next row ahead
    // is slower yet (28 to 41). Up to two rows an SM there is nothing else to hide latency with, so that as many threads as there are take a row (32 x 4096 2.1 us, 2.7 with 128).
    // A few vectors beyond what the threads keep are read again: half of twice the threads would have nothing to do.
    const unsigned rows = static_cast<unsigned>(a.rows), quarter = (rows + 3) / 4;
    if (a.rows <= 2 * 148 && a.vectors > 64) launch_chained(token_quantize_kernel<T, ANYWHERE, 512, 2>, dim3(rows), dim3(512), 0, stream, a);
    else if (a.vectors <= 72) launch_chained(token_quantize_kernel<T, ANYWHERE, 32, 2>, dim3(quarter), dim3(128), 0, stream, a);
    else if (a.vectors <= 144) launch_chained(token_quantize_kernel<T, ANYWHERE, 32, 4>, dim3(quarter), dim3(128), 0, stream, a);
    else if (a.vectors <= 288) launch_chained(token_quantize_kernel<T, ANYWHERE, 64, 4>, dim3(rows), dim3(64), 0, stream, a);
    else if (a.vectors <= 576) launch_chained(token_quantize_kernel<T, ANYWHERE, 128, 4>, dim3(rows), dim3(128), 0, stream, a);
    else if (a.vectors <= 1152) launch_chained(token_quantize_kernel<T, ANYWHERE, 256, 4>, dim3(rows), dim3(256), 0, stream, a);
    else launch_chained(token_quantize_kernel<T, ANYWHERE, 512, 4>, dim3(rows), dim3(512), 0, stream, a);
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
    const int of_vector = 16 / dtype_bytes(p->x.dtype);
    a.vectors = (a.k - 1) / of_vector + 1;
    a.flat = rank == 2;
    cudaStream_t on = as_stream(stream);
    if (p->x.dtype == DFGPU_F32) width > 1 ? launch_quantize<float, false>(a, on) : launch_quantize<float, true>(a, on);
    else if (p->x.dtype == DFGPU_F16) width > 1 ? launch_quantize<__half, false>(a, on) : launch_quantize<__half, true>(a, on);
    else width > 1 ? launch_quantize<__nv_bfloat16, false>(a, on) : launch_quantize<__nv_bfloat16, true>(a, on);
    return check_launch("TOKEN_QUANTIZE");
}
