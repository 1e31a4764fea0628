// What the kernels of rotary positions (rope.cu) and of head norms (head_norm.cu) share: vectors of a row, types, angles, and checks of
// positions.
#pragma once

#include "common.cuh"

namespace dfgpu {
namespace {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// Positions and frequencies as a kernel reads them.
struct Positions {
    const void* positions;
    const float* frequencies;
    int64_t batch, token, frequency_stride;
    int32_t wide;   // INT64
};
// (cosine, sine) of position * frequency. The product passes 2^24 for far positions, where f32 has lost the angle: it and its reduction to one turn
// are made in f64, the sine and cosine of what is left, within half a turn, in f32.
__device__ __forceinline__ float2 turn_of(const Positions& p, int64_t batch, int64_t token, int64_t pair) {
    const int64_t at = batch * p.batch + token * p.token;
    const int64_t position = p.wide ? static_cast<const int64_t*>(p.positions)[at] : static_cast<int64_t>(static_cast<const int32_t*>(p.positions)[at]);
    const double turns = static_cast<double>(position) * static_cast<double>(p.frequencies[pair * p.frequency_stride]) * 0.15915494309189533577;
    float sine, cosine;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sine, &cosine);
    return make_float2(cosine, sine);
}

inline bool aligned(const void* pointer, int64_t bytes) { return (reinterpret_cast<uintptr_t>(pointer) & static_cast<uintptr_t>(bytes - 1)) == 0; }

}  // namespace
}  // namespace dfgpu
