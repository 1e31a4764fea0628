// Vectors of rows that start anywhere: two aligned ones, shifted together.
#pragma once

#include "rotary.cuh"

namespace dfgpu {
namespace {

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
// Elements at, at + 1, ... (16 bytes of them) of a row that starts `before` elements behind a 16-byte boundary, from the aligned vectors around them, where both are all the row's (nothing
// outside it is read) ...
template <typename T>
__device__ __forceinline__ bool halves_inside(int at, int before, int length) { return at >= before && at - before + 2 * (16 / static_cast<int>(sizeof(T))) <= length; }
// ... and one by one elsewhere, zeros past the end.
template <typename T>
__device__ __noinline__ uint4 edge_vector(const T* row, int at, int length) {
    Pack<T, 16 / sizeof(T)> held;
#pragma unroll
    for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) held.v[i] = at + i < length ? row[at + i] : narrow<T>(0.0f);
    return *reinterpret_cast<const uint4*>(&held);
}
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> vector_of(const T* row, int at, int before, int length) {
    uint4 held;
    if (halves_inside<T>(at, before, length)) {
        const uint4* halves = reinterpret_cast<const uint4*>(row + at - before);
        held = shifted(halves[0], halves[1], before * static_cast<int>(sizeof(T)));
    } else {
        held = edge_vector<T>(row, at, length);
    }
    return *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(&held);
}

}  // namespace
}  // namespace dfgpu
