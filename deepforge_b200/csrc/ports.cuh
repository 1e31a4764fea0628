// Checks of the memory behind ports, for operators whose outputs must not lie on their inputs.
#pragma once

#include "common.cuh"

namespace dfgpu {
namespace {

struct Region {
    uintptr_t begin, end;
    bool dense;   // covers all of [begin, end)
};
inline Region region_of(const void* pointer, const dfgpu_tensor& t) {
    if (!pointer || t.rank == 0) return Region{0, 0, false};
    int64_t last = 0;
    for (int i = 0; i < t.rank; ++i) last += (t.dim[i] - 1) * t.stride[i];
    const uintptr_t begin = reinterpret_cast<uintptr_t>(pointer);
    return Region{begin, begin + static_cast<uintptr_t>(last + 1) * static_cast<uintptr_t>(dtype_bytes(t.dtype)), last + 1 <= element_count(t)};
}
// Whether two tensors share memory for certain: strided ones may be slices of one buffer side by side, whose spans meet although no element does.
inline bool overlaps(const Region& a, const Region& b) {
    if (a.begin == a.end || b.begin == b.end || a.begin >= b.end || b.begin >= a.end) return false;
    return a.begin == b.begin || (a.dense && b.dense);
}
// An output in which two elements have one place for certain.
inline bool overlaps_itself(const dfgpu_tensor& t) {
    for (int i = 0; i < t.rank; ++i)
        if (t.dim[i] > 1 && t.stride[i] == 0) return true;
    return false;
}

}  // namespace
}  // namespace dfgpu
