// New keys and values into a paged cache of E4M3 codes with an E8M0 scale for each block of tokens and head.
//
// Bound by HBM where prompts are written (2 or 4 bytes in, 1 out for a value), by latency where a step adds one token. The unit of work is
// what one call adds to one scale block of K or V: its largest magnitude has to be known before its first code, so a unit's vectors stay in
// registers between the two (what a block has beyond the last variant's is read again, from the cache). Small blocks take a warp each, larger
// ones a CTA of as many threads as hold it in four vectors of 16 bytes each; nothing is shared between units, and no atomic is needed. The
// chain of a unit is length -> new tokens -> largest -> codes, with the page's id on its way beside the tokens. Long prompts are next bound by
// issue slots, so that largest magnitudes go two at a time, codes four, and places are stepped to, not divided (28 to 18 us together).
// 8 sequences of up to 2048 tokens, 8 heads of 128 bf16 channels, blocks of 64: 17.9 us, 3.2 TB/s, 49 % of the copy rate; one token of 64 sequences: 7.2 us.
#include <algorithm>

#include "common.cuh"
#include "dfgpu_cache.h"
#include "scale_rule.cuh"
#include "umma_ptx.cuh"

namespace dfgpu {
namespace {

// Vectors that a thread keeps.
__host__ __device__ constexpr int held_by(int threads) { return threads == 32 ? 8 : 4; }

struct AppendSide {
    const void* x;
    uint8_t* codes;
    uint8_t* scales;
    const int32_t* table;
    int64_t x_stride[3], code_stride[3], scale_stride[3];   // batch, head, token; page, head, token or block
    int64_t table_batch, table_slot, table_len, pages;
};
struct AppendArgs {
    AppendSide side[2];
    const int32_t* lengths;
    const int32_t* added;
    int32_t* lengths_out;
    int64_t lengths_stride, added_stride, out_stride;
    int32_t heads, seq, blocks;     // blocks: the most that one sequence's new tokens meet
    int32_t page, tokens, row;      // tokens a page and a scale block; vectors a row
    int32_t capacity;               // K's, what lengths_out is clamped to
    int64_t units;
    int32_t rows, rest;             // of a unit's threads: whole rows of vectors, and the vectors beyond
    FastDivisor by_row, by_blocks, by_heads;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) AppendVector {
    T v[V];
};
__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(__half v) { return __half2float(v); }
__device__ __forceinline__ float value_of(__nv_bfloat16 v) { return __bfloat162float(v); }

// The largest |x|, of 16-bit values two at a time: without their signs they are ordered like whole numbers, a NaN above all.
template <typename T>
struct Largest {
    uint32_t bits = 0;
    template <int V>
    __device__ __forceinline__ void take(const AppendVector<T, V>& x) {
        if constexpr (sizeof(T) == 2 && V > 1) {
            const uint32_t* pairs = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) bits = __vmaxu2(bits, pairs[i] & 0x7fff7fffu);
        } else if constexpr (sizeof(T) == 2) {
            bits = max(bits, *reinterpret_cast<const uint16_t*>(&x) & 0x7fffu);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) bits = max(bits, __float_as_uint(x.v[i]) & 0x7fffffffu);
        }
    }
    __device__ __forceinline__ uint32_t as_f32() const {
        if constexpr (sizeof(T) == 2) {
            const uint16_t top = static_cast<uint16_t>(max(bits & 0xffffu, bits >> 16));
            return __float_as_uint(value_of(*reinterpret_cast<const T*>(&top))) & 0x7fffffffu;
        } else {
            return bits;
        }
    }
};

template <int V>
struct alignas(V) AppendCodes {
    uint8_t v[V];
};
template <typename T, int V>
__device__ __forceinline__ AppendCodes<V> encode(const AppendVector<T, V>& x, float inverse) {
    AppendCodes<V> codes;
    if constexpr (V == 1) {
        codes.v[0] = static_cast<uint8_t>(encode_e4m3_scalar(value_of(x.v[0]) * inverse));
    } else {
        uint32_t* words = reinterpret_cast<uint32_t*>(&codes);
        bool zeros = false;   // a code of -0: of a value that is one, or of one that rounds to it, whose code is +0
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            float v[4];
            const uint64_t by = pack2(inverse, inverse);
            unpack2(mul2(pack2(value_of(x.v[i]), value_of(x.v[i + 1])), by), v[0], v[1]);
            unpack2(mul2(pack2(value_of(x.v[i + 2]), value_of(x.v[i + 3])), by), v[2], v[3]);
            const uint32_t word = cvt_e4m3_pair(v[0], v[1]) | cvt_e4m3_pair(v[2], v[3]) << 16, turned = word ^ 0x80808080u;
            zeros = zeros || ((turned - 0x01010101u) & ~turned & 0x80808080u) != 0;
            words[i / 4] = word;
        }
        if (zeros) {   // (one value in 10^5 of normal ones)
#pragma unroll
            for (int i = 0; i < V; i += 4)
                words[i / 4] = encode_e4m3_pair(value_of(x.v[i]) * inverse, value_of(x.v[i + 1]) * inverse) | encode_e4m3_pair(value_of(x.v[i + 2]) * inverse, value_of(x.v[i + 3]) * inverse) << 16;
        }
    }
    return codes;
}

// The places of a thread's vectors in rows of `row` vectors, NT vectors apart.
struct AppendWalk {
    int column;
    int64_t at;
    __device__ __forceinline__ AppendWalk(int thread, int64_t stride, int width, const FastDivisor& by_row, int row) {
        const int first = static_cast<int>(fast_divide(static_cast<uint32_t>(thread), by_row));
        column = thread - first * row;
        at = first * stride + column * width;
    }
    // rows: NT / row of them and rest = NT % row vectors on
    __device__ __forceinline__ void next(int64_t step, int64_t wrap, int rest, int row) {
        column += rest;
        at += step;
        if (column >= row) column -= row, at += wrap;
    }
};

// NT threads a unit.
template <typename T, int V, int NT>
__global__ void __launch_bounds__(NT < 128 ? 128 : NT)
cache_append_kernel(AppendArgs a) {
    constexpr int kPerCta = NT < 128 ? 128 / NT : 1, kHeld = held_by(NT);
    __shared__ uint32_t largest_of[NT < 128 ? 1 : NT / 32];
    chain_begin();
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kPerCta + (kPerCta > 1 ? threadIdx.x / NT : 0);
    if (unit >= a.units) return;
    const int thread = kPerCta > 1 ? threadIdx.x % NT : threadIdx.x;
    const int which = static_cast<int>(unit & 1);
    const uint32_t list = fast_divide(static_cast<uint32_t>(unit >> 1), a.by_blocks);
    const int nth = static_cast<int>(unit >> 1) - static_cast<int>(list) * a.blocks;
    const int64_t batch = fast_divide(list, a.by_heads);
    const int head = static_cast<int>(list) - static_cast<int>(batch) * a.heads;
    const AppendSide& s = a.side[which];

    const int length = min(max(a.lengths[batch * a.lengths_stride], 0), 1 << 30);   // (a table's capacity is below)
    const int added = a.added ? min(max(a.added[batch * a.added_stride], 0), a.seq) : a.seq;
    if (which == 0 && nth == 0 && head == 0 && thread == 0 && a.lengths_out)
        a.lengths_out[batch * a.out_stride] = min(length + added, a.capacity);
    // (a sequence that is as long as its table has no block here: the slot below is behind it)
    const int begin = (length / a.tokens + nth) * a.tokens, first = max(begin, length), end = min(begin + a.tokens, length + added);
    if (first >= end) return;
    const int slot = begin / a.page;
    if (slot >= s.table_len) return;
    const int page = s.table[batch * s.table_batch + slot * s.table_slot];   // (asked whether it is one below, when the tokens are on their way)
    const int in_page = begin - slot * a.page;
    const T* x = static_cast<const T*>(s.x) + batch * s.x_stride[0] + head * s.x_stride[1] + (first - length) * s.x_stride[2];
    const int count = (end - first) * a.row;   // vectors
    AppendWalk from(thread, s.x_stride[2], V, a.by_row, a.row);
    const int64_t from_step = a.rows * s.x_stride[2] + a.rest * V, from_wrap = s.x_stride[2] - a.row * V;
    auto load = [&](const AppendWalk& walk) { return *reinterpret_cast<const AppendVector<T, V>*>(x + walk.at); };
    AppendVector<T, V> held[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        if (thread + k * NT < count) held[k] = load(from);
        from.next(from_step, from_wrap, a.rest, a.row);
    }
    if (page < 0 || page >= s.pages) return;
    uint8_t* codes = s.codes + page * s.code_stride[0] + head * s.code_stride[1] + (in_page + (first - begin)) * s.code_stride[2];
    uint8_t* scale = s.scales + page * s.scale_stride[0] + head * s.scale_stride[1] + (in_page / a.tokens) * s.scale_stride[2];
    const bool holds = first > begin;
    const uint32_t old = holds ? *scale : 0u;
    Largest<T> own;
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
        if (thread + k * NT < count) own.take(held[k]);
    AppendWalk beyond = from;
    for (int i = thread + kHeld * NT; i < count; i += NT) {
        own.take(load(beyond));
        beyond.next(from_step, from_wrap, a.rest, a.row);
    }
    uint32_t largest = __reduce_max_sync(0xffffffffu, own.as_f32());
    if constexpr (NT > 32) {
        if ((threadIdx.x & 31) == 0) largest_of[threadIdx.x >> 5] = largest;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) largest = max(largest, largest_of[w]);
    }
    // A block of zeros bounds nothing: the smallest scale, where the rule of a whole tensor's blocks takes 1. (So does one whose amax / 448
    // rounds to zero, at most 224 of f32's smallest steps.)
    const uint32_t code = max(largest <= 224u ? 0u : scale_code_from_amax_bits(largest), old);
    const float inverse = reciprocal_e8m0(code);
    AppendWalk to(thread, s.code_stride[2], V, a.by_row, a.row);
    const int64_t to_step = a.rows * s.code_stride[2] + a.rest * V, to_wrap = s.code_stride[2] - a.row * V;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        if (thread + k * NT < count) *reinterpret_cast<AppendCodes<V>*>(codes + to.at) = encode(held[k], inverse);
        to.next(to_step, to_wrap, a.rest, a.row);
    }
    for (int i = thread + kHeld * NT; i < count; i += NT) {
        *reinterpret_cast<AppendCodes<V>*>(codes + to.at) = encode(load(from), inverse);
        from.next(from_step, from_wrap, a.rest, a.row), to.next(to_step, to_wrap, a.rest, a.row);
    }
    if (holds && code != old) {
        // What the block holds already, in the new scale: both are powers of two (or NaN), so that the value before the rounding is exact.
        uint8_t* before = s.codes + page * s.code_stride[0] + head * s.code_stride[1] + in_page * s.code_stride[2];
        // (Scales more than 2^60 apart leave no code but zeros, as 2^-60 does; their quotient may leave f32's range. A NaN stays one.)
        const float shrink = code != 0xffu && code - old > 60u ? 0x1p-60f : decode_e8m0(old) * inverse;
        for (int i = thread; i < (first - begin) * a.row; i += NT) {
            const int row = static_cast<int>(fast_divide(static_cast<uint32_t>(i), a.by_row));
            AppendCodes<V>& at = *reinterpret_cast<AppendCodes<V>*>(before + row * s.code_stride[2] + (i - row * a.row) * V);
            AppendCodes<V> c = at;
#pragma unroll
            for (int e = 0; e < V; ++e) c.v[e] = static_cast<uint8_t>(encode_e4m3_scalar(decode_e4m3(c.v[e]) * shrink));
            at = c;
        }
    }
    if (thread == 0) *scale = static_cast<uint8_t>(code);
}

// lengths_out that is `lengths` itself: after every unit has read them.
__global__ void __launch_bounds__(256) cache_lengths_kernel(AppendArgs a, int64_t batches) {
    chain_begin();
    const int64_t batch = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (batch >= batches) return;
    const int length = min(max(a.lengths[batch * a.lengths_stride], 0), 1 << 30);
    const int added = a.added ? min(max(a.added[batch * a.added_stride], 0), a.seq) : a.seq;
    a.lengths_out[batch * a.out_stride] = min(length + added, a.capacity);
}

bool on_boundary(const void* pointer, int64_t bytes) { return (reinterpret_cast<uintptr_t>(pointer) & static_cast<uintptr_t>(bytes - 1)) == 0; }

int check_int_vector(const dfgpu_tensor& t, int64_t batch, const char* name) {
    if (!valid_tensor(t) || t.rank != 4 || t.dtype != DFGPU_I32 || t.dim[0] != batch || t.dim[1] != 1 || t.dim[2] != 1 || t.dim[3] != 1)
        return fail(kInvalidShape, "CACHE_APPEND: %s must be INT32 [B,1,1,1]", name);
    return kOk;
}

int check_append_side(const dfgpu_cache_append_params& p, const dfgpu_tensor& x, const dfgpu_tensor& cache, const dfgpu_tensor& scale, const dfgpu_tensor& table, const char* name) {
    if (!valid_tensor(x) || x.rank != 4) return fail(kInvalidShape, "CACHE_APPEND: %s must have rank 4 and positive extents", name);
    if (x.dtype != DFGPU_F32 && x.dtype != DFGPU_F16 && x.dtype != DFGPU_BF16) return fail(kUnsupported, "CACHE_APPEND: %s must be FLOAT, HALF or BFLOAT16", name);
    for (int i = 0; i < 4; ++i)
        if (x.dim[i] != p.k.dim[i]) return fail(kInvalidShape, "CACHE_APPEND: K and V differ in extent");
    if (x.dtype != p.k.dtype) return fail(kUnsupported, "CACHE_APPEND: K and V have one type");
    if (x.stride[3] != 1) return fail(kInvalidLayout, "CACHE_APPEND: the head dimension must have unit stride");
    if (!valid_tensor(cache) || cache.rank != 4 || cache.dtype != DFGPU_E4M3 || cache.dim[1] != x.dim[1] || cache.dim[3] != x.dim[3])
        return fail(kInvalidShape, "CACHE_APPEND: the container of %s must be FP8_E4M3 [pages, Hk, T, D]", name);
    if (cache.dim[2] != p.k_cache.dim[2]) return fail(kInvalidShape, "CACHE_APPEND: the pages of K and V differ in tokens");
    if (cache.stride[3] != 1) return fail(kInvalidLayout, "CACHE_APPEND: the head dimension of a container must have unit stride");
    if (!valid_tensor(scale) || scale.rank != 4 || scale.dtype != DFGPU_E8M0 || scale.reorder != DFGPU_REORDER_NONE || scale.dim[0] != cache.dim[0] || scale.dim[1] != cache.dim[1] ||
        scale.dim[3] != 1 || cache.dim[2] % scale.dim[2] != 0 || scale.dim[2] != p.k_scale.dim[2])
        return fail(kInvalidShape, "CACHE_APPEND: the scales of %s must be FP8_E8M0 [pages, Hk, T / t, 1], t a divisor of T and one for K and V", name);
    // (a stride of zero would put several heads', pages' or tokens' codes in one place)
    for (int i = 0; i < 3; ++i)
        if ((cache.dim[i] > 1 && cache.stride[i] == 0) || (scale.dim[i] > 1 && scale.stride[i] == 0)) return fail(kInvalidLayout, "CACHE_APPEND: a container or its scales overlap themselves");
    if (!valid_tensor(table) || table.rank != 4 || table.dtype != DFGPU_I32 || table.dim[0] != x.dim[0] || table.dim[1] != 1 || table.dim[3] != 1)
        return fail(kInvalidShape, "CACHE_APPEND: page tables must be INT32 [B,1,P,1]");
    if (table.dim[2] * cache.dim[2] >= (1ll << 30)) return fail(kUnsupported, "CACHE_APPEND: a page table of 2^30 tokens or more");
    return kOk;
}

int check_append(const dfgpu_cache_append_params& p, bool& vector) {
    int status = check_append_side(p, p.k, p.k_cache, p.k_scale, p.page_table_k, "K");
    if (!status) status = check_append_side(p, p.v, p.v_cache, p.v_scale, p.page_table_v, "V");
    if (!status) status = check_int_vector(p.lengths, p.k.dim[0], "lengths");
    if (!status && p.added.rank) status = check_int_vector(p.added, p.k.dim[0], "added");
    if (!status && p.lengths_out.rank) status = check_int_vector(p.lengths_out, p.k.dim[0], "lengths_out");
    if (status) return status;
    if (p.lengths_out.rank && p.lengths_out.dim[0] > 1 && p.lengths_out.stride[0] == 0) return fail(kInvalidLayout, "CACHE_APPEND: lengths_out overlaps itself");
    if (p.k.dim[2] >= (1ll << 30) || p.k.dim[3] > 8192 || p.k_cache.dim[2] * p.k.dim[3] >= (1ll << 30)) return fail(kUnsupported, "CACHE_APPEND: too many tokens or channels");
    if (p.kernel < DFGPU_CACHE_APPEND_AUTO || p.kernel > DFGPU_CACHE_APPEND_SCALAR) return fail(kInvalidArgument, "CACHE_APPEND: unknown kernel id %d", p.kernel);
    const int width = 16 / dtype_bytes(p.k.dtype);
    vector = p.kernel != DFGPU_CACHE_APPEND_SCALAR && p.k.dim[3] % width == 0;
    for (int i = 0; i < 3 && vector; ++i)
        for (const dfgpu_tensor* t : {&p.k, &p.v, &p.k_cache, &p.v_cache}) vector = vector && (t->dim[i] == 1 || t->stride[i] % width == 0);
    if (p.kernel == DFGPU_CACHE_APPEND_VECTOR && !vector) return fail(kUnsupported, "CACHE_APPEND: the vector kernel needs extents and strides of whole 16-byte vectors");
    return kOk;
}

template <typename T, int V>
void launch_append(const AppendArgs& a, int threads, cudaStream_t stream) {
    if (threads == 32) launch_chained(cache_append_kernel<T, V, 32>, dim3(static_cast<unsigned>((a.units + 3) / 4)), dim3(128), 0, stream, a);
    else if (threads == 128) launch_chained(cache_append_kernel<T, V, 128>, dim3(static_cast<unsigned>(a.units)), dim3(128), 0, stream, a);
    else if (threads == 256) launch_chained(cache_append_kernel<T, V, 256>, dim3(static_cast<unsigned>(a.units)), dim3(256), 0, stream, a);
    else launch_chained(cache_append_kernel<T, V, 512>, dim3(static_cast<unsigned>(a.units)), dim3(512), 0, stream, a);
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_cache_append(const dfgpu_cache_append_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "CACHE_APPEND: null params");
    bool vector;
    const int status = check_append(*p, vector);
    if (status) return status;
    info->kernel = vector ? DFGPU_CACHE_APPEND_VECTOR : DFGPU_CACHE_APPEND_SCALAR;
    info->launches = 1;   // (and a second one where lengths_out is lengths)
    info->scratch_bytes = 0;
    return kOk;
}

extern "C" int dfgpu_cache_append(const dfgpu_cache_append_params* p, void* const* tensors, void* scratch, void* stream) {
    (void)scratch;
    if (!p || !tensors) return fail(kInvalidArgument, "CACHE_APPEND: null params");
    bool vector;
    int status = check_append(*p, vector);
    if (status) return status;
    for (int i = 0; i < 9; ++i)
        if (!tensors[i]) return fail(kInvalidArgument, "CACHE_APPEND: port %d is null", i);
    if ((p->added.rank && !tensors[9]) || (p->lengths_out.rank && !tensors[10])) return fail(kInvalidArgument, "CACHE_APPEND: added or lengths_out is declared but null");
    const int bytes = dtype_bytes(p->k.dtype), width = 16 / bytes;
    if (!on_boundary(tensors[0], bytes) || !on_boundary(tensors[1], bytes)) return fail(kInvalidArgument, "CACHE_APPEND: K or V is not aligned to its type");
    for (int i = 6; i < 11; ++i)
        if (!on_boundary(tensors[i], 4)) return fail(kInvalidArgument, "CACHE_APPEND: port %d is not aligned to its type", i);
    if (tensors[2] == tensors[3] || tensors[4] == tensors[5]) return fail(kInvalidArgument, "CACHE_APPEND: K and V share a container or its scales");
    if (vector && !(on_boundary(tensors[0], 16) && on_boundary(tensors[1], 16) && on_boundary(tensors[2], width) && on_boundary(tensors[3], width))) {
        if (p->kernel == DFGPU_CACHE_APPEND_VECTOR) return fail(kInvalidArgument, "CACHE_APPEND: the vector kernel needs K and V on 16-byte boundaries, containers on those of a vector's codes");
        vector = false;
    }
    AppendArgs a{};
    for (int s = 0; s < 2; ++s) {
        const dfgpu_tensor &x = s ? p->v : p->k, &cache = s ? p->v_cache : p->k_cache, &scale = s ? p->v_scale : p->k_scale, &table = s ? p->page_table_v : p->page_table_k;
        AppendSide& side = a.side[s];
        side.x = tensors[s];
        side.codes = static_cast<uint8_t*>(tensors[2 + s]);
        side.scales = static_cast<uint8_t*>(tensors[4 + s]);
        side.table = static_cast<const int32_t*>(tensors[6 + s]);
        for (int i = 0; i < 3; ++i) {
            side.x_stride[i] = x.stride[i];
            side.code_stride[i] = cache.stride[i];
            side.scale_stride[i] = scale.stride[i];
        }
        side.table_batch = table.stride[0];
        side.table_slot = table.stride[2];
        side.table_len = table.dim[2];
        side.pages = cache.dim[0];
    }
    a.lengths = static_cast<const int32_t*>(tensors[8]);
    a.added = p->added.rank ? static_cast<const int32_t*>(tensors[9]) : nullptr;
    int32_t* lengths_out = p->lengths_out.rank ? static_cast<int32_t*>(tensors[10]) : nullptr;
    const bool in_place = lengths_out == a.lengths;
    a.lengths_out = in_place ? nullptr : lengths_out;
    // (`added` is still read while lengths_out is written; in place the lengths come in a launch of their own)
    if (lengths_out && !in_place && lengths_out == a.added) return fail(kInvalidArgument, "CACHE_APPEND: lengths_out is added");
    a.lengths_stride = p->lengths.stride[0];
    a.added_stride = p->added.rank ? p->added.stride[0] : 0;
    a.out_stride = p->lengths_out.rank ? p->lengths_out.stride[0] : 0;
    if (in_place && p->lengths.dim[0] > 1 && a.lengths_stride != a.out_stride) return fail(kInvalidLayout, "CACHE_APPEND: in place, lengths and lengths_out have the same stride");
    a.heads = static_cast<int>(p->k.dim[1]);
    a.seq = static_cast<int>(p->k.dim[2]);
    a.page = static_cast<int>(p->k_cache.dim[2]);
    a.tokens = static_cast<int>(p->k_cache.dim[2] / p->k_scale.dim[2]);
    a.blocks = (a.seq + a.tokens - 2) / a.tokens + 1;
    a.capacity = static_cast<int>(p->page_table_k.dim[2] * a.page);
    a.units = 2ll * a.blocks * a.heads * p->k.dim[0];
    a.row = static_cast<int>(p->k.dim[3]) / (vector ? width : 1);
    a.by_row = make_fast_divisor(static_cast<uint32_t>(a.row));
    a.by_blocks = make_fast_divisor(static_cast<uint32_t>(a.blocks));
    a.by_heads = make_fast_divisor(static_cast<uint32_t>(a.heads));
    if (a.units >= (1ll << 31)) return fail(kUnsupported, "CACHE_APPEND: too many blocks in one call");
    // As few threads as hold a whole block of new tokens in their registers. 8 x 2048 tokens of 8 heads of 128 bf16 channels: blocks of 16 tokens, a warp 16.4 us,
    // 128 threads 27.6; of 64, 256 threads 17.9, 512 32.1, a warp 19.8; of 256, 512 threads 20.2, 128 33.1, a warp 58.
    const int64_t vectors = static_cast<int64_t>(std::min(a.tokens, a.seq)) * a.row;
    int threads = 32;
    if (vectors > 32 * held_by(32))
        for (threads = 128; threads < 512 && vectors > threads * held_by(threads);) threads *= 2;
    a.rows = threads / a.row, a.rest = threads % a.row;
    cudaStream_t on = as_stream(stream);
    if (p->k.dtype == DFGPU_F32) vector ? launch_append<float, 4>(a, threads, on) : launch_append<float, 1>(a, threads, on);
    else if (p->k.dtype == DFGPU_F16) vector ? launch_append<__half, 8>(a, threads, on) : launch_append<__half, 1>(a, threads, on);
    else vector ? launch_append<__nv_bfloat16, 8>(a, threads, on) : launch_append<__nv_bfloat16, 1>(a, threads, on);
    status = check_launch("CACHE_APPEND");
    if (status || !in_place || !lengths_out) return status;
    a.lengths_out = lengths_out;
    const int64_t batches = p->k.dim[0];
    launch_chained(cache_lengths_kernel, dim3(static_cast<unsigned>((batches + 255) / 256)), dim3(256), 0, on, a, batches);
    return check_launch("CACHE_APPEND lengths");
}
