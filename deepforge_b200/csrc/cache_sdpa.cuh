// What the kernels of attention over the 8-bit cache share: arguments and the keys that a query row sees.
#pragma once

#include "common.cuh"
#include "dfgpu_cache.h"

namespace dfgpu {

struct CacheSide {   // K or V
    const uint8_t* codes;
    const uint8_t* scales;
    const int32_t* table;
    int64_t stride[3], scale_stride[3];   // page, head, token or block of tokens
    int64_t table_batch, table_slot, pages;
    int32_t table_len;
};

struct CacheSdpaArgs {
    CacheSide side[2];
    const void* q;
    void* o;
    float* stats;
    const int32_t* seq_q_data;
    const int32_t* seq_kv_data;
    float* partial;       // [part][first list, last list][row][D + 2]: the part's own O, the largest score in it, the sum against that
    int32_t* starts;      // [0] units a part, [1 + list] the list's first unit among all, -1: one part has all of it
    int64_t q_stride[3], o_stride[3], stats_stride[3], seq_q_stride, seq_kv_stride;
    int64_t left, right;
    int32_t o_type, o_vector, q_vector;
    int32_t heads_kv, group, rows, seq_q, s_kv;   // rows: (token, head of the group) pairs of a KV head
    int32_t page, box;                            // tokens a page, and of one TMA copy
    FastDivisor by_page, by_tokens, by_group;     // the first two of numbers of 16 tokens
    FastDivisor by_rows, by_heads, by_row_blocks;
    int32_t has_left, has_right, bottom_right;
    int32_t row_blocks, block_rows, entries;      // entries: (sequence, block of rows)
    float scale_log2;
    const int32_t* only_if;   // the streaming form returns at once unless one of these only_if_count integers is set; null: always runs
    int32_t only_if_count;
};

// The tcgen05 form (cache_sdpa_umma.cu). What it leaves to the streaming form it says in `flags`, one integer a piece of an item.
bool cache_sdpa_umma_supported(const dfgpu_cache_sdpa_params& p);
int64_t cache_sdpa_umma_items(const dfgpu_cache_sdpa_params& p);
int cache_sdpa_umma_pieces(const dfgpu_cache_sdpa_params& p);   // of an item
int64_t cache_sdpa_umma_partial_bytes(const dfgpu_cache_sdpa_params& p);
int launch_cache_sdpa_umma(const dfgpu_cache_sdpa_params& p, const CacheSdpaArgs& a, int32_t* flags, float* partial, cudaStream_t stream);

struct SequenceWindow {
    int64_t shift;    // key minus query position on the diagonal
    int32_t len_q, keys;
};

__device__ __forceinline__ SequenceWindow sequence_window(const CacheSdpaArgs& a, int64_t batch) {
    SequenceWindow w;
    const int length = a.seq_kv_data[batch * a.seq_kv_stride];
    w.len_q = a.seq_q_data ? min(max(a.seq_q_data[batch * a.seq_q_stride], 0), a.seq_q) : a.seq_q;
    w.shift = a.bottom_right ? static_cast<int64_t>(length) - (a.seq_q_data ? a.seq_q_data[batch * a.seq_q_stride] : a.seq_q) : 0;
    w.keys = min(max(length, 0), a.s_kv);
    return w;
}

// Keys [lo, hi) that some query from `first` to `last` sees; lo = hi = 0 where there is none.
__device__ __forceinline__ void window_of_tokens(const CacheSdpaArgs& a, const SequenceWindow& w, int first, int last, int& lo, int& hi) {
    int64_t from = 0, until = w.keys;
    if (last > w.len_q - 1) last = w.len_q - 1;
    if (a.has_right) until = min(until, last + w.shift + a.right + 1);
    if (a.has_left) from = max(from, first + w.shift - a.left + 1);
    const bool some = first <= last && from < until;
    lo = some ? static_cast<int>(from) : 0;
    hi = some ? static_cast<int>(until) : 0;
}

}  // namespace dfgpu
