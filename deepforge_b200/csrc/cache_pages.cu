// Bookkeeping of a paged cache: reserve, fork, free, compact and copy over page table, lengths, reference counts and pools.
//
// The integers are few (some 100 KB) and each operation is a handful of passes over them with an order between the passes: free pages
// are counted before they are given out, lists are searched for repetitions before they are obeyed. One thread-block cluster does all
// of it in one launch, its barriers between the passes (about a microsecond each, where a launch of its own costs each pass
// three): eight CTAs of 1024 threads read 64 K counts in eight loads a thread. Counts and ranks come from prefix sums in thread
// order, repeated entries from atomic minima and maxima of list positions, reference counts from integer sums: nothing depends on
// the order in which threads run. Contents move in a second launch (two bytes over HBM for each byte of a page), over
// a list of (source, target) pages that the first one leaves in the scratch memory; no page is both.
// Reserving for 256 sequences among 40000 pages 8.1 us; 32 forks of 64 sequences, 8.6 MB copied, 13.5 us (three more barriers: 15.7; without the one at the
// beginning, which orders the first writes into other CTAs' shared memory, 13.3); compacting 8192 pages, 337 MB moved, 65.6 us, of which the copy's 53 run at
// 6.4 TB/s, 98 % of the copy rate. With the L2 flushed before every four calls: freeing 32 of 64 sequences among 8192 pages 10.2 us, 128 of 256 among 70000 pages
// 16.4; copying 544 pages of 131 KB 37 us (143 MB: 3.8 TB/s), 4192 pages of 8 KB 30 us.
#include <algorithm>

#include "common.cuh"
#include "dfgpu_cache.h"

namespace dfgpu {
namespace {

constexpr int kPagesThreads = 1024, kPagesCtas = 8, kPagesAll = kPagesThreads * kPagesCtas;
constexpr int kCopyThreads = 256;
constexpr int kPiece = 8192;          // bytes that a warp copies at a time
constexpr int kHeader = 64;           // integers at the start of the scratch memory: the copies of the list, counters

struct PagesArgs {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* refs;
    const int32_t* list;
    int32_t* table_out;
    int32_t* lengths_out;
    int32_t* refs_out;
    int32_t* report;
    int32_t* header;      // [0] entries of `copies`, [1..3] counters
    int32_t* pages_a;     // [pages] free list, or holes, or last entries
    int32_t* pages_b;     // [pages] movers' targets
    int32_t* sequence_a;  // [batch]
    int32_t* sequence_b;  // [batch]
    int32_t* entry_a;     // [entries]
    int2* copies;         // [pages / 2 or entries]
    int32_t batch, slots, pages, entries, block;
};

// Once at the kernel's beginning, the two halves apart: nobody writes into another CTA's shared memory before that CTA is running.
__device__ __forceinline__ void cluster_arrive_first() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait_first() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    return rank;
}

struct PagesShared {
    int32_t warps[2][kPagesThreads / 32];
    int32_t totals[4][2][kPagesCtas];   // by scan: each CTA's sums, written by the CTAs themselves
};

// Sums of two values over the threads before this one, in thread order over the cluster, and their totals. One cluster barrier, so that it
// also ends a pass. `turn`: the scan's number in the operation (its own place for the totals: nobody may still read those of the scan before).
__device__ __forceinline__ int2 cluster_scan(PagesShared& shared, int turn, int2 value, int2& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 sum = value;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum.x, s), y = __shfl_up_sync(0xffffffffu, sum.y, s);
        if (lane >= s) sum.x += x, sum.y += y;
    }
    if (lane == 31) shared.warps[0][warp] = sum.x, shared.warps[1][warp] = sum.y;
    __syncthreads();
    int2 before = make_int2(0, 0), all = make_int2(0, 0);
    int2 own = make_int2(shared.warps[0][lane], shared.warps[1][lane]);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {   // (over lanes: of all warps, and of those before)
        const int x = __shfl_xor_sync(0xffffffffu, own.x, s), y = __shfl_xor_sync(0xffffffffu, own.y, s);
        own.x += x, own.y += y;
    }
    all = own;
    before = make_int2(lane < warp ? shared.warps[0][lane] : 0, lane < warp ? shared.warps[1][lane] : 0);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        before.x += __shfl_xor_sync(0xffffffffu, before.x, s);
        before.y += __shfl_xor_sync(0xffffffffu, before.y, s);
    }
    const uint32_t rank = cluster_rank();
    if (threadIdx.x < 2 * kPagesCtas) {   // this CTA's totals to every CTA
        const int which = threadIdx.x / kPagesCtas, to = threadIdx.x % kPagesCtas;
        const uint32_t own_address = static_cast<uint32_t>(__cvta_generic_to_shared(&shared.totals[turn][which][rank]));
        uint32_t address;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(own_address), "r"(to));
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(address), "r"(which ? all.y : all.x) : "memory");
    }
    cluster_barrier();
    total = make_int2(0, 0);
    int2 base = make_int2(0, 0);
#pragma unroll
    for (int c = 0; c < kPagesCtas; ++c) {
        const int x = shared.totals[turn][0][c], y = shared.totals[turn][1][c];
        if (c < static_cast<int>(rank)) base.x += x, base.y += y;
        total.x += x, total.y += y;
    }
    return make_int2(base.x + before.x + sum.x - value.x, base.y + before.y + sum.y - value.y);
}

// Thread t's share of n items, side by side.
__device__ __forceinline__ void share_of(int n, int thread, int& from, int& until) {
    const int each = (n + kPagesAll - 1) / kPagesAll;
    from = static_cast<int>(min(static_cast<int64_t>(thread) * each, static_cast<int64_t>(n)));
    until = min(from + each, n);
}

__device__ __forceinline__ int length_of(const PagesArgs& a, int sequence) {   // (the table's capacity is below 2^30)
    return min(max(a.lengths[sequence], 0), a.slots * a.block);
}
__device__ __forceinline__ int slots_of(const PagesArgs& a, int length) { return (length + a.block - 1) / a.block; }
__device__ __forceinline__ bool names_page(const PagesArgs& a, int id) { return id >= 0 && id < a.pages; }

__device__ __forceinline__ void copy_ints(int32_t* to, const int32_t* from, int64_t n, int thread) {
    if (to == from) return;
    for (int64_t i = thread; i < n; i += kPagesAll) to[i] = from[i];
}

template <int OP>
__global__ void __launch_bounds__(kPagesThreads)
cache_pages_kernel(PagesArgs a) {
    __shared__ PagesShared shared;
    const int thread = static_cast<int>(cluster_rank()) * kPagesThreads + threadIdx.x;
    const int warp = thread >> 5, lane = thread & 31;
    cluster_arrive_first();
    chain_begin();
    cluster_wait_first();   // (behind the wait for the kernel before, where the others arrive too)
    if (thread < 8) a.header[thread] = 0;
    int2 total;

    if constexpr (OP == DFGPU_CACHE_PAGES_RESERVE || OP == DFGPU_CACHE_PAGES_FORK) {
        constexpr bool kFork = OP == DFGPU_CACHE_PAGES_FORK;
        copy_ints(a.refs_out, a.refs, a.pages, thread);
        copy_ints(a.table_out, a.table, static_cast<int64_t>(a.batch) * a.slots, thread);
        if constexpr (kFork) {
            // the first entry that names a target; the lengths, which a target's new one may go over before its source's is asked for
            for (int i = thread; i < a.batch; i += kPagesAll) a.sequence_a[i] = 0x7fffffff, a.sequence_b[i] = length_of(a, i);
            copy_ints(a.lengths_out, a.lengths, a.batch, thread);
            cluster_barrier();
            for (int i = thread; i < a.entries; i += kPagesAll) {
                const int source = a.list[2 * i], target = a.list[2 * i + 1];
                const bool fine = source >= 0 && source < a.batch && target >= 0 && target < a.batch && source != target && length_of(a, target) == 0;
                if (fine) atomicMin(&a.sequence_a[target], i);
            }
            cluster_barrier();
        }
        // Free pages before this thread's, and demand before this thread's sequences or entries.
        int page0, page1, from, until;
        share_of(a.pages, thread, page0, page1);
        share_of(kFork ? a.entries : a.batch, thread, from, until);
        int2 mine = make_int2(0, 0);
        for (int i = page0; i < page1; ++i) mine.x += a.refs[i] <= 0;
        auto demand = [&](int i, bool& fine) -> int {
            if constexpr (kFork) {
                const int source = a.list[2 * i], target = a.list[2 * i + 1];
                fine = source >= 0 && source < a.batch && target >= 0 && target < a.batch && source != target && length_of(a, target) == 0 && a.sequence_a[target] == i;
                return fine && length_of(a, source) % a.block != 0;
            } else {
                const int length = length_of(a, i), more = max(a.list[i], 0);
                fine = more <= a.slots * a.block - length;
                return fine ? slots_of(a, length + more) - slots_of(a, length) : 0;
            }
        };
        int wanted_most = 0;
        for (int i = from; i < until; ++i) {
            bool fine;
            mine.y += demand(i, fine);
        }
        const int2 before = cluster_scan(shared, 0, mine, total);
        const int available = total.x;
        wanted_most = min(total.y, available);
        int rank = before.x;
        for (int i = page0; i < page1 && rank < wanted_most; ++i) {
            const int count = a.refs[i];
            if (count > 0) continue;
            a.pages_a[rank++] = i;
            if (kFork && count < 0) a.refs_out[i] = 0;   // (what is added to it below makes it one)
        }
        int ahead = before.y;
        int2 taken = make_int2(0, 0);   // pages, refused
        int copied = 0;
        for (int i = from; i < until; ++i) {
            bool fine;
            const int wanted = demand(i, fine);
            const bool served = fine && ahead + wanted <= available;
            if constexpr (kFork) {
                a.entry_a[i] = served ? ahead : -1;
                taken.y += !served && a.list[2 * i] >= 0;
                if (served && wanted) {
                    const int source = a.list[2 * i];
                    copied += names_page(a, a.table[static_cast<int64_t>(source) * a.slots + length_of(a, source) / a.block]);
                }
            } else {
                a.sequence_a[i] = ahead;
                a.sequence_b[i] = served ? wanted : 0;
                taken.y += !served;
            }
            taken.x += served ? wanted : 0;
            ahead += wanted;
        }
        if (kFork && copied) atomicAdd(&a.header[1], copied);
        cluster_scan(shared, 1, taken, total);   // (its barrier: the lists are there, and the inputs have been copied)
        if constexpr (kFork) {
            for (int i = warp; i < a.entries; i += kPagesAll / 32) {
                const int place = a.entry_a[i];
                if (place < 0) continue;
                const int source = a.list[2 * i], target = a.list[2 * i + 1];
                const int length = a.sequence_b[source], full = length / a.block;
                const bool partial = length % a.block != 0;
                if (lane == 0) a.lengths_out[target] = length;
                for (int s = lane; s < a.slots; s += 32) {
                    int id = -1;
                    if (s < full || (s == full && partial)) {
                        id = a.table[static_cast<int64_t>(source) * a.slots + s];
                        if (s == full) {
                            const int fresh = a.pages_a[place];
                            a.copies[place] = make_int2(names_page(a, id) ? id : -1, fresh);
                            id = fresh;
                        }
                        if (names_page(a, id)) atomicAdd(&a.refs_out[id], 1);
                    }
                    a.table_out[static_cast<int64_t>(target) * a.slots + s] = id;
                }
            }
            if (thread == 0) a.header[0] = total.x;
            if (thread == 0 && a.report) {
                a.report[0] = available - total.x;
                a.report[1] = total.x;
                a.report[2] = *static_cast<volatile int32_t*>(&a.header[1]);
                a.report[3] = total.y;
            }
        } else {
            for (int i = warp; i < a.batch; i += kPagesAll / 32) {
                const int base = a.sequence_a[i], count = a.sequence_b[i], used = slots_of(a, length_of(a, i));
                for (int k = lane; k < count; k += 32) {
                    const int id = a.pages_a[base + k];
                    a.table_out[static_cast<int64_t>(i) * a.slots + used + k] = id;
                    a.refs_out[id] = 1;
                }
            }
            copy_ints(a.lengths_out, a.lengths, a.batch, thread);
            if (thread == 0 && a.report) {
                a.report[0] = available - total.x;
                a.report[1] = total.x;
                a.report[2] = 0;
                a.report[3] = total.y;
            }
        }
    } else if constexpr (OP == DFGPU_CACHE_PAGES_FREE) {
        for (int i = thread; i < a.batch; i += kPagesAll) a.sequence_a[i] = 0;
        copy_ints(a.refs_out, a.refs, a.pages, thread);
        cluster_barrier();
        int2 mine = make_int2(0, 0);   // pages given back, refused
        for (int i = thread; i < a.entries; i += kPagesAll) {
            const int sequence = a.list[i];
            if (sequence >= 0 && sequence < a.batch) a.sequence_a[sequence] = 1;
            else mine.y += sequence >= a.batch;
        }
        cluster_barrier();
        for (int i = warp; i < a.batch; i += kPagesAll / 32) {
            const bool drop = a.sequence_a[i] != 0;
            if (!drop && a.table == a.table_out) continue;
            const int used = slots_of(a, length_of(a, i));
            for (int s = lane; s < a.slots; s += 32) {
                const int64_t at = static_cast<int64_t>(i) * a.slots + s;
                const int id = a.table[at];
                if (drop && s < used && names_page(a, id)) mine.x += atomicSub(&a.refs_out[id], 1) == 1;
                a.table_out[at] = drop ? -1 : id;
            }
        }
        cluster_scan(shared, 0, mine, total);
        const int2 changed = total;
        mine = make_int2(0, 0);
        for (int i = thread; i < a.pages; i += kPagesAll) {
            const int count = a.refs_out[i];
            if (count < 0) a.refs_out[i] = 0;
            mine.x += count <= 0;
        }
        for (int i = thread; i < a.batch; i += kPagesAll) {
            const int length = a.lengths[i];
            a.lengths_out[i] = a.sequence_a[i] ? 0 : length;
        }
        cluster_scan(shared, 1, mine, total);
        if (thread == 0 && a.report) {
            a.report[0] = total.x;
            a.report[1] = changed.x;
            a.report[2] = 0;
            a.report[3] = changed.y;
        }
    } else if constexpr (OP == DFGPU_CACHE_PAGES_COMPACT) {
        int page0, page1;
        share_of(a.pages, thread, page0, page1);
        int2 mine = make_int2(0, 0);
        for (int i = page0; i < page1; ++i) mine.x += a.refs[i] > 0;
        cluster_scan(shared, 0, mine, total);
        const int live = total.x;
        mine = make_int2(0, 0);   // pages that move, and places that they move to
        for (int i = page0; i < page1; ++i) {
            const bool used = a.refs[i] > 0;
            mine.x += used && i >= live;
            mine.y += !used && i < live;
        }
        const int2 before = cluster_scan(shared, 1, mine, total);
        int hole = before.y;
        for (int i = page0; i < min(page1, live); ++i)
            if (a.refs[i] <= 0) a.pages_a[hole++] = i;
        cluster_barrier();
        int mover = before.x;
        for (int i = page0; i < page1; ++i) {
            int to = i;
            if (i >= live) {
                const int count = a.refs[i];
                if (count > 0) {
                    to = a.pages_a[mover];
                    a.copies[mover++] = make_int2(i, to);
                    a.refs_out[to] = count;   // (a free page's: its own thread leaves it alone below)
                }
                a.refs_out[i] = 0;
            } else if (a.refs_out != a.refs) {
                const int count = a.refs[i];
                if (count > 0) a.refs_out[i] = count;
            }
            a.pages_b[i] = to;
        }
        cluster_barrier();
        for (int i = warp; i < a.batch; i += kPagesAll / 32) {
            const int used = slots_of(a, length_of(a, i));
            for (int s = lane; s < a.slots; s += 32) {
                const int64_t at = static_cast<int64_t>(i) * a.slots + s;
                const int id = a.table[at];
                a.table_out[at] = s < used && names_page(a, id) ? a.pages_b[id] : id;
            }
        }
        copy_ints(a.lengths_out, a.lengths, a.batch, thread);
        if (thread == 0) {
            a.header[0] = total.x;
            if (a.report) {
                a.report[0] = a.pages - live;
                a.report[1] = total.x;
                a.report[2] = total.x;
                a.report[3] = 0;
            }
        }
    } else {
        auto valid = [&](int i, int& source, int& target) {
            source = a.list[2 * i], target = a.list[2 * i + 1];
            return names_page(a, source) && names_page(a, target) && source != target;
        };
        int source, target;
        for (int i = thread; i < a.entries; i += kPagesAll)
            if (valid(i, source, target)) a.pages_a[source] = a.pages_a[target] = -1;   // the last entry that names a target
        cluster_barrier();
        for (int i = thread; i < a.entries; i += kPagesAll)
            if (valid(i, source, target)) atomicMax(&a.pages_a[target], i);
        cluster_barrier();
        int2 mine = make_int2(0, 0);   // copied, refused
        for (int i = thread; i < a.entries; i += kPagesAll) {
            const bool fine = valid(i, source, target);
            const bool is_target = fine && a.pages_a[source] >= 0, goes = fine && !is_target && a.pages_a[target] == i;
            a.copies[i] = make_int2(goes ? source : -1, target);
            mine.x += goes;
            mine.y += (!fine && source >= 0) || is_target;
        }
        int2 free_pages = make_int2(0, 0);
        if (a.refs)
            for (int i = thread; i < a.pages; i += kPagesAll) free_pages.x += a.refs[i] <= 0;
        cluster_scan(shared, 0, mine, total);
        const int2 changed = total;
        cluster_scan(shared, 1, free_pages, total);
        if (a.refs_out) copy_ints(a.refs_out, a.refs, a.pages, thread);
        if (a.table_out) copy_ints(a.table_out, a.table, static_cast<int64_t>(a.batch) * a.slots, thread);
        if (a.lengths_out) copy_ints(a.lengths_out, a.lengths, a.batch, thread);
        if (thread == 0) {
            a.header[0] = a.entries;
            if (a.report) {
                a.report[0] = total.x;
                a.report[1] = changed.x;
                a.report[2] = changed.x;
                a.report[3] = changed.y;
            }
        }
    }
}

struct CopyPool {
    uint8_t* base;
    int64_t layer_stride, page_stride, row;   // bytes
    int32_t width;                            // bytes a lane moves at a time
    int32_t pieces;                           // of a row
    int32_t first;                            // this pool's first piece in a copy's
};
struct CopyArgs {
    CopyPool pool[DFGPU_CACHE_MAX_POOLS];
    const int32_t* header;
    const int2* copies;
    int32_t pools, per_copy;
};

template <typename T>
__device__ __forceinline__ void copy_piece(uint8_t* to, const uint8_t* from, int bytes, int lane) {
    constexpr int kAhead = 8;   // loads on their way a lane
    const int count = bytes / static_cast<int>(sizeof(T));
    for (int i = lane; i < count; i += 32 * kAhead) {
        T v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + 32 * k < count) v[k] = reinterpret_cast<const T*>(from)[i + 32 * k];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + 32 * k < count) reinterpret_cast<T*>(to)[i + 32 * k] = v[k];
    }
}

__global__ void __launch_bounds__(kCopyThreads)
cache_copy_kernel(CopyArgs a) {
    chain_begin();
    const int lane = threadIdx.x & 31;
    const int64_t items = static_cast<int64_t>(a.header[0]) * a.per_copy;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5); item < items; item += static_cast<int64_t>(gridDim.x) * (kCopyThreads / 32)) {
        const int64_t nth = item / a.per_copy;
        int piece = static_cast<int>(item - nth * a.per_copy);
        const int2 copy = a.copies[nth];
        if (copy.x < 0) continue;
        int p = 0;
        while (p + 1 < a.pools && piece >= a.pool[p + 1].first) ++p;
        const CopyPool& pool = a.pool[p];
        piece -= pool.first;
        const int layer = piece / pool.pieces;
        const int64_t at = static_cast<int64_t>(piece - layer * pool.pieces) * kPiece;
        const int bytes = static_cast<int>(min(pool.row - at, static_cast<int64_t>(kPiece)));
        const uint8_t* from = pool.base + layer * pool.layer_stride + copy.x * pool.page_stride + at;
        uint8_t* to = pool.base + layer * pool.layer_stride + copy.y * pool.page_stride + at;
        if (pool.width == 16) copy_piece<uint4>(to, from, bytes, lane);
        else if (pool.width == 4) copy_piece<uint32_t>(to, from, bytes, lane);
        else copy_piece<uint8_t>(to, from, bytes, lane);
    }
}

bool moves_contents(int op) { return op == DFGPU_CACHE_PAGES_FORK || op == DFGPU_CACHE_PAGES_COMPACT || op == DFGPU_CACHE_PAGES_COPY; }

struct PagesSizes {
    int64_t batch, slots, pages, entries;
    // integers of the scratch memory: header, pages_a, pages_b, sequence_a, sequence_b, entry_a, copies
    int64_t page_ints() const { return (pages + 63) / 64 * 64; }
    int64_t batch_ints() const { return (batch + 63) / 64 * 64; }
    int64_t entry_ints() const { return (entries + 63) / 64 * 64; }
    int64_t bytes() const { return 4 * (kHeader + 2 * page_ints() + 2 * batch_ints() + entry_ints() + 2 * std::max(page_ints(), entry_ints())); }
};

int check_pages(const dfgpu_cache_pages_params& p, PagesSizes& sizes) {
    if (p.op < DFGPU_CACHE_PAGES_RESERVE || p.op > DFGPU_CACHE_PAGES_COPY) return fail(kInvalidArgument, "CACHE_PAGES: unknown operation %d", p.op);
    if (p.pool_count < 0 || p.pool_count > DFGPU_CACHE_MAX_POOLS) return fail(kInvalidArgument, "CACHE_PAGES: %d pools (at most %d)", p.pool_count, DFGPU_CACHE_MAX_POOLS);
    if (!valid_tensor(p.refs) || p.refs.rank != 1 || p.refs.dtype != DFGPU_I32 || !is_packed_row_major(p.refs)) return fail(kInvalidShape, "CACHE_PAGES: refs must be INT32 [pages]");
    const bool copy = p.op == DFGPU_CACHE_PAGES_COPY;
    sizes.pages = p.refs.dim[0];
    sizes.batch = sizes.slots = 0;
    if (p.page_table.rank || !copy) {
        const dfgpu_tensor& t = p.page_table;
        if (!valid_tensor(t) || t.rank != 4 || t.dtype != DFGPU_I32 || t.dim[1] != 1 || t.dim[3] != 1 || !is_packed_row_major(t)) return fail(kInvalidShape, "CACHE_PAGES: the page table must be packed INT32 [B,1,P,1]");
        const dfgpu_tensor& n = p.lengths;
        if (!valid_tensor(n) || n.rank != 4 || n.dtype != DFGPU_I32 || n.dim[0] != t.dim[0] || n.dim[1] != 1 || n.dim[2] != 1 || n.dim[3] != 1 || !is_packed_row_major(n))
            return fail(kInvalidShape, "CACHE_PAGES: lengths must be packed INT32 [B,1,1,1]");
        sizes.batch = t.dim[0];
        sizes.slots = t.dim[2];
    }
    if (!copy && p.block <= 0) return fail(kInvalidShape, "CACHE_PAGES: tokens per page must be positive");
    if (sizes.pages >= (1ll << 28) || sizes.batch >= (1ll << 28) || (!copy && (p.block >= (1ll << 30) || sizes.slots * p.block >= (1ll << 30))) || sizes.batch * sizes.slots >= (1ll << 40))
        return fail(kUnsupported, "CACHE_PAGES: too many pages, sequences or tokens");
    // (RESERVE adds up what all sequences lack, those that are refused too, in 32 bits: at most all slots)
    if (p.op == DFGPU_CACHE_PAGES_RESERVE && sizes.batch * sizes.slots >= (1ll << 31)) return fail(kUnsupported, "CACHE_PAGES: RESERVE over a page table of 2^31 slots or more");
    sizes.entries = 0;
    if (p.op != DFGPU_CACHE_PAGES_COMPACT) {
        const int64_t width = p.op == DFGPU_CACHE_PAGES_FORK || copy ? 2 : 1;
        if (!valid_tensor(p.list) || p.list.rank != 2 || p.list.dtype != DFGPU_I32 || p.list.dim[1] != width || !is_packed_row_major(p.list) ||
            (p.op == DFGPU_CACHE_PAGES_RESERVE && p.list.dim[0] != sizes.batch))
            return fail(kInvalidShape, "CACHE_PAGES: the list must be packed INT32 [%s, %d]", p.op == DFGPU_CACHE_PAGES_RESERVE ? "B" : "n", static_cast<int>(width));
        sizes.entries = p.list.dim[0];
        if (sizes.entries >= (1ll << 28)) return fail(kUnsupported, "CACHE_PAGES: too many entries");
    } else if (p.list.rank) {
        return fail(kInvalidArgument, "CACHE_PAGES: COMPACT takes no list");
    }
    if (p.pool_count && !moves_contents(p.op)) return fail(kInvalidArgument, "CACHE_PAGES: this operation moves no contents and takes no pools");
    int64_t pieces = 0;
    for (int i = 0; i < p.pool_count; ++i) {
        const dfgpu_tensor& t = p.pools[i];
        if (!valid_tensor(t) || t.rank != 3 || t.dim[1] != sizes.pages) return fail(kInvalidShape, "CACHE_PAGES: pool %d must be [layers, pages, n]", i);
        if (t.dtype < DFGPU_F32 || t.dtype >= DFGPU_FP4) return fail(kUnsupported, "CACHE_PAGES: pool %d has no type of whole bytes", i);
        if (t.dim[2] > 1 && t.stride[2] != 1) return fail(kInvalidLayout, "CACHE_PAGES: what lies under a page's id must be contiguous (pool %d)", i);
        // a page's content apart from every other's, layer by layer or page by page
        const int64_t n = t.dim[2], low = std::min(t.dim[0] > 1 ? t.stride[0] : INT64_MAX, t.dim[1] > 1 ? t.stride[1] : INT64_MAX);
        const bool layers_out = t.stride[0] >= t.stride[1];
        const int64_t inner = layers_out ? (t.dim[1] - 1) * t.stride[1] + n : (t.dim[0] - 1) * t.stride[0] + n;
        if ((t.dim[0] > 1 || t.dim[1] > 1) && low < n) return fail(kInvalidLayout, "CACHE_PAGES: the pages of pool %d overlap", i);
        if (t.dim[0] > 1 && t.dim[1] > 1 && (layers_out ? t.stride[0] : t.stride[1]) < inner) return fail(kInvalidLayout, "CACHE_PAGES: the pages of pool %d overlap", i);
        pieces += t.dim[0] * ((n * dtype_bytes(t.dtype) + kPiece - 1) / kPiece);
    }
    if (pieces >= (1ll << 30)) return fail(kUnsupported, "CACHE_PAGES: a page's contents are too large");
    return kOk;
}

}  // namespace
}  // namespace dfgpu

using namespace dfgpu;

extern "C" int dfgpu_query_cache_pages(const dfgpu_cache_pages_params* p, dfgpu_plan_info* info) {
    if (!p || !info) return fail(kInvalidArgument, "CACHE_PAGES: null params");
    PagesSizes sizes;
    const int status = check_pages(*p, sizes);
    if (status) return status;
    info->kernel = p->op;
    info->launches = p->pool_count ? 2 : 1;
    info->scratch_bytes = sizes.bytes();
    return kOk;
}

extern "C" int dfgpu_cache_pages(const dfgpu_cache_pages_params* p, void* const* tensors, void* scratch, void* stream) {
    if (!p || !tensors) return fail(kInvalidArgument, "CACHE_PAGES: null params");
    PagesSizes sizes;
    int status = check_pages(*p, sizes);
    if (status) return status;
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15u) != 0) return fail(kInvalidArgument, "CACHE_PAGES: needs the 16-byte aligned scratch dfgpu_query_cache_pages reports");
    const bool copy = p->op == DFGPU_CACHE_PAGES_COPY;
    for (int i = 0; i < 8; ++i) {
        const bool needed = i == 3 ? p->op != DFGPU_CACHE_PAGES_COMPACT : i < 7 && !copy;
        if (needed && !tensors[i]) return fail(kInvalidArgument, "CACHE_PAGES: port %d is null", i);
        if ((reinterpret_cast<uintptr_t>(tensors[i]) & 3u) != 0) return fail(kInvalidArgument, "CACHE_PAGES: port %d is not aligned to its type", i);
    }
    if (copy)
        for (int i : {0, 1, 2})
            if ((tensors[i] == nullptr) != (tensors[4 + i] == nullptr)) return fail(kInvalidArgument, "CACHE_PAGES: COPY takes a table, lengths or counts together with what they become, or neither");
    if (copy && (tensors[0] || tensors[1]) && p->page_table.rank == 0) return fail(kInvalidArgument, "CACHE_PAGES: a page table or lengths without a descriptor");
    PagesArgs a{};
    a.table = static_cast<const int32_t*>(tensors[0]);
    a.lengths = static_cast<const int32_t*>(tensors[1]);
    a.refs = static_cast<const int32_t*>(tensors[2]);
    a.list = static_cast<const int32_t*>(tensors[3]);
    a.table_out = static_cast<int32_t*>(tensors[4]);
    a.lengths_out = static_cast<int32_t*>(tensors[5]);
    a.refs_out = static_cast<int32_t*>(tensors[6]);
    a.report = static_cast<int32_t*>(tensors[7]);
    a.header = static_cast<int32_t*>(scratch);
    a.pages_a = a.header + kHeader;
    a.pages_b = a.pages_a + sizes.page_ints();
    a.sequence_a = a.pages_b + sizes.page_ints();
    a.sequence_b = a.sequence_a + sizes.batch_ints();
    a.entry_a = a.sequence_b + sizes.batch_ints();
    a.copies = reinterpret_cast<int2*>(a.entry_a + sizes.entry_ints());
    a.batch = static_cast<int>(sizes.batch);
    a.slots = static_cast<int>(sizes.slots);
    a.pages = static_cast<int>(sizes.pages);
    a.entries = static_cast<int>(sizes.entries);
    a.block = static_cast<int>(p->block);
    CopyArgs c{};
    c.header = a.header;
    c.copies = a.copies;
    c.pools = p->pool_count;
    for (int i = 0; i < p->pool_count; ++i) {
        const dfgpu_tensor& t = p->pools[i];
        const int bytes = dtype_bytes(t.dtype);
        CopyPool& pool = c.pool[i];
        pool.base = static_cast<uint8_t*>(tensors[8 + i]);
        if (!pool.base) return fail(kInvalidArgument, "CACHE_PAGES: pool %d is null", i);
        for (int j = 0; j < i; ++j)
            if (tensors[8 + j] == tensors[8 + i]) return fail(kInvalidArgument, "CACHE_PAGES: pools %d and %d are the same", j, i);
        pool.layer_stride = t.dim[0] > 1 ? t.stride[0] * bytes : 0;
        pool.page_stride = t.dim[1] > 1 ? t.stride[1] * bytes : 0;
        pool.row = t.dim[2] * bytes;
        const int64_t odd = static_cast<int64_t>(reinterpret_cast<uintptr_t>(pool.base)) | pool.layer_stride | pool.page_stride | pool.row;
        pool.width = (odd & 15) == 0 ? 16 : (odd & 3) == 0 ? 4 : 1;
        pool.pieces = static_cast<int>((pool.row + kPiece - 1) / kPiece);
        pool.first = c.per_copy;
        c.per_copy += static_cast<int>(t.dim[0]) * pool.pieces;
    }
    cudaStream_t on = as_stream(stream);
    const dim3 grid(kPagesCtas), block(kPagesThreads);
    switch (p->op) {
        case DFGPU_CACHE_PAGES_RESERVE: launch_chained_cluster(cache_pages_kernel<DFGPU_CACHE_PAGES_RESERVE>, grid, block, kPagesCtas, 0, on, a); break;
        case DFGPU_CACHE_PAGES_FORK: launch_chained_cluster(cache_pages_kernel<DFGPU_CACHE_PAGES_FORK>, grid, block, kPagesCtas, 0, on, a); break;
        case DFGPU_CACHE_PAGES_FREE: launch_chained_cluster(cache_pages_kernel<DFGPU_CACHE_PAGES_FREE>, grid, block, kPagesCtas, 0, on, a); break;
        case DFGPU_CACHE_PAGES_COMPACT: launch_chained_cluster(cache_pages_kernel<DFGPU_CACHE_PAGES_COMPACT>, grid, block, kPagesCtas, 0, on, a); break;
        default: launch_chained_cluster(cache_pages_kernel<DFGPU_CACHE_PAGES_COPY>, grid, block, kPagesCtas, 0, on, a); break;
    }
    status = check_launch("CACHE_PAGES");
    if (status || !p->pool_count) return status;
    launch_chained(cache_copy_kernel, dim3(static_cast<unsigned>(4 * sm_count())), dim3(kCopyThreads), 0, on, c);
    return check_launch("CACHE_PAGES copy");
}
