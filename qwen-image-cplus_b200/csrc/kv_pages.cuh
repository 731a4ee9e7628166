// Upkeep of the cache's pages, all of it on the device: no call waits, and a captured graph can hold them. `references[page]` says
// how many sequences hold a page, 0 = free; new pages are always the lowest free ones, so results do not depend on timing.
//
// One CTA decides (which pages are free is a running count over `references`; the lists are short), and a second launch copies
// what has to be copied with the whole GPU. The copies are bound by memory, page by page of every layer at once; the decision costs
// a launch and a few round trips to memory.
#pragma once
#include "kv_cache.cuh"

namespace qi {
namespace kv {

constexpr int PLAN_THREADS = 1024, PLAN_ITEMS = 4;  // references a thread takes at a time
constexpr int MOST_TABLE_PAGES = 1 << 19;           // the needs of PLAN_THREADS sequences add up in 32 bits

struct PageTables {
    int *table, *lengths, *references;
    int sequences, table_pages, pages, page_shift;
};

// The workspace: how many copies the plan found, their sources and targets, where each page went, a snapshot of tables.
struct PageWork {
    int *count;      // [4]
    int *sources;    // [lists]
    int *targets;    // [lists]
    int *moved;      // [pages]
    int *rows;       // [sequences][table_pages]
    int *held;       // [sequences]
};

// Sum over the CTA of `value` before this thread, and of all.
__device__ __forceinline__ int scan_before(int value, int *warp_sums, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = value;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
        const int below = __shfl_up_sync(0xffffffffu, sum, step);
        if (lane >= step) sum += below;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int all = warp_sums[lane];
#pragma unroll
        for (int step = 1; step < 32; step *= 2) {
            const int below = __shfl_up_sync(0xffffffffu, all, step);
            if (lane >= step) all += below;
        }
        warp_sums[lane] = all;
    }
    __syncthreads();
    const int before = (warp > 0 ? warp_sums[warp - 1] : 0) + sum - value;
    total = warp_sums[31];
    __syncthreads();
    return before;
}

// Writes the pages of [0, below) whose references are zero (or, with LIVE, not) to list[0...) in ascending order, until `most` are
// found; returns how many, at most `most`. `from`: pages before it are passed over.
template <bool LIVE>
__device__ __forceinline__ int collect(const int *references, int from, int below, int most, int *list, int *warp_sums) {
    int found = 0;
    for (int base = from; base < below && found < most; base += PLAN_THREADS * PLAN_ITEMS) {
        const int mine = base + threadIdx.x * PLAN_ITEMS;
        bool take[PLAN_ITEMS];
        int n = 0;
#pragma unroll
        for (int i = 0; i < PLAN_ITEMS; ++i) {
            take[i] = mine + i < below && (references[mine + i] > 0) == LIVE;
            n += take[i];
        }
        int total;
        int at = found + scan_before(n, warp_sums, total);
#pragma unroll
        for (int i = 0; i < PLAN_ITEMS; ++i)
            if (take[i] && at < most) list[at++] = mine + i;
        found += total;
    }
    __syncthreads();  // the list, for every thread of the CTA
    return found < most ? found : most;
}

__device__ __forceinline__ int pages_of(int tokens, int page_shift) { return static_cast<int>((static_cast<long long>(tokens) + (1 << page_shift) - 1) >> page_shift); }

__device__ __forceinline__ bool known(const PageTables &t, int slot) { return slot >= 0 && slot < t.sequences; }

// Room for counts[i] more tokens of sequence slots[i], whose length grows by that: all of them, or none when pages are too few
// (*shortage pages more are wanted; or -1: a sequence or a table that is too small for it).
__global__ void __launch_bounds__(PLAN_THREADS) reserve_kernel(PageTables t, const int *slots, const int *counts, int n, int *shortage, PageWork work) {
    __shared__ int warp_sums[32], wrong;
    grid_wait();
    if (threadIdx.x == 0) wrong = 0;
    __syncthreads();
    int wanted = 0;
    for (int base = 0; base < n; base += PLAN_THREADS) {
        const int i = base + threadIdx.x;
        int need = 0;
        if (i < n) {
            const int slot = slots[i], count = counts[i];
            if (!known(t, slot) || count < 0 || t.lengths[slot] < 0 || count > 0x7fffffff - t.lengths[slot] || pages_of(t.lengths[slot] + count, t.page_shift) > t.table_pages) {
                wrong = 1;
            } else {
                work.held[i] = t.lengths[slot];
                need = pages_of(work.held[i] + count, t.page_shift) - pages_of(work.held[i], t.page_shift);
            }
        }
        int total;
        const int before = scan_before(need, warp_sums, total);
        if (i < n) work.sources[i] = wanted + before;  // the first of its new pages
        wanted += total;
        wanted = min(wanted, 1 << 30);  // far more than there are: no sum runs over (a table has at most MOST_TABLE_PAGES)
    }
    __syncthreads();
    if (wrong) {
        if (threadIdx.x == 0) *shortage = -1, complain(0xC020);
        return;
    }
    const int found = collect<false>(t.references, 0, t.pages, wanted, work.moved, warp_sums);
    if (threadIdx.x == 0) *shortage = wanted - found;
    if (found < wanted) return;
    // A warp takes a sequence: short ones (one new token each) and long ones (a prompt) alike. Its length is the one that was checked, so
    // that a sequence that is named twice, against the rules, does not grow beyond its row or its share of the pages.
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < n; i += PLAN_THREADS / 32) {
        const int slot = slots[i], length = work.held[i], more = counts[i];
        const int have = pages_of(length, t.page_shift), want = pages_of(length + more, t.page_shift), first = work.sources[i];
        for (int j = have + lane; j < want; j += 32) t.table[static_cast<long long>(slot) * t.table_pages + j] = work.moved[first + j - have];
        __syncwarp();
        if (lane == 0) t.lengths[slot] = length + more;
    }
    for (int j = threadIdx.x; j < wanted; j += PLAN_THREADS) t.references[work.moved[j]] = 1;
}

// children[i] becomes what parents[i] was BEFORE the call: its whole pages shared, its last partial one copied to a page of the
// child's own, taken from those that were free before the call. What a child held is given back; child = parent changes nothing.
__global__ void __launch_bounds__(PLAN_THREADS) fork_kernel(PageTables t, const int *parents, const int *children, int n, int *shortage, PageWork work) {
    __shared__ int warp_sums[32], wrong;
    grid_wait();
    if (threadIdx.x == 0) wrong = 0, work.count[0] = 0;
    __syncthreads();
    int wanted = 0;
    for (int base = 0; base < n; base += PLAN_THREADS) {
        const int i = base + threadIdx.x;
        int need = 0;
        if (i < n) {
            const int parent = parents[i], child = children[i];
            if (!known(t, parent) || !known(t, child) || t.lengths[parent] < 0 || pages_of(t.lengths[parent], t.page_shift) > t.table_pages) {
                wrong = 1;
            } else {
                work.held[i] = t.lengths[parent];
                need = parent != child && (t.lengths[parent] & ((1 << t.page_shift) - 1)) != 0;
            }
        }
        int total;
        const int before = scan_before(need, warp_sums, total);
        if (i < n) work.targets[i] = need ? wanted + before : -1;
        wanted += total;
    }
    __syncthreads();
    if (wrong) {
        if (threadIdx.x == 0) *shortage = -1, complain(0xC021);
        return;
    }
    const int found = collect<false>(t.references, 0, t.pages, wanted, work.moved, warp_sums);
    if (threadIdx.x == 0) *shortage = wanted - found;
    if (found < wanted) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the rows as they are, and what is shared, before anything is rewritten
    for (int i = warp; i < n; i += PLAN_THREADS / 32) {
        if (parents[i] == children[i]) continue;
        const int have = pages_of(work.held[i], t.page_shift), whole = work.held[i] >> t.page_shift;
        const int *row = t.table + static_cast<long long>(parents[i]) * t.table_pages;
        for (int j = lane; j < have; j += 32) {
            const int page = row[j];
            work.rows[static_cast<long long>(i) * t.table_pages + j] = page;
            if (page < 0 || page >= t.pages) complain(0xC022);
            else if (j < whole) atomicAdd(t.references + page, 1);
        }
    }
    __syncthreads();
    for (int i = warp; i < n; i += PLAN_THREADS / 32) {
        const int child = children[i];
        if (parents[i] == child) continue;
        int *row = t.table + static_cast<long long>(child) * t.table_pages;
        const int have = pages_of(work.held[i], t.page_shift), whole = work.held[i] >> t.page_shift;
        const int before = min(pages_of(max(t.lengths[child], 0), t.page_shift), t.table_pages);
        // of the last page, which is copied; a parent that has none there leaves its child none either, and not what a free page happens to hold
        const int from = have > whole ? work.rows[static_cast<long long>(i) * t.table_pages + whole] : -1;
        const bool there = from >= 0 && from < t.pages;
        for (int j = lane; j < max(have, before); j += 32) {
            const int gone = j < before ? row[j] : -1;
            if (gone >= 0 && gone < t.pages) atomicSub(t.references + gone, 1);
            int page = -1;
            if (j < whole) page = work.rows[static_cast<long long>(i) * t.table_pages + j];
            else if (j < have && there) page = work.moved[work.targets[i]];
            row[j] = page;
        }
        __syncwarp();
        if (lane == 0) {
            t.lengths[child] = work.held[i];
            if (have > whole) {
                const int rank = work.targets[i];
                if (there) t.references[work.moved[rank]] = 1;
                work.sources[rank] = there ? from : work.moved[rank];
            }
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < wanted; j += PLAN_THREADS) work.targets[j] = work.moved[j];
    if (threadIdx.x == 0) work.count[0] = wanted;
}

// The sequences end: their pages are given back, their lengths become 0.
__global__ void __launch_bounds__(PLAN_THREADS) free_kernel(PageTables t, const int *slots, int n) {
    grid_wait();
    const int lane = threadIdx.x & 31;
    for (int i = (blockIdx.x * PLAN_THREADS + threadIdx.x) >> 5; i < n; i += gridDim.x * (PLAN_THREADS / 32)) {
        const int slot = slots[i];
        if (!known(t, slot)) {
            if (lane == 0) complain(0xC023);
            continue;
        }
        int *row = t.table + static_cast<long long>(slot) * t.table_pages;
        const int have = min(pages_of(max(t.lengths[slot], 0), t.page_shift), t.table_pages);
        for (int j = lane; j < have; j += 32) {
            const int page = row[j];
            if (page >= 0 && page < t.pages) atomicSub(t.references + page, 1);
            row[j] = -1;
        }
        __syncwarp();
        if (lane == 0) t.lengths[slot] = 0;
    }
}

// The live pages, *used of them, move together at the front: the k-th live page from *used on goes to the k-th free one before.
__global__ void __launch_bounds__(PLAN_THREADS) compact_kernel(PageTables t, int *used, PageWork work) {
    __shared__ int warp_sums[32];
    grid_wait();
    int live = 0;
    for (int base = 0; base < t.pages; base += PLAN_THREADS * PLAN_ITEMS) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PLAN_ITEMS; ++i) {
            const int page = base + i * PLAN_THREADS + threadIdx.x;
            n += page < t.pages && t.references[page] > 0;
        }
        live += n;
    }
    int total;
    scan_before(live, warp_sums, total);
    const int holes = collect<false>(t.references, 0, total, t.pages, work.targets, warp_sums);
    collect<true>(t.references, total, t.pages, holes, work.sources, warp_sums);  // as many: what is not below is above
    for (int j = threadIdx.x; j < holes; j += PLAN_THREADS) {
        const int from = work.sources[j], to = work.targets[j];
        work.moved[from] = to;
        t.references[to] = t.references[from];
        t.references[from] = 0;
    }
    if (threadIdx.x == 0) *used = total, work.count[0] = holes, work.count[1] = total;
}

// ---- copies --------------------------------------------------------------------------------------------------------
//
// Pairs of pages, of every layer, keys and values: pieces of 16 KB, one to a CTA at a time, and the page's scales with the first of
// them. `count` is the device's own, so the grid does not depend on it. A compaction renames the tables' pages in the same launch.

// Eight loads of 16 bytes are under way for a thread, and a CTA that ends makes room for another with the next share (COPY_CTAS to an SM, some half
// of them at a time). 180 pages of 16 layers, 379 MB read and written: 65.7 us, 5.8 TB/s; 256 threads of four loads, 8 to an SM, 68.8, and 16 to an
// SM 65.7, but those take 6.8 us for 16 pages, which are 5.9 here.
constexpr int COPY_THREADS = 128, COPY_UNROLL = 8, COPY_CTAS = 16;
constexpr int COPY_PIECE = COPY_THREADS * 16 * COPY_UNROLL;

struct Pool {
    uint8_t *codes[2];
    float *scales[2];
    long long pages;
    int layers, page_bytes, page_scales;
};

__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(Pool pool, const int *count, int fixed_count, const int *sources, const int *targets, PageTables t, const int *moved) {
    grid_wait();
    const int pairs = count != nullptr ? count[0] : fixed_count;
    const int pieces = (pool.page_bytes + COPY_PIECE - 1) / COPY_PIECE;
    const long long items = static_cast<long long>(pairs) * pool.layers * 2 * pieces;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int piece = static_cast<int>(item % pieces);
        const long long rest = item / pieces;
        const int which = static_cast<int>(rest & 1), layer = static_cast<int>((rest >> 1) % pool.layers), pair = static_cast<int>((rest >> 1) / pool.layers);
        const int from = sources[pair], to = targets[pair];
        if (from < 0 || from >= pool.pages || to < 0 || to >= pool.pages) {
            if (threadIdx.x == 0) complain(0xC024);
            continue;
        }
        const long long source = layer * pool.pages + from, target = layer * pool.pages + to;
        const uint4 *in = reinterpret_cast<const uint4 *>(pool.codes[which] + source * pool.page_bytes);
        uint4 *out = reinterpret_cast<uint4 *>(pool.codes[which] + target * pool.page_bytes);
        const int first = piece * (COPY_PIECE / 16) + threadIdx.x, end = pool.page_bytes / 16;
        uint4 words[COPY_UNROLL];
#pragma unroll
        for (int i = 0; i < COPY_UNROLL; ++i)
            if (first + i * COPY_THREADS < end) words[i] = in[first + i * COPY_THREADS];
#pragma unroll
        for (int i = 0; i < COPY_UNROLL; ++i)
            if (first + i * COPY_THREADS < end) out[first + i * COPY_THREADS] = words[i];
        if (piece == 0)
            for (int i = threadIdx.x; i < pool.page_scales; i += COPY_THREADS)
                pool.scales[which][target * pool.page_scales + i] = pool.scales[which][source * pool.page_scales + i];
    }
    if (moved != nullptr && pairs > 0) {
        const int used = count[1];
        const long long entries = static_cast<long long>(t.sequences) * t.table_pages;
        for (long long i = static_cast<long long>(blockIdx.x) * COPY_THREADS + threadIdx.x; i < entries; i += static_cast<long long>(gridDim.x) * COPY_THREADS) {
            const int page = t.table[i];
            if (page >= used && page < t.pages) t.table[i] = moved[page];
        }
    }
}

}  // namespace kv
}  // namespace qi
