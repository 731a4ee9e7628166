// C ABI of the operators between the packed linears (include/qipack_b200.h): the norms around a block, the paged 8-bit cache, the
// attention over it and the upkeep of its pages. Argument checks, plans and launches.
#pragma once
#include <algorithm>

#include "gated_norm.cuh"
#include "kv_cache.cuh"
#include "kv_decode.cuh"
#include "kv_pages.cuh"
#include "kv_prefill.cuh"

namespace qi {
namespace {

// SMs of the current device; where there is none, as many as a B200 has: plans need no device, and a launch then says what is missing.
int sms_or_usual() {
    const int device = current_device();
    return device < 0 ? 148 : sm_count(device);
}

bool aligned4(const void *pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 3) == 0; }
bool known_dtype(int dtype) { return dtype == QI_DTYPE_F32 || dtype == QI_DTYPE_F16; }

// ---- the cache --------------------------------------------------------------------------------------------------------

int page_shift_of(int page_tokens) {
    for (int shift = 4; shift <= 8; ++shift)
        if (page_tokens == 1 << shift) return shift;
    return -1;
}

bool sound(const qi_kv_cache *cache) {
    return cache && cache->k_codes && cache->v_codes && cache->k_scales && cache->v_scales && aligned16(cache->k_codes) && aligned16(cache->v_codes) &&
           aligned4(cache->k_scales) && aligned4(cache->v_scales) && cache->layers > 0 && cache->pages > 0 && cache->kv_heads > 0 &&
           cache->kv_heads <= 4096 && (cache->head_dim == 64 || cache->head_dim == 128) && page_shift_of(cache->page_tokens) > 0;
}
bool sound(const qi_kv_pages *pages) {
    return pages && pages->table && pages->lengths && pages->references && aligned4(pages->table) && aligned4(pages->lengths) && aligned4(pages->references) &&
           pages->sequences > 0 && pages->table_pages > 0 && pages->table_pages <= kv::MOST_TABLE_PAGES;
}
bool sound(const qi_kv_batch *batch) {
    return batch && batch->offsets && aligned4(batch->offsets) && aligned4(batch->slots) && aligned4(batch->shortage) && batch->entries >= 0 && batch->entries <= 65535 && batch->tokens >= 0 && batch->most >= 0;
}

kv::Cache layer_of(const qi_kv_cache *cache, int layer) {
    kv::Cache c;
    c.codes[0] = static_cast<uint8_t *>(cache->k_codes), c.codes[1] = static_cast<uint8_t *>(cache->v_codes);
    c.scales[0] = cache->k_scales, c.scales[1] = cache->v_scales;
    c.first_page = static_cast<long long>(layer) * cache->pages;
    c.pages = cache->pages, c.heads = cache->kv_heads, c.page_shift = page_shift_of(cache->page_tokens);
    return c;
}
kv::Tables tables_of(const qi_kv_pages *pages) { return {pages->table, pages->lengths, pages->references, pages->sequences, pages->table_pages}; }
kv::Batch batch_of(const qi_kv_batch *batch) { return {batch->slots, batch->offsets, batch->entries, batch->tokens, batch->most, batch->shortage}; }

// A launch of any grid. It may start while the kernel before it in the stream ends, if that one calls grid_release() (the packed linears do; the kernels of this
// file do not, so behind one another they start when the one before has ended).
template <typename... Parameters, typename... Arguments>
int launch_grid(void (*kernel)(Parameters...), dim3 grid, int threads, int smem_bytes, void *stream, const Arguments &...arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem_bytes;
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return static_cast<int>(launched(cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...)));
}

// CTAs to an entry for the kernels that take a block of a head with each warp, of keys or of values; -1: too many. `most` may be any bound, but no
// sequence has more blocks than its row of the table, so a block's first token stays below 2 * MOST_TABLE_PAGES pages, far from 2^31.
long long cache_grid(const qi_kv_cache *cache, const qi_kv_pages *pages, const qi_kv_batch *batch) {
    const long long touched = (static_cast<long long>(batch->most) + 2 * kv::BLOCK - 2) / kv::BLOCK;  // by `most` tokens in a row
    const long long blocks = std::min(touched, static_cast<long long>(pages->table_pages) * cache->page_tokens / kv::BLOCK);
    const long long grid = (blocks * cache->kv_heads * 2 + kv::UNIT_WARPS - 1) / kv::UNIT_WARPS;
    return grid > 0x7fffffff / kv::UNIT_WARPS ? -1 : grid;
}

template <typename T>
int launch_append(const qi_kv_cache *cache, const qi_kv_pages *pages, const qi_kv_batch *batch, int layer, const void *k, const void *v, long long ld_k, long long ld_v, void *stream) {
    const long long grid = cache_grid(cache, pages, batch);
    if (grid < 0) return INVALID;
    auto kernel = cache->head_dim == 128 ? kv::append_kernel<T, 128> : kv::append_kernel<T, 64>;
    return launch_grid(kernel, dim3(static_cast<unsigned>(grid), batch->entries), kv::UNIT_WARPS * 32, 0, stream, layer_of(cache, layer), tables_of(pages), batch_of(batch),
                       static_cast<const T *>(k), static_cast<const T *>(v), ld_k, ld_v);
}

template <typename T>
int launch_read(const qi_kv_cache *cache, const qi_kv_pages *pages, const qi_kv_batch *batch, int layer, void *k, void *v, long long ld_k, long long ld_v, void *stream) {
    const long long grid = cache_grid(cache, pages, batch);
    if (grid < 0) return INVALID;
    auto kernel = cache->head_dim == 128 ? kv::read_kernel<T, 128> : kv::read_kernel<T, 64>;
    return launch_grid(kernel, dim3(static_cast<unsigned>(grid), batch->entries), kv::UNIT_WARPS * 32, 0, stream, layer_of(cache, layer), tables_of(pages), batch_of(batch),
                       static_cast<T *>(k), static_cast<T *>(v), ld_k, ld_v);
}

// ---- attention ----------------------------------------------------------------------------------------------------------

struct AttentionPlan {
    int tiles;  // of 8 query rows on mma.sync; 0: of 256 on tcgen05
    int grid;   // of the former
    int row_tiles, chunk, splits;
    size_t partial_offset, bytes;
};

// Query rows to a sequence and head of the cache up to which the streaming kernel takes a call. 64 sequences of 2048 to 8192 tokens, 8 heads:
// with 4 rows 123 us there and 324 on tcgen05, with 16 rows 152 and 393; one of 8192 with 16 rows 25 and 43. It has no form for more.
constexpr int DECODE_ROWS = 16;

// A bound of lengths, cut to the tokens of a row of the table: at most 2^27, so that no piece of it leaves int and a loose bound costs nothing.
int held_length(const qi_kv_cache *cache, int table_pages, int max_length) { return std::min(max_length, table_pages * cache->page_tokens); }

// CTAs of the streaming kernel, and its workspace. One counter for each of its CTAs, or for each tile of rows that is cut into pieces (at most half as
// many as SMs), lies at the same place for every call, so that calls of different shapes may share a workspace.
size_t counter_bytes(int sms) { return (static_cast<size_t>(sms) * 3 * 4 + 255) / 256 * 256; }
int streaming_grid(const qi_kv_cache *cache, int tiles, int sms) {
    return sms * (cache->head_dim == 128 ? (tiles == 1 ? kv::Decode<128, 1>::CTAS : kv::Decode<128, 2>::CTAS) : (tiles == 1 ? kv::Decode<64, 1>::CTAS : kv::Decode<64, 2>::CTAS));
}
size_t streaming_bytes(const qi_kv_cache *cache, int tiles, int max_length, int sms) {  // units of one round each are never shared
    return max_length <= kv::ROUND ? 0 : counter_bytes(sms) + static_cast<size_t>(streaming_grid(cache, tiles, sms)) * 2 * (8 * tiles) * (cache->head_dim + 2) * 4;
}
// The workspace of so many tiles of rows, with room for as many pieces as any window gives.
size_t piece_bytes(const qi_kv_cache *cache, long long units, int max_length, int sms) {
    const long long most = std::min(sms / units, (max_length + kv::TILE_TOKENS - 1LL) / kv::TILE_TOKENS);
    return most > 1 ? counter_bytes(sms) + static_cast<size_t>(units) * most * kv::PREFILL_ROWS * (cache->head_dim + 2) * 4 : 0;
}

// How a call is cut. The streaming kernel shares the tokens out by itself. The other one takes a CTA to a tile of rows, one to an SM, and
// where there are too few tiles for the GPU, several to pieces of its tokens.
bool plan_attention(const qi_kv_cache *cache, const qi_kv_batch *batch, int heads, int max_length, int window, int sms, AttentionPlan &plan) {
    if (heads <= 0 || heads % cache->kv_heads != 0 || max_length < 0 || window < 0) return false;
    const long long rows = static_cast<long long>(batch->most) * (heads / cache->kv_heads), entries = batch->entries > 0 ? batch->entries : 1;
    plan.tiles = rows <= 8 ? 1 : rows <= DECODE_ROWS ? 2 : 0;
    plan.partial_offset = counter_bytes(sms);
    plan.grid = streaming_grid(cache, plan.tiles, sms);
    plan.row_tiles = 1, plan.chunk = 0, plan.splits = 1;
    if (plan.tiles > 0) {
        plan.bytes = streaming_bytes(cache, plan.tiles, max_length, sms);
        return true;
    }
    const long long row_tiles = (rows + kv::PREFILL_ROWS - 1) / kv::PREFILL_ROWS;
    if (row_tiles * cache->kv_heads > 65535) return false;
    plan.row_tiles = static_cast<int>(row_tiles);
    const long long units = row_tiles * cache->kv_heads * entries;
    long long span = max_length;  // of the tokens that a tile can see
    if (window > 0 && static_cast<long long>(window) + batch->most + kv::BLOCK < span) span = static_cast<long long>(window) + batch->most + kv::BLOCK;
    const long long pieces = sms / units > 1 ? sms / units : 1;
    long long chunk = (span + pieces - 1) / pieces;
    chunk = (chunk + kv::TILE_TOKENS - 1) / kv::TILE_TOKENS * kv::TILE_TOKENS;
    if (chunk < kv::TILE_TOKENS) chunk = kv::TILE_TOKENS;
    plan.chunk = static_cast<int>(chunk), plan.splits = static_cast<int>(span > 0 ? (span + chunk - 1) / chunk : 1);
    plan.bytes = piece_bytes(cache, units, max_length, sms);
    return true;
}

// What any call within the bounds of `batch` and `max_length` needs: few tiles of rows are cut into pieces, so a smaller call can need more.
bool attention_bytes(const qi_kv_cache *cache, const qi_kv_batch *batch, int heads, int max_length, int sms, size_t &bytes) {
    AttentionPlan plan;
    if (!plan_attention(cache, batch, heads, max_length, 0, sms, plan)) return false;
    bytes = std::max(plan.bytes, streaming_bytes(cache, 1, max_length, sms));
    const long long rows = static_cast<long long>(batch->most) * (heads / cache->kv_heads);
    if (rows > 8) bytes = std::max(bytes, streaming_bytes(cache, 2, max_length, sms));
    if (plan.tiles == 0)
        for (long long units = cache->kv_heads; units <= std::min(static_cast<long long>(plan.row_tiles) * cache->kv_heads * std::max(batch->entries, 1), sms / 2LL); units += cache->kv_heads)
            bytes = std::max(bytes, piece_bytes(cache, units, max_length, sms));
    return true;
}

template <int DIM, int TILES>
int launch_decode(const dim3 grid, const kv::Cache &cache, const kv::Tables &tables, const kv::Batch &batch, const kv::Attention &a, void *stream) {
    const int device = current_device();
    if (device < 0) return static_cast<int>(cudaErrorNoDevice);
    static std::atomic<bool> configured[MAX_DEVICES];
    if (const cudaError_t error = configure_once(kv::decode_kernel<DIM, TILES>, kv::Decode<DIM, TILES>::SMEM_BYTES, configured[device])) return static_cast<int>(error);
    return launch_grid(kv::decode_kernel<DIM, TILES>, grid, kv::DECODE_THREADS, kv::Decode<DIM, TILES>::SMEM_BYTES, stream, cache, tables, batch, a);
}

template <int DIM>
int launch_prefill(const dim3 grid, const kv::Cache &cache, const kv::Tables &tables, const kv::Batch &batch, const kv::Attention &a, void *stream) {
    const int device = current_device();
    if (device < 0) return static_cast<int>(cudaErrorNoDevice);
    static std::atomic<bool> configured[MAX_DEVICES];
    if (const cudaError_t error = configure_once(kv::prefill_kernel<DIM>, kv::Prefill<DIM>::SMEM_BYTES, configured[device])) return static_cast<int>(error);
    return launch_grid(kv::prefill_kernel<DIM>, grid, kv::PREFILL_THREADS, kv::Prefill<DIM>::SMEM_BYTES, stream, cache, tables, batch, a);
}

// As many CTAs as run at once, each with its share of the rows: with twice as many, a last round left SMs idle.
template <int THREADS, int PIECES>
int launch_norm(const gated_norm::Arguments &a, void *stream) {
    const int device = current_device();
    if (device < 0) return static_cast<int>(cudaErrorNoDevice);
    static std::atomic<int> cached[MAX_DEVICES];
    int ctas = cached[device].load(std::memory_order_relaxed);
    if (ctas == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, gated_norm::norm_kernel<THREADS, PIECES>, THREADS, 0) != cudaSuccess || ctas <= 0) {
            (void)cudaGetLastError();
            ctas = 1;
        }
        cached[device].store(ctas, std::memory_order_relaxed);
    }
    return launch_grid(gated_norm::norm_kernel<THREADS, PIECES>, dim3(std::min(a.rows, ctas * sm_count(device))), THREADS, 0, stream, a);
}

kv::PageTables page_tables_of(const qi_kv_cache *cache, const qi_kv_pages *pages) {
    return {pages->table, pages->lengths, pages->references, pages->sequences, pages->table_pages, cache->pages, page_shift_of(cache->page_tokens)};
}

size_t page_work_bytes(const qi_kv_cache *cache, const qi_kv_pages *pages) {
    const size_t lists = static_cast<size_t>(cache->pages > pages->sequences ? cache->pages : pages->sequences);
    return 4 * (4 + 2 * lists + cache->pages + static_cast<size_t>(pages->sequences) * pages->table_pages + pages->sequences);
}

kv::PageWork page_work_of(const qi_kv_cache *cache, const qi_kv_pages *pages, void *workspace) {
    const size_t lists = static_cast<size_t>(cache->pages > pages->sequences ? cache->pages : pages->sequences);
    kv::PageWork work;
    work.count = static_cast<int *>(workspace);
    work.sources = work.count + 4;
    work.targets = work.sources + lists;
    work.moved = work.targets + lists;
    work.rows = work.moved + cache->pages;
    work.held = work.rows + static_cast<size_t>(pages->sequences) * pages->table_pages;
    return work;
}

int launch_copies(const qi_kv_cache *cache, const kv::PageTables &tables, const int *count, long long fixed_count, const int *sources, const int *targets, const int *moved, void *stream) {
    kv::Pool pool;
    pool.codes[0] = static_cast<uint8_t *>(cache->k_codes), pool.codes[1] = static_cast<uint8_t *>(cache->v_codes);
    pool.scales[0] = cache->k_scales, pool.scales[1] = cache->v_scales;
    pool.pages = cache->pages, pool.layers = cache->layers;
    pool.page_bytes = cache->kv_heads * cache->page_tokens * cache->head_dim;
    pool.page_scales = cache->kv_heads * (cache->page_tokens / kv::BLOCK);
    return launch_grid(kv::copy_kernel, dim3(sms_or_usual() * kv::COPY_CTAS), kv::COPY_THREADS, 0, stream, pool, count, static_cast<int>(fixed_count), sources, targets, tables, moved);
}

}  // namespace
}  // namespace qi

using namespace qi;

extern "C" {

int qi_kv_append_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, const qi_kv_batch *batch, int layer, const void *k, const void *v, int dtype, long long ld_k, long long ld_v,
                    void *stream) {
    if (!sound(cache) || !sound(pages) || !sound(batch) || layer < 0 || layer >= cache->layers || !known_dtype(dtype)) return INVALID;
    const long long width = static_cast<long long>(cache->kv_heads) * cache->head_dim, step = dtype == QI_DTYPE_F16 ? 8 : 4;
    if (!k || !v || !aligned16(k) || !aligned16(v) || ld_k < width || ld_v < width || ld_k % step != 0 || ld_v % step != 0) return INVALID;
    if (batch->entries == 0 || batch->most == 0) return 0;
    return dtype == QI_DTYPE_F16 ? launch_append<__half>(cache, pages, batch, layer, k, v, ld_k, ld_v, stream) : launch_append<float>(cache, pages, batch, layer, k, v, ld_k, ld_v, stream);
}

int qi_kv_read_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, const qi_kv_batch *batch, int layer, void *k, void *v, int dtype, long long ld_k, long long ld_v, void *stream) {
    if (!sound(cache) || !sound(pages) || !sound(batch) || layer < 0 || layer >= cache->layers || !known_dtype(dtype)) return INVALID;
    const long long width = static_cast<long long>(cache->kv_heads) * cache->head_dim, step = dtype == QI_DTYPE_F16 ? 8 : 4;
    if (!k || !v || !aligned16(k) || !aligned16(v) || ld_k < width || ld_v < width || ld_k % step != 0 || ld_v % step != 0) return INVALID;
    if (batch->entries == 0 || batch->most == 0) return 0;
    return dtype == QI_DTYPE_F16 ? launch_read<__half>(cache, pages, batch, layer, k, v, ld_k, ld_v, stream) : launch_read<float>(cache, pages, batch, layer, k, v, ld_k, ld_v, stream);
}

int qi_kv_attention_workspace(const qi_kv_cache *cache, const qi_kv_batch *batch, int heads, int max_length, size_t *bytes) {
    if (!sound(cache) || !sound(batch) || !bytes || !attention_bytes(cache, batch, heads, held_length(cache, kv::MOST_TABLE_PAGES, max_length), sms_or_usual(), *bytes)) return INVALID;
    return 0;
}

int qi_kv_attention_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, const qi_kv_batch *batch, const qi_kv_attention *call, void *workspace, size_t workspace_bytes, void *stream) {
    if (!sound(cache) || !sound(pages) || !sound(batch) || !call || call->layer < 0 || call->layer >= cache->layers) return INVALID;
    if (call->heads <= 0 || call->heads % cache->kv_heads != 0 || call->heads > (1 << 20) / cache->head_dim) return INVALID;
    const long long width = static_cast<long long>(call->heads) * cache->head_dim;
    if (!call->q || !call->y || !aligned16(call->q) || !aligned16(call->y) || !aligned4(call->lse) || call->ld_q < width || call->ld_y < width || call->ld_q % 8 != 0 ||
        call->ld_y % 8 != 0 || !(call->scale > 0.0f) || !(call->scale < INFINITY))
        return INVALID;
    const int max_length = held_length(cache, pages->table_pages, call->max_length);
    AttentionPlan plan;
    if (!plan_attention(cache, batch, call->heads, max_length, call->window, sms_or_usual(), plan)) return INVALID;
    if (plan.bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < plan.bytes)) return INVALID;
    if (batch->entries == 0 || batch->most == 0) return 0;
    kv::Attention a;
    a.q = static_cast<const __half *>(call->q), a.y = static_cast<__half *>(call->y), a.lse = call->lse;
    a.ld_q = call->ld_q, a.ld_y = call->ld_y;
    a.heads = call->heads, a.group = call->heads / cache->kv_heads;
    a.scale_log2 = call->scale * 1.4426950408889634f;
    a.causal = call->causal, a.window = call->window, a.max_length = max_length;
    a.chunk = plan.chunk, a.splits = plan.splits, a.row_tiles = plan.row_tiles;
    a.arrivals = static_cast<int *>(workspace);
    a.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.partial_offset);
    const dim3 grid = plan.tiles > 0 ? dim3(plan.grid) : dim3(plan.splits, cache->kv_heads * plan.row_tiles, batch->entries);
    if (plan.tiles == 0)
        return cache->head_dim == 128 ? launch_prefill<128>(grid, layer_of(cache, call->layer), tables_of(pages), batch_of(batch), a, stream)
                                      : launch_prefill<64>(grid, layer_of(cache, call->layer), tables_of(pages), batch_of(batch), a, stream);
    auto launch = cache->head_dim == 128 ? (plan.tiles == 1 ? launch_decode<128, 1> : launch_decode<128, 2>) : (plan.tiles == 1 ? launch_decode<64, 1> : launch_decode<64, 2>);
    return launch(grid, layer_of(cache, call->layer), tables_of(pages), batch_of(batch), a, stream);
}

int qi_kv_pages_workspace(const qi_kv_cache *cache, const qi_kv_pages *pages, size_t *bytes) {
    if (!sound(cache) || !sound(pages) || !bytes) return INVALID;
    *bytes = page_work_bytes(cache, pages);
    return 0;
}

int qi_kv_pages_reserve_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, const int *slots, const int *counts, int n, int *shortage, void *workspace, size_t workspace_bytes,
                           void *stream) {
    if (!sound(cache) || !sound(pages) || !slots || !counts || !shortage || !aligned4(slots) || !aligned4(counts) || !aligned4(shortage) || n < 0 || n > pages->sequences ||
        !workspace || !aligned16(workspace) || workspace_bytes < page_work_bytes(cache, pages))
        return INVALID;
    return launch_grid(kv::reserve_kernel, dim3(1), kv::PLAN_THREADS, 0, stream, page_tables_of(cache, pages), slots, counts, n, shortage, page_work_of(cache, pages, workspace));
}

int qi_kv_pages_fork_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, const int *parents, const int *children, int n, int *shortage, void *workspace, size_t workspace_bytes,
                        void *stream) {
    if (!sound(cache) || !sound(pages) || !parents || !children || !shortage || !aligned4(parents) || !aligned4(children) || !aligned4(shortage) || n < 0 || n > pages->sequences ||
        !workspace || !aligned16(workspace) || workspace_bytes < page_work_bytes(cache, pages))
        return INVALID;
    const kv::PageTables tables = page_tables_of(cache, pages);
    const kv::PageWork work = page_work_of(cache, pages, workspace);
    const int status = launch_grid(kv::fork_kernel, dim3(1), kv::PLAN_THREADS, 0, stream, tables, parents, children, n, shortage, work);
    return status != 0 ? status : launch_copies(cache, tables, work.count, 0, work.sources, work.targets, nullptr, stream);
}

int qi_kv_pages_free_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, const int *slots, int n, void *stream) {
    if (!sound(cache) || !sound(pages) || !slots || !aligned4(slots) || n < 0 || n > pages->sequences) return INVALID;
    if (n == 0) return 0;
    const int grid = (n + kv::PLAN_THREADS / 32 - 1) / (kv::PLAN_THREADS / 32);
    return launch_grid(kv::free_kernel, dim3(grid), kv::PLAN_THREADS, 0, stream, page_tables_of(cache, pages), slots, n);
}

int qi_kv_pages_compact_ex(const qi_kv_cache *cache, const qi_kv_pages *pages, int *used, void *workspace, size_t workspace_bytes, void *stream) {
    if (!sound(cache) || !sound(pages) || !used || !aligned4(used) || !workspace || !aligned16(workspace) || workspace_bytes < page_work_bytes(cache, pages)) return INVALID;
    const kv::PageTables tables = page_tables_of(cache, pages);
    const kv::PageWork work = page_work_of(cache, pages, workspace);
    const int status = launch_grid(kv::compact_kernel, dim3(1), kv::PLAN_THREADS, 0, stream, tables, used, work);
    return status != 0 ? status : launch_copies(cache, tables, work.count, 0, work.sources, work.targets, work.moved, stream);
}

int qi_kv_pages_copy_ex(const qi_kv_cache *cache, const int *sources, const int *targets, int n, void *stream) {
    if (!sound(cache) || !sources || !targets || !aligned4(sources) || !aligned4(targets) || n < 0 || n > cache->pages) return INVALID;
    if (n == 0) return 0;
    return launch_copies(cache, kv::PageTables{}, nullptr, n, sources, targets, nullptr, stream);
}

int qi_gated_norm_ex(const qi_gated_norm *call, void *stream) {
    if (!call || call->rows < 0 || call->width <= 0 || call->width > gated_norm::MOST_WIDTH || call->width % 8 != 0) return INVALID;
    if (call->kind != QI_NORM_LAYER && call->kind != QI_NORM_RMS) return INVALID;
    if (!known_dtype(call->residual_dtype) || !known_dtype(call->branch_dtype) || !known_dtype(call->vector_dtype) || !known_dtype(call->y_dtype)) return INVALID;
    if (!call->residual || (!call->y && !call->residual_out) || !(call->epsilon >= 0.0f) || !(call->epsilon < INFINITY)) return INVALID;
    const void *pointers[] = {call->residual, call->branch, call->branch_weight, call->gate, call->scale, call->shift, call->weight, call->residual_out, call->y};
    for (const void *pointer : pointers)
        if (!aligned16(pointer)) return INVALID;
    if (!call->branch && (call->branch_norm || call->branch_weight || call->gate)) return INVALID;  // nothing to apply them to
    if (call->gate || call->scale || call->shift)
        if (call->rows_per_vector <= 0 || call->ld_vector < call->width || call->ld_vector % 8 != 0) return INVALID;
    if (call->rows == 0) return 0;
    gated_norm::Arguments a;
    a.residual = call->residual, a.branch = call->branch, a.branch_weight = call->branch_weight;
    a.gate = call->gate, a.scale = call->scale, a.shift = call->shift, a.weight = call->weight;
    a.residual_out = call->residual_out, a.y = call->y;
    a.ld_vector = call->ld_vector, a.rows = call->rows, a.width = call->width;
    a.rows_per_vector = call->rows_per_vector > 0 ? call->rows_per_vector : call->rows;
    a.residual_scale = call->residual_scale, a.epsilon = call->epsilon;
    a.residual_f16 = call->residual_dtype == QI_DTYPE_F16, a.branch_f16 = call->branch_dtype == QI_DTYPE_F16;
    a.vector_f16 = call->vector_dtype == QI_DTYPE_F16, a.y_f16 = call->y_dtype == QI_DTYPE_F16;
    a.branch_norm = call->branch_norm != 0, a.layer = call->kind == QI_NORM_LAYER;
    // Threads for whole widths: idle ones hold registers that a row in flight could have. 16384 rows of 512 columns with 64 threads 21 us, with 128
    // 28; of 768 with 96 28, with 128 31; of 1280 with 160 46, with 256 58; of 1536 with 192 53, with 256 62. 8192 rows of 2560 with 160 48, with
    // 256 56; of 3072 with 192 57, with 256 61. 4096 rows of 5120 with 320 55, with 512 65; of 6144 with 384 63, with 512 70. Of 224 or 448 no more
    // fit than of 256 or 512, and nothing was gained.
    if (a.width <= 512) return launch_norm<64, 1>(a, stream);
    if (a.width <= 768) return launch_norm<96, 1>(a, stream);
    if (a.width <= 1024) return launch_norm<128, 1>(a, stream);
    if (a.width <= 1280) return launch_norm<160, 1>(a, stream);
    if (a.width <= 1536) return launch_norm<192, 1>(a, stream);
    if (a.width <= 2048) return launch_norm<256, 1>(a, stream);
    if (a.width <= 2560) return launch_norm<160, 2>(a, stream);
    if (a.width <= 3072) return launch_norm<192, 2>(a, stream);
    if (a.width <= 4096) return launch_norm<256, 2>(a, stream);
    if (a.width <= 5120) return launch_norm<320, 2>(a, stream);
    if (a.width <= 6144) return launch_norm<384, 2>(a, stream);
    if (a.width <= 8192) return launch_norm<512, 2>(a, stream);
    return launch_norm<512, 4>(a, stream);
}

}  // extern "C"
