// The paged 8-bit cache of keys and values: its layout, and the two kernels that fill it and read it back.
//
//   codes   uint8   [layers][pages][kv_heads][page_tokens][head_dim]   value = (code - 128) * scale
//   scales  float32 [layers][pages][kv_heads][page_tokens / 16]        one for 16 consecutive tokens of one head
//
// keys and values alike. A sequence is a row of the table, the pages of its tokens in order. All heads of a page lie together, so
// that a page is one piece of memory per layer when it is copied, and the tokens of one head within it lie together, so that the
// attention of a head reads whole lines.
//
// Codes have an offset of 128 and not a sign: a byte beside 0x64 is then the float16 1024 + code, and one subtraction of 1152
// gives the exact whole number, two codes an instruction. Scales are float32: they are 0.2 % of the bytes.
#pragma once
#include "ptx.cuh"
#include "w4a16_gemm.cuh"

namespace qi {
namespace kv {

constexpr int BLOCK = 16;      // tokens that share a scale
constexpr int ZERO_CODE = 128;

struct Cache {
    uint8_t *codes[2];   // keys, values
    float *scales[2];
    long long first_page;  // of the layer: layer * pages
    int pages, heads, page_shift;
};

struct Tables {
    const int *table, *lengths, *references;
    int sequences, table_pages;
};

struct Batch {
    const int *slots, *offsets;
    int entries, tokens, most;
    const int *shortage;
};

// One entry of a batch: the last `count` tokens of a sequence of `length` tokens, `first` of the batch's token rows on.
struct Entry {
    int slot, first, count, length;
};

__device__ __forceinline__ void complain(uint32_t detail) { atomicCAS(&g_status, 0u, STATUS_BAD_ARGUMENT | detail); }

// The batch's tokens have no pages, and lengths do not count them.
__device__ __forceinline__ bool no_room(const Batch &batch) { return batch.shortage != nullptr && __ldg(batch.shortage) != 0; }

// What the host cannot check without waiting for the device is checked here, by every CTA: nothing is read or written through
// an entry that is not sound, and the status word says so.
__device__ __forceinline__ bool read_entry(const Batch &batch, const Tables &tables, int page_shift, int b, int max_length, Entry &entry) {
    entry.first = __ldg(batch.offsets + b);
    const int end = __ldg(batch.offsets + b + 1);
    entry.count = end - entry.first;
    entry.slot = batch.slots != nullptr ? __ldg(batch.slots + b) : b;
    if (entry.first < 0 || end < entry.first || end > batch.tokens || entry.count > batch.most || entry.slot < 0 || entry.slot >= tables.sequences) return false;
    entry.length = __ldg(tables.lengths + entry.slot);
    return entry.length >= 0 && entry.length <= max_length && ((static_cast<long long>(entry.length) - 1) >> page_shift) < tables.table_pages;
}

// Rows of `dim` codes (and, divided by 16 * dim, blocks) before the one of `token` within page `page` of a head.
__device__ __forceinline__ long long token_row(const Cache &cache, int page, int head, int token) {
    return (((cache.first_page + page) * cache.heads + head) << cache.page_shift) + (token & ((1 << cache.page_shift) - 1));
}

// ---- append ------------------------------------------------------------------------------------------------------
//
// scale = max |new value| * (1 / 127) over the new tokens of a block of 16 and all of a head's channels; where the block holds earlier
// tokens, at least the scale that they have, and if it is more, they are rounded again: rint(code * (old / new)). New codes are
// rint(value / scale). A block's scale never falls while it holds earlier tokens, so writing the same tokens again changes nothing.
//
// A warp takes one block of one head, of the keys or of the values: the maximum is one reduction over the warp, and a lane holds 16 bytes
// of every (32 / (DIM / CHANNELS))-th token, so that loads and stores are whole lines. Bound by memory.
//
// rint(x / scale) is taken as x * (1 / scale), rounded by adding 1.5 * 2^23; the reciprocal is off by 2^-24 and the product by another, so a
// quotient up to 127 is known to 2^-15, and a lane with one that near to a tie takes its eight or four again with the division. (With
// divisions alone, 12 instructions each, 5700 tokens of 32 heads took 30 us more.)

constexpr int UNIT_WARPS = 4;

// What one warp does: block `block` of the batch's entry, tokens [early, end) of it, and where its codes and its scale are.
struct Unit {
    Entry entry;
    int which, head, block, start, early, end;
    uint8_t *codes;  // of the block's first token
    float *scale;
};

// Which tokens of which block; false: nothing to do, or nothing that may be done.
__device__ __forceinline__ bool read_unit(const Cache &cache, const Tables &tables, const Batch &batch, uint32_t detail, Unit &u) {
    if (no_room(batch)) return false;
    const int unit = blockIdx.x * UNIT_WARPS + (threadIdx.x >> 5);  // (block, head, keys or values)
    u.which = unit & 1, u.head = (unit >> 1) % cache.heads;
    const bool sound = read_entry(batch, tables, cache.page_shift, blockIdx.y, 0x7fffffff, u.entry);
    if (!sound || u.entry.count > u.entry.length) {
        if ((threadIdx.x & 31) == 0) complain(detail);
        return false;
    }
    u.start = u.entry.length - u.entry.count, u.block = u.start / BLOCK + (unit >> 1) / cache.heads;
    const int first = u.block * BLOCK;
    u.early = max(u.start - first, 0), u.end = min(u.entry.length - first, BLOCK);
    return u.entry.count > 0 && first < u.entry.length;
}

// Where the block is. The page's number and what it says about others are two trips to memory after the entry's two, so what does not depend
// on them is asked for before.
__device__ __forceinline__ bool place_unit(const Cache &cache, const Tables &tables, int dim, bool writes, uint32_t detail, Unit &u) {
    const int first = u.block * BLOCK;
    const int page = __ldg(tables.table + static_cast<long long>(u.entry.slot) * tables.table_pages + (first >> cache.page_shift));
    if (page < 0 || page >= cache.pages || (writes && __ldg(tables.references + page) != 1)) {  // no page, or one that others hold too
        if ((threadIdx.x & 31) == 0) complain(detail);
        return false;
    }
    const long long row = token_row(cache, page, u.head, first);
    u.codes = (u.which == 0 ? cache.codes[0] : cache.codes[1]) + row * dim;
    u.scale = (u.which == 0 ? cache.scales[0] : cache.scales[1]) + row / BLOCK;
    return true;
}

template <typename T>
__device__ __forceinline__ void load_values(const T *source, float (&x)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(source));
        const uint32_t pairs[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&pairs[j]));
            x[2 * j] = f.x, x[2 * j + 1] = f.y;
        }
    } else {
        const float4 w = __ldg(reinterpret_cast<const float4 *>(source));
        x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
    }
}

// The larger one in magnitude; NaN where either is.
__device__ __forceinline__ float larger_or_nan(float peak, float x) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(peak), "f"(fabsf(x)));
    return y;
}

constexpr uint32_t INFINITE = 0x7f800000u;  // as bits: NaN's are above
constexpr float ROUND_MAGIC = 12582912.0f, NEAR_TIE = 0.5f - 1.0f / 16384.0f, LEAST_NORMAL_SCALE = 1e-36f;

template <typename T, int DIM>
__global__ void __launch_bounds__(UNIT_WARPS * 32) append_kernel(Cache cache, Tables tables, Batch batch, const T *k, const T *v, long long ld_k, long long ld_v) {
    constexpr int CHANNELS = 16 / sizeof(T), LANES = DIM / CHANNELS, TOKENS = 32 / LANES, PASSES = BLOCK / TOKENS;  // lanes to a token, tokens of a pass
    grid_wait();
    const int lane = threadIdx.x & 31;
    Unit u;
    if (!read_unit(cache, tables, batch, 0xC000, u)) return;
    const int within = lane / LANES, channel = lane % LANES * CHANNELS;
    const T *source = (u.which == 0 ? k : v) + static_cast<long long>(u.head) * DIM + channel;
    const long long ld = u.which == 0 ? ld_k : ld_v, row0 = u.entry.first + static_cast<long long>(u.block) * BLOCK - u.start;
    float x[PASSES][CHANNELS];
    float peak;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int token = i * TOKENS + within;
#pragma unroll
        for (int j = 0; j < CHANNELS; ++j) x[i][j] = 0.0f;
        if (token >= u.early && token < u.end) load_values(source + (row0 + token) * ld, x[i]);
    }
    if (!place_unit(cache, tables, DIM, true, 0xC001, u)) return;
    const float old = u.early > 0 ? *u.scale : 0.0f;
    // no negative ones: ordered as whole numbers
    auto largest = [&]() {
        peak = 0.0f;
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
#pragma unroll
            for (int j = 0; j < CHANNELS; ++j) peak = larger_or_nan(peak, x[i][j]);
        peak = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(peak)));
    };
    largest();
    if (__float_as_uint(peak) >= INFINITE) {  // what no scale could hold is 0, and its neighbours stay what they are
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
#pragma unroll
            for (int j = 0; j < CHANNELS; ++j)
                if ((__float_as_uint(x[i][j]) & INFINITE) == INFINITE) x[i][j] = 0.0f;
        largest();
        if (lane == 0) complain(0xC002);
    }
    const float scale = fmaxf(old, __fmul_rn(peak, 1.0f / 127.0f));
    if (u.early > 0 && scale > old) {
        const float factor = __fdiv_rn(old, scale);
        for (int item = lane; item < u.early * (DIM / 4); item += 32) {
            uint32_t *at = reinterpret_cast<uint32_t *>(u.codes) + item;
            const uint32_t w = *at;
            uint32_t out = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int code = static_cast<int>(w >> 8 * b & 255u) - ZERO_CODE;
                out |= static_cast<uint32_t>(__float2int_rn(static_cast<float>(code) * factor) + ZERO_CODE) << 8 * b;
            }
            *at = out;
        }
    }
    const bool normal = scale >= LEAST_NORMAL_SCALE;
    const float inverse = normal ? __frcp_rn(scale) : 0.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int token = i * TOKENS + within;
        if (token < u.early || token >= u.end) continue;
        uint32_t bits[CHANNELS];
        float furthest = 0.0f;
#pragma unroll
        for (int j = 0; j < CHANNELS; ++j) {
            const float q = x[i][j] * inverse, rounded = q + ROUND_MAGIC;
            furthest = fmaxf(furthest, fabsf(q - (rounded - ROUND_MAGIC)));
            bits[j] = __float_as_uint(rounded);
        }
        if (!(furthest < NEAR_TIE) || !normal) {
#pragma unroll
            for (int j = 0; j < CHANNELS; ++j) bits[j] = scale > 0.0f ? static_cast<uint32_t>(min(max(__float2int_rn(__fdiv_rn(x[i][j], scale)), -127), 127)) : 0u;
        }
        uint32_t words[CHANNELS / 4];
#pragma unroll
        for (int j = 0; j < CHANNELS / 4; ++j)  // the lowest bytes; two's complement becomes an offset of 128
            words[j] = __byte_perm(__byte_perm(bits[4 * j], bits[4 * j + 1], 0x0040), __byte_perm(bits[4 * j + 2], bits[4 * j + 3], 0x0040), 0x5410) ^ 0x80808080u;
        uint8_t *at = u.codes + token * DIM + channel;
        if constexpr (CHANNELS == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(words[0], words[1]);
        else *reinterpret_cast<uint32_t *>(at) = words[0];
    }
    __syncwarp();
    if (lane == 0) *u.scale = scale;
}

// ---- read back -----------------------------------------------------------------------------------------------------
//
// (code - 128) * scale of the last tokens of each entry, rounded once. The same units as above; a lane takes four adjacent channels, so
// that a warp writes whole lines.

template <typename T, int DIM>
__global__ void __launch_bounds__(UNIT_WARPS * 32) read_kernel(Cache cache, Tables tables, Batch batch, T *k, T *v, long long ld_k, long long ld_v) {
    constexpr int LANES = DIM / 4, TOKENS = 32 / LANES, PASSES = BLOCK / TOKENS;
    grid_wait();
    const int lane = threadIdx.x & 31;
    Unit u;
    if (!read_unit(cache, tables, batch, 0xC010, u) || !place_unit(cache, tables, DIM, false, 0xC011, u)) return;
    const int within = lane / LANES, channel = lane % LANES * 4;
    const float scale = *u.scale;
    uint32_t words[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) words[i] = *reinterpret_cast<const uint32_t *>(u.codes + (i * TOKENS + within) * DIM + channel);
    const long long ld = u.which == 0 ? ld_k : ld_v, row0 = u.entry.first + static_cast<long long>(u.block) * BLOCK - u.start;
    T *out = (u.which == 0 ? k : v) + static_cast<long long>(u.head) * DIM + channel;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int token = i * TOKENS + within;
        if (token < u.early || token >= u.end) continue;
        float x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = static_cast<float>(static_cast<int>(words[i] >> 8 * b & 255u) - ZERO_CODE) * scale;
        T *at = out + (row0 + token) * ld;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(at) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
            const __half2 low = __floats2half2_rn(x[0], x[1]), high = __floats2half2_rn(x[2], x[3]);
            *reinterpret_cast<uint2 *>(at) = make_uint2(*reinterpret_cast<const uint32_t *>(&low), *reinterpret_cast<const uint32_t *>(&high));
        }
    }
}

}  // namespace kv
}  // namespace qi
