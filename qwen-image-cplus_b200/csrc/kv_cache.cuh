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
};

// One entry of a batch: the last `count` tokens of a sequence of `length` tokens, `first` of the batch's token rows on.
struct Entry {
    int slot, first, count, length;
};

__device__ __forceinline__ void complain(uint32_t detail) { atomicCAS(&g_status, 0u, STATUS_BAD_ARGUMENT | detail); }

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
// A warp takes one block of one head, of the keys or of the values: a lane holds 16 adjacent channels of every
// (32 / (DIM / 16))-th token, so that codes leave in 16-byte pieces and the maximum is one reduction over the warp.

constexpr int APPEND_WARPS = 4;

template <typename T, int DIM>
__device__ __forceinline__ void load16(const T *source, float (&x)[16]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 *words = reinterpret_cast<const uint4 *>(source);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = __ldg(words + i);
            const uint32_t pairs[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&pairs[j]));
                x[8 * i + 2 * j] = f.x, x[8 * i + 2 * j + 1] = f.y;
            }
        }
    } else {
        const float4 *words = reinterpret_cast<const float4 *>(source);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 w = __ldg(words + i);
            x[4 * i] = w.x, x[4 * i + 1] = w.y, x[4 * i + 2] = w.z, x[4 * i + 3] = w.w;
        }
    }
}

// rint(x / scale) as a code, for |x| <= 127.5 * scale or so; a NaN becomes the code of zero.
__device__ __forceinline__ uint32_t to_code(float x, float scale) {
    const int code = __float2int_rn(__fdiv_rn(x, scale));
    return static_cast<uint32_t>(min(max(code, -127), 127) + ZERO_CODE);
}

template <typename T, int DIM>
__global__ void __launch_bounds__(APPEND_WARPS * 32) append_kernel(Cache cache, Tables tables, Batch batch, const T *k, const T *v, long long ld_k, long long ld_v) {
    constexpr int LANES = DIM / 16, TOKENS = 32 / LANES, PASSES = BLOCK / TOKENS;  // lanes to a token, tokens and passes of a warp
    grid_wait();
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);  // (block, head, keys or values)
    const int which = unit & 1, head = (unit >> 1) % cache.heads, nth = (unit >> 1) / cache.heads;
    Entry entry;
    const bool sound = read_entry(batch, tables, cache.page_shift, blockIdx.y, 0x7fffffff, entry);
    if (!sound || entry.count > entry.length) {
        if (lane == 0) complain(0xC000);
        return;
    }
    const int start = entry.length - entry.count, block = start / BLOCK + nth;
    if (entry.count == 0 || block * BLOCK >= entry.length) return;
    const int page = __ldg(tables.table + static_cast<long long>(entry.slot) * tables.table_pages + (block * BLOCK >> cache.page_shift));
    if (page < 0 || page >= cache.pages || __ldg(tables.references + page) != 1) {  // no page, or one that others hold too
        if (lane == 0) complain(0xC001);
        return;
    }
    const int within = lane / LANES, channel = lane % LANES * 16;
    const int early = max(start - block * BLOCK, 0), end = min(entry.length - block * BLOCK, BLOCK);  // tokens of the block: [early, end) are new
    const T *source = (which == 0 ? k : v) + static_cast<long long>(head) * DIM + channel;
    const long long ld = which == 0 ? ld_k : ld_v;
    float x[PASSES][16];
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int token = i * TOKENS + within;
        if (token >= early && token < end) {
            load16<T, DIM>(source + (entry.first + static_cast<long long>(block) * BLOCK + token - start) * ld, x[i]);
#pragma unroll
            for (int j = 0; j < 16; ++j) peak = fmaxf(peak, fabsf(x[i][j]));
        }
    }
    const long long row = token_row(cache, page, head, block * BLOCK);
    uint8_t *codes = (which == 0 ? cache.codes[0] : cache.codes[1]) + row * DIM + channel;
    float *held = (which == 0 ? cache.scales[0] : cache.scales[1]) + row / BLOCK;
    peak = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(peak)));  // no negative ones: ordered as whole numbers
    const float old = early > 0 ? *held : 0.0f;
    const float scale = fmaxf(old, __fmul_rn(peak, 1.0f / 127.0f));
    if (early > 0 && scale > old) {
        const float factor = __fdiv_rn(old, scale);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int token = i * TOKENS + within;
            if (token >= early) continue;
            uint4 *at = reinterpret_cast<uint4 *>(codes + token * DIM);
            const uint4 w = *at;
            uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t out = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int code = static_cast<int>(words[j] >> 8 * b & 255u) - ZERO_CODE;
                    out |= static_cast<uint32_t>(__float2int_rn(static_cast<float>(code) * factor) + ZERO_CODE) << 8 * b;
                }
                words[j] = out;
            }
            *at = make_uint4(words[0], words[1], words[2], words[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int token = i * TOKENS + within;
        if (token < early || token >= end) continue;
        uint32_t words[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            words[j] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) words[j] |= to_code(x[i][4 * j + b], scale) << 8 * b;
        }
        *reinterpret_cast<uint4 *>(codes + token * DIM) = make_uint4(words[0], words[1], words[2], words[3]);
    }
    __syncwarp();
    if (lane == 0) *held = scale;
}

// ---- read back -----------------------------------------------------------------------------------------------------
//
// (code - 128) * scale of the last tokens of each entry, rounded once. A thread takes four adjacent channels, so that a warp
// writes whole lines; ROWS tokens a thread keep enough loads in flight.

constexpr int READ_THREADS = 256, READ_ROWS = 4;

template <typename T, int DIM>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(Cache cache, Tables tables, Batch batch, T *k, T *v, long long ld_k, long long ld_v) {
    grid_wait();
    Entry entry;
    const bool sound = read_entry(batch, tables, cache.page_shift, blockIdx.y, 0x7fffffff, entry);
    if (!sound || entry.count > entry.length) {
        if (threadIdx.x == 0) complain(0xC010);
        return;
    }
    constexpr int QUADS = DIM / 4;
    const int row_quads = cache.heads * QUADS;
    const int which = blockIdx.z;
    T *out = which == 0 ? k : v;
    const long long ld = which == 0 ? ld_k : ld_v, total = static_cast<long long>(entry.count) * row_quads;
    const long long begin = static_cast<long long>(blockIdx.x) * (READ_THREADS * READ_ROWS) + threadIdx.x;
    const int *pages = tables.table + static_cast<long long>(entry.slot) * tables.table_pages;
    uint32_t words[READ_ROWS];
    float scales[READ_ROWS];
#pragma unroll
    for (int i = 0; i < READ_ROWS; ++i) {
        const long long item = begin + i * READ_THREADS;
        words[i] = 0x80808080u, scales[i] = 0.0f;
        if (item >= total) continue;
        const int t = static_cast<int>(item / row_quads), rest = static_cast<int>(item % row_quads), head = rest / QUADS;
        const int token = entry.length - entry.count + t;
        const int page = __ldg(pages + (token >> cache.page_shift));
        if (page < 0 || page >= cache.pages) {
            complain(0xC011);
            continue;
        }
        const long long row = token_row(cache, page, head, token);
        words[i] = *reinterpret_cast<const uint32_t *>((which == 0 ? cache.codes[0] : cache.codes[1]) + row * DIM + rest % QUADS * 4);
        scales[i] = (which == 0 ? cache.scales[0] : cache.scales[1])[row / BLOCK];
    }
#pragma unroll
    for (int i = 0; i < READ_ROWS; ++i) {
        const long long item = begin + i * READ_THREADS;
        if (item >= total) continue;
        float x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = static_cast<float>(static_cast<int>(words[i] >> 8 * b & 255u) - ZERO_CODE) * scales[i];
        T *at = out + (entry.first + item / row_quads) * ld + item % row_quads * 4;
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
