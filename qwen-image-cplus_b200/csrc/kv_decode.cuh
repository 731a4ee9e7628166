// Attention over the paged 8-bit cache for few queries to a sequence: one token of each request, or a handful.
//
//   y_i = sum_j softmax_j(scale * q_i . k_j) v_j       k_j = (c_j - 128) * sk, v_j = (d_j - 128) * sv, sk and sv one for 16 tokens
//
// The work is a list of rounds of 128 tokens: those of each unit (an entry and a head of the cache, with up to 8 * TILES query rows: group
// heads times tokens) one after the other, unit after unit. Two or three CTAs an SM share it evenly, whatever the lengths, so that all
// end together and each pays only once for its start; a ring of copies runs on from one unit into the next. A CTA's warps take 32 tokens of a round each,
// with sums of their own; warps are joined in shared memory, and a unit that several CTAs share in a workspace, where the CTA that
// arrives last adds the pieces up in their order (the same bits whichever is last). 64 sequences of
// 2048 to 8192 tokens, 8 heads: 120 us, 5.3 TB/s (a CTA to each piece of a unit: 143); one of 131071: 57 us. The slope with the length is 6.2 TB/s; what is left are 10 us of starting, joining
// and launching. What bounds it: HBM, and the instructions that widen codes: 733 for 32 tokens and a warp, 48 % of the issue slots.
//
// The products run transposed on m16n8k16: S^T = K Q^T and O^T = V^T P^T, so that the 16 rows of an instruction are tokens and channels
// of the cache, of which there are always enough, and the 8 columns are queries, of which there may be one. Which channel or
// token stands at which place of a sum is free as long as both operands agree, and is chosen so that every load is 16 adjacent
// codes of a token: codes go as they are through shared memory and are widened in registers.
//
// Scales cost nothing per element. With base-2 logarithms, x_j = (scale * log2 e * sk) * raw_j + log2 sv, m = max x_j, p_j = 2^(x_j - m):
//   O = sum p_j d_j (d_j whole numbers),  l = sum p_j / sv,  y = O / l
// so sk and log2 sv enter one fused multiply-add, and 1 / sv once for the sum of a block. p_j is rounded to float16 for the tensor
// cores; queries are float16 as they come, codes are exact, all sums are float32. m is not the maximum of what has been seen so far but an
// older one: weights are computed with the m that there is, as 2^(x - m + 7), and only where one of them could be more than 2^15 is
// the maximum taken anew and O rescaled. So float16 weights neither run over nor lose digits above 2^-21 of the largest, and what every
// step would spend on a maximum over the warp (shuffles, one after the other) is spent in the first. A block of zeros has sv = 0:
// log2 is taken of max(sv, 2^-60), which changes nothing that float16 results could hold.
#pragma once
#include "kv_cache.cuh"

namespace qi {
namespace kv {

constexpr float P_SHIFT = 7.0f, MOST_SUM = 32768.0f, LEAST_SCALE = 8.6736174e-19f;  // 2^-60
constexpr float LEAST_FACTOR = 1e-30f;  // in place of a key scale of zero: what is hidden stays -infinity times it, every score 0
constexpr int DECODE_WARPS = 4, DECODE_THREADS = DECODE_WARPS * 32, STEP = 32, ROUND = DECODE_WARPS * STEP;
constexpr int JOIN_ROUNDS = 3;

struct Attention {
    const __half *q;
    __half *y;
    float *lse;
    long long ld_q, ld_y;
    int heads, group;   // query heads, and how many of them share a head of the cache
    float scale_log2;
    int causal, window, max_length;
    int chunk, splits, row_tiles;  // of the kernel for many queries
    int *arrivals;      // how many pieces are there, zero between calls: one for each CTA, for the unit that begins in it and goes on in the next, or for each tile of rows
    float *partial;     // what pieces leave: [piece][rows][head_dim + 2]
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3, const uint32_t b0, const uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Two codes, at bytes SELECT of `word`, as float16 whole numbers.
template <uint32_t SELECT>
__device__ __forceinline__ uint32_t widen2(uint32_t word) {
    const uint32_t magic = __byte_perm(word, 0x64646464u, SELECT);  // 1024 + code
    const __half2 value = __hsub2(*reinterpret_cast<const __half2 *>(&magic), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&value);
}

__device__ __forceinline__ uint4 load_codes(const uint8_t *at) {  // read once by this call
    uint4 w;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(at));
    return w;
}
// Quotients of what may need 64 bits but hardly ever does.
__device__ __forceinline__ long long divide(long long a, long long b) {
    if (static_cast<unsigned long long>(a | b) >> 32 == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// The keys that row `row` of an entry (row = token * group + head of the group) sees: [low, high).
__device__ __forceinline__ void visible(const Attention &a, const Entry &entry, int row, int &low, int &high) {
    const int position = entry.length - entry.count + row / a.group;
    low = a.window > 0 && position >= a.window ? position - a.window + 1 : 0;  // (where there are more rows than tokens, positions go below zero)
    high = a.causal ? min(entry.length, position + 1) : entry.length;
}

template <int DIM, int TILES>
struct Decode {
    // CTAs to an SM, rounds of a ring, and rounds that are worth a CTA of their own (joining a piece costs as much). 64 sequences of 2048 to
    // 8192 tokens, 8 heads: 128 channels, three CTAs with rings of two 124 us, two with three the same, but 131071 tokens of one 70 and 62;
    // 64 channels 78 with three, 89 with two. With 16 rows two rounds, so that two CTAs fit: 152 us, 234 with one.
    static constexpr int CTAS = DIM == 64 ? 3 : 2, LEAST_ROUNDS = TILES == 1 ? 2 : 4;
    static constexpr int STAGES = (DIM == 64 ? 4 : 3) - (TILES == 1 ? 0 : 1), STAGE_BYTES = 2 * STEP * DIM + 32;  // codes of keys, of values, scales
    struct Join {
        float o[DECODE_WARPS][8 * TILES][DIM], m[DECODE_WARPS][8 * TILES], l[DECODE_WARPS][8 * TILES];
    };
    static constexpr int JOIN_AT = DECODE_WARPS * STAGES * STAGE_BYTES, SMEM_BYTES = JOIN_AT + sizeof(Join);
    static_assert(CTAS * (SMEM_BYTES + 1024 + 128) <= 228 * 1024, "so many CTAs to an SM");
};

// Where piece `piece` (16 bytes) of a token's codes lies in its row: keys are read by lanes of two tokens in turn with four pieces each, values
// by lanes of four tokens, two apart, with two pieces each.
template <int DIM>
__device__ __forceinline__ int key_place(int token, int piece) { return DIM == 128 ? piece ^ (token & 1) << 2 : piece; }
template <int DIM>
__device__ __forceinline__ int value_place(int token, int piece) { return DIM == 128 ? piece ^ (token >> 1 & 3) << 1 : piece ^ (token >> 1 & 3); }

template <int DIM, int TILES>
__global__ void __launch_bounds__(DECODE_THREADS, Decode<DIM, TILES>::CTAS) decode_kernel(Cache cache, Tables tables, Batch batch, Attention a) {
    constexpr int ROWS = 8 * TILES, K_WORDS = DIM / 16;            // K_WORDS: 32-bit words of a token's codes that a lane holds (keys)
    constexpr int V_WORDS = DIM / 32, BLOCKS = STEP / BLOCK;       // and of values, of each of four tokens
    constexpr int STAGES = Decode<DIM, TILES>::STAGES, STAGE_BYTES = Decode<DIM, TILES>::STAGE_BYTES;
    constexpr int PIECE = ROWS * (DIM + 2);                        // floats that a CTA leaves of a unit it shares
    extern __shared__ __align__(16) uint8_t smem[];
    using Join = typename Decode<DIM, TILES>::Join;
    Join *join = reinterpret_cast<Join *>(smem + Decode<DIM, TILES>::JOIN_AT);
    auto &join_o = join->o;
    auto &join_m = join->m, &join_l = join->l;
    __shared__ int is_last, first_entry;
    __shared__ long long warp_rounds[DECODE_WARPS], first_before, bounds[2];
    __shared__ int warp_entries[DECODE_WARPS], warp_longest[DECODE_WARPS];
    grid_wait();
    if (no_room(batch)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row8 = lane >> 2, quad = lane & 3;

    // ---- which rounds are this CTA's ----
    struct Span {
        Entry entry;
        int low, high, rounds;  // the tokens that any row sees, low a multiple of 16; their rounds, at least one where there are rows
    };
    auto span_of = [&](int b, Span &u) {
        u.rounds = 0, u.low = 0, u.high = 0;
        if (!read_entry(batch, tables, cache.page_shift, b, a.max_length, u.entry)) {
            complain(0xC030);
            return;
        }
        if (u.entry.count == 0) return;
        int unused;
        visible(a, u.entry, 0, u.low, unused);
        visible(a, u.entry, u.entry.count * a.group - 1, unused, u.high);
        u.low = u.low / BLOCK * BLOCK;
        u.rounds = max((max(u.high - u.low, 0) + ROUND - 1) / ROUND, 1);
    };
    Span span;
    int b = 0, longest = 0;
    long long total = 0, units = 0, unit_round = 0;  // of rounds, of units; the first round of this CTA's first unit
    long long ctas = 1, first_round = 0, end_round = 0;
    // Either all rounds are shared out evenly, no more CTAs than have LEAST_ROUNDS each or a unit, or CTAs take whole units: that is chosen where
    // the one with the most to do is done sooner so, a join being worth JOIN_ROUNDS. (32 sequences of up to 500 tokens: 13 us with whole units, 18 shared.)
    bool whole_units = false;
    auto share = [&]() {
        constexpr int LEAST_ROUNDS = Decode<DIM, TILES>::LEAST_ROUNDS;
        const long long most = gridDim.x, shared = min(most, max((total + LEAST_ROUNDS - 1) / LEAST_ROUNDS, units)), apart = min(most, units);
        whole_units = longest * divide(units + apart - 1, apart) <= divide(total + shared - 1, shared) + JOIN_ROUNDS;
        ctas = whole_units ? apart : shared;
        if (blockIdx.x >= ctas) return false;
        const long long work = whole_units ? units : total;  // in units, or in rounds
        first_round = divide(blockIdx.x * work, ctas), end_round = divide((blockIdx.x + 1) * work, ctas);
        return true;
    };
    if (batch.entries == 1) {
        span_of(0, span);
        longest = span.rounds, total = static_cast<long long>(span.rounds) * cache.heads, units = cache.heads;
        if (total == 0 || !share()) return;
        if (whole_units) first_round *= span.rounds, end_round *= span.rounds;
    } else {
        const int each = (batch.entries + DECODE_THREADS - 1) / DECODE_THREADS, from = threadIdx.x * each, to = min(from + each, batch.entries);
        long long rounds = 0, before;
        int entries = 0, entries_before;  // with rows
        for (int i = from; i < to; ++i) span_of(i, span), rounds += span.rounds, entries += span.rounds > 0, longest = max(longest, span.rounds);
        before = rounds, entries_before = entries;
#pragma unroll
        for (int step = 1; step < 32; step *= 2) {
            const long long below = __shfl_up_sync(0xffffffffu, before, step);
            const int entries_below = __shfl_up_sync(0xffffffffu, entries_before, step);
            if (lane >= step) before += below, entries_before += entries_below;
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        if (lane == 31) warp_rounds[warp] = before, warp_entries[warp] = entries_before, warp_longest[warp] = longest;
        __syncthreads();
        before -= rounds, entries_before -= entries;
        total = units = 0;
#pragma unroll
        for (int w = 0; w < DECODE_WARPS; ++w) {
            if (w < warp) before += warp_rounds[w], entries_before += warp_entries[w];
            total += warp_rounds[w], units += warp_entries[w], longest = max(longest, warp_longest[w]);
        }
        total *= cache.heads, units *= cache.heads;
        if (total == 0 || !share()) return;
        // whoever has the entry that a bound falls into knows the round that it is
        const long long first = first_round, end = end_round;
        const long long mine_from = (whole_units ? entries_before : before) * cache.heads, mine_to = (whole_units ? entries_before + entries : before + rounds) * cache.heads;
        auto find = [&](long long bound, int &entry, long long &rounds_before, long long &round) {
            long long so_far = before;
            int i = from, entries_so_far = entries_before;
            for (span_of(i, span); (whole_units ? entries_so_far + (span.rounds > 0) : so_far + span.rounds) * cache.heads <= bound && i + 1 < to; span_of(++i, span))
                so_far += span.rounds, entries_so_far += span.rounds > 0;
            entry = i, rounds_before = so_far;
            round = whole_units ? so_far * cache.heads + (bound - static_cast<long long>(entries_so_far) * cache.heads) * span.rounds : bound;
        };
        if (mine_from <= first && first < mine_to) find(first, first_entry, first_before, bounds[0]);
        if (whole_units && mine_from <= end && end < mine_to) {
            int entry;
            long long rounds_before;
            find(end, entry, rounds_before, bounds[1]);
        }
        __syncthreads();
        first_round = bounds[0], end_round = !whole_units ? end : end == units ? total : bounds[1];
        b = first_entry, unit_round = first_before * cache.heads;
        span_of(b, span);
        if (span.rounds == 0) return;
    }
    auto cta_of = [&](long long round) { return divide((round + 1) * ctas - 1, total); };
    int head = static_cast<int>(divide(first_round - unit_round, span.rounds)), r = static_cast<int>(first_round - unit_round - static_cast<long long>(head) * span.rounds);
    unit_round += static_cast<long long>(head) * span.rounds;

    // Each warp has a ring of STAGES steps of its own in shared memory, filled by 16-byte asynchronous copies, all rounds but one of
    // them under way at any time: 16 KB with 128 channels, 12 with 64, 8 with 16 rows. Pieces of a row are stored where eight lanes that read together meet no bank twice (DIM 64, values: two of them do).
    uint8_t *ring = smem + warp * (STAGES * STAGE_BYTES);
    // what is fetched next: it runs STAGES - 1 rounds ahead
    Span ahead = span;
    int ahead_entry = b, ahead_head = head, ahead_round = r;
    long long left = end_round - first_round;
    long long place[BLOCKS];  // token rows of its blocks; -1: none, NO_PAGE: tokens whose page is no page of the pool, which nothing is read for
    constexpr long long NO_PAGE = -2;
    auto look_up = [&]() {
        const int token = ahead.low + ahead_round * ROUND + warp * STEP;
        const int *pages = tables.table + static_cast<long long>(ahead.entry.slot) * tables.table_pages;
        auto place_of = [&](int token) -> long long {
            if (left <= 0 || token >= ahead.high) return -1;
            const int page = __ldg(pages + (token >> cache.page_shift));
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(cache.pages)) {
                complain(0xC031);
                return NO_PAGE;
            }
            return token_row(cache, page, ahead_head, token);
        };
        place[0] = place_of(token);
        if (cache.page_shift >= 5 && ahead.low % STEP == 0) place[1] = token + BLOCK < ahead.high ? place[0] + (place[0] >= 0 ? BLOCK : 0) : -1;  // in the same page
        else place[1] = place_of(token + BLOCK);
    };
    static_assert(BLOCKS == 2, "look_up");
    auto go_on = [&]() {
        --left;
        if (++ahead_round == ahead.rounds && left > 0) {
            ahead_round = 0;
            if (++ahead_head == cache.heads) {
                ahead_head = 0;
                do span_of(++ahead_entry, ahead);
                while (ahead.rounds == 0 && ahead_entry + 1 < batch.entries);
            }
        }
        look_up();
    };
    auto fetch = [&](int step) {  // the round's codes and scales, from `place`
        uint8_t *stage = ring + step % STAGES * STAGE_BYTES;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            if (place[k] >= 0) {
                constexpr int PIECES = DIM / 16, TOKENS = 32 / PIECES;  // 16-byte pieces of a token, tokens a pass
                const int piece = lane % PIECES, row = lane / PIECES;
#pragma unroll
                for (int i = 0; i < BLOCK / TOKENS; ++i) {
                    const int t = i * TOKENS + row;
                    cp_async_16(stage + (k * BLOCK + t) * DIM + key_place<DIM>(t, piece) * 16, cache.codes[0] + (place[k] + t) * DIM + piece * 16);
                    cp_async_16(stage + (STEP + k * BLOCK + t) * DIM + value_place<DIM>(t, piece) * 16, cache.codes[1] + (place[k] + t) * DIM + piece * 16);
                }
                if (lane < 2) cp_async_4(stage + 2 * STEP * DIM + (2 * k + lane) * 4, (lane == 0 ? cache.scales[0] : cache.scales[1]) + place[k] / BLOCK);
            } else if (place[k] == NO_PAGE && lane == 0) {
                *reinterpret_cast<float2 *>(stage + 2 * STEP * DIM + 8 * k) = make_float2(0.0f, -1.0f);  // no scale is negative
            }
        }
        cp_async_commit();
    };
    look_up();
    for (int step = 0; step < STAGES - 1; ++step) {
        fetch(step);
        go_on();
    }
    uint32_t q[TILES][K_WORDS][2];
    auto fetch_queries = [&](const Entry &entry, int head) {
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            const int row = n * 8 + row8;
            const __half *source = a.q + (entry.first + static_cast<long long>(row / a.group)) * a.ld_q + (head * a.group + row % a.group) * DIM;
#pragma unroll
            for (int j = 0; j < DIM / 64; ++j) {
                uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (row < entry.count * a.group) {
                    const uint4 *at = reinterpret_cast<const uint4 *>(source + (quad + 4 * j) * 16);
                    w[0] = __ldg(at), w[1] = __ldg(at + 1);
                }
                q[n][4 * j][0] = w[0].x, q[n][4 * j][1] = w[0].y, q[n][4 * j + 1][0] = w[0].z, q[n][4 * j + 1][1] = w[0].w;
                q[n][4 * j + 2][0] = w[1].x, q[n][4 * j + 2][1] = w[1].y, q[n][4 * j + 3][0] = w[1].z, q[n][4 * j + 3][1] = w[1].w;
            }
        }
    };
    fetch_queries(span.entry, head);
    int step = 0;
    for (long long round = first_round; round < end_round;) {
        // ---- one unit ----
        const Entry entry = span.entry;
        const int rows = entry.count * a.group, end = span.high;
        const int first = r, last = static_cast<int>(min(static_cast<long long>(span.rounds), r + end_round - round));  // rounds of it that are this CTA's
        int row_low[TILES][2], row_high[TILES][2];  // of this lane's columns of S^T
        int all_low, all_high, unused;              // what every row sees
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) visible(a, entry, min(n * 8 + quad * 2 + i, rows - 1), row_low[n][i], row_high[n][i]);
        visible(a, entry, rows - 1, all_low, unused);
        visible(a, entry, 0, unused, all_high);
        float o[TILES][DIM / 16][4], m[TILES][2], l[TILES][2];
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int t = 0; t < DIM / 16; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.0f;
        }
        for (; r < last; ++r, ++round, ++step) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();  // the round is there for every lane, and the one before it is done with
            fetch(step + STAGES - 1);
            go_on();
            const int token = span.low + r * ROUND + warp * STEP;
            if (token >= end) continue;
            const uint8_t *stage = ring + step % STAGES * STAGE_BYTES;
            float s[TILES][BLOCKS][4];
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
                for (int n = 0; n < TILES; ++n) s[n][k][0] = s[n][k][1] = s[n][k][2] = s[n][k][3] = 0.0f;
                uint32_t key[2][K_WORDS];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < DIM / 64; ++j) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(stage + (k * BLOCK + row8 + 8 * i) * DIM + key_place<DIM>(row8, quad + 4 * j) * 16);
                        key[i][4 * j] = w.x, key[i][4 * j + 1] = w.y, key[i][4 * j + 2] = w.z, key[i][4 * j + 3] = w.w;
                    }
#pragma unroll
                for (int j = 0; j < K_WORDS; ++j) {
                    const uint32_t a0 = widen2<0x4140>(key[0][j]), a1 = widen2<0x4140>(key[1][j]), a2 = widen2<0x4342>(key[0][j]), a3 = widen2<0x4342>(key[1][j]);
#pragma unroll
                    for (int n = 0; n < TILES; ++n) mma_16x8x16(s[n][k], a0, a1, a2, a3, q[n][j][0], q[n][j][1]);
                }
            }
            float factor[BLOCKS], offset[BLOCKS], inverse[BLOCKS];
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) {
                const float2 scales = *reinterpret_cast<const float2 *>(stage + 2 * STEP * DIM + 8 * k);
                const bool there = token + k * BLOCK < end && !(scales.y < 0.0f);
                const float scale = there ? fmaxf(scales.y, LEAST_SCALE) : 1.0f;  // else weights of 0, whatever the scores
                factor[k] = there ? scales.x * a.scale_log2 : 0.0f, offset[k] = there ? log2_fast(scale) : -INFINITY, inverse[k] = reciprocal_fast(scale);
            }
            if (!(token >= all_low && token + STEP <= min(all_high, end))) {
                // what is hidden: its score becomes -infinity, and the block's factor, if it is 0, something that leaves it that
#pragma unroll
                for (int k = 0; k < BLOCKS; ++k) {
                    factor[k] = fmaxf(factor[k], LEAST_FACTOR);
#pragma unroll
                    for (int n = 0; n < TILES; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = token + k * BLOCK + row8 + i / 2 * 8;
                            if (at < row_low[n][i & 1] || at >= min(row_high[n][i & 1], end)) s[n][k][i] = -INFINITY;
                        }
                }
            }
            float weight[TILES][BLOCKS][4], l_next[TILES][2];
            bool nothing = false;  // a row that has seen nothing yet
#pragma unroll
            for (int n = 0; n < TILES; ++n) nothing |= m[n][0] == -INFINITY || m[n][1] == -INFINITY;
            bool again = __any_sync(0xffffffffu, nothing);
            while (true) {
                if (again) {
#pragma unroll
                    for (int n = 0; n < TILES; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float top = m[n][i];
#pragma unroll
                            for (int k = 0; k < BLOCKS; ++k) top = fmaxf(top, fmaf(fmaxf(s[n][k][i], s[n][k][2 + i]), factor[k], offset[k]));
#pragma unroll
                            for (int step = 4; step < 32; step *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
                            const float shrink = m[n][i] == -INFINITY ? 1.0f : exp2_fast(m[n][i] - top);
                            m[n][i] = top, l[n][i] *= shrink;
#pragma unroll
                            for (int t = 0; t < DIM / 16; ++t) o[n][t][i] *= shrink, o[n][t][2 + i] *= shrink;
                        }
                }
                float worst = 0.0f;
#pragma unroll
                for (int n = 0; n < TILES; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float base = (m[n][i] == -INFINITY ? 0.0f : m[n][i]) - P_SHIFT;
                        l_next[n][i] = l[n][i];
#pragma unroll
                        for (int k = 0; k < BLOCKS; ++k) {
                            weight[n][k][i] = exp2_fast(fmaf(s[n][k][i], factor[k], offset[k] - base)), weight[n][k][2 + i] = exp2_fast(fmaf(s[n][k][2 + i], factor[k], offset[k] - base));
                            const float sum = weight[n][k][i] + weight[n][k][2 + i];
                            worst = fmaxf(worst, sum);
                            l_next[n][i] = fmaf(sum, inverse[k], l_next[n][i]);
                        }
                    }
                if (again || __all_sync(0xffffffffu, worst <= MOST_SUM)) break;
                again = true;
            }
            uint32_t p[TILES][BLOCKS][2];
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                l[n][0] = l_next[n][0], l[n][1] = l_next[n][1];
#pragma unroll
                for (int k = 0; k < BLOCKS; ++k)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const __half2 pair = __floats2half2_rn(weight[n][k][2 * r], weight[n][k][2 * r + 1]);
                        p[n][k][r] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&pair));
                    }
            }
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) {
                uint32_t value[4][V_WORDS];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = quad * 2 + (i & 1) + 8 * (i >> 1);
                    const uint8_t *at = stage + (STEP + k * BLOCK + t) * DIM + value_place<DIM>(t, row8 * DIM / 128) * 16;
                    if constexpr (DIM == 128) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(at);
                        value[i][0] = w.x, value[i][1] = w.y, value[i][2] = w.z, value[i][3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2 *>(at + row8 % 2 * 8);
                        value[i][0] = w.x, value[i][1] = w.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < V_WORDS; ++w) {
                    // [channel 4w of two tokens, channel 4w + 1 of both], and 4w + 2, 4w + 3; tokens 8 further on likewise
                    const uint32_t low0 = __byte_perm(value[0][w], value[1][w], 0x5140), high0 = __byte_perm(value[0][w], value[1][w], 0x7362);
                    const uint32_t low8 = __byte_perm(value[2][w], value[3][w], 0x5140), high8 = __byte_perm(value[2][w], value[3][w], 0x7362);
                    const uint32_t a0 = widen2<0x4140>(low0), a1 = widen2<0x4342>(low0), a2 = widen2<0x4140>(low8), a3 = widen2<0x4342>(low8);
                    const uint32_t c0 = widen2<0x4140>(high0), c1 = widen2<0x4342>(high0), c2 = widen2<0x4140>(high8), c3 = widen2<0x4342>(high8);
#pragma unroll
                    for (int n = 0; n < TILES; ++n) {
                        mma_16x8x16(o[n][2 * w], a0, a1, a2, a3, p[n][k][0], p[n][k][1]);
                        mma_16x8x16(o[n][2 * w + 1], c0, c1, c2, c3, p[n][k][0], p[n][k][1]);
                    }
                }
            }
        }
        __syncthreads();  // the unit before has been read from where warps are joined
        // the next unit's queries are asked for before this one's warps are joined
        const bool whole = first == 0 && last == span.rounds;
        const long long unit_begin = unit_round, unit_end = unit_round + span.rounds;
        const int unit_head = head;
        unit_round = unit_end, r = 0;
        bool more = round < end_round;
        if (more && ++head == cache.heads) {
            head = 0;
            do {
                ++b;
                if (b == ahead_entry) span = ahead;  // which has been looked up already
                else span_of(b, span);
            } while (span.rounds == 0 && b + 1 < batch.entries);
            more = span.rounds > 0;  // else lengths changed while the kernel ran
        }
        if (more) fetch_queries(span.entry, head);
        // warps, then pieces
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int step = 4; step < 32; step *= 2) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], step);
                const int row = n * 8 + quad * 2 + i;
                if (row8 == 0) join_m[warp][row] = m[n][i], join_l[warp][row] = l[n][i];
#pragma unroll
                for (int t = 0; t < DIM / 16; ++t) *reinterpret_cast<float2 *>(&join_o[warp][row][row8 * (DIM / 8) + 2 * t]) = make_float2(o[n][t][i], o[n][t][2 + i]);
            }
        __syncthreads();
        // a CTA has at most two units that it shares: the one that goes on from the CTA before, and the one that goes on in the next
        float *piece = a.partial + (2LL * blockIdx.x + (first == 0)) * PIECE;
        const int owned = rows;
        auto finish = [&](int row, int channel, float2 sum, float top, float total) {  // channels `channel`, `channel` + 1
            const long long out_row = entry.first + row / a.group;
            const int out_head = unit_head * a.group + row % a.group;
            const float factor = total > 0.0f ? __frcp_rn(total) : (total == 0.0f ? 0.0f : total);
            *reinterpret_cast<__half2 *>(a.y + out_row * a.ld_y + out_head * DIM + channel) = __floats2half2_rn(sum.x * factor, sum.y * factor);
            if (channel == 0 && a.lse != nullptr)
                a.lse[out_row * a.heads + out_head] = total == 0.0f ? -INFINITY : 0.6931471805599453f * (top - P_SHIFT + log2f(total));
        };
        for (int item = threadIdx.x; item < owned * (DIM / 2); item += DECODE_THREADS) {
            const int row = item / (DIM / 2), channel = item % (DIM / 2) * 2;
            float top = -INFINITY, total = 0.0f;
#pragma unroll
            for (int w = 0; w < DECODE_WARPS; ++w) top = fmaxf(top, join_m[w][row]);
            const float base = top == -INFINITY ? 0.0f : top;
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < DECODE_WARPS; ++w) {
                const float weight = exp2_fast(join_m[w][row] - base);
                const float2 part = *reinterpret_cast<const float2 *>(&join_o[w][row][channel]);
                total = fmaf(join_l[w][row], weight, total), sum.x = fmaf(part.x, weight, sum.x), sum.y = fmaf(part.y, weight, sum.y);
            }
            if (whole) {
                finish(row, channel, sum, top, total);
            } else {
                *reinterpret_cast<float2 *>(piece + 2 * ROWS + row * DIM + channel) = sum;
                if (channel == 0) piece[row] = top, piece[ROWS + row] = total;
            }
        }
        if (!whole) {
            const long long first_cta = cta_of(unit_begin);
            const int used = static_cast<int>(cta_of(unit_end - 1) - first_cta) + 1;
            auto piece_at = [&](int i) { return a.partial + (2 * (first_cta + i) + (i == 0)) * PIECE; };
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) is_last = atomicAdd(a.arrivals + first_cta, 1) == used - 1;
            __syncthreads();
            if (is_last) {
                __threadfence();
                // Warps share the pieces, lanes the channels, four rows at a time (the last again where there are fewer: no branch stands between
                // one load and the next, of which there have to be many under way; with a walk over rows one by one this took 17 us for 37 pieces).
                constexpr int EACH = DIM / 32, AT_ONCE = 4;
                for (int base = 0; base < owned; base += AT_ONCE) {
                    float top[AT_ONCE], totals[AT_ONCE], sum[AT_ONCE][EACH];
                    int rows_of[AT_ONCE];
#pragma unroll
                    for (int n = 0; n < AT_ONCE; ++n) {
                        rows_of[n] = min(base + n, owned - 1);
                        top[n] = -INFINITY, totals[n] = 0.0f;
#pragma unroll
                        for (int c = 0; c < EACH; ++c) sum[n][c] = 0.0f;
                    }
                    for (int i = lane; i < used; i += 32)
#pragma unroll
                        for (int n = 0; n < AT_ONCE; ++n) top[n] = fmaxf(top[n], __ldcg(piece_at(i) + rows_of[n]));
#pragma unroll
                    for (int n = 0; n < AT_ONCE; ++n) {
#pragma unroll
                        for (int step = 16; step > 0; step /= 2) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], step));
                    }
#pragma unroll 4
                    for (int i = warp; i < used; i += DECODE_WARPS) {
                        const float *one = piece_at(i);
#pragma unroll
                        for (int n = 0; n < AT_ONCE; ++n) {
                            const int row = rows_of[n];
                            const float weight = exp2_fast(__ldcg(one + row) - (top[n] == -INFINITY ? 0.0f : top[n]));
                            totals[n] = fmaf(__ldcg(one + ROWS + row), weight, totals[n]);
                            float part[EACH];
                            if constexpr (EACH == 4) {
                                const float4 f = __ldcg(reinterpret_cast<const float4 *>(one + 2 * ROWS + row * DIM + lane * EACH));
                                part[0] = f.x, part[1] = f.y, part[2] = f.z, part[3] = f.w;
                            } else {
                                const float2 f = __ldcg(reinterpret_cast<const float2 *>(one + 2 * ROWS + row * DIM + lane * EACH));
                                part[0] = f.x, part[1] = f.y;
                            }
#pragma unroll
                            for (int c = 0; c < EACH; ++c) sum[n][c] = fmaf(part[c], weight, sum[n][c]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < AT_ONCE; ++n) {
                        if (lane == 0) join_m[warp][rows_of[n]] = top[n], join_l[warp][rows_of[n]] = totals[n];
#pragma unroll
                        for (int c = 0; c < EACH; ++c) join_o[warp][rows_of[n]][lane * EACH + c] = sum[n][c];
                    }
                }
                __syncthreads();
                for (int item = threadIdx.x; item < owned * (DIM / 2); item += DECODE_THREADS) {
                    const int row = item / (DIM / 2), channel = item % (DIM / 2) * 2;
                    float all = 0.0f;
                    float2 both = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < DECODE_WARPS; ++w) {
                        const float2 part = *reinterpret_cast<const float2 *>(&join_o[w][row][channel]);
                        all += join_l[w][row], both.x += part.x, both.y += part.y;
                    }
                    finish(row, channel, both, join_m[0][row], all);
                }
                if (threadIdx.x == 0) a.arrivals[first_cta] = 0;
            }
        }
        if (!more) break;
    }
    cp_async_wait<0>();
}

}  // namespace kv
}  // namespace qi
