// Attention over the paged 8-bit cache for many queries to a sequence (a prompt, the image tokens of a denoising step), on tcgen05.
//
// The mathematics are those of kv_decode.cuh: x_j = (scale * log2 e * sk) * raw_j + log2 sv, p_j = 2^(x_j - m), O = sum p_j d_j,
// l = sum p_j / sv, y = O / l, with the scales constant over 16 tokens, so that they enter once per block.
//
// A CTA takes 2 x 128 query rows that share a head of the cache and walks over its tokens in tiles of 128:
//   warps 0-3, 4-7   the softmax of one half of the rows each, a row to a thread: scores from TMEM, weights back into TMEM where the
//                    scores were, the running maximum and sum in registers
//   warps 8-11       widen codes: HBM -> registers -> float16 whole numbers in shared memory (exact), a tile ahead
//   warp 12          issues the MMAs: S = Q K^T and O += P V, operands K and V from shared memory, P from TMEM
//   warp 13          looks up pages and scales, up to four tiles ahead: page number, then scale, are two trips to memory in a row, and
//                    where the widening warps made them they set the pace (4.3 us a tile and CTA instead of 2.5)
// so that the two halves alternate: while one's weights are computed the tensor cores have the other's products. Values are stored as
// they lie in the cache, a token a row, and enter their product "MN-major"; nothing is transposed.
//
// m is not the maximum of what has been seen so far but an older one: weights are computed in one pass with the m that there is, and only
// where those of 16 tokens add up to more than 2^15 (they are 2^7 where x = m, so that needs a growth by 2^4 to 2^8) is the tile's
// maximum taken, O rescaled (which waits for the product before) and the pass repeated. So no weight is more than 2^15 in float16, and
// all its digits are kept down to 2^-21 of the largest; sums are float32. Only the first tile pays for a pass over its maximum.
//
// Two guided sequences, 4096 queries over 4173 tokens and 2691 over 2999, 32 heads: 505 us, 816 TFLOP/s, call after call (463 us and 890 in the first
// hundred calls, before the power limit); one round of CTAs over 65536 tokens 1030. A
// tile takes a CTA 2.3 us, of which the products alone would be 1.6 (two thirds of the tensor cores' rate: Q and K from shared memory are
// 128 bytes a clock, and the widened codes are written beside them); the rest is the chain scores - weights - product - next scores,
// which two halves of rows overlap and do not fill (issue slots 38 %, special functions 40 %, tensor cores 42 % busy). A CTA starts for 5 us
// and ends for 3. Tried without gain: scores in halves of 64 columns, so that no softmax waits (521 us: Q is read twice); an issuing warp for
// each half (568); a quarter or half of the exponentials as polynomials (531, 564); the maximum taken first (493); predicated MMAs (550);
// serving whichever half is ready (641: asking two barriers in turn takes longer); waits with pauses, or by all lanes (470 to 500).
//
// TMEM: S and P of the halves at columns 0 and 128, O at 256 and 384.
#pragma once
#include "kv_decode.cuh"

namespace qi {
namespace kv {

constexpr int PREFILL_THREADS = 512, TILE_ROWS = 128, TILE_TOKENS = 128, PREFILL_ROWS = 2 * TILE_ROWS;
constexpr int WIDEN_WARP0 = 8, ISSUE_WARP = 12, LOOK_UP_WARP = 13, TILE_BLOCKS = TILE_TOKENS / BLOCK, SLOTS = 4;
constexpr int HALF_TOKENS = TILE_TOKENS / 2, HALF_BLOCKS = TILE_BLOCKS / 2;
constexpr uint32_t TMEM_S = 0, TMEM_O = 256;

template <int DIM>
struct Prefill {
    static constexpr int HALVES = DIM / 64;                            // 128-byte rows of 64 channels
    static constexpr int OPERAND_BYTES = TILE_TOKENS * DIM * 2;        // of K, V, or half of Q
    static constexpr int Q_AT = 0, K_AT = 2 * OPERAND_BYTES, V_AT = 4 * OPERAND_BYTES, SCALES_AT = 6 * OPERAND_BYTES;
    static constexpr int PLACES_AT = SCALES_AT + SLOTS * TILE_BLOCKS * 16, BARRIERS_AT = PLACES_AT + SLOTS * TILE_BLOCKS * 8;
    static constexpr int BARRIERS = 8 + 3 * SLOTS + 10 + 1;
    static constexpr int SMEM_BYTES = BARRIERS_AT + BARRIERS * 8 + 16 + 1024;
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
};

// A shared-memory operand stored as rows of 64 channels (128 bytes, swizzled by the row's last three bits), a token a row, for a product that
// sums over tokens: 8 tokens 1024 bytes apart, 64 channels `OPERAND / HALVES` bytes apart.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t address, uint32_t channel_stride) {
    uint64_t descriptor = 0;
    descriptor |= static_cast<uint64_t>((address & 0x3FFFFu) >> 4);
    descriptor |= static_cast<uint64_t>(channel_stride >> 4) << 16;
    descriptor |= static_cast<uint64_t>(1024 >> 4) << 32;
    descriptor |= static_cast<uint64_t>(1) << 46;
    descriptor |= static_cast<uint64_t>(2) << 61;
    return descriptor;
}

// D[tmem] (+)= A[tmem] * B[smem], A float16, two of a row's values in a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_store_32x32(uint32_t address, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store_32x16(uint32_t address, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(address), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Uses of what tcgen05.ld gave stay behind the wait for it.
template <int N>
__device__ __forceinline__ void arrived(uint32_t (&r)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) asm volatile("" : "+r"(r[j]));
}

// Pieces of a tile's tokens: the CTA that arrives last adds them up in their order. All softmax warps.
template <int DIM>
__device__ __forceinline__ void join_pieces(const Attention &a, const Entry &entry, int head, long long unit, int first_row, int last_row, int used, int *is_last) {
    constexpr int PIECE = PREFILL_ROWS * (DIM + 2);
    __threadfence();
    named_barrier_sync(1, PREFILL_ROWS);
    if (threadIdx.x == 0) *is_last = atomicAdd(a.arrivals + unit, 1) == used - 1;
    named_barrier_sync(1, PREFILL_ROWS);
    if (!*is_last) return;
    __threadfence();
    const int local = threadIdx.x, row = first_row + local;
    if (local == 0) a.arrivals[unit] = 0;
    if (row > last_row) return;
    const float *partial = a.partial + unit * a.splits * PIECE + local;
    float top = -INFINITY, total = 0.0f;
    for (int i = 0; i < used; ++i) top = fmaxf(top, __ldcg(partial + static_cast<long long>(i) * PIECE));
    const float base = top == -INFINITY ? 0.0f : top;
    for (int i = 0; i < used; ++i) {
        const float *one = partial + static_cast<long long>(i) * PIECE;
        total = fmaf(__ldcg(one + PREFILL_ROWS), exp2_fast(__ldcg(one) - base), total);
    }
    const float factor = total > 0.0f ? __frcp_rn(total) : (total == 0.0f ? 0.0f : total);
    const long long out_row = entry.first + row / a.group;
    const int out_head = head * a.group + row % a.group;
    for (int channel = 0; channel < DIM; channel += 16) {
        float sum[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) sum[c] = 0.0f;
        for (int i = 0; i < used; ++i) {
            const float *one = partial + static_cast<long long>(i) * PIECE;
            const float weight = exp2_fast(__ldcg(one) - base);
#pragma unroll
            for (int c = 0; c < 16; ++c) sum[c] = fmaf(__ldcg(one + (2 + channel + c) * PREFILL_ROWS), weight, sum[c]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t pairs[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __half2 pair = __floats2half2_rn(sum[8 * half + 2 * e] * factor, sum[8 * half + 2 * e + 1] * factor);
                pairs[e] = *reinterpret_cast<const uint32_t *>(&pair);
            }
            *reinterpret_cast<uint4 *>(a.y + out_row * a.ld_y + out_head * DIM + channel + 8 * half) = make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
        }
    }
    if (a.lse != nullptr) a.lse[out_row * a.heads + out_head] = total == 0.0f ? -INFINITY : 0.6931471805599453f * (top - P_SHIFT + log2f(total));
}

template <int DIM>
__global__ void __launch_bounds__(PREFILL_THREADS, 1) prefill_kernel(Cache cache, Tables tables, Batch batch, Attention a) {
    using P = Prefill<DIM>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float4(*scales)[TILE_BLOCKS] = reinterpret_cast<float4(*)[TILE_BLOCKS]>(smem + P::SCALES_AT);  // factor, offset, 1 / sv of each block
    long long(*places)[TILE_BLOCKS] = reinterpret_cast<long long(*)[TILE_BLOCKS]>(smem + P::PLACES_AT);  // its token row
    uint64_t *barriers = reinterpret_cast<uint64_t *>(smem + P::BARRIERS_AT);
    uint64_t *k_full = barriers, *k_empty = barriers + 2, *v_full = barriers + 4, *v_empty = barriers + 6, *place_full = barriers + 8, *slot_full = place_full + SLOTS, *slot_empty = slot_full + SLOTS;
    uint64_t *s_full = slot_empty + SLOTS, *p_full = s_full + 2, *o_done = s_full + 6, *q_full = s_full + 10;  // of p and o [half of a tile][half of the rows]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(barriers + P::BARRIERS);
    __shared__ int is_last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == ISSUE_WARP) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbarrier_init(k_full + i, 4), mbarrier_init(v_full + i, 4);
            mbarrier_init(k_empty + i, 1), mbarrier_init(v_empty + i, 1);
            mbarrier_init(s_full + i, 1);
        }
        for (int i = 0; i < 4; ++i) mbarrier_init(p_full + i, 4), mbarrier_init(o_done + i, 1);
        for (int i = 0; i < SLOTS; ++i) mbarrier_init(place_full + i, 1), mbarrier_init(slot_full + i, 1), mbarrier_init(slot_empty + i, 1);
        mbarrier_init(q_full, 8);
        fence_barrier_init();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto wait = [lane](uint64_t *barrier, uint32_t parity, uint32_t code) { return mbarrier_wait_warp(barrier, parity, &g_status, code, lane); };
    grid_wait();

    // the last rows first: under a causal mask they see the most tokens, and what is short fills up the end
    const int split = blockIdx.x, head = blockIdx.y % cache.heads, tile = a.row_tiles - 1 - blockIdx.y / cache.heads, b = blockIdx.z;
    Entry entry;
    const bool sound = read_entry(batch, tables, cache.page_shift, b, a.max_length, entry);
    if (!sound && threadIdx.x == 0) complain(0xC040);
    const int rows = sound && !no_room(batch) ? entry.count * a.group : 0, first_row = tile * PREFILL_ROWS;
    const int last_row = min(first_row + PREFILL_ROWS, rows) - 1;
    int low = 0, high = 0, unused, used = 0;
    if (first_row < rows) {
        visible(a, entry, first_row, low, unused);
        visible(a, entry, last_row, unused, high);
        low = low / BLOCK * BLOCK;
        used = max((max(high - low, 0) + a.chunk - 1) / a.chunk, 1);
    }
    // this CTA's tokens; a CTA without any still writes its rows if it is the first of its tile
    const int begin = low + split * a.chunk, end = min(begin + a.chunk, high);
    const int tiles = split < used && end > begin ? (end - begin + TILE_TOKENS - 1) / TILE_TOKENS : 0;
    const int parts = first_row + TILE_ROWS <= last_row ? 2 : 1;  // halves that hold rows

    if (split < used) {
        if (warp >= WIDEN_WARP0 && warp < ISSUE_WARP) {
            // ---- codes ----
            setmaxnreg_dec<104>();
            // A thread takes 16 codes of a token, the same ones of every TOKENS-th token. Eight threads that store together have four
            // pieces of one 128-byte row and four of the next, so that they meet no bank twice.
            constexpr int LANES = DIM / 16, TOKENS = 128 / LANES, LOADS = TILE_TOKENS / TOKENS;  // threads to a token, tokens and loads of a pass
            const int t = threadIdx.x - WIDEN_WARP0 * 32;
            const int pair = t / (2 * LANES), row0 = pair * 2 + t / 4 % 2, chunk = t % 4 + t % (2 * LANES) / 8 * 4;
            const uint32_t piece = chunk % 4 * 2, at0 = smem_u32(smem) + chunk / 4 * (TILE_TOKENS * 128) + row0 * 128;
            const uint32_t first_at = at0 + ((piece ^ (row0 & 7)) << 4), second_at = at0 + (((piece + 1) ^ (row0 & 7)) << 4);
            static_assert(TOKENS % 8 == 0, "a thread's rows have their last three bits in common");
            const uint8_t *sources[2] = {cache.codes[0] + row0 % BLOCK * DIM + chunk * 16, cache.codes[1] + row0 % BLOCK * DIM + chunk * 16};
            uint4 words[2][LOADS];  // of keys, of values
            auto fetch = [&](int which, int j) {
                const long long *place = places[j % SLOTS] + row0 / BLOCK;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) words[which][i] = load_codes(sources[which] + place[i * TOKENS / BLOCK] * DIM);
            };
            auto widen = [&](int which, uint32_t offset) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const uint4 w = words[which][i];
                    const uint32_t to = offset + i * (TOKENS * 128);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(first_at + to), "r"(widen2<0x4140>(w.x)), "r"(widen2<0x4342>(w.x)), "r"(widen2<0x4140>(w.y)), "r"(widen2<0x4342>(w.y)) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(second_at + to), "r"(widen2<0x4140>(w.z)), "r"(widen2<0x4342>(w.z)), "r"(widen2<0x4140>(w.w)), "r"(widen2<0x4342>(w.w)) : "memory");
                }
            };
            bool alive = tiles > 0 && wait(place_full, 0, STATUS_WAIT_FULL | 0xC020);
            if (alive) fetch(0, 0), fetch(1, 0);
            for (int j = 0; j < tiles && alive; ++j) {
                const int stage = j & 1, phase = j >> 1 & 1;
                if (!wait(k_empty + stage, phase ^ 1, STATUS_WAIT_EMPTY | 0xC000 | stage)) { alive = false; break; }
                widen(0, P::K_AT + stage * P::OPERAND_BYTES);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbarrier_arrive(k_full + stage);
                if (j + 1 == tiles) {
                    if (!wait(v_empty + stage, phase ^ 1, STATUS_WAIT_EMPTY | 0xC100 | stage)) break;
                    widen(1, P::V_AT + stage * P::OPERAND_BYTES);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(v_full + stage);
                    break;
                }
                if (!wait(place_full + (j + 1) % SLOTS, (j + 1) / SLOTS & 1, STATUS_WAIT_FULL | 0xC020)) { alive = false; break; }
                fetch(0, j + 1);
                if (!wait(v_empty + stage, phase ^ 1, STATUS_WAIT_EMPTY | 0xC100 | stage)) { alive = false; break; }
                widen(1, P::V_AT + stage * P::OPERAND_BYTES);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbarrier_arrive(v_full + stage);
                fetch(1, j + 1);
            }
        } else if (warp >= ISSUE_WARP) {
            // ---- products ----
            setmaxnreg_dec<40>();
            if (warp == ISSUE_WARP) {
                // One lane by itself: a vote of the warp or a hand-over to it at every step would be in the chain of the whole tile (471 us, so 464).
                if (tiles > 0 && elect_one()) {
                    constexpr uint32_t IDESC_S = umma_idesc_f16_f32(TILE_ROWS, TILE_TOKENS), IDESC_O = umma_idesc_f16_f32(TILE_ROWS, DIM) | 1u << 16;  // B is MN-major
                    const uint32_t q_at = smem_u32(smem + P::Q_AT), k_at = smem_u32(smem + P::K_AT), v_at = smem_u32(smem + P::V_AT);
                    auto scores = [&](int i, int j) {
                        const uint32_t q = q_at + i * P::OPERAND_BYTES, k = k_at + (j & 1) * P::OPERAND_BYTES;
#pragma unroll
                        for (int s = 0; s < DIM / 16; ++s) {
                            const uint32_t step = s / 4 * (TILE_TOKENS * 128) + s % 4 * 32;
                            umma_f16(tmem + TMEM_S + i * 128, umma_desc_k_sw128(q + step), umma_desc_k_sw128(k + step), IDESC_S, s > 0);
                        }
                        tcgen05_commit(s_full + i);
                    };
                    bool alive = mbarrier_wait(q_full, 0, &g_status, STATUS_WAIT_FULL | 0xC200) && mbarrier_wait(k_full, 0, &g_status, STATUS_WAIT_FULL | 0xC210);
                    tcgen05_fence_after();
                    if (alive) {
                        for (int i = 0; i < parts; ++i) scores(i, 0);
                        tcgen05_commit(k_empty);
                    }
                    for (int j = 0; j < tiles && alive; ++j) {
                        const int stage = j & 1, next = (j + 1) & 1;
                        alive = mbarrier_wait(v_full + stage, j >> 1 & 1, &g_status, STATUS_WAIT_FULL | 0xC220 | stage);
                        for (int i = 0; i < parts && alive; ++i) {
                            for (int h = 0; h < 2; ++h) {
                                alive = mbarrier_wait(p_full + 2 * h + i, j & 1, &g_status, STATUS_WAIT_READY | 0xC230 | i);
                                if (!alive) break;
                                tcgen05_fence_after();
                                const uint32_t v = v_at + stage * P::OPERAND_BYTES + h * (HALF_TOKENS * 128), weights = tmem + TMEM_S + i * 128 + h * 32;
#pragma unroll
                                for (int s = 0; s < HALF_TOKENS / 16; ++s)
                                    umma_f16_ts(tmem + TMEM_O + i * 128, weights + s * 8, umma_desc_mn_sw128(v + s * 2048, TILE_TOKENS * 128), IDESC_O, j + h > 0 || s > 0);
                                tcgen05_commit(o_done + 2 * h + i);
                            }
                            if (alive && i == 0 && j + 1 < tiles) alive = mbarrier_wait(k_full + next, (j + 1) >> 1 & 1, &g_status, STATUS_WAIT_FULL | 0xC240 | next);
                            if (!alive) break;
                            tcgen05_fence_after();
                            if (j + 1 < tiles) scores(i, j + 1);
                            if (i == parts - 1) {
                                tcgen05_commit(v_empty + stage), tcgen05_commit(slot_empty + j % SLOTS);
                                if (j + 1 < tiles) tcgen05_commit(k_empty + next);
                            }
                        }
                    }
                }
                __syncwarp();
            } else if (warp == LOOK_UP_WARP) {
                const int *pages = tables.table + static_cast<long long>(entry.slot) * tables.table_pages;
                auto page_at = [&](int j) {  // of this lane's block of tile j
                    const int token = begin + j * TILE_TOKENS + lane * BLOCK;
                    return lane < TILE_BLOCKS && token < end ? __ldg(pages + (token >> cache.page_shift)) : 0;
                };
                int page = page_at(0);
                for (int j = 0; j < tiles; ++j) {
                    const int next_page = page_at(j + 1), token = begin + j * TILE_TOKENS + lane * BLOCK;
                    const bool known = page >= 0 && page < cache.pages, there = lane < TILE_BLOCKS && token < end && known;
                    if (!known) complain(0xC041);
                    // What is fetched for nothing (the pool's first codes) is finite, and its weights are 0: 2^-infinity, whatever the scores
                    const long long place = there ? token_row(cache, page, head, token) : 0;
                    const float k_scale = there ? __ldg(cache.scales[0] + place / BLOCK) : 0.0f, v_scale = there ? fmaxf(__ldg(cache.scales[1] + place / BLOCK), LEAST_SCALE) : 1.0f;
                    if (j >= SLOTS && !wait(slot_empty + j % SLOTS, (j / SLOTS - 1) & 1, STATUS_WAIT_EMPTY | 0xC240)) break;
                    if (lane < TILE_BLOCKS) places[j % SLOTS][lane] = place;
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(place_full + j % SLOTS);  // codes can be fetched while the scales are on their way
                    if (lane < TILE_BLOCKS) scales[j % SLOTS][lane] = make_float4(fmaxf(k_scale * a.scale_log2, LEAST_FACTOR), there ? log2_fast(v_scale) : -INFINITY, reciprocal_fast(v_scale), 0.0f);
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(slot_full + j % SLOTS);
                    page = next_page;
                }
            }
        } else {
            // ---- softmax ----
            setmaxnreg_inc<184>();
            const int part = warp >> 2, row = first_row + part * TILE_ROWS + (warp & 3) * 32 + lane;
            const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
            const uint32_t s_at = tmem + lanes + TMEM_S + part * 128, o_at = tmem + lanes + TMEM_O + part * 128;
            int row_low, row_high;
            visible(a, entry, min(row, last_row), row_low, row_high);
            // rows of Q and y in whole lines: a lane has piece `piece` of rows row0, row0 + ROWS_AT_ONCE, ... of its warp's 32
            constexpr int PIECES = DIM / 8, ROWS_AT_ONCE = 32 / PIECES, WARP_PASSES = 32 / ROWS_AT_ONCE;
            const int piece = lane % PIECES, y_row0 = first_row + part * TILE_ROWS + (warp & 3) * 32 + lane / PIECES, row0 = min(y_row0, rows - 1);
            struct Walk {  // token and head of the group of a row, without a division a row
                int token, member, tokens, members, group;
                __device__ Walk(int row, int group) : token(row / group), member(row % group), tokens(ROWS_AT_ONCE / group), members(ROWS_AT_ONCE % group), group(group) {}
                __device__ void go_on() {
                    token += tokens, member += members;
                    if (member >= group) member -= group, ++token;
                }
            };
            {
                // this warp's rows of Q, whole lines at a time: with a row to a thread the loads alone took 2 us
                const uint32_t at = smem_u32(smem + P::Q_AT) + part * P::OPERAND_BYTES + piece / 8 * (TILE_ROWS * 128);
                uint4 w[WARP_PASSES];
                Walk walk(row0, a.group);
#pragma unroll
                for (int i = 0; i < WARP_PASSES; ++i) {
                    w[i] = __ldg(reinterpret_cast<const uint4 *>(a.q + (entry.first + static_cast<long long>(walk.token)) * a.ld_q + (head * a.group + walk.member) * DIM) + piece);
                    if (row0 + (i + 1) * ROWS_AT_ONCE < rows) walk.go_on();  // beyond the last row: some row again, whose results are not written
                }
#pragma unroll
                for (int i = 0; i < WARP_PASSES; ++i) {
                    const uint32_t r = (warp & 3) * 32 + i * ROWS_AT_ONCE + lane / PIECES;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + r * 128 + ((piece % 8 ^ (r & 7)) << 4)), "r"(w[i].x), "r"(w[i].y), "r"(w[i].z), "r"(w[i].w) : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbarrier_arrive(q_full);
            }
            float m = -INFINITY, l = 0.0f;
            bool alive = true;
            if (part < parts) {
                for (int j = 0; j < tiles; ++j) {
                    if (!wait(slot_full + j % SLOTS, j / SLOTS & 1, STATUS_WAIT_FULL | 0xC300 | part) ||
                        !wait(s_full + part, j & 1, STATUS_WAIT_TMEM_FULL | 0xC300 | part)) { alive = false; break; }
                    tcgen05_fence_after();
                    const int token = begin + j * TILE_TOKENS;
                    const int seen_low = row_low - token, seen_high = min(row_high, end) - token;
                    if (!__all_sync(0xffffffffu, seen_low <= 0 && seen_high >= TILE_TOKENS)) {
                        // scores of hidden tokens become -infinity where they are: few tiles need it, and the others' code stays short
#pragma unroll 1
                        for (int k = 0; k < TILE_BLOCKS; ++k) {
                            uint32_t hidden[BLOCK];
                            tmem_load_32x16(s_at + k * BLOCK, hidden);
                            tmem_load_wait();
                            arrived(hidden);
#pragma unroll
                            for (int c = 0; c < BLOCK; ++c)
                                if (k * BLOCK + c < seen_low || k * BLOCK + c >= seen_high) hidden[c] = 0xff800000u;
                            tmem_store_32x16(s_at + k * BLOCK, hidden);
                        }
                        tmem_store_wait();
                    }
                    // Half a tile at a time: the product of its first 64 tokens runs while the weights of the others are computed.
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t half_at = s_at + h * HALF_TOKENS;
                        const float4 *scale = &scales[j % SLOTS][h * HALF_BLOCKS];
                        uint32_t s[HALF_BLOCKS / 2][32], p[32];  // scores, weights in pairs
                        auto take = [&]() {
#pragma unroll
                            for (int i = 0; i < HALF_BLOCKS / 2; ++i) tmem_load_32x32(half_at + i * 32, s[i]);
                            tmem_load_wait();
#pragma unroll
                            for (int i = 0; i < HALF_BLOCKS / 2; ++i) arrived(s[i]);
                        };
                        float l_next;
                        bool again = __any_sync(0xffffffffu, m == -INFINITY);  // a row that has seen nothing yet
#pragma unroll 1
                        while (true) {
                            if (again) {  // the maximum of every row, so that none can be over it below
                                float top = m;
                                take();
#pragma unroll
                                for (int k = 0; k < HALF_BLOCKS; ++k) {
                                    float most = -INFINITY;
#pragma unroll
                                    for (int c = 0; c < BLOCK; ++c) most = fmaxf(most, __uint_as_float(s[k / 2][k % 2 * BLOCK + c]));
                                    top = fmaxf(top, fmaf(most, scale[k].x, scale[k].y));
                                }
                                const float shrink = m != -INFINITY ? exp2_fast(m - top) : 1.0f;
                                m = top;
                                if (j + h > 0) {
                                    alive = wait(o_done + 2 * (h ^ 1) + part, (h ? j : j - 1) & 1, STATUS_WAIT_TMEM_FULL | 0xC310 | part);
                                    if (!alive) break;
                                    tcgen05_fence_after();
#pragma unroll 1
                                    for (int i = 0; i < DIM / 32; ++i) {
                                        uint32_t o[32];
                                        tmem_load_32x32(o_at + i * 32, o);
                                        tmem_load_wait();
                                        arrived(o);
#pragma unroll
                                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * shrink);
                                        tmem_store_32x32(o_at + i * 32, o);
                                    }
                                    l *= shrink;
                                }
                            }
                            const float base = (m == -INFINITY ? 0.0f : m) - P_SHIFT;
                            float worst = 0.0f;
                            l_next = l;
                            take();
#pragma unroll
                            for (int k = 0; k < HALF_BLOCKS; ++k) {
                                const float4 f = scale[k];
                                const float factor = f.x, offset = f.y - base;
                                const uint64_t factor2 = pack_f32x2(factor, factor), offset2 = pack_f32x2(offset, offset);
                                uint64_t sums = pack_f32x2(0.0f, 0.0f);
#pragma unroll
                                for (int c = 0; c < BLOCK; c += 2) {
                                    float low, high;
                                    unpack_f32x2(fma_f32x2(pack_u32x2(s[k / 2][k % 2 * BLOCK + c], s[k / 2][k % 2 * BLOCK + c + 1]), factor2, offset2), low, high);
                                    low = exp2_fast(low), high = exp2_fast(high);
                                    sums = add_f32x2(sums, pack_f32x2(low, high));
                                    const __half2 pair = __floats2half2_rn(low, high);
                                    p[(k * BLOCK + c) / 2] = *reinterpret_cast<const uint32_t *>(&pair);
                                }
                                float even, odd;
                                unpack_f32x2(sums, even, odd);
                                worst = fmaxf(worst, even + odd);
                                l_next = fmaf(even + odd, f.z, l_next);
                            }
                            if (again || __all_sync(0xffffffffu, worst <= MOST_SUM)) break;
                            again = true;
                        }
                        if (!alive) break;
                        l = l_next;
                        tmem_store_32x32(s_at + h * 32, p);
                        tmem_store_wait();
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbarrier_arrive(p_full + 2 * h + part);
                    }
                    if (!alive) break;
                }
                if (alive && tiles > 0) {
                    alive = wait(o_done + 2 + part, (tiles - 1) & 1, STATUS_WAIT_TMEM_FULL | 0xC320 | part);
                    tcgen05_fence_after();
                }
                const long long unit = (static_cast<long long>(b) * cache.heads + head) * a.row_tiles + tile;
                float *partial = a.partial + (unit * a.splits + split) * (PREFILL_ROWS * (DIM + 2));
                const int local = row - first_row;
                const float factor = l > 0.0f ? __frcp_rn(l) : (l == 0.0f ? 0.0f : l);
                const long long out_row = entry.first + row / a.group;
                const int out_head = head * a.group + row % a.group;
                if (alive) {
#pragma unroll
                    for (int i = 0; i < DIM / 32; ++i) {
                        uint32_t o[32];
                        if (tiles > 0) {
                            tmem_load_32x32(o_at + i * 32, o);
                            tmem_load_wait();
                            arrived(o);
                        } else {
#pragma unroll
                            for (int c = 0; c < 32; ++c) o[c] = 0;
                        }
                        if (used == 1) {
                            // through this warp's rows of Q, which is done with, so that rows leave in whole lines
                            const uint32_t r = (warp & 3) * 32 + lane, at = smem_u32(smem + P::Q_AT) + part * P::OPERAND_BYTES + r * 128 + i / 2 * (TILE_ROWS * 128);
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t pairs[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const __half2 pair = __floats2half2_rn(__uint_as_float(o[8 * c + 2 * e]) * factor, __uint_as_float(o[8 * c + 2 * e + 1]) * factor);
                                    pairs[e] = *reinterpret_cast<const uint32_t *>(&pair);
                                }
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + (((i % 2 * 4 + c) ^ (r & 7)) << 4)), "r"(pairs[0]), "r"(pairs[1]), "r"(pairs[2]), "r"(pairs[3]) : "memory");
                            }
                        } else if (row >= rows) {
                            continue;
                        } else {
                            // a column's rows together: threads of a warp write adjacent words
#pragma unroll
                            for (int c = 0; c < 32; ++c) partial[(2 + i * 32 + c) * PREFILL_ROWS + local] = __uint_as_float(o[c]);
                        }
                    }
                    if (used == 1) {
                        const uint32_t at = smem_u32(smem + P::Q_AT) + part * P::OPERAND_BYTES + piece / 8 * (TILE_ROWS * 128);
                        Walk walk(row0, a.group);
                        __syncwarp();
#pragma unroll
                        for (int n = 0; n < WARP_PASSES; ++n) {
                            const uint32_t r = (warp & 3) * 32 + n * ROWS_AT_ONCE + lane / PIECES;
                            uint4 w;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at + r * 128 + ((piece % 8 ^ (r & 7)) << 4)) : "memory");
                            if (y_row0 + n * ROWS_AT_ONCE < rows)
                                *(reinterpret_cast<uint4 *>(a.y + (entry.first + static_cast<long long>(walk.token)) * a.ld_y + (head * a.group + walk.member) * DIM) + piece) = w;
                            walk.go_on();
                        }
                    }
                    if (row < rows && used == 1) {
                        if (a.lse != nullptr) a.lse[out_row * a.heads + out_head] = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m - P_SHIFT + log2f(l));
                    } else if (row < rows) {
                        partial[local] = m, partial[PREFILL_ROWS + local] = l;
                    }
                }
            }
            if (used > 1) join_pieces<DIM>(a, entry, head, (static_cast<long long>(b) * cache.heads + head) * a.row_tiles + tile, first_row, last_row, used, &is_last);
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == ISSUE_WARP) tmem_dealloc(tmem, 512);
}

}  // namespace kv
}  // namespace qi
