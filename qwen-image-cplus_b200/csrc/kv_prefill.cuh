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
// so that the two halves alternate: while one's weights are computed the tensor cores have the other's products. Values are stored as
// they lie in the cache, a token a row, and enter their product "MN-major"; nothing is transposed.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time (which then waits for the product before):
// weights are at most 2^(8 + 7) in float16 and keep all their digits down to 2^-21 of that maximum; sums are float32.
//
// TMEM: S and P of the halves at columns 0 and 128, O at 256 and 384.
#pragma once
#include "kv_decode.cuh"

namespace qi {
namespace kv {

constexpr int PREFILL_THREADS = 512, TILE_ROWS = 128, TILE_TOKENS = 128, PREFILL_ROWS = 2 * TILE_ROWS;
constexpr int WIDEN_WARP0 = 8, ISSUE_WARP = 12, TILE_BLOCKS = TILE_TOKENS / BLOCK, SCALE_SLOTS = 4;
constexpr float PREFILL_SHIFT = 7.0f, GROWTH = 8.0f;
constexpr float LEAST_FACTOR = 1e-30f;  // in place of a key scale of zero: what is hidden stays -infinity times it, every score 0
constexpr uint32_t TMEM_S = 0, TMEM_O = 256;

template <int DIM>
struct Prefill {
    static constexpr int HALVES = DIM / 64;                            // 128-byte rows of 64 channels
    static constexpr int OPERAND_BYTES = TILE_TOKENS * DIM * 2;        // of K, V, or half of Q
    static constexpr int Q_AT = 0, K_AT = 2 * OPERAND_BYTES, V_AT = 4 * OPERAND_BYTES, SCALES_AT = 6 * OPERAND_BYTES;
    static constexpr int BARRIERS_AT = SCALES_AT + SCALE_SLOTS * 3 * TILE_BLOCKS * 4;
    static constexpr int BARRIERS = 8 + SCALE_SLOTS + 6 + 1;
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
    if (a.lse != nullptr) a.lse[out_row * a.heads + out_head] = total == 0.0f ? -INFINITY : 0.6931471805599453f * (top - PREFILL_SHIFT + log2f(total));
}

template <int DIM>
__global__ void __launch_bounds__(PREFILL_THREADS, 1) prefill_kernel(Cache cache, Tables tables, Batch batch, Attention a) {
    using P = Prefill<DIM>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float(*scales)[3][TILE_BLOCKS] = reinterpret_cast<float(*)[3][TILE_BLOCKS]>(smem + P::SCALES_AT);
    uint64_t *barriers = reinterpret_cast<uint64_t *>(smem + P::BARRIERS_AT);
    uint64_t *k_full = barriers, *k_empty = barriers + 2, *v_full = barriers + 4, *v_empty = barriers + 6, *scale_full = barriers + 8;
    uint64_t *s_full = barriers + 8 + SCALE_SLOTS, *p_full = s_full + 2, *o_done = s_full + 4, *q_full = s_full + 6;
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
            mbarrier_init(s_full + i, 1), mbarrier_init(p_full + i, 4), mbarrier_init(o_done + i, 1);
        }
        for (int i = 0; i < SCALE_SLOTS; ++i) mbarrier_init(scale_full + i, 1);
        mbarrier_init(q_full, 8);
        fence_barrier_init();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_wait();

    const int split = blockIdx.x, head = blockIdx.y / a.row_tiles, tile = blockIdx.y % a.row_tiles, b = blockIdx.z;
    Entry entry;
    const bool sound = read_entry(batch, tables, cache.page_shift, b, a.max_length, entry);
    if (!sound && threadIdx.x == 0) complain(0xC040);
    const int rows = sound ? entry.count * a.group : 0, first_row = tile * PREFILL_ROWS;
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
            constexpr int LANES = DIM / 16, TOKENS = 128 / LANES, LOADS = TILE_TOKENS / TOKENS;  // threads to a token, tokens and loads of a pass
            const int t = threadIdx.x - WIDEN_WARP0 * 32, row0 = t / LANES, chunk = t % LANES;
            const int *pages = tables.table + static_cast<long long>(entry.slot) * tables.table_pages;
            uint4 words[2][LOADS];  // of keys, of values
            auto place_of = [&](int token) -> long long {  // token row of a block; -1: none
                if (token >= end) return -1;
                int page = __ldg(pages + (token >> cache.page_shift));
                if (page < 0 || page >= cache.pages) complain(0xC041), page = 0;
                return token_row(cache, page, head, token);
            };
            auto fetch = [&](int which, int j) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int token = begin + j * TILE_TOKENS + i * TOKENS + row0;
                    const long long place = j < tiles ? place_of(token / BLOCK * BLOCK) : -1;
                    words[which][i] = place < 0 ? make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u)
                                                : load_codes(cache.codes[which] + (place + token % BLOCK) * DIM + chunk * 16);
                }
            };
            auto widen = [&](int which, uint32_t base) {
                // the two 16-byte pieces in the other order for every second half, so that eight threads meet no bank twice
                const uint32_t half = chunk / 4, piece = chunk % 4 * 2, swap = half;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const uint32_t row = i * TOKENS + row0;
                    const uint32_t w[4] = {words[which][i].x, words[which][i].y, words[which][i].z, words[which][i].w};
                    uint32_t out[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) out[2 * k] = widen2<0x4140>(w[k]), out[2 * k + 1] = widen2<0x4342>(w[k]);
                    const uint32_t at = base + half * (TILE_TOKENS * 128) + row * 128;
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        const uint32_t p = k ^ swap;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + (((piece + p) ^ (row & 7)) << 4)), "r"(p ? out[4] : out[0]), "r"(p ? out[5] : out[1]),
                                     "r"(p ? out[6] : out[2]), "r"(p ? out[7] : out[3]) : "memory");
                    }
                }
            };
            bool alive = true;
            fetch(0, 0);
            fetch(1, 0);
            for (int j = 0; j < tiles && alive; ++j) {
                const int stage = j & 1, phase = j >> 1 & 1;
                if (warp == WIDEN_WARP0) {
                    if (lane < TILE_BLOCKS) {
                        const long long place = place_of(begin + j * TILE_TOKENS + lane * BLOCK);
                        const float k_scale = place < 0 ? 0.0f : __ldg(cache.scales[0] + place / BLOCK), v_scale = place < 0 ? 1.0f : fmaxf(__ldg(cache.scales[1] + place / BLOCK), LEAST_SCALE);
                        scales[j % SCALE_SLOTS][0][lane] = fmaxf(k_scale * a.scale_log2, LEAST_FACTOR);
                        scales[j % SCALE_SLOTS][1][lane] = log2f(v_scale);
                        scales[j % SCALE_SLOTS][2][lane] = __frcp_rn(v_scale);
                    }
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(scale_full + j % SCALE_SLOTS);
                }
                if (!mbarrier_wait_warp(k_empty + stage, phase ^ 1, &g_status, STATUS_WAIT_EMPTY | 0xC000 | stage, lane)) { alive = false; break; }
                widen(0, smem_u32(smem + P::K_AT + stage * P::OPERAND_BYTES));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbarrier_arrive(k_full + stage);
                fetch(0, j + 1);
                if (!mbarrier_wait_warp(v_empty + stage, phase ^ 1, &g_status, STATUS_WAIT_EMPTY | 0xC100 | stage, lane)) { alive = false; break; }
                widen(1, smem_u32(smem + P::V_AT + stage * P::OPERAND_BYTES));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbarrier_arrive(v_full + stage);
                fetch(1, j + 1);
            }
        } else if (warp >= ISSUE_WARP) {
            // ---- products ----
            setmaxnreg_dec<40>();
            if (warp == ISSUE_WARP && tiles > 0) {
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
                bool alive = mbarrier_wait_warp(q_full, 0, &g_status, STATUS_WAIT_FULL | 0xC200, lane) && mbarrier_wait_warp(k_full, 0, &g_status, STATUS_WAIT_FULL | 0xC210, lane);
                tcgen05_fence_after();
                const bool elected = elect_one();
                if (alive && elected) {
                    for (int i = 0; i < parts; ++i) scores(i, 0);
                    tcgen05_commit(k_empty);
                }
                __syncwarp();
                for (int j = 0; j < tiles && alive; ++j) {
                    const int stage = j & 1, next = (j + 1) & 1;
                    alive = mbarrier_wait_warp(v_full + stage, j >> 1 & 1, &g_status, STATUS_WAIT_FULL | 0xC220 | stage, lane);
                    for (int i = 0; i < parts && alive; ++i) {
                        alive = mbarrier_wait_warp(p_full + i, j & 1, &g_status, STATUS_WAIT_READY | 0xC230 | i, lane);
                        if (alive && i == 0 && j + 1 < tiles) alive = mbarrier_wait_warp(k_full + next, (j + 1) >> 1 & 1, &g_status, STATUS_WAIT_FULL | 0xC240 | next, lane);
                        if (!alive) break;
                        tcgen05_fence_after();
                        if (elected) {
                            const uint32_t v = v_at + stage * P::OPERAND_BYTES;
#pragma unroll
                            for (int s = 0; s < TILE_TOKENS / 16; ++s)
                                umma_f16_ts(tmem + TMEM_O + i * 128, tmem + TMEM_S + i * 128 + s * 8, umma_desc_mn_sw128(v + s * 2048, TILE_TOKENS * 128), IDESC_O, j > 0 || s > 0);
                            tcgen05_commit(o_done + i);
                            if (j + 1 < tiles) scores(i, j + 1);
                            if (i == parts - 1) {
                                tcgen05_commit(v_empty + stage);
                                if (j + 1 < tiles) tcgen05_commit(k_empty + next);
                            }
                        }
                        __syncwarp();
                    }
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
            {
                // this thread's row of Q
                const __half *source = a.q + (entry.first + static_cast<long long>(row / a.group)) * a.ld_q + (head * a.group + row % a.group) * DIM;
                const uint32_t r = (warp & 3) * 32 + lane, at = smem_u32(smem + P::Q_AT) + part * P::OPERAND_BYTES + r * 128;
#pragma unroll
                for (int c = 0; c < DIM / 8; ++c) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (row < rows) w = __ldg(reinterpret_cast<const uint4 *>(source) + c);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + c / 8 * (TILE_ROWS * 128) + ((c % 8 ^ (r & 7)) << 4)), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbarrier_arrive(q_full);
            }
            float m = -INFINITY, l = 0.0f;
            bool alive = true;
            if (part < parts) {
                for (int j = 0; j < tiles; ++j) {
                    if (!mbarrier_wait_warp(scale_full + j % SCALE_SLOTS, j / SCALE_SLOTS & 1, &g_status, STATUS_WAIT_FULL | 0xC300 | part, lane) ||
                        !mbarrier_wait_warp(s_full + part, j & 1, &g_status, STATUS_WAIT_TMEM_FULL | 0xC300 | part, lane)) { alive = false; break; }
                    tcgen05_fence_after();
                    uint32_t s[4][32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_load_32x32(s_at + i * 32, s[i]);
                    tmem_load_wait();
#pragma unroll
                    for (int i = 0; i < 4; ++i) arrived(s[i]);
                    const float(&scale)[3][TILE_BLOCKS] = scales[j % SCALE_SLOTS];
                    const int token = begin + j * TILE_TOKENS;
                    const int seen_low = row_low - token, seen_high = min(row_high, end) - token;
                    if (!__all_sync(0xffffffffu, seen_low <= 0 && seen_high >= TILE_TOKENS)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (i * 32 + c < seen_low || i * 32 + c >= seen_high) s[i][c] = 0xff800000u;  // -infinity
                    }
                    float top = m;
#pragma unroll
                    for (int k = 0; k < TILE_BLOCKS; ++k) {
                        float most = -INFINITY;
#pragma unroll
                        for (int c = 0; c < BLOCK; ++c) most = fmaxf(most, __uint_as_float(s[k / 2][k % 2 * BLOCK + c]));
                        top = fmaxf(top, fmaf(most, scale[0][k], scale[1][k]));
                    }
                    const bool grown = top > m + GROWTH || (m == -INFINITY && top > m);
                    if (__any_sync(0xffffffffu, grown)) {
                        const float shrink = grown ? exp2_fast(m - top) : 1.0f;
                        if (grown) m = top;
                        if (j > 0) {
                            if (!mbarrier_wait_warp(o_done + part, (j - 1) & 1, &g_status, STATUS_WAIT_TMEM_FULL | 0xC310 | part, lane)) { alive = false; break; }
                            tcgen05_fence_after();
#pragma unroll
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
                    const float base = m == -INFINITY ? 0.0f : m;
                    uint32_t p[2][32];
#pragma unroll
                    for (int k = 0; k < TILE_BLOCKS; ++k) {
                        const float factor = scale[0][k], offset = scale[1][k] - base + PREFILL_SHIFT;
                        float sum = 0.0f;
#pragma unroll
                        for (int c = 0; c < BLOCK; c += 2) {
                            float x[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float raw = __uint_as_float(s[k / 2][k % 2 * BLOCK + c + e]);
                                x[e] = exp2_fast(fmaf(raw, factor, offset));
                                sum += x[e];
                            }
                            const __half2 pair = __floats2half2_rn(x[0], x[1]);
                            p[k / 4][k % 4 * 8 + c / 2] = *reinterpret_cast<const uint32_t *>(&pair);
                        }
                        l = fmaf(sum, scale[2][k], l);
                    }
                    tmem_store_32x32(s_at, p[0]);
                    tmem_store_32x32(s_at + 32, p[1]);
                    tmem_store_wait();
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(p_full + part);
                }
                if (alive && tiles > 0) {
                    alive = mbarrier_wait_warp(o_done + part, (tiles - 1) & 1, &g_status, STATUS_WAIT_TMEM_FULL | 0xC320 | part, lane);
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
                        if (row >= rows) continue;
                        if (used == 1) {
                            uint4 *at = reinterpret_cast<uint4 *>(a.y + out_row * a.ld_y + out_head * DIM + i * 32);
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t pairs[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const __half2 pair = __floats2half2_rn(__uint_as_float(o[8 * c + 2 * e]) * factor, __uint_as_float(o[8 * c + 2 * e + 1]) * factor);
                                    pairs[e] = *reinterpret_cast<const uint32_t *>(&pair);
                                }
                                at[c] = make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
                            }
                        } else {
                            // a column's rows together: threads of a warp write adjacent words
#pragma unroll
                            for (int c = 0; c < 32; ++c) partial[(2 + i * 32 + c) * PREFILL_ROWS + local] = __uint_as_float(o[c]);
                        }
                    }
                    if (row < rows && used == 1) {
                        if (a.lse != nullptr) a.lse[out_row * a.heads + out_head] = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m - PREFILL_SHIFT + log2f(l));
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
