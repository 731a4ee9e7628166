// Attention over the paged 8-bit cache for few queries to a sequence: one token of each request, or a handful.
//
//   y_i = sum_j softmax_j(scale * q_i . k_j) v_j       k_j = (c_j - 128) * sk, v_j = (d_j - 128) * sv, sk and sv one for 16 tokens
//
// A CTA takes up to 8 * TILES query rows that share a head of the cache (group heads times tokens) and a piece of that head's
// tokens. Each of its warps walks over steps of 32 tokens with sums of its own; warps are joined in shared memory, pieces in
// a workspace, where the CTA that arrives last adds them up in their order (the same bits whichever is last).
//
// The products run transposed on m16n8k16: S^T = K Q^T and O^T = V^T P^T, so that the 16 rows of an instruction are tokens and channels
// of the cache, of which there are always enough, and the 8 columns are queries, of which there may be one. Which channel or
// token stands at which place of a sum is free as long as both operands agree, and is chosen so that every load is 16 adjacent
// codes of a token: codes go from HBM to registers and from there, widened, into the tensor cores, never through shared memory.
//
// Scales cost nothing per element. With base-2 logarithms, x_j = (scale * log2 e * sk) * raw_j + log2 sv, m = max x_j, p_j = 2^(x_j - m):
//   O = sum p_j d_j (d_j whole numbers),  l = sum p_j / sv,  y = O / l
// so sk and log2 sv enter one fused multiply-add, and 1 / sv once for the sum of a block. p_j is rounded to float16 for the tensor
// cores, in a range shifted up by 2^12 so that it keeps all its digits down to 2^-26 of the largest; queries are float16 as they
// come, codes are exact, all sums are float32. A block of zeros has sv = 0: log2 is taken of max(sv, 2^-60), which changes
// nothing that float16 results could hold.
#pragma once
#include "kv_cache.cuh"

namespace qi {
namespace kv {

constexpr float P_SHIFT = 12.0f, LEAST_SCALE = 8.6736174e-19f;  // 2^-60
constexpr int DECODE_WARPS = 4, DECODE_THREADS = DECODE_WARPS * 32, STEP = 32;

struct Attention {
    const __half *q;
    __half *y;
    float *lse;
    long long ld_q, ld_y;
    int heads, group;   // query heads, and how many of them share a head of the cache
    float scale_log2;
    int causal, window, max_length;
    int chunk, splits, row_tiles;
    int *arrivals;      // [entries][kv_heads][row_tiles], zero between calls
    float *partial;     // [entries][kv_heads][row_tiles][splits][rows][head_dim + 2]
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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
__device__ __forceinline__ uint2 load_codes8(const uint8_t *at) {
    uint2 w;
    asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(at));
    return w;
}

// The keys that row `row` of an entry (row = token * group + head of the group) sees: [low, high).
__device__ __forceinline__ void visible(const Attention &a, const Entry &entry, int row, int &low, int &high) {
    const int position = entry.length - entry.count + row / a.group;
    low = a.window > 0 ? max(0, position - a.window + 1) : 0;
    high = a.causal ? min(entry.length, position + 1) : entry.length;
}

template <int DIM, int TILES>
__global__ void __launch_bounds__(DECODE_THREADS, TILES == 1 ? 3 : 2) decode_kernel(Cache cache, Tables tables, Batch batch, Attention a) {
    constexpr int ROWS = 8 * TILES, K_WORDS = DIM / 16;            // K_WORDS: 32-bit words of a token's codes that a lane holds (keys)
    constexpr int V_WORDS = DIM / 32, BLOCKS = STEP / BLOCK;       // and of values, of each of four tokens
    constexpr int PITCH = DIM + 4;
    __shared__ float join_o[DECODE_WARPS][ROWS][PITCH];
    __shared__ float join_m[DECODE_WARPS][ROWS], join_l[DECODE_WARPS][ROWS];
    __shared__ int is_last;
    grid_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row8 = lane >> 2, quad = lane & 3;
    const int split = blockIdx.x, head = blockIdx.y / a.row_tiles, tile = blockIdx.y % a.row_tiles, b = blockIdx.z;
    Entry entry;
    if (!read_entry(batch, tables, cache.page_shift, b, a.max_length, entry)) {
        if (threadIdx.x == 0) complain(0xC030);
        return;
    }
    const int rows = entry.count * a.group, first_row = tile * ROWS;
    if (first_row >= rows) return;
    const int last_row = min(first_row + ROWS, rows) - 1;
    int low, high, unused;
    visible(a, entry, first_row, low, unused);
    visible(a, entry, last_row, unused, high);
    low = low / BLOCK * BLOCK;
    const int span = max(high - low, 0), used = max((span + a.chunk - 1) / a.chunk, 1);
    if (split >= used) return;
    const int begin = low + split * a.chunk, end = min(begin + a.chunk, high);  // this CTA's tokens

    uint32_t q[TILES][K_WORDS][2];
    int row_low[TILES][2], row_high[TILES][2];  // of this lane's columns of S^T
    int all_low = 0, all_high = 0x7fffffff;     // what every row sees
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
        const int row = first_row + n * 8 + row8;
        const __half *source = a.q + (entry.first + static_cast<long long>(row / a.group)) * a.ld_q + (head * a.group + row % a.group) * DIM;
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j) {
            uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if (row < rows) {
                const uint4 *at = reinterpret_cast<const uint4 *>(source + (quad + 4 * j) * 16);
                w[0] = __ldg(at), w[1] = __ldg(at + 1);
            }
            q[n][4 * j][0] = w[0].x, q[n][4 * j][1] = w[0].y, q[n][4 * j + 1][0] = w[0].z, q[n][4 * j + 1][1] = w[0].w;
            q[n][4 * j + 2][0] = w[1].x, q[n][4 * j + 2][1] = w[1].y, q[n][4 * j + 3][0] = w[1].z, q[n][4 * j + 3][1] = w[1].w;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) visible(a, entry, min(first_row + n * 8 + quad * 2 + i, last_row), row_low[n][i], row_high[n][i]);
    }
    visible(a, entry, last_row, all_low, unused);
    visible(a, entry, first_row, unused, all_high);

    float o[TILES][DIM / 16][4], m[TILES][2], l[TILES][2];
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
        m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int t = 0; t < DIM / 16; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.0f;
    }

    const int *pages = tables.table + static_cast<long long>(entry.slot) * tables.table_pages;
    long long place[BLOCKS];   // token row of each block of the step whose codes are fetched next; -1: none
    auto look_up = [&](int token) {
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            place[k] = -1;
            if (token + k * BLOCK < end) {
                int page = __ldg(pages + (token + k * BLOCK >> cache.page_shift));
                if (page < 0 || page >= cache.pages) complain(0xC031), page = 0;
                place[k] = token_row(cache, page, head, token + k * BLOCK);
            }
        }
    };
    uint32_t key[BLOCKS][2][K_WORDS], value[BLOCKS][4][V_WORDS];
    float k_scale[BLOCKS], v_scale[BLOCKS];
    long long value_place[BLOCKS];
    auto fetch_keys = [&]() {
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            value_place[k] = place[k];
            k_scale[k] = 0.0f, v_scale[k] = 1.0f;
            if (place[k] < 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < K_WORDS; ++j) key[k][i][j] = 0x80808080u;
                continue;
            }
            k_scale[k] = __ldg(cache.scales[0] + place[k] / BLOCK), v_scale[k] = __ldg(cache.scales[1] + place[k] / BLOCK);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < DIM / 64; ++j) {
                    const uint4 w = load_codes(cache.codes[0] + (place[k] + row8 + 8 * i) * DIM + (quad + 4 * j) * 16);
                    key[k][i][4 * j] = w.x, key[k][i][4 * j + 1] = w.y, key[k][i][4 * j + 2] = w.z, key[k][i][4 * j + 3] = w.w;
                }
        }
    };
    auto fetch_values = [&]() {
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (value_place[k] < 0) {
#pragma unroll
                    for (int j = 0; j < V_WORDS; ++j) value[k][i][j] = 0x80808080u;
                    continue;
                }
                const uint8_t *at = cache.codes[1] + (value_place[k] + quad * 2 + (i & 1) + 8 * (i >> 1)) * DIM + row8 * (DIM / 8);
                if constexpr (DIM == 128) {
                    const uint4 w = load_codes(at);
                    value[k][i][0] = w.x, value[k][i][1] = w.y, value[k][i][2] = w.z, value[k][i][3] = w.w;
                } else {
                    const uint2 w = load_codes8(at);
                    value[k][i][0] = w.x, value[k][i][1] = w.y;
                }
            }
    };

    int token = begin + warp * STEP;
    look_up(token);
    fetch_keys();
    fetch_values();
    look_up(token + DECODE_THREADS);
    for (; token < end; token += DECODE_THREADS) {
        float s[TILES][BLOCKS][4];
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
            for (int n = 0; n < TILES; ++n) s[n][k][0] = s[n][k][1] = s[n][k][2] = s[n][k][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < K_WORDS; ++j) {
                const uint32_t a0 = widen2<0x4140>(key[k][0][j]), a1 = widen2<0x4140>(key[k][1][j]), a2 = widen2<0x4342>(key[k][0][j]), a3 = widen2<0x4342>(key[k][1][j]);
#pragma unroll
                for (int n = 0; n < TILES; ++n) mma_16x8x16(s[n][k], a0, a1, a2, a3, q[n][j][0], q[n][j][1]);
            }
        }
        float factor[BLOCKS], offset[BLOCKS], inverse[BLOCKS];
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            const float scale = fmaxf(v_scale[k], LEAST_SCALE);
            factor[k] = k_scale[k] * a.scale_log2, offset[k] = log2f(scale), inverse[k] = __frcp_rn(scale);
        }
        fetch_keys();
        const bool whole = token >= all_low && token + STEP <= min(all_high, end);
        uint32_t p[TILES][BLOCKS][2];
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = m[n][i];
#pragma unroll
                for (int k = 0; k < BLOCKS; ++k)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float &x = s[n][k][2 * r + i];
                        x = fmaf(x, factor[k], offset[k]);
                        const int at = token + k * BLOCK + row8 + 8 * r;
                        if (!whole && (at < row_low[n][i] || at >= min(row_high[n][i], end))) x = -INFINITY;
                        top = fmaxf(top, x);
                    }
#pragma unroll
                for (int step = 4; step < 32; step *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
                const float base = top == -INFINITY ? 0.0f : top;
                const float shrink = exp2_fast(m[n][i] - base);
                m[n][i] = top;
                l[n][i] *= shrink;
#pragma unroll
                for (int t = 0; t < DIM / 16; ++t) o[n][t][i] *= shrink, o[n][t][2 + i] *= shrink;
#pragma unroll
                for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) s[n][k][2 * r + i] = exp2_fast(s[n][k][2 * r + i] - (base - P_SHIFT));
                    l[n][i] = fmaf(s[n][k][i] + s[n][k][2 + i], inverse[k], l[n][i]);
                }
            }
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const __half2 pair = __floats2half2_rn(s[n][k][2 * r], s[n][k][2 * r + 1]);
                    p[n][k][r] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&pair));
                }
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k)
#pragma unroll
            for (int w = 0; w < V_WORDS; ++w) {
                // [channel 4w of two tokens, channel 4w + 1 of both], and 4w + 2, 4w + 3; tokens 8 further on likewise
                const uint32_t low0 = __byte_perm(value[k][0][w], value[k][1][w], 0x5140), high0 = __byte_perm(value[k][0][w], value[k][1][w], 0x7362);
                const uint32_t low8 = __byte_perm(value[k][2][w], value[k][3][w], 0x5140), high8 = __byte_perm(value[k][2][w], value[k][3][w], 0x7362);
                const uint32_t a0 = widen2<0x4140>(low0), a1 = widen2<0x4342>(low0), a2 = widen2<0x4140>(low8), a3 = widen2<0x4342>(low8);
                const uint32_t c0 = widen2<0x4140>(high0), c1 = widen2<0x4342>(high0), c2 = widen2<0x4140>(high8), c3 = widen2<0x4342>(high8);
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    mma_16x8x16(o[n][2 * w], a0, a1, a2, a3, p[n][k][0], p[n][k][1]);
                    mma_16x8x16(o[n][2 * w + 1], c0, c1, c2, c3, p[n][k][0], p[n][k][1]);
                }
            }
        fetch_values();
        look_up(token + 2 * DECODE_THREADS);
    }

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
    const long long unit = (static_cast<long long>(b) * cache.heads + head) * a.row_tiles + tile;
    float *partial = a.partial + unit * a.splits * (ROWS * (DIM + 2));
    const int owned = last_row - first_row + 1;
    auto finish = [&](int row, int channel, float2 sum, float top, float total) {  // channels `channel`, `channel` + 1
        const long long out_row = entry.first + (first_row + row) / a.group;
        const int out_head = head * a.group + (first_row + row) % a.group;
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
        if (used == 1) {
            finish(row, channel, sum, top, total);
        } else {
            float *mine = partial + static_cast<long long>(split) * (ROWS * (DIM + 2));
            *reinterpret_cast<float2 *>(mine + 2 * ROWS + row * DIM + channel) = sum;
            if (channel == 0) mine[row] = top, mine[ROWS + row] = total;
        }
    }
    if (used == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) is_last = atomicAdd(a.arrivals + unit, 1) == used - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    // Warps share the pieces, lanes the channels: many loads on their way at once, where a thread that walked through all pieces of
    // its channels took 70 us for 200 of them.
    constexpr int PIECE = ROWS * (DIM + 2), EACH = DIM / 32;
    float top[ROWS], total[ROWS], sum[ROWS][EACH];
#pragma unroll
    for (int row = 0; row < ROWS; ++row) {
        top[row] = -INFINITY, total[row] = 0.0f;
#pragma unroll
        for (int c = 0; c < EACH; ++c) sum[row][c] = 0.0f;
    }
    for (int i = lane; i < used; i += 32)
#pragma unroll
        for (int row = 0; row < ROWS; ++row)
            if (row < owned) top[row] = fmaxf(top[row], __ldcg(partial + static_cast<long long>(i) * PIECE + row));
#pragma unroll
    for (int row = 0; row < ROWS; ++row)
#pragma unroll
        for (int step = 16; step > 0; step /= 2) top[row] = fmaxf(top[row], __shfl_xor_sync(0xffffffffu, top[row], step));
#pragma unroll 2
    for (int i = warp; i < used; i += DECODE_WARPS) {
        const float *one = partial + static_cast<long long>(i) * PIECE;
#pragma unroll
        for (int row = 0; row < ROWS; ++row) {
            if (row >= owned) break;
            const float weight = exp2_fast(__ldcg(one + row) - (top[row] == -INFINITY ? 0.0f : top[row]));
            total[row] = fmaf(__ldcg(one + ROWS + row), weight, total[row]);
            float part[EACH];
            if constexpr (EACH == 4) {
                const float4 f = __ldcg(reinterpret_cast<const float4 *>(one + 2 * ROWS + row * DIM + lane * EACH));
                part[0] = f.x, part[1] = f.y, part[2] = f.z, part[3] = f.w;
            } else {
                const float2 f = __ldcg(reinterpret_cast<const float2 *>(one + 2 * ROWS + row * DIM + lane * EACH));
                part[0] = f.x, part[1] = f.y;
            }
#pragma unroll
            for (int c = 0; c < EACH; ++c) sum[row][c] = fmaf(part[c], weight, sum[row][c]);
        }
    }
#pragma unroll
    for (int row = 0; row < ROWS; ++row) {
        if (lane == 0) join_m[warp][row] = top[row], join_l[warp][row] = total[row];
#pragma unroll
        for (int c = 0; c < EACH; ++c) join_o[warp][row][lane * EACH + c] = sum[row][c];
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
    if (threadIdx.x == 0) a.arrivals[unit] = 0;
}

}  // namespace kv
}  // namespace qi
