// The norms on both sides of a block with the block's gate, in one pass over the rows:
//
//   r' = r + residual_scale * gate * post(branch)          post: a norm of the block's result times its weight, or nothing
//   y  = norm(r') * weight * (1 + scale) + shift           norm: x / rms(x), or (x - mean) / deviation
//
// Each row is read once and written once; the values stay in registers between the sums, which are float32 and taken about the
// mean (passes over registers, so that a large mean costs no digits). r' enters the second norm unrounded, also where it is
// stored as float16. Bound by memory, and by what stands between a row's loads and its stores: up to four sums over the CTA. So each CTA
// walks over its share of the rows with the next row's loads under way, and keeps what the vectors (gate, scale, shift, weights) come to
// for a column in registers: two CTAs of 256 threads to an SM, 16384 rows of 4096: 132 us, 6.1 TB/s, 4096 rows 37.5. With the vectors
// read from L1 for each row 156 (62 % of the issue slots were taken, most of them by that); five CTAs without loads ahead 163, eight that do
// not all run at once 174; a ring of rows in shared memory, filled by bulk copies, leaves no L1 for the vectors: 203.
#pragma once
#include "ptx.cuh"

namespace qi {
namespace gated_norm {

constexpr int MOST_WIDTH = 16384;

struct Arguments {
    const void *residual, *branch;
    const float *branch_weight;
    const void *gate, *scale, *shift;
    const float *weight;
    void *residual_out, *y;
    long long ld_vector;
    int rows, width, rows_per_vector;
    float residual_scale, epsilon;
    bool residual_f16, branch_f16, vector_f16, y_f16, branch_norm, layer;
};

// Eight values from `at` on as they lie in memory: of a row, which are read once (STREAM), or of a vector, which other rows read too.
struct Raw8 {
    uint4 w[2];
};
template <bool STREAM>
__device__ __forceinline__ void fetch8(const void *base, bool f16, long long at, Raw8 &raw) {
    const uint4 *words = reinterpret_cast<const uint4 *>(static_cast<const char *>(base) + at * (f16 ? 2 : 4));
    raw.w[0] = STREAM ? __ldcs(words) : __ldg(words);
    if (!f16) raw.w[1] = STREAM ? __ldcs(words + 1) : __ldg(words + 1);
}
__device__ __forceinline__ void widen8(const Raw8 &raw, bool f16, float (&x)[8]) {
    if (f16) {
        const uint32_t pairs[4] = {raw.w[0].x, raw.w[0].y, raw.w[0].z, raw.w[0].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&pairs[j]));
            x[2 * j] = f.x, x[2 * j + 1] = f.y;
        }
    } else {
        const uint32_t words[8] = {raw.w[0].x, raw.w[0].y, raw.w[0].z, raw.w[0].w, raw.w[1].x, raw.w[1].y, raw.w[1].z, raw.w[1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(words[j]);
    }
}
__device__ __forceinline__ void load8(const void *base, bool f16, long long at, float (&x)[8]) {
    Raw8 raw;
    fetch8<false>(base, f16, at, raw);
    widen8(raw, f16, x);
}

__device__ __forceinline__ void store8(void *base, bool f16, long long at, const float (&x)[8]) {
    if (f16) {
        uint32_t pairs[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
            pairs[j] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(static_cast<__half *>(base) + at) = make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
    } else {
        float4 *words = reinterpret_cast<float4 *>(static_cast<float *>(base) + at);
        words[0] = make_float4(x[0], x[1], x[2], x[3]);
        words[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

// Two sums over the CTA. Two rows of `sums` in turn: a thread that writes the next sums' has passed the barrier behind which all have
// read the ones before the last.
template <int WARPS>
__device__ __forceinline__ float2 block_sums(float2 value, float2 (&sums)[2][WARPS], int &turn) {
#pragma unroll
    for (int step = 16; step > 0; step /= 2) value.x += __shfl_xor_sync(0xffffffffu, value.x, step), value.y += __shfl_xor_sync(0xffffffffu, value.y, step);
    if ((threadIdx.x & 31) == 0) sums[turn][threadIdx.x >> 5] = value;
    __syncthreads();
    float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total.x += sums[turn][w].x, total.y += sums[turn][w].y;
    turn ^= 1;
    return total;
}

// With two pieces a thread needs 110 to 128 registers: fewer, and what is fetched ahead is spilled, which waits for it (three CTAs of 192: 74 us
// instead of 57 for 8192 rows of 3072). The compiler spills 16 bytes of the one with 160 threads all the same.
template <int THREADS, int PIECES>
__global__ void __launch_bounds__(THREADS, PIECES == 1 ? 768 / THREADS : THREADS <= 256 ? 512 / THREADS : 1) norm_kernel(const Arguments a) {
    constexpr int WARPS = THREADS / 32;
    __shared__ float2 sums[2][WARPS];
    grid_wait();
    int turn = 0;
    const float per_value = 1.0f / static_cast<float>(a.width);
    // x becomes (x - mean if it is a layer norm) and its factor is returned. The mean is taken twice, the second time of what the first
    // left, together with the squares: a float32 sum of values around 10^4 knows their mean to 10^-3 only.
    auto normalise = [&](float (&x)[PIECES][8]) {
        auto shift_by = [&](float mean) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                if ((p * THREADS + static_cast<int>(threadIdx.x)) * 8 < a.width)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[p][j] -= mean;
        };
        float2 sum = make_float2(0.0f, 0.0f);
        if (a.layer) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum.x += x[p][j];
            shift_by(block_sums<WARPS>(sum, sums, turn).x * per_value);
            sum.x = 0.0f;
        }
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (a.layer) sum.x += x[p][j];
                sum.y = fmaf(x[p][j], x[p][j], sum.y);
            }
        sum = block_sums<WARPS>(sum, sums, turn);
        if (!a.layer) return rsqrtf(fmaf(sum.y, per_value, a.epsilon));
        const float rest = sum.x * per_value;
        shift_by(rest);
        return rsqrtf(fmaxf(fmaf(sum.y, per_value, -rest * rest), 0.0f) + a.epsilon);
    };
    constexpr bool KEEP = PIECES <= 2;  // a thread that has 32 columns has no registers for what follows, nor for a row ahead
    Raw8 raw_r[PIECES], raw_b[PIECES];  // the next row's values: on their way while this row's sums are waited for
    auto fetch = [&](long long row) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int column = (p * THREADS + threadIdx.x) * 8;
            raw_r[p].w[0] = raw_r[p].w[1] = raw_b[p].w[0] = raw_b[p].w[1] = make_uint4(0, 0, 0, 0);
            if (row < a.rows && column < a.width) {
                fetch8<true>(a.residual, a.residual_f16, row * a.width + column, raw_r[p]);
                if (a.branch != nullptr) fetch8<true>(a.branch, a.branch_f16, row * a.width + column, raw_b[p]);
            }
        }
    };
    // What a column's values are multiplied by and what is added to them. They are kept for the rows to come, which mostly have the same vectors.
    auto read_into = [&](int column, long long vector, float (&into)[8]) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) into[j] = a.residual_scale;
        if (a.branch_weight != nullptr) {
            load8(a.branch_weight, false, column, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) into[j] *= v[j];
        }
        if (a.gate != nullptr) {
            load8(a.gate, a.vector_f16, vector + column, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) into[j] *= v[j];
        }
    };
    auto read_out = [&](int column, long long vector, float (&scale)[8], float (&shift)[8]) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) scale[j] = 1.0f, shift[j] = 0.0f;
        if (a.scale != nullptr) {
            load8(a.scale, a.vector_f16, vector + column, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] += v[j];
        }
        if (a.weight != nullptr) {
            load8(a.weight, false, column, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] *= v[j];
        }
        if (a.shift != nullptr) load8(a.shift, a.vector_f16, vector + column, shift);
    };
    constexpr int KEPT = KEEP ? PIECES : 1;
    float into[KEPT][8], scale[KEPT][8], shift[KEPT][8];
    if (KEEP) fetch(blockIdx.x);
    long long held = -1;
    for (int row = blockIdx.x; static_cast<unsigned>(row) < static_cast<unsigned>(a.rows); row += gridDim.x) {  // a sum that leaves int ends it
        const long long start = static_cast<long long>(row) * a.width, vector = static_cast<long long>(row / a.rows_per_vector) * a.ld_vector;
        if (KEEP && vector != held) {
            held = vector;
#pragma unroll
            for (int p = 0; p < KEPT; ++p) {
                const int column = (p * THREADS + threadIdx.x) * 8;
                if (column < a.width) read_into(column, vector, into[p]), read_out(column, vector, scale[p], shift[p]);
            }
        }
        if (!KEEP) fetch(row);
        float r[PIECES][8], b[PIECES][8];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) widen8(raw_r[p], a.residual_f16, r[p]), widen8(raw_b[p], a.branch_f16, b[p]);
        if (KEEP) fetch(static_cast<long long>(row) + gridDim.x);
        if (a.branch != nullptr) {
            const float factor = a.branch_norm ? normalise(b) : 1.0f;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int column = (p * THREADS + threadIdx.x) * 8;
                if (column >= a.width) continue;
                float w[8];
                if constexpr (!KEEP) read_into(column, vector, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) r[p][j] = fmaf(b[p][j] * factor, KEEP ? into[p % KEPT][j] : w[j], r[p][j]);
            }
        }
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int column = (p * THREADS + threadIdx.x) * 8;
            if (column < a.width && a.residual_out != nullptr) store8(a.residual_out, a.residual_f16, start + column, r[p]);
        }
        if (a.y == nullptr) continue;
        const float factor = normalise(r);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int column = (p * THREADS + threadIdx.x) * 8;
            if (column >= a.width) continue;
            float w[8], v[8];
            if constexpr (!KEEP) read_out(column, vector, w, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) r[p][j] = fmaf(r[p][j] * factor, KEEP ? scale[p % KEPT][j] : w[j], KEEP ? shift[p % KEPT][j] : v[j]);
            store8(a.y, a.y_f16, start + column, r[p]);
        }
    }
}

}  // namespace gated_norm
}  // namespace qi
