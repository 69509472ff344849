/*
 * Attention of one new token per sequence over a key-value cache kept in pages.
 *
 *   out[b,h] = sum_t softmax_t(scale q[b,h].k_t) v_t
 * over the visible tokens t of sequence b: t < length, and with a window
 * t >= length - window or t < sinks. Query head h reads key head
 * h / (heads / kv_heads). Token t of sequence b lies in page table[b][t / page]
 * at slot t % page. A token whose page number is outside [0, pages) is not
 * visible; a head that sees nothing gives zeros.
 *
 * Bound: every visible key and value has to be read once, 2 * depth values per
 * token and key head, for 4 * depth * (heads / kv_heads) operations, so HBM
 * bounds it for any group of heads that one pass serves; the products go to the
 * tensor cores because eight heads per key on CUDA cores would not keep up. The work of a warp is 16
 * tokens: S^T[16 tokens, 8 heads] = K Q^T and O^T[depth, 8 heads] += V^T P^T
 * with mma.m16n8k16. Tokens (and depth) take the 16-row side, so that a group
 * of up to eight heads fills the 8-column side, and the softmax statistics of a
 * head sit on the lanes that hold the head's column in both products. P^T turns
 * from the accumulator's to the operand's layout by movmatrix, without shared
 * memory. (tcgen05 would want 128 rows of M and bring nothing to a kernel that
 * waits for HBM.) Scores, statistics, sums and the joined result are FP32; P is
 * rounded to BF16 (to FP16 over an 8-bit cache), at most half a step relative
 * to each weight, like the operands of any BF16 product.
 *
 * Work split. All (sequence, key head, block of 8 or 16 query heads) items are
 * laid end to end in tiles of 64 visible tokens and cut into equal contiguous
 * ranges, one per CTA, so ragged lengths load every SM alike. Every CTA finds
 * its range from the lengths on the device: no plan on the host, and a captured
 * call follows the lengths of the replay. A range that covers an item whole
 * writes its result; a piece of an item leaves maximum, sum and unscaled result
 * in the workspace (at most two pieces per CTA, its first and its last), and
 * attend_join adds the pieces of an item in token order. No atomics: the same
 * call gives the same bits.
 *
 * Each of the four warps of a CTA copies its own 16 tokens of a tile into its
 * own shared-memory ring with cp.async and reads nothing of the others until
 * the segment of an item ends, so the main loop has no barrier. Tokens that are
 * not visible are filled with zeros instead of being read: a weight of zero
 * times a NaN would be NaN.
 */
#pragma once

#include "context.cuh"
#include "head_rotate.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace attend
{

constexpr int kWarps = 4;
constexpr int kWarpTokens = 16;
constexpr int kTile = kWarps * kWarpTokens;

struct AttendTask {
    int batch, heads, kv_heads, group, head_blocks, depth;
    int page_size, page_shift, pages, table_width; /* page_shift < 0: not a power of two */
    int window, sinks;
    long long q_batch, q_head, table_row;
    const __nv_bfloat16 *q;
    heads::CacheLayout keys, values;
    const int32_t *table, *lengths;
    float score_scale; /* scale * key scale * log2(e) */
    float value_scale;
    __nv_bfloat16 *out; /* [batch, heads, depth] contiguous */
    float *pieces;      /* [grid][2][head slots][depth], then statistics */
    float *statistics;  /* [grid][2][head slots][2] */
};

/* Tokens of a sequence that are visible, before bad pages are taken out. */
__device__ __forceinline__ int visible_tokens(const AttendTask &task, int length)
{
    const long long room = (long long)task.table_width * task.page_size;
    int seen = length < 0 ? 0 : (length < room ? length : int(room));
    if (task.window > 0 && seen > task.window) {
        const int rest = seen - task.window;
        seen = task.window + (task.sinks < rest ? task.sinks : rest);
    }
    return seen;
}

__device__ __forceinline__ int clamped_length(const AttendTask &task, int length)
{
    const long long room = (long long)task.table_width * task.page_size;
    return length < 0 ? 0 : (length < room ? length : int(room));
}

/* Tiles of one item of sequence b; an empty one keeps a tile so that its zeros
 * get written. */
__device__ __forceinline__ int tiles_of(const AttendTask &task, int b)
{
    const int seen = visible_tokens(task, task.lengths[b]);
    return seen ? (seen - 1) / kTile + 1 : 1;
}

/* Called by whole warps. Sum of tiles_of over the batch. */
__device__ __forceinline__ long long total_tiles(const AttendTask &task)
{
    long long sum = 0;
    for (int b = threadIdx.x & 31; b < task.batch; b += 32)
        sum += tiles_of(task, b);
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2)
        sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    return sum * task.kv_heads * task.head_blocks;
}

/* Called by whole warps. The sequence that holds tile `tile` of the whole list
 * and the number of the sequence's first tile. */
__device__ __forceinline__ void locate(const AttendTask &task, long long tile, int &sequence,
                                       long long &first)
{
    const int lane = threadIdx.x & 31;
    const long long per = (long long)task.kv_heads * task.head_blocks;
    long long before = 0;
    for (int base = 0; base < task.batch; base += 32) {
        const long long mine = base + lane < task.batch ? per * tiles_of(task, base + lane) : 0;
        long long upto = mine;
#pragma unroll
        for (int offset = 1; offset < 32; offset *= 2) {
            const long long other = __shfl_up_sync(0xffffffffu, upto, offset);
            if (lane >= offset)
                upto += other;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + lane < task.batch &&
                                                             before + upto > tile);
        if (past) {
            const int at = __ffs(past) - 1;
            sequence = base + at;
            first = before + __shfl_sync(0xffffffffu, upto - mine, at);
            return;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    sequence = task.batch, first = before;
}

__device__ __forceinline__ long long range_start(long long total, int grid, int cta)
{
    return total / grid * cta + total % grid * cta / grid;
}

/* ---- tensor-core pieces ---- */

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t address)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t address)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <bool Half>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (Half)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, "
                     "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, "
                     "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy_16(uint32_t shared, const void *global, bool real)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(global),
                 "r"(real ? 16 : 0)
                 : "memory");
}

template <bool Half> __device__ __forceinline__ uint32_t pack(float low, float high)
{
    if constexpr (Half) {
        const __half2 pair = __floats2half2_rn(low, high);
        return *reinterpret_cast<const uint32_t *>(&pair);
    } else {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
        return *reinterpret_cast<const uint32_t *>(&pair);
    }
}

/* two E4M3 values (exact in FP16), the lower byte in the lower half */
__device__ __forceinline__ uint32_t widen(uint32_t two_bytes)
{
    const __half2_raw pair =
        __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two_bytes), __NV_E4M3);
    return uint32_t(pair.x) | (uint32_t(pair.y) << 16);
}

/* ---- the kernel ---- */

/* Depth: 64, 128 or 256, the stored depth rounded up. Blocks: 8-head column
 * blocks served by one pass over the keys. Eight: 8-bit cache. */
template <int Depth, int Blocks, bool Eight> struct Shape {
    static constexpr int kRowBytes = Depth * (Eight ? 1 : 2);
    static constexpr int kChunks = kRowBytes / 16;
    /* Byte offset in its row of a 16-byte chunk: permuted so that eight consecutive rows hold a
     * chunk in different banks (rows of 64 bytes lie two to a line of banks). Rows r and r + 8
     * have the same order. */
    static __device__ __forceinline__ uint32_t place(int row, int chunk)
    {
        return 16u * uint32_t(kChunks >= 8 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3));
    }
    static constexpr int kStageBytes = 2 * kWarpTokens * kRowBytes; /* keys and values */
    static constexpr int kStages = kStageBytes >= 16384 ? 3 : (kStageBytes >= 8192 ? 3 : 4);
    static constexpr int kHeads = 8 * Blocks;
    static constexpr int kJoinPitch = Depth + 4; /* heads two apart fall eight banks apart */
    static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
    static constexpr int kJoinBytes = kWarps * kHeads * kJoinPitch * 4;
    static constexpr int kBytes = kRingBytes + kJoinBytes + kWarps * kHeads * 8 + kWarps * kStages * 4;
    /* CTAs whose shared memory fits an SM: 228 KB, of which each CTA takes 1 KB more than it asks for */
    static constexpr int kResident = 228 * 1024 / (kBytes + 1024);
};

template <int Depth, int Blocks, bool Eight>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const AttendTask task)
{
    using S = Shape<Depth, Blocks, Eight>;
    extern __shared__ __align__(128) uint8_t shared[];
    float *join = reinterpret_cast<float *>(shared + S::kRingBytes);
    float *join_stats = reinterpret_cast<float *>(shared + S::kRingBytes + S::kJoinBytes);
    uint32_t *stage_seen = reinterpret_cast<uint32_t *>(join_stats + kWarps * S::kHeads * 2);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int g = lane / 4, t = lane % 4;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(shared)) +
                          warp * S::kStages * S::kStageBytes;
    uint32_t *seen_words = stage_seen + warp * S::kStages;

    const long long total = total_tiles(task);
    const long long begin = range_start(total, gridDim.x, blockIdx.x);
    const long long end = range_start(total, gridDim.x, blockIdx.x + 1);
    if (begin >= end)
        return;
    int sequence;
    long long sequence_first;
    locate(task, begin, sequence, sequence_first);

    for (long long tile = begin; tile < end;) {
        /* the item and the segment [from, upto) of its tiles */
        const int length = clamped_length(task, task.lengths[sequence]);
        const int seen = visible_tokens(task, length);
        const int tiles = seen ? (seen - 1) / kTile + 1 : 1;
        const int item = int((tile - sequence_first) / tiles);
        const long long item_first = sequence_first + (long long)item * tiles;
        const int from = int(tile - item_first);
        const int upto = int(end - item_first < tiles ? end - item_first : tiles);
        const int kv_head = item / task.head_blocks;
        const int head_block = item % task.head_blocks;
        const int first_head = kv_head * task.group + head_block * S::kHeads;
        const int live_heads = min(S::kHeads, task.group - head_block * S::kHeads);
        const int jump_at = task.window > 0 && length > task.window ? seen - task.window : 0;
        const int jump = length - seen; /* tokens between the sinks and the window */
        const int32_t *table_row = task.table + sequence * task.table_row;

        const auto issue = [&](int j) {
            const int stage = (j - from) % S::kStages;
            const uint32_t base = ring + stage * S::kStageBytes;
            int page = -1, slot = 0;
            if (lane < kWarpTokens && j < upto) {
                int v = j * kTile + warp * kWarpTokens + lane;
                if (v < seen) {
                    v += v >= jump_at ? jump : 0;
                    const int number = task.page_shift >= 0 ? v >> task.page_shift : v / task.page_size;
                    slot = v - number * task.page_size;
                    page = table_row[number];
                    if (page < 0 || page >= task.pages)
                        page = -1;
                }
            }
            const uint32_t real = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0)
                seen_words[stage] = real;
            if (real) {
                constexpr int kRows = 32 / S::kChunks; /* rows a warp copies at once */
                const int chunk = lane % S::kChunks;
                const bool inside = chunk * 16 < task.depth * (Eight ? 1 : 2);
                constexpr int kElement = Eight ? 1 : 2;
#pragma unroll
                for (int r = 0; r < kWarpTokens; r += kRows) {
                    const int row = r + lane / S::kChunks;
                    const int row_page = __shfl_sync(0xffffffffu, page, row);
                    const int row_slot = __shfl_sync(0xffffffffu, slot, row);
                    const bool load = row_page >= 0 && inside;
                    const uint32_t to = base + row * S::kRowBytes + S::place(row, chunk);
                    const uint8_t *k = static_cast<const uint8_t *>(task.keys.base);
                    const uint8_t *v = static_cast<const uint8_t *>(task.values.base);
                    if (load) {
                        k += (row_page * task.keys.page_stride + row_slot * task.keys.slot_stride +
                              kv_head * task.keys.head_stride) * kElement + chunk * 16;
                        v += (row_page * task.values.page_stride + row_slot * task.values.slot_stride +
                              kv_head * task.values.head_stride) * kElement + chunk * 16;
                    }
                    copy_16(to, k, load);
                    copy_16(to + kWarpTokens * S::kRowBytes, v, load);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

#pragma unroll
        for (int s = 0; s < S::kStages - 1; ++s)
            issue(from + s);

        /* Q^T as the column operand: lane (g, t) holds head g */
        uint32_t qf[Blocks][Depth / 16][2];
        float head_scale[Blocks][2]; /* of heads 2t and 2t+1 of the block */
#pragma unroll
        for (int n = 0; n < Blocks; ++n) {
            const bool live = 8 * n + g < live_heads;
            const __nv_bfloat16 *q = task.q + sequence * task.q_batch +
                                     (live ? first_head + 8 * n + g : 0) * task.q_head;
            if constexpr (!Eight) {
#pragma unroll
                for (int kk = 0; kk < Depth / 16; ++kk)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int d = 16 * kk + 8 * i + 2 * t;
                        qf[n][kk][i] = live && d < task.depth
                                           ? *reinterpret_cast<const uint32_t *>(q + d)
                                           : 0u;
                    }
                head_scale[n][0] = head_scale[n][1] = task.score_scale;
            } else {
                /* To FP16, whose mantissa holds a BF16 but whose range does not: divided by
                 * a power of two that brings the head's largest element to [1, 2). */
                uint2 raw[Depth / 16];
                float largest = 0.f;
#pragma unroll
                for (int kk = 0; kk < Depth / 16; ++kk) {
                    const int d = 16 * kk + 4 * t;
                    raw[kk] = live && d < task.depth ? *reinterpret_cast<const uint2 *>(q + d)
                                                     : make_uint2(0, 0);
                    const heads::Piece p = heads::load_piece(
                        reinterpret_cast<const __nv_bfloat16 *>(&raw[kk]));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        largest = fmaxf(largest, fabsf(p.e[i]));
                }
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                int exponent = 0;
                if (largest > 0.f && largest < INFINITY)
                    exponent = ilogbf(largest);
                exponent = max(-126, min(126, exponent));
                const float down = exp2f(float(-exponent)), up = exp2f(float(exponent));
#pragma unroll
                for (int kk = 0; kk < Depth / 16; ++kk) {
                    const heads::Piece p = heads::load_piece(
                        reinterpret_cast<const __nv_bfloat16 *>(&raw[kk]));
                    qf[n][kk][0] = pack<true>(p.e[0] * down, p.e[1] * down);
                    qf[n][kk][1] = pack<true>(p.e[2] * down, p.e[3] * down);
                }
                /* lane (g, t) needs the factors of heads 2t and 2t+1, held by lanes 4*(2t + i) */
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    head_scale[n][i] =
                        task.score_scale * __shfl_sync(0xffffffffu, up, 4 * (2 * t + i));
            }
        }

        float o[Blocks][Depth / 16][4];
        float top[Blocks][2], sum[Blocks][2];
#pragma unroll
        for (int n = 0; n < Blocks; ++n) {
#pragma unroll
            for (int j = 0; j < Depth / 16; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[n][j][i] = 0.f;
            top[n][0] = top[n][1] = -INFINITY;
            sum[n][0] = sum[n][1] = 0.f;
        }

        for (int j = from; j < upto; ++j) {
            issue(j + S::kStages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            __syncwarp();
            const int stage = (j - from) % S::kStages;
            const uint32_t keys = ring + stage * S::kStageBytes;
            const uint32_t values = keys + kWarpTokens * S::kRowBytes;
            const uint32_t real = seen_words[stage];
            if (real) {
                float s[Blocks][4];
#pragma unroll
                for (int n = 0; n < Blocks; ++n)
                    s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int kk = 0; kk < Depth / 16; ++kk) {
                    uint32_t a[4];
                    if constexpr (!Eight) {
                        const int row = lane & 15, chunk = 2 * kk + lane / 16;
                        ldmatrix_x4(a, keys + row * S::kRowBytes + S::place(row, chunk));
                    } else {
                        /* lane (g, t) takes depths 16 kk + 4t .. + 3 of tokens g and g + 8; the
                         * query operand is in the same order */
                        const uint32_t at = S::place(g, kk) + 4 * t;
                        uint32_t low, high;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(low) : "r"(keys + g * S::kRowBytes + at));
                        asm volatile("ld.shared.u32 %0, [%1];"
                                     : "=r"(high)
                                     : "r"(keys + (g + 8) * S::kRowBytes + at));
                        a[0] = widen(low & 0xffff), a[1] = widen(high & 0xffff);
                        a[2] = widen(low >> 16), a[3] = widen(high >> 16);
                    }
#pragma unroll
                    for (int n = 0; n < Blocks; ++n)
                        mma_16816<Eight>(s[n], a, qf[n][kk][0], qf[n][kk][1]);
                }
                const bool low_real = (real >> g) & 1, high_real = (real >> (g + 8)) & 1;
                uint32_t p[Blocks][2];
                bool rescale = false;
                float factor[Blocks][2];
#pragma unroll
                for (int n = 0; n < Blocks; ++n) {
                    float weight[4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float a = low_real ? s[n][i] * head_scale[n][i] : -INFINITY;
                        const float b = high_real ? s[n][i + 2] * head_scale[n][i] : -INFINITY;
                        float best = fmaxf(a, b);
#pragma unroll
                        for (int offset = 4; offset < 32; offset *= 2)
                            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, offset));
                        best = fmaxf(best, top[n][i]);
                        const float reference = best == -INFINITY ? 0.f : best;
                        factor[n][i] = exp2f(top[n][i] - reference);
                        rescale = rescale || best != top[n][i];
                        top[n][i] = best;
                        weight[i] = exp2f(a - reference), weight[i + 2] = exp2f(b - reference);
                        sum[n][i] = sum[n][i] * factor[n][i] + weight[i] + weight[i + 2];
                    }
                    p[n][0] = transpose_8x8(pack<Eight>(weight[0], weight[1]));
                    p[n][1] = transpose_8x8(pack<Eight>(weight[2], weight[3]));
                }
                if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                    for (int n = 0; n < Blocks; ++n)
#pragma unroll
                        for (int jj = 0; jj < Depth / 16; ++jj)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                o[n][jj][i] *= factor[n][i & 1];
                }
                if constexpr (!Eight) {
#pragma unroll
                    for (int jj = 0; jj < Depth / 16; ++jj) {
                        uint32_t a[4];
                        const int row = (lane & 7) + (lane / 16) * 8, chunk = 2 * jj + ((lane / 8) & 1);
                        ldmatrix_x4_trans(a, values + row * S::kRowBytes + S::place(row, chunk));
#pragma unroll
                        for (int n = 0; n < Blocks; ++n)
                            mma_16816<false>(o[n][jj], a, p[n][0], p[n][1]);
                    }
                } else {
                    /* lane (g, t): depths 32 J + 4g + i, i = 0..3, of tokens 2t, 2t+1, 2t+8, 2t+9:
                     * row g of product 2J is depth 32 J + 4g, row g + 8 the next one, and so on */
#pragma unroll
                    for (int J = 0; J < Depth / 32; ++J) {
                        uint32_t word[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = 2 * t + (i & 1) + (i / 2) * 8;
                            const uint32_t at = values + row * S::kRowBytes +
                                                S::place(row, 2 * J + g / 4) + 4 * (g % 4);
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(word[i]) : "r"(at));
                        }
                        const uint32_t low01 = __byte_perm(word[0], word[1], 0x5140);
                        const uint32_t high01 = __byte_perm(word[0], word[1], 0x7362);
                        const uint32_t low23 = __byte_perm(word[2], word[3], 0x5140);
                        const uint32_t high23 = __byte_perm(word[2], word[3], 0x7362);
                        const uint32_t even[4] = {widen(low01 & 0xffff), widen(low01 >> 16),
                                                  widen(low23 & 0xffff), widen(low23 >> 16)};
                        const uint32_t odd[4] = {widen(high01 & 0xffff), widen(high01 >> 16),
                                                 widen(high23 & 0xffff), widen(high23 >> 16)};
#pragma unroll
                        for (int n = 0; n < Blocks; ++n) {
                            mma_16816<true>(o[n][2 * J], even, p[n][0], p[n][1]);
                            mma_16816<true>(o[n][2 * J + 1], odd, p[n][0], p[n][1]);
                        }
                    }
                }
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        /* join the four warps, then write the result or this CTA's piece of it */
#pragma unroll
        for (int n = 0; n < Blocks; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int offset = 4; offset < 32; offset *= 2)
                    sum[n][i] += __shfl_xor_sync(0xffffffffu, sum[n][i], offset);
                const int head = 8 * n + 2 * t + i;
                if (g == 0) {
                    join_stats[(warp * S::kHeads + head) * 2] = top[n][i];
                    join_stats[(warp * S::kHeads + head) * 2 + 1] = sum[n][i];
                }
                float *to = join + (warp * S::kHeads + head) * S::kJoinPitch;
#pragma unroll
                for (int jj = 0; jj < Depth / 16; ++jj) {
                    /* rows g and g + 8 of product jj */
                    const int d = Eight ? 32 * (jj / 2) + 4 * g + 2 * (jj & 1) : 16 * jj + g;
                    to[d] = o[n][jj][i];
                    to[d + (Eight ? 1 : 8)] = o[n][jj][i + 2];
                }
            }
        __syncthreads();
        const bool whole = from == 0 && upto == tiles;
        const long long piece = 2ll * blockIdx.x + (tile == begin ? 0 : 1);
        for (int at = threadIdx.x; at < live_heads * task.depth; at += kWarps * 32) {
            const int head = at / task.depth, d = at - head * task.depth;
            float best = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                best = fmaxf(best, join_stats[(w * S::kHeads + head) * 2]);
            const float reference = best == -INFINITY ? 0.f : best;
            float value = 0.f, weight = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float factor = exp2f(join_stats[(w * S::kHeads + head) * 2] - reference);
                weight += factor * join_stats[(w * S::kHeads + head) * 2 + 1];
                value += factor * join[(w * S::kHeads + head) * S::kJoinPitch + d];
            }
            if (whole) {
                const long long row = (long long)sequence * task.heads + first_head + head;
                task.out[row * task.depth + d] = __float2bfloat16_rn(
                    weight != 0.f ? value * task.value_scale / weight : 0.f);
            } else {
                task.pieces[(piece * S::kHeads + head) * task.depth + d] = value;
                if (d == 0) {
                    task.statistics[(piece * S::kHeads + head) * 2] = best;
                    task.statistics[(piece * S::kHeads + head) * 2 + 1] = weight;
                }
            }
        }
        __syncthreads();
        tile = item_first + upto;
        if (tile >= sequence_first + (long long)tiles * task.kv_heads * task.head_blocks) {
            sequence_first += (long long)tiles * task.kv_heads * task.head_blocks;
            ++sequence;
        }
    }
}

/* Adds the pieces of every item that more than one CTA worked on, in token
 * order. One CTA per item; `grid` and `slots` (heads per piece) are those of the
 * attend kernel, whose programmatic dependent this kernel is. */
__global__ void __launch_bounds__(128) attend_join(const AttendTask task, int grid, int slots)
{
    const int per = task.kv_heads * task.head_blocks;
    const int sequence = blockIdx.x / per, item = blockIdx.x % per;
    const long long total = total_tiles(task);
    long long before = 0;
    for (int b = threadIdx.x & 31; b < sequence; b += 32)
        before += tiles_of(task, b);
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2)
        before += __shfl_xor_sync(0xffffffffu, before, offset);
    const int tiles = tiles_of(task, sequence);
    const long long first = before * per + (long long)item * tiles, last = first + tiles - 1;
    /* the CTA of a tile: the last one whose range starts at or before it */
    const auto owner = [&](long long tile) {
        int low = 0, high = grid - 1;
        while (low < high) {
            const int middle = (low + high + 1) / 2;
            if (range_start(total, grid, middle) <= tile)
                low = middle;
            else
                high = middle - 1;
        }
        return low;
    };
    const int from = owner(first), upto = owner(last);
    if (from == upto)
        return; /* written whole */
    const int kv_head = item / task.head_blocks, head_block = item % task.head_blocks;
    const int first_head = kv_head * task.group + head_block * slots;
    const int live_heads = min(slots, task.group - head_block * slots);
    const int first_slot = range_start(total, grid, from) < first ? 1 : 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int at = threadIdx.x; at < live_heads * task.depth; at += blockDim.x) {
        const int head = at / task.depth, d = at - head * task.depth;
        float best = -INFINITY, weight = 0.f, value = 0.f;
        for (int cta = from; cta <= upto; ++cta) {
            if (cta != from && cta != upto && range_start(total, grid, cta) == range_start(total, grid, cta + 1))
                continue;
            const long long piece = (2ll * cta + (cta == from ? first_slot : 0)) * slots + head;
            const float top = task.statistics[piece * 2], part = task.statistics[piece * 2 + 1];
            const float higher = fmaxf(best, top);
            const float reference = higher == -INFINITY ? 0.f : higher;
            const float old = exp2f(best - reference), fresh = exp2f(top - reference);
            weight = weight * old + part * fresh;
            value = value * old + task.pieces[piece * task.depth + d] * fresh;
            best = higher;
        }
        const long long row = (long long)sequence * task.heads + first_head + head;
        task.out[row * task.depth + d] =
            __float2bfloat16_rn(weight != 0.f ? value * task.value_scale / weight : 0.f);
    }
}

/* How one call is cut: kernel instance, CTAs, workspace. */
struct Plan {
    int depth_class = 0; /* 64, 128 or 256 */
    int blocks = 1;
    int head_blocks = 1;
    long long tiles_bound = 0; /* most tiles an item can have */
    int grid = 0;
    size_t bytes = 0;
};

/* Calls work(Shape<...>) for the instance that a call uses. */
template <typename Work> auto with_shape(int depth_class, int blocks, bool eight, Work work)
{
    if (eight) {
        if (depth_class == 64)
            return blocks == 1 ? work(Shape<64, 1, true>{}) : work(Shape<64, 2, true>{});
        if (depth_class == 128)
            return blocks == 1 ? work(Shape<128, 1, true>{}) : work(Shape<128, 2, true>{});
        return work(Shape<256, 1, true>{});
    }
    if (depth_class == 64)
        return blocks == 1 ? work(Shape<64, 1, false>{}) : work(Shape<64, 2, false>{});
    if (depth_class == 128)
        return blocks == 1 ? work(Shape<128, 1, false>{}) : work(Shape<128, 2, false>{});
    return work(Shape<256, 1, false>{});
}

inline Plan make_plan(int sm_count, int batch, int heads_count, int kv_heads, int depth, int cache_type,
                      int page_size, int table_width, int window, int sinks)
{
    Plan plan;
    const int group = heads_count / kv_heads;
    plan.depth_class = depth <= 64 ? 64 : (depth <= 128 ? 128 : 256);
    /* Sixteen heads per pass where a group has more than eight: half the reads. Their result
     * does not fit the registers at 256 columns; there the second block of heads reads again. */
    plan.blocks = group > 8 && plan.depth_class <= 128 ? 2 : 1;
    plan.head_blocks = (group + 8 * plan.blocks - 1) / (8 * plan.blocks);
    long long bound = (long long)page_size * table_width;
    if (window > 0 && bound > (long long)window + sinks)
        bound = (long long)window + sinks;
    plan.tiles_bound = bound > kTile ? (bound + kTile - 1) / kTile : 1;
    const int resident = with_shape(plan.depth_class, plan.blocks, cache_type == 3,
                                    [](auto shape) { return decltype(shape)::kResident; });
    const long long most = plan.tiles_bound * batch * kv_heads * plan.head_blocks;
    const long long full = (long long)sm_count * resident;
    plan.grid = int(most < full ? most : full);
    plan.bytes = size_t(plan.grid) * 2 * 8 * plan.blocks * (size_t(depth) + 2) * 4;
    return plan;
}

template <int Depth, int Blocks, bool Eight>
void launch(camblas_cuda_context *context, const AttendTask &task, const Plan &plan, Shape<Depth, Blocks, Eight>)
{
    attend_kernel<Depth, Blocks, Eight>
        <<<plan.grid, kWarps * 32, Shape<Depth, Blocks, Eight>::kBytes, context->stream>>>(task);
}

template <int Depth, int Blocks, bool Eight> int allow_shared(Shape<Depth, Blocks, Eight>)
{
    return int(cudaFuncSetAttribute(attend_kernel<Depth, Blocks, Eight>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Shape<Depth, Blocks, Eight>::kBytes));
}

/* Raises the shared-memory limit of every instance on the current device. */
inline int prepare_kernels()
{
    int status = 0;
    for (int eight = 0; eight < 2; ++eight)
        for (int depth_class = 64; depth_class <= 256; depth_class *= 2)
            for (int blocks = 1; blocks <= (depth_class < 256 ? 2 : 1); ++blocks)
                status |= with_shape(depth_class, blocks, eight != 0,
                                     [](auto shape) { return allow_shared(shape); });
    return status;
}

inline bool sizes_bad(int batch, int heads_count, int kv_heads, int depth, int cache_type, int page_size,
                      int table_width, int window, int sinks)
{
    return batch < 0 || kv_heads < 1 || heads_count < 1 || heads_count > 65536 || heads_count % kv_heads ||
           depth < 8 || depth > 256 || (cache_type != 2 && cache_type != 3) ||
           depth % (cache_type == 3 ? 16 : 8) || page_size < 1 || table_width < 0 || window < 0 || sinks < 0 ||
           (long long)batch * heads_count > INT_MAX;
}

} // namespace attend

extern "C" size_t camblas_cuda_paged_attention_workspace(const camblas_cuda_context *context, int batch,
                                                         int heads_count, int kv_heads, int depth,
                                                         int cache_type, int page_size, int table_width,
                                                         int window, int sinks)
{
    if (!context || batch == 0 ||
        attend::sizes_bad(batch, heads_count, kv_heads, depth, cache_type, page_size, table_width, window, sinks))
        return 0;
    return attend::make_plan(context->sm_count, batch, heads_count, kv_heads, depth, cache_type, page_size,
                             table_width, window, sinks)
        .bytes;
}

extern "C" int camblas_cuda_paged_attention(
    camblas_cuda_context *context, int batch, int heads_count, int kv_heads, int depth, float scale,
    const void *q, int cache_type, const void *key_cache, const void *value_cache,
    const long long *strides, int pages, int page_size, float key_scale, float value_scale,
    const void *table, int table_width, const void *lengths, int window, int sinks, void *workspace,
    size_t workspace_bytes, void *output)
{
    return host::guarded(context, [&] {
        if (attend::sizes_bad(batch, heads_count, kv_heads, depth, cache_type, page_size, table_width, window,
                              sinks) ||
            pages < 0 || !std::isfinite(scale) || !std::isfinite(key_scale) || !std::isfinite(value_scale))
            return host::fail(context, "invalid paged attention dimensions", 1);
        if (batch == 0)
            return 0;
        const int element = cache_type == 3 ? 1 : 2;
        attend::AttendTask task{};
        bool bad = !q || !strides || !lengths || !output ||
                   (table_width > 0 && !table) || (pages > 0 && (!key_cache || !value_cache));
        bad = bad || heads::misaligned(q, 8) || heads::misaligned(table, 4) || heads::misaligned(lengths, 4) ||
              heads::misaligned(output, 2) || q == output || key_cache == output || value_cache == output;
        if (!bad) {
            task.keys = {const_cast<void *>(key_cache), strides[2], strides[3], strides[4]};
            task.values = {const_cast<void *>(value_cache), strides[5], strides[6], strides[7]};
            bad = strides[0] % 4 || strides[1] % 4 || (batch > 1 && strides[8] < 0) ||
                  (pages > 0 && (heads::cache_bad(task.keys, element, 16) ||
                                 heads::cache_bad(task.values, element, 16)));
        }
        if (bad)
            return host::fail(context, "invalid paged attention operands", 1);
        const attend::Plan plan = attend::make_plan(context->sm_count, batch, heads_count, kv_heads, depth,
                                                    cache_type, page_size, table_width, window, sinks);
        if (workspace_bytes < plan.bytes || !workspace || heads::misaligned(workspace, 16))
            return host::fail(context, "paged attention workspace too small", 1);
        task.batch = batch, task.heads = heads_count, task.kv_heads = kv_heads;
        task.group = heads_count / kv_heads, task.head_blocks = plan.head_blocks, task.depth = depth;
        task.page_size = page_size, task.pages = pages, task.table_width = table_width;
        task.page_shift = -1;
        for (int shift = 0; shift < 31; ++shift)
            if (page_size == 1 << shift)
                task.page_shift = shift;
        task.window = window, task.sinks = sinks;
        task.q = static_cast<const __nv_bfloat16 *>(q);
        task.q_batch = strides[0], task.q_head = strides[1];
        task.table = static_cast<const int32_t *>(table), task.table_row = strides[8];
        task.lengths = static_cast<const int32_t *>(lengths);
        task.score_scale = scale * key_scale * 1.4426950408889634f;
        task.value_scale = value_scale;
        task.out = static_cast<__nv_bfloat16 *>(output);
        task.pieces = static_cast<float *>(workspace);
        task.statistics = task.pieces + size_t(plan.grid) * 2 * 8 * plan.blocks * depth;
        context->counts[6]++;
        attend::with_shape(plan.depth_class, plan.blocks, cache_type == 3, [&](auto shape) {
            attend::launch(context, task, plan, shape);
            return 0;
        });
        const int status = host::launched(context, "paged attention");
        if (status != 0 || plan.tiles_bound == 1)
            return status;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(unsigned(batch) * kv_heads * plan.head_blocks);
        config.blockDim = dim3(128);
        config.stream = context->stream;
        cudaLaunchAttribute attribute[1];
        attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attribute[0].val.programmaticStreamSerializationAllowed = 1;
        config.attrs = attribute;
        config.numAttrs = 1;
        const cudaError_t error = cudaLaunchKernelEx(&config, attend::attend_join, task, plan.grid, 8 * plan.blocks);
        if (error != cudaSuccess)
            return host::fail(context, "paged attention join", error);
        context->kernel_launches.fetch_add(1, std::memory_order_relaxed);
        return 0;
    });
}
