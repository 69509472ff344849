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
 * tensor cores because eight heads per key on CUDA cores would not keep up. A
 * warp's tile is 16, 32 or 64 tokens, 8 KB (16 KB at 256 BF16 columns): S^T[16
 * tokens, 8 heads] = K Q^T and O^T[depth, 8 heads] += V^T P^T with mma.m16n8k16.
 * Tokens (and depth) take the 16-row side, so that a group of up to eight heads
 * fills the 8-column side, and the softmax statistics of a head sit on the lanes
 * that hold the head's column in both products. P^T turns from the accumulator's
 * to the operand's layout by movmatrix, without shared memory. (tcgen05 would
 * want 128 rows of M and bring nothing to a kernel that waits for HBM; mma.sync
 * does a product in 8 cycles per sub-core here, the 24 of 16 tokens of 128 columns
 * in a seventh of the time that HBM gives.) Scores, statistics, sums and the joined result are FP32; P goes to the
 * value product in two parts, of BF16 the upper half and what that leaves, rounded
 * (over an 8-bit cache FP16, both rounded): at most 2^-16 (2^-22) of each weight is
 * lost. In one part the 2^-8 (2^-11) of each weight made the result's error against
 * 64 bits 3 to 13 % larger than its last rounding alone. FP16 keeps its bits only
 * down to 2^-14, and a result can be made of weights far below the largest (a first
 * token that takes the weight and has next to no value), so over an 8-bit cache P is
 * 2^15 times the weights, and what lies below 2^-40 of the largest is lost.
 *
 * Measured, 64 query and 8 key heads of 128 in BF16: one sequence of 130977
 * tokens 98 us (0.83 of the measured copy rate), 48 sequences of 0 to 8191 tokens
 * 60 us (0.61; some 5 us are the way from the lengths to the first keys, and 11
 * the join), one of 300 tokens 9.6 us. Over an 8-bit cache widening to FP16 and the
 * products of the weights' second part show: 69 and 50 us, 0.59 and 0.37.
 *
 * Work split. A warp works alone. The slots of a sequence (key heads times
 * blocks of 8 or 16 query heads) are taken in teams of four neighbours, two or
 * one, whichever divides their number, one warp each, so that the warps of a
 * team read neighbouring heads of the same tokens at the same time: the rows
 * they fetch lie side by side in a page. The tiles of all (sequence, team)
 * items are laid end to end and cut into equal contiguous ranges, one per team
 * of warps of the grid, so ragged lengths load every SM alike. Every warp finds
 * its range from the lengths on the device: no plan on the host, and a captured
 * call follows the lengths of the replay. An item that one range covers whole is
 * written at once; a piece of an item leaves maximum, sum and unscaled result
 * in the workspace (at most two pieces per warp, its first and its last), and
 * attend_join adds the pieces of an item in token order. No atomics: the same
 * call gives the same bits.
 *
 * A warp copies its tiles into its own shared-memory ring with cp.async, the
 * page numbers one tile further ahead, running on into the next item while the
 * present one is summed; there is no barrier in the kernel. Tokens that are not
 * visible are filled with zeros instead of being read: a weight of zero times a
 * NaN would be NaN.
 */
#pragma once

#include "context.cuh"
#include "head_rotate.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace attend
{

constexpr int kWarps = 4; /* of a CTA */
constexpr float kRaised = 0x1p15f; /* the largest weight in FP16 */

struct AttendTask {
    int batch, heads, group, depth;      /* group: query heads per key head */
    int head_blocks, team, teams;        /* slots = kv_heads * head_blocks = team * teams */
    int page_size, page_shift, pages; /* page_shift < 0: not a power of two */
    int room;                         /* tokens that a row of the table can hold */
    int window, sinks;
    int tile_shift; /* log2 of the tokens of a tile */
    int workers; /* teams of warps in the grid */
    long long q_batch, q_head, table_row;
    const __nv_bfloat16 *q;
    heads::CacheLayout keys, values; /* strides in bytes */
    const int32_t *table, *lengths;
    float score_scale; /* scale * key scale * log2(e) */
    float value_scale; /* over an 8-bit cache divided by kRaised */
    __nv_bfloat16 *out;    /* [batch, heads, depth] contiguous */
    long long *first_tile; /* [batch + 1]: number of the first tile of a sequence, then the total */
    float4 *pieces;        /* [2 * warps][column block][depth class / 16][32 lanes] */
    float2 *statistics;    /* [2 * warps][column block][8 heads]: maximum, sum */
};

/* The visible tokens of one sequence: `seen` of them, numbered from 0; number v
 * is token v, or v + jump from number jump_at on. */
struct Visible {
    int seen, jump_at, jump, tiles;
};

__device__ __forceinline__ Visible visible(const AttendTask &task, int length)
{
    length = max(0, min(length, task.room));
    Visible v{length, 0, 0, 1};
    if (task.window > 0 && length > task.window) {
        const int rest = length - task.window;
        v.jump_at = task.sinks < rest ? task.sinks : rest;
        v.seen = task.window + v.jump_at;
        v.jump = length - v.seen;
    }
    /* an empty sequence keeps a tile so that its zeros get written */
    v.tiles = v.seen ? ((v.seen - 1) >> task.tile_shift) + 1 : 1;
    return v;
}

/* Quotient of numbers that are not negative: the 64-bit division, some hundred instructions, only
 * where it is needed. */
__device__ __forceinline__ long long divide(long long a, long long b)
{
    return (a | b) >> 32 ? a / b : (long long)(unsigned(a) / unsigned(b));
}

/* The range of tiles of a worker: `total` in equal parts, the first ones a tile longer. */
struct Cut {
    long long each;
    long long longer; /* workers with one tile more */

    __device__ __forceinline__ Cut(long long total, int workers)
    {
        each = divide(total, workers), longer = total - each * workers;
    }
    __device__ __forceinline__ long long start(int worker) const
    {
        return each * worker + (worker < longer ? worker : longer);
    }
    __device__ __forceinline__ int owner(long long tile) const
    {
        const long long in_longer = longer * (each + 1);
        return int(tile < in_longer ? divide(tile, each + 1) : longer + divide(tile - in_longer, each));
    }
};

/* Called by whole warps: inclusive prefix sum over the lanes. */
__device__ __forceinline__ long long running_sum(long long mine)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int offset = 1; offset < 32; offset *= 2) {
        const long long other = __shfl_up_sync(0xffffffffu, mine, offset);
        if (lane >= offset)
            mine += other;
    }
    return mine;
}

/* Called by whole warps. Tiles of all items; the first warp of the grid leaves
 * the first tile of every sequence for attend_join. */
__device__ __forceinline__ long long count_tiles(const AttendTask &task, bool keep)
{
    const int lane = threadIdx.x & 31;
    if (!keep) {
        long long sum = 0;
        for (int b = lane; b < task.batch; b += 32)
            sum += visible(task, task.lengths[b]).tiles;
#pragma unroll
        for (int offset = 16; offset > 0; offset /= 2)
            sum += __shfl_xor_sync(0xffffffffu, sum, offset);
        return sum * task.teams;
    }
    long long before = 0;
    for (int base = 0; base < task.batch; base += 32) {
        const bool live = base + lane < task.batch;
        const long long mine =
            live ? (long long)task.teams * visible(task, task.lengths[base + lane]).tiles : 0;
        const long long upto = running_sum(mine);
        if (live)
            task.first_tile[base + lane] = before + upto - mine;
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0)
        task.first_tile[task.batch] = before;
    return before;
}

/* Called by whole warps. The sequence that holds tile number `tile` of the whole
 * list, and the number of the sequence's first tile. */
__device__ __forceinline__ void locate(const AttendTask &task, long long tile, int &sequence,
                                       long long &first)
{
    const int lane = threadIdx.x & 31;
    long long before = 0;
    for (int base = 0; base < task.batch; base += 32) {
        const bool live = base + lane < task.batch;
        const long long mine =
            live ? (long long)task.teams * visible(task, task.lengths[base + lane]).tiles : 0;
        const long long upto = running_sum(mine);
        const unsigned past = __ballot_sync(0xffffffffu, live && before + upto > tile);
        if (past) {
            const int at = __ffs(past) - 1;
            sequence = base + at;
            first = before + __shfl_sync(0xffffffffu, upto - mine, at);
            return;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    sequence = task.batch - 1, first = before; /* not reached: tile is below the total */
}

/* A place in a worker's range, for the warp that is number `member` of its team. */
struct Cursor {
    int sequence, team, tile;
    int kv_head, head_block;
    Visible view;

    __device__ __forceinline__ void enter(const AttendTask &task, int b, int member)
    {
        sequence = b;
        if (b < task.batch)
            view = visible(task, task.lengths[b]);
        choose(task, 0, member);
    }
    __device__ __forceinline__ void choose(const AttendTask &task, int of_teams, int member)
    {
        team = of_teams;
        const int slot = team * task.team + member;
        kv_head = task.head_blocks == 1 ? slot : slot / task.head_blocks;
        head_block = slot - kv_head * task.head_blocks;
    }
    __device__ __forceinline__ void advance(const AttendTask &task, int member)
    {
        if (++tile < view.tiles)
            return;
        tile = 0;
        if (team + 1 < task.teams)
            choose(task, team + 1, member);
        else
            enter(task, sequence + 1, member);
    }
};

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

/* Two weights as the sums of two 16-bit parts each. A BF16 value may be infinite, and its weight's parts
 * have to be positive then: the first part is cut off, not rounded, and the rest is 2^-24 of the weight at
 * least. (E4M3 has no infinities.) */
struct Parts {
    uint32_t first, rest;
};

template <bool Half> __device__ __forceinline__ Parts in_parts(float low, float high)
{
    if constexpr (Half) {
        const uint32_t first = pack<true>(low, high);
        const float2 taken = __half22float2(*reinterpret_cast<const __half2 *>(&first));
        return {first, pack<true>(low - taken.x, high - taken.y)};
    } else {
        const float low_rest = low - __uint_as_float(__float_as_uint(low) & 0xffff0000u);
        const float high_rest = high - __uint_as_float(__float_as_uint(high) & 0xffff0000u);
        return {__byte_perm(__float_as_uint(low), __float_as_uint(high), 0x7632),
                pack<false>(fmaxf(low_rest, low * 0x1p-24f), fmaxf(high_rest, high * 0x1p-24f))};
    }
}

/* 2^x; 0 for -infinity */
__device__ __forceinline__ float power_of_two(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* The exponent of the power of two that is divided out of BF16 numbers, the largest of which is
 * `largest`, to bring that to [2^14, 2^15), the top of FP16's range; 0 for zero and for what is not
 * finite. Both 2^exponent and 2^-exponent are normal numbers. */
__device__ __forceinline__ int half_exponent(float largest)
{
    if (!(largest > 0.f && largest < INFINITY))
        return 0;
    return max(-126, (__float_as_int(largest) >> 23) - 127 - 14);
}

/* two E4M3 values (exact in FP16), the lower byte in the lower half */
__device__ __forceinline__ uint32_t widen(uint32_t two_bytes)
{
    const __half2_raw pair =
        __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two_bytes), __NV_E4M3);
    return uint32_t(pair.x) | (uint32_t(pair.y) << 16);
}

/* ---- the kernels ---- */

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
    static constexpr int kPieces = Depth / 16; /* 16-row products along the depth */
    /* Tokens of a tile: 8 KB of keys and values where rows are short, so that what a tile costs
     * beside its products (page numbers, maxima across lanes) is spread over as many bytes. */
    static constexpr int kTile = kRowBytes >= 256 ? 16 : (kRowBytes == 128 ? 32 : 64);
    static constexpr int kGroups = kTile / 16; /* of 16 tokens */
    static constexpr int kTileShift = kTile == 16 ? 4 : (kTile == 32 ? 5 : 6);
    static constexpr int kTileBytes = 2 * kTile * kRowBytes; /* keys and values */
    /* The copies in flight on an SM have to cover the latency of HBM at its share of the bandwidth,
     * some 45 KB. Two stages do, and let more warps share the SM (48 ragged sequences of 128 BF16
     * columns: 60 us, three stages 64), unless registers keep the third CTA away or make it spill:
     * sixteen heads at 128 BF16 columns (eight sequences, one key head: 28.5 us with three, 34.4 with
     * two). At 256 BF16 columns three are within 5 % of two (sixteen sequences: 31.5 and 29.9). */
    static constexpr int kStages = kRowBytes >= 512 || (kRowBytes == 256 && Blocks == 2) ? 3 : 2;
    static constexpr int kNoteBytes = 16 * kTile + 16; /* where the rows of a stage lie, which are real */
    static constexpr int kWarpBytes = kStages * (kTileBytes + kNoteBytes);
    static constexpr int kBytes = kWarps * kWarpBytes;
    /* CTAs on an SM: shared memory is 228 KB, of which each CTA takes 1 KB more than it asks for */
    static constexpr int kResident = 228 * 1024 / (kBytes + 1024);
    static_assert(kResident >= 1 && kResident <= 4, "registers");
};

/* Result of 16 depths and 8 heads, `o` in the accumulator layout (rows g and
 * g + 8, heads 2t and 2t + 1), times factor[head]: BF16 rows of the heads at
 * `out`, of which `live` exist. */
template <bool Eight>
__device__ __forceinline__ void store_heads(__nv_bfloat16 *out, int depth, int live, int piece,
                                            const float (&o)[4], const float (&factor)[2])
{
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
    const uint32_t low = transpose_8x8(pack<false>(o[0] * factor[0], o[1] * factor[1]));
    const uint32_t high = transpose_8x8(pack<false>(o[2] * factor[0], o[3] * factor[1]));
    /* now head g, rows 2t and 2t + 1 of the lower and of the upper half */
    if (g >= live)
        return;
    uint32_t *row = reinterpret_cast<uint32_t *>(out + (long long)g * depth);
    if constexpr (Eight) { /* see the value product of attend_kernel */
        const int d = 32 * (piece / 2) + 8 * t + 2 * (piece & 1);
        if (d < depth) {
            row[d / 2] = __byte_perm(low, high, 0x5410);
            row[d / 2 + 2] = __byte_perm(low, high, 0x7632);
        }
    } else {
        const int d = 16 * piece + 2 * t;
        if (d < depth)
            row[d / 2] = low;
        if (d + 8 < depth)
            row[d / 2 + 4] = high;
    }
}

template <int Depth, int Blocks, bool Eight>
__global__ void __launch_bounds__(kWarps * 32, Shape<Depth, Blocks, Eight>::kResident)
    attend_kernel(const __grid_constant__ AttendTask task)
{
    using S = Shape<Depth, Blocks, Eight>;
    extern __shared__ __align__(128) uint8_t shared[];

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int g = lane / 4, t = lane % 4;
    const int global_warp = blockIdx.x * kWarps + warp;
    const int worker = global_warp / task.team, member = global_warp % task.team;
    /* the ring of this warp, then the notes of its stages: byte offsets of keys and values of the
     * rows, and the mask of the real ones */
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(shared)) + warp * S::kStages * S::kTileBytes;
    uint8_t *notes = shared + kWarps * S::kStages * S::kTileBytes + warp * S::kStages * S::kNoteBytes;

    const long long total = count_tiles(task, global_warp == 0);
    const Cut cut(total, task.workers);
    const long long begin = cut.start(worker);
    if (worker >= task.workers || begin >= total)
        return;
    const int count = int(min(cut.start(worker + 1), total) - begin);
    Cursor use;
    {
        long long first;
        int sequence;
        locate(task, begin, sequence, first);
        use.enter(task, sequence, member);
        const int item = int(divide(begin - first, use.view.tiles));
        use.choose(task, item, member);
        use.tile = int(begin - first - (long long)item * use.view.tiles);
    }
    Cursor ahead = use; /* the tile whose page numbers are fetched next */
    int fetched = 0;
    constexpr int kOwn = (S::kTile + 31) / 32; /* rows of a tile that a lane looks up: lane, lane + 32 */
    int page[kOwn], place_in_page[kOwn], page_head = 0; /* of the tile that is copied next */

    const auto fetch = [&] {
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            page[i] = -1;
        if (fetched < count) {
            page_head = ahead.kv_head;
            const int32_t *row = task.table + ahead.sequence * task.table_row;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                int v = ahead.tile * S::kTile + 32 * i + lane;
                if ((S::kTile >= 32 || lane < S::kTile) && v < ahead.view.seen) {
                    v += v >= ahead.view.jump_at ? ahead.view.jump : 0;
                    const int number = task.page_shift >= 0 ? v >> task.page_shift : v / task.page_size;
                    place_in_page[i] = v - number * task.page_size;
                    page[i] = row[number];
                }
            }
            ahead.advance(task, member);
        }
        ++fetched;
    };
    const int chunk = lane % S::kChunks, sub = lane / S::kChunks;
    const bool inside = chunk * 16 < task.depth * (Eight ? 1 : 2);
    const uint8_t *const key_base = static_cast<const uint8_t *>(task.keys.base) + chunk * 16;
    const uint8_t *const value_base = static_cast<const uint8_t *>(task.values.base) + chunk * 16;
    const auto copy = [&](int stage) {
        uint8_t *note = notes + stage * S::kNoteBytes;
        uint32_t real[kOwn], any = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const bool real_row = unsigned(page[i]) < unsigned(task.pages);
            real[i] = __ballot_sync(0xffffffffu, real_row);
            any |= real[i];
            if (S::kTile >= 32 || lane < S::kTile) {
                longlong2 at = make_longlong2(0, 0);
                if (real_row) {
                    at.x = page[i] * task.keys.page_stride + place_in_page[i] * task.keys.slot_stride +
                           page_head * task.keys.head_stride;
                    at.y = page[i] * task.values.page_stride + place_in_page[i] * task.values.slot_stride +
                           page_head * task.values.head_stride;
                }
                reinterpret_cast<longlong2 *>(note)[32 * i + lane] = at;
            }
            if (lane == 0)
                reinterpret_cast<uint32_t *>(note + 16 * S::kTile)[i] = real[i];
        }
        __syncwarp();
        if (any) {
            constexpr int kRows = 32 / S::kChunks; /* rows the warp copies at once */
            const uint32_t base = ring + stage * S::kTileBytes + sub * S::kRowBytes;
#pragma unroll
            for (int r = 0; r < S::kTile; r += kRows) {
                const longlong2 at = reinterpret_cast<const longlong2 *>(note)[r + sub];
                const bool load = inside && (real[r / 32] >> (r % 32 + sub)) & 1;
                const uint32_t to = base + r * S::kRowBytes + S::place(r + sub, chunk);
                copy_16(to, key_base + at.x, load);
                copy_16(to + S::kTile * S::kRowBytes, value_base + at.y, load);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        fetch();
    };
    fetch();
#pragma unroll
    for (int s = 0; s < S::kStages - 1; ++s)
        copy(s);

    uint32_t qf[Blocks][S::kPieces][2]; /* Q^T as the column operand: lane (g, t) holds head g */
    float head_scale[Blocks][2];        /* of heads 2t and 2t+1 of the block */
    float o[Blocks][S::kPieces][4];
    float top[Blocks][2], sum[Blocks][2];
    bool entered = false, at_first = true;
    int from = 0, stage = 0, first_head = 0, live_heads = 0;
    for (int done = 0; done < count; ++done) {
        if (!entered) { /* a new item */
            entered = true, from = use.tile;
            first_head = use.kv_head * task.group + use.head_block * 8 * Blocks;
            live_heads = task.group - use.head_block * 8 * Blocks;
#pragma unroll
            for (int n = 0; n < Blocks; ++n) {
                const bool live = 8 * n + g < live_heads;
                const __nv_bfloat16 *q = task.q + use.sequence * task.q_batch +
                                         (live ? first_head + 8 * n + g : 0) * task.q_head;
                if constexpr (!Eight) {
#pragma unroll
                    for (int kk = 0; kk < S::kPieces; ++kk)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int d = 16 * kk + 8 * i + 2 * t;
                            qf[n][kk][i] =
                                live && d < task.depth ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
                        }
                    head_scale[n][0] = head_scale[n][1] = task.score_scale;
                } else {
                    /* To FP16, whose mantissa holds a BF16 but whose range does not: divided by a
                     * power of two of the head's largest element. */
                    uint2 raw[S::kPieces];
                    float largest = 0.f;
#pragma unroll
                    for (int kk = 0; kk < S::kPieces; ++kk) {
                        const int d = 16 * kk + 4 * t;
                        raw[kk] = live && d < task.depth ? *reinterpret_cast<const uint2 *>(q + d)
                                                         : make_uint2(0, 0);
                        const heads::Piece p = heads::unpack_piece(raw[kk]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            largest = fmaxf(largest, fabsf(p.e[i]));
                    }
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                    const int exponent = half_exponent(largest);
                    const float down = __int_as_float((127 - exponent) << 23);
                    const float up = __int_as_float((127 + exponent) << 23);
#pragma unroll
                    for (int kk = 0; kk < S::kPieces; ++kk) {
                        const heads::Piece p = heads::unpack_piece(raw[kk]);
                        qf[n][kk][0] = pack<true>(p.e[0] * down, p.e[1] * down);
                        qf[n][kk][1] = pack<true>(p.e[2] * down, p.e[3] * down);
                    }
                    /* lane (g, t) needs the factors of heads 2t and 2t+1, held by lanes 4*(2t + i) */
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        head_scale[n][i] = task.score_scale * __shfl_sync(0xffffffffu, up, 4 * (2 * t + i));
                }
#pragma unroll
                for (int j = 0; j < S::kPieces; ++j)
                    o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
                top[n][0] = top[n][1] = -INFINITY;
                sum[n][0] = sum[n][1] = 0.f;
            }
        }

        copy(stage == 0 ? S::kStages - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
        __syncwarp();
        const uint32_t keys = ring + stage * S::kTileBytes;
        const uint32_t values = keys + S::kTile * S::kRowBytes;
        uint32_t real[kOwn], any = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            real[i] = reinterpret_cast<const uint32_t *>(notes + stage * S::kNoteBytes + 16 * S::kTile)[i];
            any |= real[i];
        }
        if (any) {
            /* scores of tokens 16m + g and 16m + g + 8; a single group has two chains of products,
             * added afterwards */
            constexpr int kChains = S::kGroups == 1 ? 2 : 1;
            float s[Blocks][S::kGroups][kChains][4];
#pragma unroll
            for (int n = 0; n < Blocks; ++n)
#pragma unroll
                for (int m = 0; m < S::kGroups; ++m)
#pragma unroll
                    for (int c = 0; c < kChains; ++c)
                        s[n][m][c][0] = s[n][m][c][1] = s[n][m][c][2] = s[n][m][c][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < S::kPieces; ++kk)
#pragma unroll
                for (int m = 0; m < S::kGroups; ++m) {
                    uint32_t a[4];
                    if constexpr (!Eight) {
                        const int row = 16 * m + (lane & 15), part = 2 * kk + lane / 16;
                        ldmatrix_x4(a, keys + row * S::kRowBytes + S::place(row, part));
                    } else {
                        /* lane (g, t) takes depths 16 kk + 4t .. + 3 of tokens g and g + 8; the
                         * query operand is in the same order */
                        const uint32_t at = keys + (16 * m + g) * S::kRowBytes + S::place(g, kk) + 4 * t;
                        uint32_t low, high;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(low) : "r"(at));
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(high) : "r"(at + 8 * S::kRowBytes));
                        a[0] = widen(low & 0xffff), a[1] = widen(high & 0xffff);
                        a[2] = widen(low >> 16), a[3] = widen(high >> 16);
                    }
#pragma unroll
                    for (int n = 0; n < Blocks; ++n)
                        mma_16816<Eight>(s[n][m][kk % kChains], a, qf[n][kk][0], qf[n][kk][1]);
                }
            uint32_t p[Blocks][S::kGroups][2], rest[Blocks][S::kGroups][2];
            bool rescale = false;
            float factor[Blocks][2];
#pragma unroll
            for (int n = 0; n < Blocks; ++n) {
                float score[S::kGroups][4], best[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int m = 0; m < S::kGroups; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float value = s[n][m][0][i];
                        if constexpr (kChains == 2)
                            value += s[n][m][1][i];
                        const bool seen = (real[m / 2] >> (16 * (m % 2) + g + 8 * (i / 2))) & 1;
                        score[m][i] = seen ? value * head_scale[n][i & 1] : -INFINITY;
                        best[i & 1] = fmaxf(best[i & 1], score[m][i]);
                    }
                float reference[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int offset = 4; offset < 32; offset *= 2)
                        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], offset));
                    best[i] = fmaxf(best[i], top[n][i]);
                    reference[i] = best[i] == -INFINITY ? 0.f : best[i];
                    factor[n][i] = power_of_two(top[n][i] - reference[i]);
                    rescale = rescale || best[i] != top[n][i];
                    top[n][i] = best[i];
                    sum[n][i] *= factor[n][i];
                }
#pragma unroll
                for (int m = 0; m < S::kGroups; ++m) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        score[m][i] = power_of_two(score[m][i] - reference[i & 1]);
                        sum[n][i & 1] += score[m][i];
                    }
                    constexpr float kFactor = Eight ? kRaised : 1.f;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const Parts parts =
                            in_parts<Eight>(score[m][2 * i] * kFactor, score[m][2 * i + 1] * kFactor);
                        p[n][m][i] = transpose_8x8(parts.first), rest[n][m][i] = transpose_8x8(parts.rest);
                    }
                }
            }
            if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (int n = 0; n < Blocks; ++n)
#pragma unroll
                    for (int j = 0; j < S::kPieces; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            o[n][j][i] *= factor[n][i & 1];
            }
#pragma unroll
            for (int m = 0; m < S::kGroups; ++m) {
                if constexpr (!Eight) {
#pragma unroll
                    for (int j = 0; j < S::kPieces; ++j) {
                        uint32_t a[4];
                        const int row = 16 * m + (lane & 7) + (lane / 16) * 8, part = 2 * j + ((lane / 8) & 1);
                        ldmatrix_x4_trans(a, values + row * S::kRowBytes + S::place(row, part));
#pragma unroll
                        for (int n = 0; n < Blocks; ++n) {
                            mma_16816<false>(o[n][j], a, p[n][m][0], p[n][m][1]);
                            mma_16816<false>(o[n][j], a, rest[n][m][0], rest[n][m][1]);
                        }
                    }
                } else {
                    /* lane (g, t): depths 32 J + 4g + i, i = 0..3, of tokens 2t, 2t+1, 2t+8, 2t+9:
                     * row g of product 2J is depth 32 J + 4g, row g + 8 the next one, and so on */
#pragma unroll
                    for (int J = 0; J < S::kPieces / 2; ++J) {
                        uint32_t word[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = 16 * m + 2 * t + (i & 1) + (i / 2) * 8;
                            const uint32_t at =
                                values + row * S::kRowBytes + S::place(row, 2 * J + g / 4) + 4 * (g % 4);
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(word[i]) : "r"(at));
                        }
                        const uint32_t low01 = __byte_perm(word[0], word[1], 0x5140);
                        const uint32_t high01 = __byte_perm(word[0], word[1], 0x7362);
                        const uint32_t low23 = __byte_perm(word[2], word[3], 0x5140);
                        const uint32_t high23 = __byte_perm(word[2], word[3], 0x7362);
                        const uint32_t even[4] = {widen(low01 & 0xffff), widen(low01 >> 16), widen(low23 & 0xffff),
                                                  widen(low23 >> 16)};
                        const uint32_t odd[4] = {widen(high01 & 0xffff), widen(high01 >> 16), widen(high23 & 0xffff),
                                                 widen(high23 >> 16)};
#pragma unroll
                        for (int n = 0; n < Blocks; ++n) {
                            mma_16816<true>(o[n][2 * J], even, p[n][m][0], p[n][m][1]);
                            mma_16816<true>(o[n][2 * J + 1], odd, p[n][m][0], p[n][m][1]);
                            mma_16816<true>(o[n][2 * J], even, rest[n][m][0], rest[n][m][1]);
                            mma_16816<true>(o[n][2 * J + 1], odd, rest[n][m][0], rest[n][m][1]);
                        }
                    }
                }
            }
        }
        __syncwarp(); /* all lanes are done with the stage that the next copy fills */
        stage = stage + 1 == S::kStages ? 0 : stage + 1;

        const bool item_ends = use.tile + 1 == use.view.tiles;
        if (item_ends || done + 1 == count) {
            const bool whole = item_ends && from == 0;
            const long long piece = 2ll * global_warp + (at_first ? 0 : 1);
#pragma unroll
            for (int n = 0; n < Blocks; ++n) {
                float inverse[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int offset = 4; offset < 32; offset *= 2)
                        sum[n][i] += __shfl_xor_sync(0xffffffffu, sum[n][i], offset);
                    inverse[i] = sum[n][i] != 0.f ? task.value_scale / sum[n][i] : 0.f;
                    if (!whole && g == 0)
                        task.statistics[(piece * Blocks + n) * 8 + 2 * t + i] = make_float2(top[n][i], sum[n][i]);
                }
                __nv_bfloat16 *out =
                    task.out + ((long long)use.sequence * task.heads + first_head + 8 * n) * task.depth;
#pragma unroll
                for (int j = 0; j < S::kPieces; ++j) {
                    if (whole)
                        store_heads<Eight>(out, task.depth, live_heads - 8 * n, j, o[n][j], inverse);
                    else
                        task.pieces[((piece * Blocks + n) * S::kPieces + j) * 32 + lane] =
                            make_float4(o[n][j][0], o[n][j][1], o[n][j][2], o[n][j][3]);
                }
            }
            entered = false, at_first = false;
        }
        use.advance(task, member);
    }
}

/* Adds the pieces of an item that more than one worker took part in, in token
 * order; a programmatic dependent of attend_kernel. blockIdx.x: item and column
 * block. A warp adds `Products` 16-depth products; `parts` warps each take a
 * contiguous share of the pieces, `AtOnce` in flight, and their sums are added
 * through shared memory. The products that do not fit a CTA are blockIdx.y's. */
constexpr int kJoinWarps = 16; /* at most */

template <bool Eight, int Products, int AtOnce>
__global__ void __launch_bounds__(kJoinWarps * 32)
    attend_join(const __grid_constant__ AttendTask task, int blocks, int depth_pieces, int parts)
{
    __shared__ float4 shared_sum[kJoinWarps][Products][32];
    __shared__ float shared_stats[kJoinWarps][2][8];
    const int warp = threadIdx.x / 32, part = warp % parts;
    const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n = blockIdx.x % blocks, item = blockIdx.x / blocks;
    const int product = (blockIdx.y * (blockDim.x / 32 / parts) + warp / parts) * Products;
    const int slots = task.team * task.teams;
    const int sequence = item / slots, slot = item % slots;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long sequence_first = __ldcg(&task.first_tile[sequence]);
    const long long sequence_end = __ldcg(&task.first_tile[sequence + 1]);
    const Cut cut(__ldcg(&task.first_tile[task.batch]), task.workers);
    const int tiles = int(divide(sequence_end - sequence_first, task.teams));
    const long long first = sequence_first + (long long)(slot / task.team) * tiles;
    const int from = cut.owner(first), upto = cut.owner(first + tiles - 1);
    if (from == upto)
        return; /* written whole */
    const int member = slot % task.team;
    const int first_place = cut.start(from) < first ? 1 : 0;
    const int share = (upto - from + parts) / parts;
    const int begin = from + part * share, end = min(upto + 1, begin + share);
    float sum[Products][4] = {};
    float top[2] = {-INFINITY, -INFINITY}, weight[2] = {0.f, 0.f};
    for (int base = begin; base < end; base += AtOnce) {
        float4 value[AtOnce][Products];
        float2 stats[AtOnce][2];
#pragma unroll
        for (int i = 0; i < AtOnce; ++i) {
            const int worker = min(base + i, end - 1);
            const long long piece =
                (2ll * (worker * task.team + member) + (worker == from ? first_place : 0)) * blocks + n;
#pragma unroll
            for (int c = 0; c < Products; ++c)
                value[i][c] = __ldcg(&task.pieces[(piece * depth_pieces + product + c) * 32 + lane]);
            stats[i][0] = __ldcg(&task.statistics[piece * 8 + 2 * t]);
            stats[i][1] = __ldcg(&task.statistics[piece * 8 + 2 * t + 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float best = top[h];
#pragma unroll
            for (int i = 0; i < AtOnce; ++i)
                best = fmaxf(best, stats[i][h].x);
            const float reference = best == -INFINITY ? 0.f : best;
            const float factor = power_of_two(top[h] - reference);
            top[h] = best, weight[h] *= factor;
#pragma unroll
            for (int c = 0; c < Products; ++c)
                sum[c][h] *= factor, sum[c][h + 2] *= factor;
#pragma unroll
            for (int i = 0; i < AtOnce; ++i) {
                if (base + i >= end)
                    break;
                const float share_of = power_of_two(stats[i][h].x - reference);
                weight[h] += share_of * stats[i][h].y;
#pragma unroll
                for (int c = 0; c < Products; ++c) {
                    sum[c][h] += share_of * (h == 0 ? value[i][c].x : value[i][c].y);
                    sum[c][h + 2] += share_of * (h == 0 ? value[i][c].z : value[i][c].w);
                }
            }
        }
    }
    if (parts > 1) {
#pragma unroll
        for (int c = 0; c < Products; ++c)
            shared_sum[warp][c][lane] = make_float4(sum[c][0], sum[c][1], sum[c][2], sum[c][3]);
        if (g == 0)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                shared_stats[warp][0][2 * t + h] = top[h], shared_stats[warp][1][2 * t + h] = weight[h];
        __syncthreads();
        if (part != 0)
            return;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float best = -INFINITY;
            for (int other = 0; other < parts; ++other)
                best = fmaxf(best, shared_stats[warp + other][0][2 * t + h]);
            const float reference = best == -INFINITY ? 0.f : best;
            weight[h] = 0.f;
#pragma unroll
            for (int c = 0; c < Products; ++c)
                sum[c][h] = sum[c][h + 2] = 0.f;
            for (int other = 0; other < parts; ++other) {
                const float factor = power_of_two(shared_stats[warp + other][0][2 * t + h] - reference);
                weight[h] += factor * shared_stats[warp + other][1][2 * t + h];
#pragma unroll
                for (int c = 0; c < Products; ++c) {
                    const float4 v = shared_sum[warp + other][c][lane];
                    sum[c][h] += factor * (h == 0 ? v.x : v.y);
                    sum[c][h + 2] += factor * (h == 0 ? v.z : v.w);
                }
            }
        }
    }
    float inverse[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        inverse[h] = weight[h] != 0.f ? task.value_scale / weight[h] : 0.f;
    const int head_block = slot % task.head_blocks;
    const int first_head = slot / task.head_blocks * task.group + (head_block * blocks + n) * 8;
    const int live_heads = task.group - (head_block * blocks + n) * 8;
#pragma unroll
    for (int c = 0; c < Products; ++c)
        store_heads<Eight>(task.out + ((long long)sequence * task.heads + first_head) * task.depth, task.depth,
                           live_heads, product + c, sum[c], inverse);
}

/* How one call is cut: kernel instance, CTAs, workspace. */
struct Plan {
    int depth_class = 0; /* 64, 128 or 256 */
    int blocks = 1, head_blocks = 1, team = 1, teams = 1;
    long long tiles_bound = 0; /* most tiles an item can have */
    int grid = 0, workers = 0, tile_shift = 0;
    size_t first_bytes = 0, piece_bytes = 0, bytes = 0;
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
    const int slots = kv_heads * plan.head_blocks;
    plan.team = slots % 4 == 0 ? 4 : (slots % 2 == 0 ? 2 : 1);
    plan.teams = slots / plan.team;
    long long bound = (long long)page_size * table_width;
    if (window > 0 && bound > (long long)window + sinks)
        bound = (long long)window + sinks;
    bound = bound < INT_MAX ? bound : INT_MAX;
    const bool eight = cache_type == 3;
    plan.tile_shift =
        with_shape(plan.depth_class, plan.blocks, eight, [](auto shape) { return decltype(shape)::kTileShift; });
    plan.tiles_bound = bound > 0 ? ((bound - 1) >> plan.tile_shift) + 1 : 1;
    const int resident =
        with_shape(plan.depth_class, plan.blocks, eight, [](auto shape) { return decltype(shape)::kResident; });
    const long long warps = plan.tiles_bound * batch * slots;
    const long long most = (warps + kWarps - 1) / kWarps;
    const long long full = (long long)sm_count * resident;
    plan.grid = int(most < full ? most : full);
    plan.workers = plan.grid * kWarps / plan.team;
    plan.first_bytes = (size_t(batch) + 1 + 1) / 2 * 16;
    const size_t held = plan.tiles_bound > 1 ? size_t(plan.grid) * kWarps * 2 * plan.blocks : 0;
    plan.piece_bytes = held * (plan.depth_class / 16) * 32 * 16;
    plan.bytes = plan.first_bytes + plan.piece_bytes + held * 8 * 8;
    return plan;
}

template <int Depth, int Blocks, bool Eight>
void launch(camblas_cuda_context *context, const AttendTask &task, const Plan &plan, Shape<Depth, Blocks, Eight>)
{
    attend_kernel<Depth, Blocks, Eight>
        <<<plan.grid, kWarps * 32, Shape<Depth, Blocks, Eight>::kBytes, context->stream>>>(task);
}

template <bool Eight, int Products, int AtOnce>
cudaError_t launch_join_of(camblas_cuda_context *context, const AttendTask &task, const Plan &plan, int parts)
{
    const int depth_pieces = plan.depth_class / 16, shares = depth_pieces / Products;
    const int held = shares < kJoinWarps / parts ? shares : kJoinWarps / parts; /* of a CTA; powers of two */
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(task.batch) * plan.team * plan.teams * plan.blocks, shares / held);
    config.blockDim = dim3(held * parts * 32);
    config.stream = context->stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, attend_join<Eight, Products, AtOnce>, task, plan.blocks, depth_pieces, parts);
}

template <bool Eight>
cudaError_t launch_join(camblas_cuda_context *context, const AttendTask &task, const Plan &plan)
{
    /* Pieces per item if the lengths are alike. Few items with many pieces each: a product per warp,
     * sixteen warps to its pieces. More items: two products per warp and fewer warps per item, so that
     * the items fit one wave; ragged lengths still give long items more pieces than this. */
    const int items = task.batch * plan.team * plan.teams;
    const int expected = plan.grid * kWarps / items + 2;
    if (expected > 32)
        return launch_join_of<Eight, 1, 8>(context, task, plan, 16);
    return launch_join_of<Eight, 2, 4>(context, task, plan,
                                       expected > 16 ? 8 : (expected > 8 ? 4 : (expected > 4 ? 2 : 1)));
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

/* Query heads of a call: the scans of the lengths count up to the next multiple of 32, in 32 bits. */
constexpr int kMostHeads = INT_MAX - 63;

inline bool sizes_bad(int batch, int heads_count, int kv_heads, int depth, int cache_type, int page_size,
                      int table_width, int window, int sinks)
{
    return batch < 0 || kv_heads < 1 || heads_count < 1 || heads_count > 65536 || heads_count % kv_heads ||
           depth < 8 || depth > 256 || (cache_type != 2 && cache_type != 3) ||
           depth % (cache_type == 3 ? 16 : 8) || page_size < 1 || table_width < 0 || window < 0 || sinks < 0 ||
           (long long)batch * heads_count > kMostHeads;
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
              heads::misaligned(output, 4) /* stored in pairs */ || q == output || key_cache == output || value_cache == output;
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
        task.batch = batch, task.heads = heads_count, task.group = heads_count / kv_heads, task.depth = depth;
        task.head_blocks = plan.head_blocks, task.team = plan.team, task.teams = plan.teams;
        task.workers = plan.workers;
        for (heads::CacheLayout *cache : {&task.keys, &task.values})
            cache->page_stride *= element, cache->slot_stride *= element, cache->head_stride *= element;
        task.page_size = page_size, task.pages = pages, task.tile_shift = plan.tile_shift;
        task.room = int(std::min<long long>((long long)table_width * page_size, INT_MAX));
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
        task.value_scale = cache_type == 3 ? value_scale / attend::kRaised : value_scale;
        task.out = static_cast<__nv_bfloat16 *>(output);
        char *held = static_cast<char *>(workspace);
        task.first_tile = reinterpret_cast<long long *>(held);
        task.pieces = reinterpret_cast<float4 *>(held + plan.first_bytes);
        task.statistics = reinterpret_cast<float2 *>(held + plan.first_bytes + plan.piece_bytes);
        context->counts[6]++;
        attend::with_shape(plan.depth_class, plan.blocks, cache_type == 3, [&](auto shape) {
            attend::launch(context, task, plan, shape);
            return 0;
        });
        const int status = host::launched(context, "paged attention");
        if (status != 0 || plan.tiles_bound == 1)
            return status;
        const cudaError_t error = cache_type == 3 ? attend::launch_join<true>(context, task, plan)
                                                  : attend::launch_join<false>(context, task, plan);
        if (error != cudaSuccess)
            return host::fail(context, "paged attention join", error);
        context->kernel_launches.fetch_add(1, std::memory_order_relaxed);
        return 0;
    });
}
