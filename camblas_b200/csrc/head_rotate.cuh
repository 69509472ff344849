/*
 * RMS norm of every query and key head, position rotation, and the write of the
 * new keys and values into a paged cache, in one pass.
 *
 * For one head x[depth] at position p:
 *   y = x * rsqrt(mean(x^2) + eps) * weight           (weight NULL: y = x)
 *   (a, b) -> (a cos - b sin, b cos + a sin)          over the first `rotary` elements
 * with pair i = (i, i + rotary/2), or (2i, 2i+1) when interleaved, and cos/sin row
 * p of a table the caller computed (angles of far positions lose their
 * fraction in FP32, so they are not formed here). Everything between the load
 * and the store is FP32; the result, divided by the scale of its cache, is rounded
 * once, to BF16 or, for an 8-bit cache, from FP32 straight to E4M3. A head whose
 * squares leave FP32's range is done again, divided by a power of two.
 *
 * The reads and writes of the heads bound the kernel: seven operations per
 * element against four bytes, as long as issue keeps up: a head's eight elements
 * of a lane take about 140 instructions here; the first form, which divided by
 * the heads per token and multiplied weight, cosine and sine for every head, took
 * 250 and 117 us where this takes 60 (8192 tokens of 64 + 8 heads of 128; 0.77 of
 * the measured copy rate). As many lanes as a depth needs at eight elements per
 * lane, rounded up to a power of two, share a head; a lane holds both members of
 * its pairs, so the rotation needs no exchange and the norm one shuffle tree. A
 * lane's eight elements are two 8-byte pieces, which for the half-split form lie
 * rotary/2 apart.
 */
#pragma once

#include "context.cuh"

#include <cuda_fp8.h>

#include <climits>
#include <cmath>
#include <type_traits>

namespace heads
{

/* Two warps: with 64 + 8 heads of 128 a lane turns 16 query heads and 2 key heads, over which its
 * preparation is spread (8192 tokens: 85 us with 256 threads, 68 with 128, 62 with 64). */
constexpr int kThreads = 64;
constexpr int kBatch = 4; /* heads of a lane that are fetched together */

/* Address of head h of one cached token: base + page*page_stride +
 * slot*slot_stride + h*head_stride, in elements. */
struct CacheLayout {
    void *base;
    long long page_stride, slot_stride, head_stride;
};

struct RotateTask {
    int tokens, heads, kv_heads, depth, rotary, table_rows, page_size;
    int interleaved, eight_bit;
    float epsilon, inverse_depth, key_scale, value_scale;
    const __nv_bfloat16 *q, *k, *v; /* v NULL: no cache */
    long long q_token, k_token, v_token; /* strides */
    int q_head, k_head, v_head;
    const __nv_bfloat16 *q_weight, *k_weight;
    const int64_t *positions, *slots;
    const float *table;
    __nv_bfloat16 *q_out, *k_out;
    CacheLayout key_cache, value_cache;
    long long slot_count;
};

struct Piece { /* four elements of a head */
    float e[4];
};

__device__ __forceinline__ Piece unpack_piece(const uint2 &raw)
{
    const float2 low = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw.x));
    const float2 high = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw.y));
    return {{low.x, low.y, high.x, high.y}};
}

__device__ __forceinline__ void store_piece(__nv_bfloat16 *to, const Piece &p)
{
    const __nv_bfloat162 low = __floats2bfloat162_rn(p.e[0], p.e[1]);
    const __nv_bfloat162 high = __floats2bfloat162_rn(p.e[2], p.e[3]);
    uint2 raw;
    raw.x = *reinterpret_cast<const uint32_t *>(&low);
    raw.y = *reinterpret_cast<const uint32_t *>(&high);
    *reinterpret_cast<uint2 *>(to) = raw;
}

/* rounded to the nearest E4M3, at most 448 in magnitude */
__device__ __forceinline__ void store_piece_e4m3(uint8_t *to, const Piece &p)
{
    const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(p.e[0], p.e[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(p.e[2], p.e[3]), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint32_t *>(to) = low | (high << 16);
}

/* Two FP32 numbers in a register pair, and the packed arithmetic on them. */
typedef unsigned long long Two;

__device__ __forceinline__ Two two(float low, float high)
{
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(low), "f"(high));
    return r;
}

__device__ __forceinline__ float2 both(Two x)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}

__device__ __forceinline__ Two multiply(Two x, Two y)
{
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

__device__ __forceinline__ Two multiply_add(Two x, Two y, Two z)
{
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}

__device__ __forceinline__ Two swapped(Two x)
{
    const float2 v = both(x);
    return two(v.y, v.x);
}

/* a BF16 pair as FP32 */
__device__ __forceinline__ Two widen_pair(uint32_t raw)
{
    return two(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u));
}

/* A lane's eight elements of one head: pieces a and b of four. */
struct Eight {
    Two a[2], b[2];
};

__device__ __forceinline__ Piece as_piece(const Two (&x)[2])
{
    const float2 low = both(x[0]), high = both(x[1]);
    return {{low.x, low.y, high.x, high.y}};
}

/* What a lane multiplies its elements by: a' = a * straight.a + (b, or a with its
 * pairs swapped) * cross.a, and b' likewise; the products of the norm's weight
 * (NULL: 1) and the cosines and sines of its angles. */
template <bool Interleaved> struct Turn {
    Eight straight, cross;

    __device__ __forceinline__ Turn(const __nv_bfloat16 *weight, const float *cosines, int half, bool turns,
                                    int first, int second)
    {
        straight = {{two(1.f, 1.f), two(1.f, 1.f)}, {two(1.f, 1.f), two(1.f, 1.f)}};
        cross = {};
        if (weight) {
            const uint2 a = *reinterpret_cast<const uint2 *>(weight + first);
            const uint2 b = *reinterpret_cast<const uint2 *>(weight + second);
            straight = {{widen_pair(a.x), widen_pair(a.y)}, {widen_pair(b.x), widen_pair(b.y)}};
        }
        if (!turns)
            return;
        const float4 c = *reinterpret_cast<const float4 *>(cosines);
        const float4 s = *reinterpret_cast<const float4 *>(cosines + half);
        if constexpr (Interleaved) {
            /* pair (x, y): x' = x wx c - y wy s, y' = y wy c + x wx s; pairs 0, 1 in a, 2, 3 in b */
            cross.a[0] = multiply(swapped(straight.a[0]), two(-s.x, s.x));
            cross.a[1] = multiply(swapped(straight.a[1]), two(-s.y, s.y));
            cross.b[0] = multiply(swapped(straight.b[0]), two(-s.z, s.z));
            cross.b[1] = multiply(swapped(straight.b[1]), two(-s.w, s.w));
            straight.a[0] = multiply(straight.a[0], two(c.x, c.x));
            straight.a[1] = multiply(straight.a[1], two(c.y, c.y));
            straight.b[0] = multiply(straight.b[0], two(c.z, c.z));
            straight.b[1] = multiply(straight.b[1], two(c.w, c.w));
        } else {
            const Two low = two(c.x, c.y), high = two(c.z, c.w);
            cross.a[0] = multiply(straight.b[0], two(-s.x, -s.y));
            cross.a[1] = multiply(straight.b[1], two(-s.z, -s.w));
            cross.b[0] = multiply(straight.a[0], two(s.x, s.y));
            cross.b[1] = multiply(straight.a[1], two(s.z, s.w));
            straight.a[0] = multiply(straight.a[0], low), straight.a[1] = multiply(straight.a[1], high);
            straight.b[0] = multiply(straight.b[0], low), straight.b[1] = multiply(straight.b[1], high);
        }
    }

    __device__ __forceinline__ Eight apply(const Eight &x, bool turns, float scale) const
    {
        Eight y;
        const Two scales = two(scale, scale);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            y.a[i] = multiply(x.a[i], straight.a[i]), y.b[i] = multiply(x.b[i], straight.b[i]);
            if (turns) { /* elsewhere cross is 0, but 0 times an infinity is not */
                y.a[i] = multiply_add(Interleaved ? swapped(x.a[i]) : x.b[i], cross.a[i], y.a[i]);
                y.b[i] = multiply_add(Interleaved ? swapped(x.b[i]) : x.a[i], cross.b[i], y.b[i]);
            }
            y.a[i] = multiply(y.a[i], scales), y.b[i] = multiply(y.b[i], scales);
        }
        return y;
    }
};

/* Bits of 2^-90 and 2^120: means of squares between them are of squares that FP32 holds. */
constexpr unsigned kLeastMean = (127 - 90) << 23, kMostMean = (127 + 120) << 23;

/* The norm's factor of a head whose squares leave FP32's range or its normal numbers: from squares of the
 * elements divided by the power of two of the largest, or of the root of epsilon where that is larger, which
 * `x` then is too. A head of zeros, or with an element that is not finite, keeps the factor it has. */
template <int Lanes>
__device__ __forceinline__ float far_scale(unsigned sharing, Eight &x, float scale, float inverse_depth, float epsilon)
{
    float largest = 0.f;
    bool broken = false;
    const Two parts[4] = {x.a[0], x.a[1], x.b[0], x.b[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = both(parts[i]);
        largest = fmaxf(largest, fmaxf(fabsf(v.x), fabsf(v.y)));
        broken = broken || !(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY);
    }
#pragma unroll
    for (int offset = Lanes / 2; offset > 0; offset /= 2)
        largest = fmaxf(largest, __shfl_xor_sync(sharing, largest, offset, Lanes));
    if (__any_sync(sharing, broken) || largest == 0.f)
        return scale;
    int exponent = ilogbf(largest);
    if (epsilon > 0.f)
        exponent = max(exponent, ilogbf(epsilon) / 2);
    const float down = ldexpf(1.f, -exponent / 2), rest = ldexpf(1.f, -exponent - -exponent / 2);
    float square = 0.f;
    Eight y = x;
    Two *const out[4] = {&y.a[0], &y.a[1], &y.b[0], &y.b[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        *out[i] = multiply(multiply(parts[i], two(down, down)), two(rest, rest));
        const float2 v = both(*out[i]);
        square += v.x * v.x + v.y * v.y;
    }
#pragma unroll
    for (int offset = Lanes / 2; offset > 0; offset /= 2)
        square += __shfl_xor_sync(sharing, square, offset, Lanes);
    x = y;
    return rsqrtf(square * inverse_depth + epsilon * down * rest * down * rest);
}

/* `Lanes` lanes share a head; a CTA takes one token's query heads, key heads and,
 * with a cache, value heads, or every gridDim.y-th round of them. What does not
 * depend on the head (the products of weight and cosine or sine) is done once
 * per lane and kind, and `Batch` heads of a lane are fetched before the first
 * is worked on. */
template <int Lanes, int Batch, bool Interleaved>
__global__ void __launch_bounds__(kThreads, Batch > 1 ? 16 : 1) rotate_kernel(const __grid_constant__ RotateTask task)
{
    constexpr int kGroups = kThreads / Lanes;
    constexpr unsigned kSharing = Lanes == 32 ? 0xffffffffu : (1u << (Lanes % 32)) - 1;
    const unsigned sharing = kSharing << (threadIdx.x % 32 / Lanes * Lanes); /* the lanes of this head */
    const int token = blockIdx.x;
    const int unit = threadIdx.x % Lanes;
    const bool live = 8 * unit < task.depth;
    const bool turns = 8 * unit < task.rotary;
    const int first = !Interleaved && turns ? 4 * unit : 8 * unit;
    const int second = !Interleaved && turns ? first + task.rotary / 2 : first + 4;
    const int step = gridDim.y * kGroups, group = blockIdx.y * kGroups + threadIdx.x / Lanes;
    const long long position = task.positions[token];
    const bool placed = position >= 0 && position < task.table_rows;
    const float *cosines = task.table + position * task.rotary + 4 * unit;

    /* Works on heads h = begin, begin + step, ... below count, the first at `source`: turns them
     * (nullptr: leaves them as they are) and hands each to store(h, a, b). Returns whether a norm left
     * the range, and the heads are to be done again with `careful`. */
    const auto run = [&](int begin, int count, const __nv_bfloat16 *source, int head_stride, const auto *turn,
                         bool normalise, auto store, auto careful) {
        constexpr int kAtOnce = careful.value ? 1 : Batch;
        bool far = false;
        const __nv_bfloat16 *at_first = source + (long long)begin * head_stride + first;
        const __nv_bfloat16 *at_second = at_first + (second - first);
        const long long ahead = (long long)step * head_stride;
        for (int head = begin; head < count; head += kAtOnce * step) {
            uint2 raw[kAtOnce][2];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                raw[i][0] = raw[i][1] = make_uint2(0, 0);
                if (live && head + i * step < count) {
                    raw[i][0] = *reinterpret_cast<const uint2 *>(at_first);
                    raw[i][1] = *reinterpret_cast<const uint2 *>(at_second);
                }
                at_first += ahead, at_second += ahead;
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (head + i * step >= count)
                    break;
                Eight x = {{widen_pair(raw[i][0].x), widen_pair(raw[i][0].y)},
                           {widen_pair(raw[i][1].x), widen_pair(raw[i][1].y)}};
                if (turn) {
                    float scale = 1.f;
                    if (normalise) {
                        const Two square_two = multiply_add(
                            x.b[1], x.b[1],
                            multiply_add(x.b[0], x.b[0], multiply_add(x.a[1], x.a[1], multiply(x.a[0], x.a[0]))));
                        float square = both(square_two).x + both(square_two).y;
#pragma unroll
                        for (int offset = Lanes / 2; offset > 0; offset /= 2)
                            square += __shfl_xor_sync(sharing, square, offset, Lanes);
                        const float mean = square * task.inverse_depth + task.epsilon;
                        scale = rsqrtf(mean);
                        /* the same for all lanes of the head; a NaN is outside too */
                        const bool outside = __float_as_uint(mean) - kLeastMean >= kMostMean - kLeastMean;
                        if constexpr (careful.value) {
                            if (outside)
                                scale = far_scale<Lanes>(sharing, x, scale, task.inverse_depth, task.epsilon);
                        } else {
                            far = far || outside;
                        }
                    }
                    x = turn->apply(x, turns, scale);
                }
                if (live)
                    store(head + i * step, as_piece(x.a), as_piece(x.b));
            }
        }
        return far;
    };
    /* The careful loop stands apart: its code within the other's takes registers that the heads in flight
     * need (8192 tokens: 61.7 us, apart 60.3). */
    const auto run_normed = [&](int begin, int count, const __nv_bfloat16 *source, int head_stride, const auto *turn,
                                bool normalise, auto store) {
        if (run(begin, count, source, head_stride, turn, normalise, store, std::false_type{}))
            run(begin, count, source, head_stride, turn, normalise, store, std::true_type{});
    };

    if (!placed) { /* a padding row: zeros, and nothing enters the cache */
        const Piece zero{};
        for (int head = group; live && head < task.heads; head += step) {
            __nv_bfloat16 *to = task.q_out + ((long long)token * task.heads + head) * task.depth;
            store_piece(to + first, zero), store_piece(to + second, zero);
        }
        for (int head = group; live && task.k_out && head < task.kv_heads; head += step) {
            __nv_bfloat16 *to = task.k_out + ((long long)token * task.kv_heads + head) * task.depth;
            store_piece(to + first, zero), store_piece(to + second, zero);
        }
        return;
    }
    if (group < task.heads) {
        const Turn<Interleaved> turn(live ? task.q_weight : nullptr, cosines, task.rotary / 2, turns, first,
                                     second);
        __nv_bfloat16 *out = task.q_out + (long long)token * task.heads * task.depth;
        run_normed(
            group, task.heads, task.q + token * task.q_token, task.q_head, &turn, task.q_weight != nullptr,
            [&](int head, const Piece &a, const Piece &b) {
                store_piece(out + head * task.depth + first, a), store_piece(out + head * task.depth + second, b);
            });
    }
    /* where the token's keys and values go in the caches; -1: nowhere */
    long long page = -1, place = 0;
    if (task.v) {
        const long long slot = task.slots[token];
        if (slot >= 0 && slot < task.slot_count)
            page = slot / task.page_size, place = slot - page * task.page_size;
    }
    const auto cache = [&](const CacheLayout &to, int head, float scale, Piece a, Piece b) {
        if (page < 0)
            return;
        if (scale != 1.f)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a.e[i] /= scale, b.e[i] /= scale;
        const long long at = page * to.page_stride + place * to.slot_stride + head * to.head_stride;
        if (task.eight_bit) {
            uint8_t *row = static_cast<uint8_t *>(to.base) + at;
            store_piece_e4m3(row + first, a), store_piece_e4m3(row + second, b);
        } else {
            __nv_bfloat16 *row = static_cast<__nv_bfloat16 *>(to.base) + at;
            store_piece(row + first, a), store_piece(row + second, b);
        }
    };
    /* keys follow the queries in the rounds, values the keys */
    const auto first_after = [&](int before) { return group >= before ? group - before : step - 1 - (before - group - 1) % step; };
    int begin = first_after(task.heads);
    if (begin < task.kv_heads) {
        const Turn<Interleaved> turn(live ? task.k_weight : nullptr, cosines, task.rotary / 2, turns, first,
                                     second);
        __nv_bfloat16 *out =
            task.k_out ? task.k_out + (long long)token * task.kv_heads * task.depth : nullptr;
        run_normed(
            begin, task.kv_heads, task.k + token * task.k_token, task.k_head, &turn, task.k_weight != nullptr,
            [&](int head, const Piece &a, const Piece &b) {
                if (out)
                    store_piece(out + head * task.depth + first, a), store_piece(out + head * task.depth + second, b);
                cache(task.key_cache, head, task.key_scale, a, b);
            });
    }
    begin = first_after(task.heads + task.kv_heads);
    if (task.v && begin < task.kv_heads && page >= 0)
        run(
            begin, task.kv_heads, task.v + token * task.v_token, task.v_head,
            static_cast<const Turn<Interleaved> *>(nullptr), false,
            [&](int head, const Piece &a, const Piece &b) { cache(task.value_cache, head, task.value_scale, a, b); },
            std::false_type{});
}

template <int Lanes, int Batch> void launch_batch(camblas_cuda_context *context, const RotateTask &task, int parts)
{
    const dim3 grid(task.tokens, parts < 65535 ? parts : 65535); /* the kernel goes round for more */
    if (task.interleaved)
        rotate_kernel<Lanes, Batch, true><<<grid, kThreads, 0, context->stream>>>(task);
    else
        rotate_kernel<Lanes, Batch, false><<<grid, kThreads, 0, context->stream>>>(task);
}

template <int Lanes> void launch(camblas_cuda_context *context, const RotateTask &task)
{
    /* Enough tokens to fill the chip: a CTA takes all heads of a token. Fewer: a head per lane, and
     * as many CTAs per token as that takes. */
    const int all_heads = task.heads + (task.v ? 2 : 1) * task.kv_heads;
    const int groups = kThreads / Lanes, rounds = (all_heads + groups - 1) / groups;
    if (task.tokens < 2 * context->sm_count)
        launch_batch<Lanes, 1>(context, task, rounds);
    else
        launch_batch<Lanes, kBatch>(context, task, 1);
}

inline bool misaligned(const void *pointer, unsigned bytes)
{
    return (reinterpret_cast<uintptr_t>(pointer) & (bytes - 1)) != 0;
}

/* Whether a cache can be written (and read) in whole pieces of `bytes` bytes. */
inline bool cache_bad(const CacheLayout &cache, int element_bytes, int bytes)
{
    const int elements = bytes / element_bytes;
    return !cache.base || misaligned(cache.base, bytes) || cache.page_stride % elements ||
           cache.slot_stride % elements || cache.head_stride % elements;
}

} // namespace heads

extern "C" int camblas_cuda_qk_norm_rope(
    camblas_cuda_context *context, int tokens, int heads_count, int kv_heads, int depth, int rotary,
    int interleaved, float epsilon, const void *q, const void *k, const void *v,
    const long long *strides, const void *q_weight, const void *k_weight, const void *positions,
    const float *table, int table_rows, void *q_out, void *k_out, int cache_type, void *key_cache,
    void *value_cache, long long pages, int page_size, float key_scale, float value_scale,
    const void *slots)
{
    return host::guarded(context, [&] {
        const bool cached = cache_type != 0;
        if (tokens < 0 || heads_count < 1 || kv_heads < 1 || heads_count > 65536 ||
            kv_heads > 65536 || depth < 8 || depth > 256 || depth % 8 || rotary < 0 ||
            rotary > depth || rotary % 8 || table_rows < 0 || !std::isfinite(epsilon) ||
            epsilon < 0 || (interleaved != 0 && interleaved != 1) ||
            (cached && cache_type != 2 && cache_type != 3))
            return host::fail(context, "invalid head rotation dimensions", 1);
        if (cached && (pages < 0 || page_size < 1 || pages > LLONG_MAX / page_size ||
                       !(key_scale > 0) || !(value_scale > 0) || !std::isfinite(key_scale) ||
                       !std::isfinite(value_scale)))
            return host::fail(context, "invalid cache arguments of the head rotation", 1);
        if (tokens == 0)
            return 0;
        bool bad = !q || !k || !strides || !positions || (rotary && table_rows && !table) || !q_out ||
                   (!cached && !k_out) || (cached && (!v || !slots)) ||
                   heads::misaligned(positions, 8) || heads::misaligned(slots, 8) ||
                   heads::misaligned(table, 16);
        const void *pieces[7] = {q, k, cached ? v : nullptr, q_weight, k_weight, q_out, k_out};
        for (const void *pointer : pieces)
            bad = bad || heads::misaligned(pointer, 8);
        for (int i = 0; i < (cached ? 6 : 4) && !bad; ++i)
            bad = strides[i] % 4 != 0 || (i % 2 == 1 && (strides[i] < INT_MIN || strides[i] > INT_MAX));
        if (bad || q_out == q || q_out == k || q_out == v || (k_out && (k_out == q || k_out == k)) ||
            q_out == k_out)
            return host::fail(context, "invalid head rotation operands", 1);
        heads::RotateTask task{};
        task.tokens = tokens, task.heads = heads_count, task.kv_heads = kv_heads;
        task.depth = depth, task.rotary = rotary, task.table_rows = table_rows;
        task.interleaved = interleaved, task.epsilon = epsilon, task.inverse_depth = 1.f / depth;
        task.q = static_cast<const __nv_bfloat16 *>(q);
        task.k = static_cast<const __nv_bfloat16 *>(k);
        task.q_token = strides[0], task.q_head = int(strides[1]);
        task.k_token = strides[2], task.k_head = int(strides[3]);
        task.q_weight = static_cast<const __nv_bfloat16 *>(q_weight);
        task.k_weight = static_cast<const __nv_bfloat16 *>(k_weight);
        task.positions = static_cast<const int64_t *>(positions);
        task.table = table;
        task.q_out = static_cast<__nv_bfloat16 *>(q_out);
        task.k_out = static_cast<__nv_bfloat16 *>(k_out);
        task.page_size = 1;
        if (cached) {
            task.eight_bit = cache_type == 3;
            task.v = static_cast<const __nv_bfloat16 *>(v);
            task.v_token = strides[4], task.v_head = int(strides[5]);
            task.slots = static_cast<const int64_t *>(slots);
            task.key_cache = {key_cache, strides[6], strides[7], strides[8]};
            task.value_cache = {value_cache, strides[9], strides[10], strides[11]};
            task.page_size = page_size, task.slot_count = pages * page_size;
            task.key_scale = key_scale, task.value_scale = value_scale;
            const int element = cache_type == 3 ? 1 : 2;
            if (pages > 0 && (heads::cache_bad(task.key_cache, element, 4 * element) ||
                              heads::cache_bad(task.value_cache, element, 4 * element) ||
                              key_cache == value_cache))
                return host::fail(context, "invalid cache layout of the head rotation", 1);
        }
        if (depth <= 64)
            heads::launch<8>(context, task);
        else if (depth <= 128)
            heads::launch<16>(context, task);
        else
            heads::launch<32>(context, task);
        return host::launched(context, "head rotation");
    });
}
