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
 * and the store is FP32; the result is rounded once, to BF16 or, for an 8-bit
 * cache, from FP32 straight to E4M3.
 *
 * The reads and writes of the heads bound the kernel: seven operations per
 * element against four bytes. The
 * largest power of two of lanes that a depth needs (eight elements per lane)
 * shares a head; a lane holds both members of its pairs, so the rotation needs
 * no exchange and the norm one shuffle tree. A lane's eight elements are two
 * 8-byte pieces, which for the half-split form lie rotary/2 apart.
 */
#pragma once

#include "context.cuh"

#include <cuda_fp8.h>

#include <climits>
#include <cmath>

namespace heads
{

constexpr int kThreads = 256;

/* Address of head h of one cached token: base + page*page_stride +
 * slot*slot_stride + h*head_stride, in elements. */
struct CacheLayout {
    void *base;
    long long page_stride, slot_stride, head_stride;
};

struct RotateTask {
    int tokens, heads, kv_heads, depth, rotary, table_rows, page_size;
    int interleaved, eight_bit;
    float epsilon, key_scale, value_scale;
    const __nv_bfloat16 *q, *k, *v; /* v NULL: no cache */
    long long q_token, q_head, k_token, k_head, v_token, v_head;
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

__device__ __forceinline__ Piece load_piece(const __nv_bfloat16 *from)
{
    return unpack_piece(*reinterpret_cast<const uint2 *>(from));
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

/* value / scale, rounded to the nearest E4M3, at most 448 in magnitude */
__device__ __forceinline__ void store_piece_e4m3(uint8_t *to, const Piece &p, float scale)
{
    const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(p.e[0] / scale, p.e[1] / scale),
                                                  __NV_SATFINITE, __NV_E4M3);
    const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(p.e[2] / scale, p.e[3] / scale),
                                                   __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint32_t *>(to) = low | (high << 16);
}

/* `Lanes` lanes share a head. Work item = one head of one token, query heads
 * first, then key heads, then (with a cache) value heads. */
template <int Lanes>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const RotateTask task)
{
    const int per_token = task.heads + (task.v ? 2 : 1) * task.kv_heads;
    const long long items = (long long)task.tokens * per_token;
    const int unit = threadIdx.x % Lanes;
    const int turned = task.rotary / 8; /* units that rotate */
    /* the two 4-element pieces of this lane */
    const bool split_pair = !task.interleaved && unit < turned;
    const int first = split_pair ? 4 * unit : 8 * unit;
    const int second = split_pair ? first + task.rotary / 2 : first + 4;
    const bool live_unit = 8 * unit < task.depth;
    constexpr int kPerBlock = kThreads / Lanes;
    for (long long start = (long long)blockIdx.x * kPerBlock; start < items;
         start += (long long)gridDim.x * kPerBlock) {
        const long long item = start + threadIdx.x / Lanes;
        const bool live = item < items && live_unit;
        const int token = live ? int(item / per_token) : 0;
        int head = live ? int(item - (long long)token * per_token) : 0;
        const __nv_bfloat16 *source, *weight;
        int kind = 0;
        if (head < task.heads) {
            source = task.q + token * task.q_token + head * task.q_head;
            weight = task.q_weight;
        } else if (head < task.heads + task.kv_heads) {
            kind = 1, head -= task.heads;
            source = task.k + token * task.k_token + head * task.k_head;
            weight = task.k_weight;
        } else {
            kind = 2, head -= task.heads + task.kv_heads;
            source = task.v + token * task.v_token + head * task.v_head;
            weight = nullptr;
        }
        Piece a{}, b{};
        long long position = 0, slot = -1;
        if (live) {
            a = load_piece(source + first), b = load_piece(source + second);
            position = task.positions[token];
            if (kind != 0 && task.v)
                slot = task.slots[token];
        }
        const bool placed = position >= 0 && position < task.table_rows;
        float square = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            square += a.e[i] * a.e[i] + b.e[i] * b.e[i];
#pragma unroll
        for (int offset = Lanes / 2; offset > 0; offset /= 2)
            square += __shfl_xor_sync(0xffffffffu, square, offset, Lanes);
        if (!live)
            continue;
        if (weight) {
            const float scale = rsqrtf(square / task.depth + task.epsilon);
            const Piece wa = load_piece(weight + first), wb = load_piece(weight + second);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a.e[i] *= scale * wa.e[i], b.e[i] *= scale * wb.e[i];
        }
        if (kind != 2 && unit < turned && placed) {
            const float *row = task.table + position * task.rotary + 4 * unit;
            const float4 c4 = *reinterpret_cast<const float4 *>(row);
            const float4 s4 = *reinterpret_cast<const float4 *>(row + task.rotary / 2);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
            if (task.interleaved) {
                Piece *both[2] = {&a, &b};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float &x = both[i / 2]->e[2 * (i & 1)], &y = both[i / 2]->e[2 * (i & 1) + 1];
                    const float turned_x = x * c[i] - y * s[i];
                    y = y * c[i] + x * s[i], x = turned_x;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float turned_x = a.e[i] * c[i] - b.e[i] * s[i];
                    b.e[i] = b.e[i] * c[i] + a.e[i] * s[i], a.e[i] = turned_x;
                }
            }
        }
        if (!placed) /* a padding row: zeros, and nothing enters the cache */
            a = Piece{}, b = Piece{};
        if (kind == 0 || (kind == 1 && task.k_out)) {
            const int count = kind == 0 ? task.heads : task.kv_heads;
            __nv_bfloat16 *to = (kind == 0 ? task.q_out : task.k_out) +
                                ((long long)token * count + head) * task.depth;
            store_piece(to + first, a), store_piece(to + second, b);
        }
        if (kind != 0 && placed && slot >= 0 && slot < task.slot_count) {
            const CacheLayout &cache = kind == 1 ? task.key_cache : task.value_cache;
            const long long page = slot / task.page_size;
            const long long at = page * cache.page_stride +
                                 (slot - page * task.page_size) * cache.slot_stride +
                                 head * cache.head_stride;
            if (task.eight_bit) {
                uint8_t *to = static_cast<uint8_t *>(cache.base) + at;
                const float scale = kind == 1 ? task.key_scale : task.value_scale;
                store_piece_e4m3(to + first, a, scale), store_piece_e4m3(to + second, b, scale);
            } else {
                __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(cache.base) + at;
                store_piece(to + first, a), store_piece(to + second, b);
            }
        }
    }
}

template <int Lanes> void launch(camblas_cuda_context *context, const RotateTask &task)
{
    const long long items =
        (long long)task.tokens * (task.heads + (task.v ? 2 : 1) * task.kv_heads);
    const long long blocks = (items + kThreads / Lanes - 1) / (kThreads / Lanes);
    rotate_kernel<Lanes><<<unsigned(blocks < (1 << 30) ? blocks : (1 << 30)), kThreads, 0,
                           context->stream>>>(task);
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
            bad = strides[i] % 4 != 0;
        if (bad || q_out == q || q_out == k || q_out == v || (k_out && (k_out == q || k_out == k)) ||
            q_out == k_out)
            return host::fail(context, "invalid head rotation operands", 1);
        heads::RotateTask task{};
        task.tokens = tokens, task.heads = heads_count, task.kv_heads = kv_heads;
        task.depth = depth, task.rotary = rotary, task.table_rows = table_rows;
        task.interleaved = interleaved, task.epsilon = epsilon;
        task.q = static_cast<const __nv_bfloat16 *>(q);
        task.k = static_cast<const __nv_bfloat16 *>(k);
        task.q_token = strides[0], task.q_head = strides[1];
        task.k_token = strides[2], task.k_head = strides[3];
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
            task.v_token = strides[4], task.v_head = strides[5];
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
