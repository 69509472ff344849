/*
 * Linear layer for a few tokens with 4-bit weights and group scales.
 *
 *   out[r,o] = sum over groups G of s[o,G] * sum_{k in G} (c[o,k] - z[o,G]) x[r,k]
 *              (+ bias[o]) (+ residual[r,o]),
 * codes c and zero points z in 0..15 (z = 8 without zero points), groups of 32,
 * 64 or 128 input features. c - z is a whole number of at most 15, exact in 16
 * bits, so the products run on the tensor cores over exact operands; the FP32
 * sums of a group are scaled in FP32, and the result is rounded once. Scaling
 * the weights themselves to BF16 before the product would round each of them.
 *
 * HBM bounds it as long as unpacking keeps up: half a byte per weight, two
 * operations per weight and token. Warp tiles of 16 outputs with mma.m16n8k16:
 * the outputs take the 16-row side, eight tokens the column side, so one token
 * costs the tensor cores no more than eight. The codes are laid out once, when
 * the weight is loaded, in the order the lanes want them: a lane's 16 bytes hold
 * its row operands of four products, 64 input features of 16 outputs are 512
 * contiguous bytes per warp.
 *
 * Unpacking. A nibble n, alone in the low bits of an FP16, is the subnormal
 * n * 2^-24, exact, and in the next four bits 16 n * 2^-24; so a pair of codes is
 * one AND of the word, or of the word shifted by 8, and the zero point, in the same
 * form, is subtracted from both at once, which is exact: nine instructions for a
 * product's operand. The factors 2^24 and 1/16 go to the scales. (128 + n in BF16,
 * less 128 + z, takes eleven: 70 us for one token, 28672 -> 8192, where this takes
 * 30. Taking z sum x from a group's sum of c x afterwards takes five, but what is
 * left where c is near z is the rounding of sums that are far larger.)
 *
 * The tokens are brought to FP16 first, in a small kernel of their own:
 * spread_tokens multiplies each 128 inputs of a token by a power of two that
 * brings the largest to [2^14, 2^15), where an FP16 holds a BF16 exactly down to
 * 2^-31 of the largest (its least step is 2^-24, a BF16's 2^-7 of its own power of
 * two) and below that to within 2^-39 of it, and leaves the power. The product is its programmatic dependent and has its first
 * weights in flight before it waits for the tokens. A token element that
 * is infinite or NaN makes the power, and so the token's outputs, NaN.
 *
 * Layout: [block of 64 outputs][unit of 128 inputs][4 tiles of 16 outputs], a
 * tile of a unit being 1024 bytes of codes, then its scales, then its zero points
 * (when there are any). Codes [2 halves of 64 inputs][lane = 4g + t][word i = 2h +
 * m]; word i holds for inputs k = 64 half + 32h + 8t + 4m + j, j = 0..3, and
 * outputs g + 8r, r = 0..1, the code at nibble r + 2 (j / 2) + 4 (j % 2). Scales,
 * and zero points of one byte, [group][g][r]. Outputs are padded to 64 and inputs
 * to 128, with scale zero. A unit of 64 outputs is one contiguous piece, one bulk
 * copy.
 */
#pragma once

#include "context.cuh"
#include "head_rotate.cuh"
#include "paged_attention.cuh"
#include "sm100_primitives.cuh"

#include <cuda_fp16.h>

namespace nibble
{

constexpr int kWarps = 4;   /* of a CTA that multiply */
constexpr int kUnit = 128;  /* inputs that are worked on at once: two blocks */
constexpr int kTokenBytes = kUnit * 2;

struct LinearTask {
    int rows, inner, outputs, units, split;
    const __nv_bfloat16 *x;
    long long ldx;
    const uint8_t *weights;
    const __nv_bfloat16 *bias, *residual;
    long long ldr;
    __nv_bfloat16 *out;
    long long ldo;
    /* Workspace. Tokens are taken in passes of `pass_rows`; for every unit a pass has the powers
     * of its tokens, pass_rows of them, and then its tokens in FP16, 256 bytes each. Odd tokens have the 64-byte halves of each 128
     * bytes swapped, so that the operand reads of two tokens meet different banks. */
    int pass_rows;
    uint8_t *tokens;
    unsigned *status;
};

/* Bytes of a tile of a unit, and of a unit's powers. */
template <int Group, typename Scale, bool Zeros> __host__ __device__ constexpr int tile_bytes()
{
    return 16 * kUnit / 2 + kUnit / Group * 16 * (int(sizeof(Scale)) + (Zeros ? 1 : 0));
}

__host__ __device__ constexpr int power_bytes(int rows) { return rows * 4; }

/* One warp per unit of a token: 16 lanes with eight inputs each, two units per warp. */
__global__ void __launch_bounds__(256) spread_tokens(const __grid_constant__ LinearTask task)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x % 32, piece = lane % 16;
    const int unit = (blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * 2 + lane / 16;
    const int row = blockIdx.y;
    const bool live = unit < task.units;
    const int k = unit * kUnit + 8 * piece;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live && k < task.inner)
        raw = *reinterpret_cast<const uint4 *>(task.x + row * task.ldx + k);
    const heads::Piece low = heads::unpack_piece(make_uint2(raw.x, raw.y));
    const heads::Piece high = heads::unpack_piece(make_uint2(raw.z, raw.w));
    float largest = 0.f;
    bool broken = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        largest = fmaxf(largest, fmaxf(fabsf(low.e[i]), fabsf(high.e[i])));
        broken = broken || !(fabsf(low.e[i]) < INFINITY) || !(fabsf(high.e[i]) < INFINITY);
    }
#pragma unroll
    for (int offset = 1; offset < 16; offset *= 2)
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
    const unsigned broken_lanes = __ballot_sync(0xffffffffu, broken) >> (lane & 16) & 0xffff; /* of this unit */
    const int exponent = attend::half_exponent(largest);
    const float down = __int_as_float((127 - exponent) << 23), up = __int_as_float((127 + exponent) << 23);
    uint4 halves;
    halves.x = attend::pack<true>(low.e[0] * down, low.e[1] * down);
    halves.y = attend::pack<true>(low.e[2] * down, low.e[3] * down);
    halves.z = attend::pack<true>(high.e[0] * down, high.e[1] * down);
    halves.w = attend::pack<true>(high.e[2] * down, high.e[3] * down);
    if (!live)
        return;
    const int pass = row / task.pass_rows, column = row - pass * task.pass_rows;
    const int pass_live = min(task.pass_rows, task.rows - pass * task.pass_rows);
    const int ahead = power_bytes(task.pass_rows);
    uint8_t *base = task.tokens + (long long)pass * task.units * (ahead + task.pass_rows * kTokenBytes) +
                    (long long)unit * (ahead + pass_live * kTokenBytes);
    *reinterpret_cast<uint4 *>(base + ahead + column * kTokenBytes + (piece ^ (column & 1) * 4) * 16) = halves;
    if (piece == 0)
        reinterpret_cast<float *>(base)[column] = broken_lanes ? NAN : up;
}

/* A zero point of output g and of g + 8 as an operand's codes have theirs, twice. */
struct ZeroPair {
    uint32_t low, high;
};

__device__ __forceinline__ ZeroPair zero_pair(uint32_t two_bytes)
{
    return {(two_bytes & 0xff) * 0x00010001u, (two_bytes >> 8) * 0x00100010u};
}

constexpr uint32_t kNoZeros = 0x0808; /* the zero points without any */

__device__ __forceinline__ uint32_t subtract(uint32_t codes, uint32_t zeros)
{
    uint32_t r; /* exact: subnormal numbers, which this form does not flush */
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(codes), "r"(zeros));
    return r;
}

/* Row operand of one product: registers 0 and 2 are 2^-24 times the codes less the
 * zero point of output g, 1 and 3 are 2^-20 times those of output g + 8. */
__device__ __forceinline__ void unpack(uint32_t (&a)[4], uint32_t word, const ZeroPair &zero)
{
    a[0] = subtract(word & 0x000f000fu, zero.low), a[1] = subtract(word & 0x00f000f0u, zero.high);
    a[2] = subtract((word >> 8) & 0x000f000fu, zero.low), a[3] = subtract((word >> 8) & 0x00f000f0u, zero.high);
}

__device__ __forceinline__ float2 scale_pair(const float *from) { return *reinterpret_cast<const float2 *>(from); }
__device__ __forceinline__ float2 scale_pair(const __nv_bfloat16 *from)
{
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(from));
}

/* The scales of outputs g and g + 8 with the factors of their codes taken back, before a token's power
 * comes in: a small power times 2^-24 would leave FP32's normal numbers. */
__device__ __forceinline__ float2 raised(float2 scales) { return make_float2(scales.x * 0x1p24f, scales.y * 0x1p20f); }

/* C = 0 form of the product, for the first of a group. */
__device__ __forceinline__ void multiply_fresh(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float read_of_rank(uint32_t address, uint32_t rank)
{
    uint32_t there;
    float value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(there) : "memory");
    return value;
}

__device__ __forceinline__ void bulk_load(uint32_t to, const void *from, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                 "l"(from), "r"(bytes), "r"(sm100::smem_u32(bar))
                 : "memory");
}

/* What a stage of the ring holds: kUnits units of 64 outputs' weights, then of the
 * powers and tokens of the pass, `live` tokens each. */
template <int Columns, int Group, typename Scale, bool Zeros> struct Stage {
    static constexpr int kGroups = kUnit / Group;
    static constexpr int kTokens = 8 * Columns;
    static constexpr int kUnits = Columns > 2 ? 1 : 2;
    static constexpr int kStages = Columns > 2 ? 3 : 4;
    static constexpr int kTileBytes = tile_bytes<Group, Scale, Zeros>();
    static constexpr int kScalesAt = 16 * kUnit / 2, kZerosAt = kScalesAt + kGroups * 16 * int(sizeof(Scale));
    static constexpr int kPowerBytes = power_bytes(kTokens);
    static constexpr int kTokensAt = kUnits * kWarps * kTileBytes;
    /* The sums that the cluster exchanges, [token][output]: a warp reads 128 contiguous bytes of
     * another CTA (lane by lane from rows of their own took 12 us of 39 at 37 tokens, 42 of 66 at
     * 64), and the rows of two tokens apart start eight banks apart for the stores. */
    static constexpr int kPitch = kWarps * 16 + 4;
    static constexpr int kExchange = kTokens * kPitch * 4;
    static constexpr int kFitRegisters = Columns > 2 ? 3 : (Columns > 1 ? 5 : 7); /* CTAs on an SM */

    static __host__ __device__ constexpr int pass_bytes(int live) { return kPowerBytes + live * kTokenBytes; }
    static __host__ __device__ constexpr int bytes(int live) { return kTokensAt + kUnits * pass_bytes(live); }
    /* The ring; then room for the tokens that the last stage's columns without a token read (what
     * they give goes nowhere), so that every read stays in the allocation; then the barriers. */
    static __host__ __device__ constexpr int ring(int live)
    {
        return kStages * bytes(live) + (kTokens - live) * kTokenBytes > kExchange
                   ? kStages * bytes(live) + (kTokens - live) * kTokenBytes
                   : (kExchange + 15) / 16 * 16;
    }
    static __host__ __device__ constexpr int shared(int live) { return ring(live) + 16 * kStages + 16; }
    /* Whether every read of the products from the last stage, for columns without a token too, lies in
     * the ring, and a launch asks for no more than allow_shared_kernel does. A later pass of fewer tokens
     * reads less far in the ring of a full one. */
    static constexpr bool reads_inside()
    {
        for (int live = 1; live <= kTokens; ++live) {
            const int last_unit = (kStages - 1) * bytes(live) + kTokensAt + (kUnits - 1) * pass_bytes(live);
            const int tokens_end = last_unit + kPowerBytes + kTokens * kTokenBytes;
            if (tokens_end > ring(live) || kExchange > ring(live) || ring(live) % 16 ||
                shared(live) > shared(kTokens) || shared(live) > 227 * 1024)
                return false;
        }
        return true;
    }
    static int resident(int live)
    {
        const int fit = 228 * 1024 / (shared(live) + 1024);
        return fit < kFitRegisters ? fit : kFitRegisters;
    }
};

/* One CTA: 16 outputs per warp, up to 8 * Columns tokens, and the share of the
 * units that its rank in the cluster gives it. The last warp's first lane keeps
 * a ring of stages full with bulk copies, which cost the multiplying warps
 * nothing; a full and an empty barrier per stage hand it over. */
template <int Columns, int Group, typename Scale, bool Zeros>
__global__ void __launch_bounds__(kWarps * 32 + 32, Stage<Columns, Group, Scale, Zeros>::kFitRegisters)
    linear_kernel(const __grid_constant__ LinearTask task)
{
    typedef Stage<Columns, Group, Scale, Zeros> S;
    constexpr int kGroups = S::kGroups, kPerGroup = 8 / kGroups; /* groups of a unit, products of a group */
    constexpr int kStages = S::kStages, kUnits = S::kUnits;
    extern __shared__ __align__(16) uint8_t shared[];
    const int stage_bytes = S::bytes(min(S::kTokens, task.rows)); /* of the first pass, the fullest */
    uint64_t *full = reinterpret_cast<uint64_t *>(shared + S::ring(min(S::kTokens, task.rows)));
    uint64_t *empty = full + kStages;
    uint32_t *abort_word = reinterpret_cast<uint32_t *>(empty + kStages);
    volatile uint32_t *abort = abort_word;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int rank = blockIdx.x % task.split, block = blockIdx.x / task.split, pass = blockIdx.y;
    const int columns = pass * S::kTokens, live = min(S::kTokens, task.rows - columns);
    const int begin = int((long long)task.units * rank / task.split);
    const int end = int((long long)task.units * (rank + 1) / task.split);
    const int steps = (end - begin + kUnits - 1) / kUnits;
    /* Every CTA reads the same tokens; taken in the same order, all would ask one slice of the L2 for
     * the same lines at once. So a block of outputs starts at a step of its own and goes round. */
    const int turn = block % steps;
    const auto first_unit = [&](int step) {
        return begin + (step + turn < steps ? step + turn : step + turn - steps) * kUnits;
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s)
            sm100::mbar_init(&full[s], 1), sm100::mbar_init(&empty[s], kWarps);
        *abort = 0;
        sm100::fence_barrier_init();
    }
    __syncthreads();

    float sum[Columns][4];
#pragma unroll
    for (int n = 0; n < Columns; ++n)
        sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;

    int issued = 0; /* stages, by the producing thread */
    if (warp == kWarps) {
        if (lane == 0) {
            const uint8_t *weights = task.weights + (long long)block * task.units * (kWarps * S::kTileBytes);
            const uint8_t *tokens = task.tokens + (long long)pass * task.units * S::pass_bytes(S::kTokens);
            const uint32_t ring = sm100::smem_u32(shared);
            const auto load_weights = [&](int step) { /* after announcing the whole stage */
                const int stage = step % kStages, unit = first_unit(step), units = min(kUnits, end - unit);
                const uint32_t bytes = units * (kWarps * S::kTileBytes);
                sm100::mbar_arrive_expect_tx(&full[stage], bytes + units * S::pass_bytes(live));
                bulk_load(ring + stage * stage_bytes, weights + (long long)unit * (kWarps * S::kTileBytes), bytes,
                          &full[stage]);
            };
            const auto load_tokens = [&](int step) {
                const int stage = step % kStages, unit = first_unit(step), units = min(kUnits, end - unit);
                bulk_load(ring + stage * stage_bytes + S::kTokensAt, tokens + (long long)unit * S::pass_bytes(live),
                          units * S::pass_bytes(live), &full[stage]);
            };
            /* the weights are there already, the tokens when the kernel before this one has run */
            const int ahead = min(steps, kStages);
            for (int step = 0; step < ahead; ++step)
                load_weights(step);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int step = 0; step < ahead; ++step)
                load_tokens(step);
            issued = ahead;
            for (int step = ahead; step < steps; ++step) {
                if (!sm100::mbar_wait(&empty[step % kStages], (step / kStages - 1) & 1, abort)) {
                    sm100::report(task.status, abort, sm100::kRoleProducer);
                    break;
                }
                load_weights(step);
                load_tokens(step);
                ++issued;
            }
        }
        __syncwarp();
    } else {
        for (int step = 0; step < steps; ++step) {
            const int stage = step % kStages;
            if (!sm100::mbar_wait(&full[stage], (step / kStages) & 1, abort)) {
                sm100::report(task.status, abort, sm100::kRoleEpilogueFull);
                break;
            }
            const int unit = first_unit(step), units = min(kUnits, end - unit);
            const uint8_t *held = shared + stage * stage_bytes;
            /* odd tokens have their halves of 128 bytes swapped */
            const int even = 64 * (g & 1), odd = 64 - even;
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                if (u >= units)
                    break;
                const uint8_t *own = held + (u * kWarps + warp) * S::kTileBytes;
                const uint8_t *pass_unit = held + S::kTokensAt + u * S::pass_bytes(live);
                const uint8_t *token = pass_unit + S::kPowerBytes + g * kTokenBytes + 16 * t;
                const float *powers = reinterpret_cast<const float *>(pass_unit) + 2 * t;
                float part_sum[Columns][4]; /* of outputs g (0, 1) and g + 8, before the token's power */
#pragma unroll
                for (int n = 0; n < Columns; ++n)
                    part_sum[n][0] = part_sum[n][1] = part_sum[n][2] = part_sum[n][3] = 0.f;
                uint4 words;
#pragma unroll
                for (int i = 0; i < kGroups; ++i) {
                    const float2 s =
                        raised(scale_pair(reinterpret_cast<const Scale *>(own + S::kScalesAt) + 16 * i + 2 * g));
                    ZeroPair z = zero_pair(kNoZeros);
                    if constexpr (Zeros)
                        z = zero_pair(*reinterpret_cast<const uint16_t *>(own + S::kZerosAt + 16 * i + 2 * g));
                    float part[Columns][4];
#pragma unroll
                    for (int half = 0; half < kPerGroup / 2; ++half) { /* 32 inputs, two products */
                        const int piece = i * (kPerGroup / 2) + half;
                        if (piece % 2 == 0)
                            words = *reinterpret_cast<const uint4 *>(own + 512 * (piece / 2) + 16 * lane);
                        uint32_t a[2][4];
                        unpack(a[0], piece % 2 ? words.z : words.x, z), unpack(a[1], piece % 2 ? words.w : words.y, z);
#pragma unroll
                        for (int n = 0; n < Columns; ++n) {
                            const uint4 in = *reinterpret_cast<const uint4 *>(
                                token + 8 * n * kTokenBytes + (piece & 1 ? odd : even) + 128 * (piece / 2));
                            if (half == 0)
                                multiply_fresh(part[n], a[0], in.x, in.y);
                            else
                                attend::mma_16816<true>(part[n], a[0], in.x, in.y);
                            attend::mma_16816<true>(part[n], a[1], in.z, in.w);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < Columns; ++n) {
                        part_sum[n][0] = fmaf(s.x, part[n][0], part_sum[n][0]);
                        part_sum[n][1] = fmaf(s.x, part[n][1], part_sum[n][1]);
                        part_sum[n][2] = fmaf(s.y, part[n][2], part_sum[n][2]);
                        part_sum[n][3] = fmaf(s.y, part[n][3], part_sum[n][3]);
                    }
                }
#pragma unroll
                for (int n = 0; n < Columns; ++n) {
                    const float2 power = *reinterpret_cast<const float2 *>(powers + 8 * n);
                    sum[n][0] = fmaf(power.x, part_sum[n][0], sum[n][0]), sum[n][1] = fmaf(power.y, part_sum[n][1], sum[n][1]);
                    sum[n][2] = fmaf(power.x, part_sum[n][2], sum[n][2]), sum[n][3] = fmaf(power.y, part_sum[n][3], sum[n][3]);
                }
            }
            __syncwarp();
            if (lane == 0)
                sm100::mbar_arrive(&empty[stage]);
        }
    }
    /* The ring becomes the place where the cluster's sums meet. Every rank adds the ranges, in their
     * order, for its share of the outputs. */
    __syncthreads();
    const bool ok = *abort == 0;
    if (!ok && threadIdx.x == kWarps * 32) { /* a wait gave up: the copies under way get as long again */
        volatile uint32_t never = 0;
        for (int step = max(0, issued - kStages); step < issued; ++step)
            sm100::mbar_wait(&full[step % kStages], (step / kStages) & 1, &never);
    }
    float *exchange = reinterpret_cast<float *>(shared);
    if (ok && warp < kWarps) {
#pragma unroll
        for (int n = 0; n < Columns; ++n) {
            float *to = exchange + (8 * n + 2 * t) * S::kPitch + warp * 16 + g;
            to[0] = sum[n][0], to[S::kPitch] = sum[n][1];
            to[8] = sum[n][2], to[S::kPitch + 8] = sum[n][3];
        }
    }
    if (task.split > 1)
        cluster_barrier();
    else
        __syncthreads();
    constexpr int kOutputs = kWarps * 16;
    const uint32_t exchange_at = sm100::smem_u32(shared);
    for (int at = rank * int(blockDim.x) + threadIdx.x; ok && at < kOutputs * live; at += task.split * blockDim.x) {
        const int o = at % kOutputs, n = at / kOutputs;
        const int row = columns + n;
        const long long output = (long long)block * kOutputs + o;
        if (output >= task.outputs)
            continue;
        const uint32_t from = exchange_at + (n * S::kPitch + o) * 4;
        float range[8]; /* all ranks' sums are under way before the first is added */
#pragma unroll
        for (int r = 0; r < 8; ++r)
            range[r] = r < task.split ? read_of_rank(from, r) : 0.f;
        float value = range[0];
#pragma unroll
        for (int r = 1; r < 8; ++r)
            value += range[r];
        if (task.bias)
            value += __bfloat162float(task.bias[output]);
        if (task.residual)
            value += __bfloat162float(task.residual[row * task.ldr + output]);
        task.out[row * task.ldo + output] = __float2bfloat16_rn(value);
    }
    if (task.split > 1)
        cluster_barrier(); /* nobody's sums go while another rank reads them */
}

/* The scales of outputs g and g + 8. */
template <typename Scale> struct __align__(2 * sizeof(Scale)) ScalePair {
    Scale low, high;
};

/* The codes, scales and zero points of a unit of 16 outputs, as a lane holds them. */
template <int Groups, typename Scale, bool Zeros> struct Weights {
    uint4 words[2];
    ScalePair<Scale> scales[Groups];
    uint16_t zeros[Zeros ? Groups : 1];
};

/* Up to eight tokens. A CTA's four warps share 16 outputs and a rank's share of
 * the units, each a contiguous quarter of it; a warp streams its weights through
 * registers, kAhead units in flight, straight past the L1, and takes the tokens'
 * operands from the L1. */
template <int Group, typename Scale, bool Zeros>
__global__ void __launch_bounds__(kWarps * 32, 7) few_kernel(const __grid_constant__ LinearTask task)
{
    constexpr int kGroups = kUnit / Group, kPerGroup = 8 / kGroups, kAhead = 2;
    __shared__ float exchange[kWarps][8][16 + 4];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int rank = blockIdx.x % task.split;
    const long long tile = blockIdx.x / task.split;
    const int part = rank * kWarps + warp, parts = task.split * kWarps;
    const int begin = int((long long)task.units * part / parts), end = int((long long)task.units * (part + 1) / parts);

    constexpr int kTileBytes = tile_bytes<Group, Scale, Zeros>(), kScalesAt = 16 * kUnit / 2;
    const uint8_t *weights = task.weights + ((tile / 4 * task.units + begin) * 4 + tile % 4) * kTileBytes;
    Weights<kGroups, Scale, Zeros> held[kAhead];
    const auto fetch = [&](Weights<kGroups, Scale, Zeros> &to, int unit) {
        if (unit >= end)
            return;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(to.words[i].x), "=r"(to.words[i].y), "=r"(to.words[i].z), "=r"(to.words[i].w)
                         : "l"(weights + 512 * i + 16 * lane));
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            to.scales[i] = *reinterpret_cast<const ScalePair<Scale> *>(weights + kScalesAt +
                                                                       (16 * i + 2 * g) * int(sizeof(Scale)));
            if constexpr (Zeros)
                to.zeros[i] = *reinterpret_cast<const uint16_t *>(
                    weights + kScalesAt + kGroups * 16 * int(sizeof(Scale)) + 16 * i + 2 * g);
        }
        weights += 4 * kTileBytes;
    };
#pragma unroll
    for (int d = 0; d < kAhead; ++d)
        fetch(held[d], begin + d);
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int row = min(g, task.rows - 1); /* columns behind the last token repeat it */
    const int pitch = power_bytes(8) + task.rows * kTokenBytes;
    const uint8_t *unit_tokens = task.tokens + (long long)begin * pitch;
    const int token_at = power_bytes(8) + row * kTokenBytes + 16 * t, swap = row & 1;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int base = begin; base < end; base += kAhead) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            if (base + d >= end)
                break;
            uint4 in[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                in[i] = *reinterpret_cast<const uint4 *>(unit_tokens + token_at + 64 * (i ^ swap));
            const float2 power = *reinterpret_cast<const float2 *>(unit_tokens + 8 * t);
            float2 low = make_float2(0.f, 0.f), high = make_float2(0.f, 0.f); /* outputs g and g + 8 */
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                ZeroPair z = zero_pair(kNoZeros);
                if constexpr (Zeros)
                    z = zero_pair(held[d].zeros[i]);
                float part_sum[kPerGroup > 2 ? 2 : 1][4];
#pragma unroll
                for (int j = 0; j < kPerGroup; ++j) {
                    const int product = i * kPerGroup + j, chain = kPerGroup > 2 ? j % 2 : 0;
                    const uint4 &w = held[d].words[product / 4], &v = in[product / 2];
                    const uint32_t word = product % 4 == 0 ? w.x : (product % 4 == 1 ? w.y : (product % 4 == 2 ? w.z : w.w));
                    const uint32_t b0 = product % 2 ? v.z : v.x, b1 = product % 2 ? v.w : v.y;
                    uint32_t a[4];
                    unpack(a, word, z);
                    if (j == chain)
                        multiply_fresh(part_sum[chain], a, b0, b1);
                    else
                        attend::mma_16816<true>(part_sum[chain], a, b0, b1);
                }
                if constexpr (kPerGroup > 2) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        part_sum[0][e] += part_sum[1][e];
                }
                const float2 s = raised(make_float2(float(held[d].scales[i].low), float(held[d].scales[i].high)));
                low.x = fmaf(s.x, part_sum[0][0], low.x), low.y = fmaf(s.x, part_sum[0][1], low.y);
                high.x = fmaf(s.y, part_sum[0][2], high.x), high.y = fmaf(s.y, part_sum[0][3], high.y);
            }
            fetch(held[d], base + d + kAhead);
            sum[0] = fmaf(power.x, low.x, sum[0]), sum[1] = fmaf(power.y, low.y, sum[1]);
            sum[2] = fmaf(power.x, high.x, sum[2]), sum[3] = fmaf(power.y, high.y, sum[3]);
            unit_tokens += pitch;
        }
    }
    exchange[warp][2 * t][g] = sum[0], exchange[warp][2 * t + 1][g] = sum[1];
    exchange[warp][2 * t][g + 8] = sum[2], exchange[warp][2 * t + 1][g + 8] = sum[3];
    if (task.split > 1)
        cluster_barrier();
    else
        __syncthreads();
    /* rank 0 adds the quarters of all ranks in the order of the units */
    const int o = threadIdx.x % 16, n = threadIdx.x / 16;
    const long long output = tile * 16 + o;
    if (rank == 0 && n < task.rows && output < task.outputs) {
        float value = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r >= task.split)
                break;
            float quarter[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                quarter[w] = read_of_rank(sm100::smem_u32(&exchange[w][n][o]), r);
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                value += quarter[w];
        }
        if (task.bias)
            value += __bfloat162float(task.bias[output]);
        if (task.residual)
            value += __bfloat162float(task.residual[n * task.ldr + output]);
        task.out[n * task.ldo + output] = __float2bfloat16_rn(value);
    }
    if (task.split > 1)
        cluster_barrier(); /* nobody's sums go while another rank reads them */
}

/* Ranges of the units per block of outputs (the ranks of a cluster), by a rough
 * model of the time: a CTA alone on an SM takes `alone` for a unit, k CTAs
 * together `shared` each (what HBM gives an SM, or the products of the columns),
 * and CTAs that do not fit wait. Measured (37 tokens, 7168 -> 4992, groups of
 * 128): 39.8, 30.9, 22.9, 21.2 and 24.9 us with 1, 2, 3, 4 and 7 ranges, the
 * chosen number 20.4; 64 outputs alone would leave 147 SMs without work. */
inline int choose_split(int blocks, int units, int step, int columns, int sm_count, int resident)
{
    const double alone = 0.15 + 0.06 * columns, shared = 0.05 * columns > 0.1 ? 0.05 * columns : 0.1;
    int best = 1;
    double best_time = 1e30;
    for (int split = 1; split <= 8 && (split == 1 || units / split >= 2 * step); ++split) {
        const long long per_sm = ((long long)blocks * split + sm_count - 1) / sm_count;
        const long long rounds = per_sm / resident, rest = per_sm % resident;
        const auto together = [&](long long k) { return k == 0 ? 0. : (k * shared > alone ? k * shared : alone); };
        const double time = double((units + split - 1) / split) * (rounds * together(resident) + together(rest)) +
                            (split > 1 ? 0.5 + 0.1 * split : 0.);
        if (time < best_time)
            best = split, best_time = time;
    }
    return best;
}

template <int Columns, int Group, typename Scale, bool Zeros>
cudaError_t launch_kernel(camblas_cuda_context *context, LinearTask task)
{
    typedef Stage<Columns, Group, Scale, Zeros> S;
    static_assert(S::reads_inside(), "shared memory of a stage");
    const int blocks = (task.outputs + kWarps * 16 - 1) / (kWarps * 16);
    const int passes = (task.rows + S::kTokens - 1) / S::kTokens;
    const int live = task.rows < S::kTokens ? task.rows : S::kTokens;
    task.split = choose_split(blocks * passes, task.units, S::kUnits, (live + 7) / 8, context->sm_count,
                              S::resident(live));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks * task.split, passes);
    config.blockDim = dim3(kWarps * 32 + 32);
    config.dynamicSmemBytes = S::shared(live);
    config.stream = context->stream;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = task.split;
    attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, linear_kernel<Columns, Group, Scale, Zeros>, task);
}

/* Ranges of the units per tile for up to eight tokens: as many as load the SMs
 * most evenly within the seven CTAs of an SM, at least three units to a warp. */
inline int choose_few_split(int tiles, int units, int sm_count)
{
    int best = 1;
    double best_load = 0;
    for (int split = 1; split <= 8 && (split == 1 || units / (split * kWarps) >= 3); ++split) {
        const long long ctas = (long long)tiles * split, full = 7ll * sm_count;
        const long long per_sm = (ctas + sm_count - 1) / sm_count;
        const long long slots = per_sm <= 7 ? per_sm * sm_count : (ctas + full - 1) / full * full;
        /* even, and four CTAs on an SM at least: fewer do not keep HBM busy */
        const double load = double(ctas) / double(slots) * (per_sm < 4 ? per_sm / 4. : 1.);
        if (load > best_load + 0.02)
            best = split, best_load = load;
    }
    return best;
}

template <int Group, typename Scale> cudaError_t launch_few(camblas_cuda_context *context, LinearTask task, bool zeros)
{
    const int tiles = (task.outputs + 15) / 16;
    task.split = choose_few_split(tiles, task.units, context->sm_count);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(tiles * task.split);
    config.blockDim = dim3(kWarps * 32);
    config.stream = context->stream;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = task.split;
    attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 2;
    return zeros ? cudaLaunchKernelEx(&config, few_kernel<Group, Scale, true>, task)
                 : cudaLaunchKernelEx(&config, few_kernel<Group, Scale, false>, task);
}

template <int Columns, int Group, typename Scale>
cudaError_t launch(camblas_cuda_context *context, const LinearTask &task, bool zeros)
{
    return zeros ? launch_kernel<Columns, Group, Scale, true>(context, task)
                      : launch_kernel<Columns, Group, Scale, false>(context, task);
}

template <int Columns, int Group, typename Scale, bool Zeros> int allow_shared_kernel()
{
    const auto kernel = linear_kernel<Columns, Group, Scale, Zeros>;
    /* without the preference the driver sets up the SMs for one CTA of a cluster launch each */
    return int(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Stage<Columns, Group, Scale, Zeros>::shared(8 * Columns))) |
           int(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared));
}

template <int Columns, int Group, typename Scale> int allow_shared()
{
    return allow_shared_kernel<Columns, Group, Scale, true>() | allow_shared_kernel<Columns, Group, Scale, false>();
}

template <int Group, typename Scale> int allow_shared_group()
{
    return allow_shared<1, Group, Scale>() | allow_shared<2, Group, Scale>() | allow_shared<4, Group, Scale>() |
           allow_shared<6, Group, Scale>() | allow_shared<8, Group, Scale>();
}

/* Raises the shared-memory limit of every instance on the current device. */
inline int prepare_kernels()
{
    return allow_shared_group<32, float>() | allow_shared_group<64, float>() | allow_shared_group<128, float>() |
           allow_shared_group<32, __nv_bfloat16>() | allow_shared_group<64, __nv_bfloat16>() |
           allow_shared_group<128, __nv_bfloat16>();
}

template <int Group, typename Scale>
cudaError_t launch_rows(camblas_cuda_context *context, const LinearTask &task, bool zeros)
{
    /* few_kernel while one wave of its CTAs has a place for every tile of outputs (16576 outputs); with
     * more, the block kernel keeps its ring full where few_kernel would start anew. One token, groups of
     * 128, few_kernel and block kernel in us:
     *   outputs            8192        12288       16384       18432       20480       24576       28672
     *   4096 inputs     8.4   8.9   10.1  10.9  11.4  15.7  18.1  14.2  18.7  18.5  20.7  17.0  18.1  23.5
     *   8192 inputs    12.4  16.9   24.6  19.2  18.1  23.7  37.6  22.8  37.0  27.7  31.4  32.1  48.7  41.4
     *   16384 inputs   19.5  25.1   37.0  31.4  31.4  37.9  67.1  36.7  56.1  43.6  52.6  50.4  74.5  63.6
     * and the same order with two, four and eight, except where they are within a tenth. The rule is wrong
     * at 12288 outputs of wide inputs, whose split few_kernel chooses over several waves, and at 28672
     * outputs of 4096 inputs. */
    if (task.rows <= 8)
        return (task.outputs + 15) / 16 <= 7ll * context->sm_count ? launch_few<Group, Scale>(context, task, zeros)
                                                                   : launch<1, Group, Scale>(context, task, zeros);
    if (task.rows <= 16)
        return launch<2, Group, Scale>(context, task, zeros);
    if (task.rows <= 32)
        return launch<4, Group, Scale>(context, task, zeros);
    if (task.rows <= 48)
        return launch<6, Group, Scale>(context, task, zeros);
    return launch<8, Group, Scale>(context, task, zeros);
}

template <int Group> int run(camblas_cuda_context *context, const LinearTask &task, int scale_type, bool zeros)
{
    const dim3 grid((task.units + 15) / 16, task.rows);
    spread_tokens<<<grid, 256, 0, context->stream>>>(task);
    int status = host::launched(context, "4-bit linear tokens");
    if (status != 0)
        return status;
    const cudaError_t error = scale_type == 0 ? launch_rows<Group, float>(context, task, zeros)
                                              : launch_rows<Group, __nv_bfloat16>(context, task, zeros);
    if (error != cudaSuccess)
        return host::fail(context, "4-bit linear", error);
    context->kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return 0;
}

inline bool sizes_bad(int rows, int inner, int group)
{
    return rows < 0 || rows > 65535 || inner < 32 || inner > INT_MAX - 128 ||
           (group != 32 && group != 64 && group != 128) || inner % group;
}

/* Tokens of a pass: all of them where that goes. */
inline int rows_of_pass(int rows)
{
    return rows <= 8 ? 8 : (rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 48 ? 48 : 64)));
}

inline size_t workspace_bytes(int rows, int inner)
{
    const size_t units = (inner + kUnit - 1) / kUnit, pass_rows = rows_of_pass(rows);
    const size_t passes = (rows + pass_rows - 1) / pass_rows;
    return units * (passes * power_bytes(int(pass_rows)) + size_t(rows) * kTokenBytes);
}

} // namespace nibble

extern "C" size_t camblas_cuda_int4_linear_workspace(const camblas_cuda_context *context, int rows, int inner,
                                                     int group)
{
    if (!context || rows == 0 || nibble::sizes_bad(rows, inner, group))
        return 0;
    return nibble::workspace_bytes(rows, inner);
}

extern "C" int camblas_cuda_int4_linear(camblas_cuda_context *context, int rows, int inner, int outputs,
                                        int group, const void *x, long long ldx, const void *weights,
                                        int scale_type, int zeros, const void *bias, const void *residual,
                                        long long ldr, void *workspace, size_t workspace_bytes, void *out,
                                        long long ldo)
{
    return host::guarded(context, [&] {
        if (nibble::sizes_bad(rows, inner, group) || outputs < 1 || outputs > INT_MAX - 64 ||
            (scale_type != 0 && scale_type != 2) || (zeros != 0 && zeros != 1) ||
            (rows > 1 && (ldx < inner || ldo < outputs || (residual && ldr < outputs))))
            return host::fail(context, "invalid 4-bit linear dimensions", 1);
        if (rows == 0)
            return 0;
        if (!x || !weights || !out || heads::misaligned(x, 16) || (rows > 1 && ldx % 8) ||
            heads::misaligned(weights, 16) || heads::misaligned(bias, 2) || heads::misaligned(residual, 2) ||
            heads::misaligned(out, 2) || out == x || out == weights || (bias && out == bias))
            return host::fail(context, "invalid 4-bit linear operands", 1);
        if (!workspace || workspace_bytes < nibble::workspace_bytes(rows, inner) ||
            heads::misaligned(workspace, 16) || workspace == out)
            return host::fail(context, "4-bit linear workspace too small", 1);
        nibble::LinearTask task{};
        task.rows = rows, task.inner = inner, task.outputs = outputs;
        task.units = (inner + nibble::kUnit - 1) / nibble::kUnit, task.pass_rows = nibble::rows_of_pass(rows);
        task.x = static_cast<const __nv_bfloat16 *>(x), task.ldx = ldx;
        task.weights = static_cast<const uint8_t *>(weights);
        task.bias = static_cast<const __nv_bfloat16 *>(bias);
        task.residual = static_cast<const __nv_bfloat16 *>(residual), task.ldr = ldr;
        task.out = static_cast<__nv_bfloat16 *>(out), task.ldo = ldo;
        task.tokens = static_cast<uint8_t *>(workspace);
        task.status = context->status;
        context->counts[0]++;
        if (group == 32)
            return nibble::run<32>(context, task, scale_type, zeros != 0);
        if (group == 64)
            return nibble::run<64>(context, task, scale_type, zeros != 0);
        return nibble::run<128>(context, task, scale_type, zeros != 0);
    });
}
