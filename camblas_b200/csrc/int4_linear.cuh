/*
 * Linear layer for a few tokens with 4-bit weights and group scales.
 *
 *   out[r,o] = sum over groups G of s[o,G] * sum_{k in G} (c[o,k] - z[o,G]) x[r,k]
 *              (+ bias[o]) (+ residual[r,o]),
 * codes c and zero points z in 0..15 (z = 8 without zero points), groups of 32,
 * 64 or 128 input features. c - z is a whole number of at most 15 and exact in
 * BF16, so the products run on the tensor cores over exact operands; the FP32
 * sums of a group are scaled in FP32, and the result is rounded once. Scaling
 * the weights themselves to BF16 before the product would round each of them.
 *
 * HBM bounds it: half a byte per weight and two operations per weight and
 * token. Warp tiles of 16 outputs with mma.m16n8k16: the outputs take the
 * 16-row side, up to eight tokens the column side, so one token costs the
 * tensor cores no more than eight. The codes are laid out once, when the weight
 * is loaded, in the order the lanes want them: a lane's 16 bytes hold its row
 * operands of four products, 64 input features of 16 outputs are 512 contiguous
 * bytes per warp, and the word of a product is unpacked by
 *   (word >> 4e) & 0x000f000f | 0x43004300 = the BF16 pair 128 + c,
 * less the BF16 pair 128 + z, both exact. The input features of a product are
 * assigned to the operand's k positions so that a lane's four products want
 * eight contiguous inputs of a token from each half of the 64: two 16-byte
 * loads of x as it lies.
 *
 * Layout: codes [tile of 16 outputs][block of 64 inputs][lane = 4g + t][word
 * i = 2h + m]; word i holds for inputs k = 64 block + 32h + 8t + 4m + j,
 * j = 0..3, and outputs 16 tile + g + 8r, r = 0..1, the code at nibble
 * r + 2 (j / 2) + 4 (j % 2). Scales (and zero points, one byte each)
 * [tile][group][g][r]. Outputs are padded to 16 and inputs to 64 with any code
 * and scale zero.
 */
#pragma once

#include "context.cuh"
#include "head_rotate.cuh"
#include "paged_attention.cuh"

namespace nibble
{

constexpr int kWarps = 8;

struct LinearTask {
    int rows, inner, outputs, group_shift, groups, blocks; /* group = 1 << group_shift, blocks of 64 */
    const __nv_bfloat16 *x;
    long long ldx;
    const uint4 *codes;
    const void *scales;
    const uint8_t *zeros;
    const __nv_bfloat16 *bias, *residual;
    long long ldr;
    __nv_bfloat16 *out;
    long long ldo;
};

__device__ __forceinline__ float2 load_scales(const float *from) { return *reinterpret_cast<const float2 *>(from); }
__device__ __forceinline__ float2 load_scales(const __nv_bfloat16 *from)
{
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(from));
}

/* BF16 pair 128 + n for a whole number n below 128 */
__device__ __forceinline__ uint32_t shifted_pair(uint32_t n) { return (n | (n << 16)) | 0x43004300u; }

__device__ __forceinline__ uint32_t subtract_pairs(uint32_t a, uint32_t b)
{
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                     *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&d);
}

/* Row operand of one product: registers 0 and 2 are output g, 1 and 3 output g + 8. */
__device__ __forceinline__ void unpack(uint32_t (&a)[4], uint32_t word, uint32_t zero_low, uint32_t zero_high)
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
        a[e] = subtract_pairs(((word >> (4 * e)) & 0x000f000fu) | 0x43004300u, e & 1 ? zero_high : zero_low);
}

/* One CTA: 16 outputs, up to 8*Columns tokens; its warps take the blocks of 64
 * inputs in turn and are added at the end in warp order. */
template <int Columns, typename Scale, bool Zeros>
__global__ void __launch_bounds__(kWarps * 32) linear_kernel(const LinearTask task)
{
    __shared__ float sums[kWarps][16][8 * Columns + 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const long long tile = blockIdx.x;
    const int first_row = blockIdx.y * 8 * Columns;
    const uint4 *codes = task.codes + tile * task.blocks * 32 + lane;
    const Scale *scales = static_cast<const Scale *>(task.scales) + tile * task.groups * 16 + 2 * g;
    const uint8_t *zeros = Zeros ? task.zeros + tile * task.groups * 16 + 2 * g : nullptr;
    const __nv_bfloat16 *x[Columns];
    bool live[Columns];
#pragma unroll
    for (int n = 0; n < Columns; ++n) {
        const int row = first_row + 8 * n + g;
        live[n] = row < task.rows;
        x[n] = task.x + (live[n] ? row : 0) * task.ldx + 8 * t;
    }
    float sum[Columns][4];
#pragma unroll
    for (int n = 0; n < Columns; ++n)
        sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;

#pragma unroll 4
    for (int block = warp; block < task.blocks; block += kWarps) {
        const uint4 word = codes[(long long)block * 32];
        const uint32_t words[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = 64 * block + 32 * half;
            if (k >= task.inner)
                break;
            const int group = k >> task.group_shift;
            const float2 scale = load_scales(scales + group * 16);
            uint32_t zero_low = 0x43084308u, zero_high = 0x43084308u;
            if constexpr (Zeros) {
                const uchar2 zero = *reinterpret_cast<const uchar2 *>(zeros + group * 16);
                zero_low = shifted_pair(zero.x), zero_high = shifted_pair(zero.y);
            }
            uint32_t a[2][4];
            unpack(a[0], words[2 * half], zero_low, zero_high);
            unpack(a[1], words[2 * half + 1], zero_low, zero_high);
#pragma unroll
            for (int n = 0; n < Columns; ++n) {
                uint4 in = make_uint4(0, 0, 0, 0);
                if (live[n])
                    in = *reinterpret_cast<const uint4 *>(x[n] + k);
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                attend::mma_16816<false>(part, a[0], in.x, in.y);
                attend::mma_16816<false>(part, a[1], in.z, in.w);
                sum[n][0] = fmaf(part[0], scale.x, sum[n][0]), sum[n][1] = fmaf(part[1], scale.x, sum[n][1]);
                sum[n][2] = fmaf(part[2], scale.y, sum[n][2]), sum[n][3] = fmaf(part[3], scale.y, sum[n][3]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < Columns; ++n) {
        sums[warp][g][8 * n + 2 * t] = sum[n][0], sums[warp][g][8 * n + 2 * t + 1] = sum[n][1];
        sums[warp][g + 8][8 * n + 2 * t] = sum[n][2], sums[warp][g + 8][8 * n + 2 * t + 1] = sum[n][3];
    }
    __syncthreads();
    for (int at = threadIdx.x; at < 16 * 8 * Columns; at += kWarps * 32) {
        const int o = at % 16, n = at / 16;
        const int row = first_row + n;
        const long long output = tile * 16 + o;
        if (row >= task.rows || output >= task.outputs)
            continue;
        float value = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            value += sums[w][o][n];
        if (task.bias)
            value += __bfloat162float(task.bias[output]);
        if (task.residual)
            value += __bfloat162float(task.residual[row * task.ldr + output]);
        task.out[row * task.ldo + output] = __float2bfloat16_rn(value);
    }
}

template <int Columns, typename Scale> void launch(camblas_cuda_context *context, const LinearTask &task)
{
    const dim3 grid((task.outputs + 15) / 16, (task.rows + 8 * Columns - 1) / (8 * Columns));
    if (task.zeros)
        linear_kernel<Columns, Scale, true><<<grid, kWarps * 32, 0, context->stream>>>(task);
    else
        linear_kernel<Columns, Scale, false><<<grid, kWarps * 32, 0, context->stream>>>(task);
}

template <typename Scale> void launch_rows(camblas_cuda_context *context, const LinearTask &task)
{
    if (task.rows <= 8)
        launch<1, Scale>(context, task);
    else if (task.rows <= 16)
        launch<2, Scale>(context, task);
    else
        launch<4, Scale>(context, task);
}

} // namespace nibble

extern "C" int camblas_cuda_int4_linear(camblas_cuda_context *context, int rows, int inner, int outputs,
                                        int group, const void *x, long long ldx, const void *codes,
                                        int scale_type, const void *scales, const void *zeros,
                                        const void *bias, const void *residual, long long ldr, void *out,
                                        long long ldo)
{
    return host::guarded(context, [&] {
        if (rows < 0 || rows > 65535 || outputs < 1 || inner < 32 || (group != 32 && group != 64 && group != 128) ||
            inner % group || inner > INT_MAX - 64 || outputs > INT_MAX - 16 ||
            (scale_type != 0 && scale_type != 2) ||
            (rows > 1 && (ldx < inner || ldo < outputs || (residual && ldr < outputs))))
            return host::fail(context, "invalid 4-bit linear dimensions", 1);
        if (rows == 0)
            return 0;
        if (!x || !codes || !scales || !out || heads::misaligned(x, 16) || ldx % 8 || heads::misaligned(codes, 16) ||
            heads::misaligned(scales, 8) || heads::misaligned(zeros, 2) || heads::misaligned(bias, 2) ||
            heads::misaligned(residual, 2) || heads::misaligned(out, 2) || out == x || out == codes ||
            out == scales || (bias && out == bias))
            return host::fail(context, "invalid 4-bit linear operands", 1);
        nibble::LinearTask task{};
        task.rows = rows, task.inner = inner, task.outputs = outputs;
        task.group_shift = group == 32 ? 5 : (group == 64 ? 6 : 7);
        task.groups = inner / group, task.blocks = (inner + 63) / 64;
        task.x = static_cast<const __nv_bfloat16 *>(x), task.ldx = ldx;
        task.codes = static_cast<const uint4 *>(codes), task.scales = scales;
        task.zeros = static_cast<const uint8_t *>(zeros);
        task.bias = static_cast<const __nv_bfloat16 *>(bias);
        task.residual = static_cast<const __nv_bfloat16 *>(residual), task.ldr = ldr;
        task.out = static_cast<__nv_bfloat16 *>(out), task.ldo = ldo;
        context->counts[0]++;
        if (scale_type == 0)
            nibble::launch_rows<float>(context, task);
        else
            nibble::launch_rows<__nv_bfloat16>(context, task);
        return host::launched(context, "4-bit linear");
    });
}
