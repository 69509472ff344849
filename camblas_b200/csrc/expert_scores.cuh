/*
 * Router of a mixture of experts: scores, choice and weights.
 *
 * For a token's logits x[experts]:
 *   score s = softmax(x) or 1/(1+exp(-x)),   rank r = s + bias (bias NULL: r = s);
 *   the experts lie in `groups` equal groups; a group's rank is the sum of its
 *   two largest r (its only one when it has one expert); the `kept` groups of
 *   largest rank stay;
 *   the `choices` experts of largest r in them are chosen, in descending order;
 *   weight = s (renormalised: s / sum of the chosen s) * scale.
 * Equal ranks go to the lower index. Ranks are compared in FP64: scores of
 * different experts may lie closer than FP32 can tell, and which expert is
 * chosen is a whole number that no tolerance covers. A NaN ranks behind every
 * number.
 *
 * One warp per token, expert e on lane e % 32.
 */
#pragma once

#include "context.cuh"

namespace routing
{

constexpr int kMostExperts = 1024;
constexpr int kMostChoices = 32;

struct ScoreTask {
    int tokens, experts, choices, groups, kept;
    int sigmoid, renormalise;
    float scale;
    const void *logits;
    long long ld_logits;
    const float *bias;
    int64_t *chosen;
    float *weights;
};

__device__ __forceinline__ float load_logit(const float *from) { return *from; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16 *from) { return __bfloat162float(*from); }

constexpr long long kRemoved = -0x7fffffffffffffffll - 1;
constexpr long long kNan = kRemoved + 1;

/* Integer whose order is that of the numbers (-0 and +0 are one number). */
__device__ __forceinline__ long long order_of(double x)
{
    if (x != x)
        return kNan;
    const long long bits = __double_as_longlong(x + 0.0);
    return bits < 0 ? bits ^ 0x7fffffffffffffffll : bits;
}

__device__ __forceinline__ double shuffle_xor(double x, int offset)
{
    return __shfl_xor_sync(0xffffffffu, x, offset);
}

/* The lane and index of the largest key of the warp, the lowest index among
 * equals; index is an expert number or INT_MAX. */
__device__ __forceinline__ void warp_best(long long &key, int &index)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) {
        const long long other = __shfl_xor_sync(0xffffffffu, key, offset);
        const int other_index = __shfl_xor_sync(0xffffffffu, index, offset);
        if (other > key || (other == key && other_index < index))
            key = other, index = other_index;
    }
}

template <int PerLane, typename T>
__global__ void __launch_bounds__(128) score_kernel(const ScoreTask task)
{
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (blockDim.x / 32);
    for (int token = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; token < task.tokens;
         token += warps) {
        const T *row = static_cast<const T *>(task.logits) + token * task.ld_logits;
        double score[PerLane];
        long long key[PerLane];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < PerLane; ++i) {
            const int e = i * 32 + lane;
            const float x = e < task.experts ? load_logit(row + e) : -INFINITY;
            score[i] = x;
            top = fmaxf(top, x);
        }
        if (task.sigmoid) {
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                score[i] = 1.0 / (1.0 + exp(-score[i]));
        } else {
#pragma unroll
            for (int offset = 16; offset > 0; offset /= 2)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
            if (top == -INFINITY) /* no expert is open: all scores are zero */
                top = 0.f;
            double sum = 0;
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                score[i] = exp(score[i] - top), sum += score[i];
#pragma unroll
            for (int offset = 16; offset > 0; offset /= 2)
                sum += shuffle_xor(sum, offset);
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                score[i] = sum != 0 ? score[i] / sum : 0.0;
        }
#pragma unroll
        for (int i = 0; i < PerLane; ++i) {
            const int e = i * 32 + lane;
            key[i] = e < task.experts ? order_of(score[i] + (task.bias ? double(task.bias[e]) : 0.0))
                                      : kRemoved;
        }
        if (task.groups > 1) {
            const int size = task.experts / task.groups;
            long long mine = kRemoved; /* lane g: the rank of group g */
            for (int group = 0; group < task.groups; ++group) {
                long long first = kRemoved, second = kRemoved;
#pragma unroll
                for (int i = 0; i < PerLane; ++i) {
                    const int e = i * 32 + lane;
                    if (e >= group * size && e < (group + 1) * size) {
                        if (key[i] > first)
                            second = first, first = key[i];
                        else if (key[i] > second)
                            second = key[i];
                    }
                }
#pragma unroll
                for (int offset = 16; offset > 0; offset /= 2) {
                    const long long a = __shfl_xor_sync(0xffffffffu, first, offset);
                    const long long b = __shfl_xor_sync(0xffffffffu, second, offset);
                    const long long lower = a < first ? a : first;
                    first = a > first ? a : first;
                    second = second > b ? second : b;
                    second = second > lower ? second : lower;
                }
                const auto value = [](long long k) {
                    return k <= kNan ? double(NAN)
                                     : __longlong_as_double(k < 0 ? k ^ 0x7fffffffffffffffll : k);
                };
                const long long rank =
                    order_of(size > 1 ? value(first) + value(second) : value(first));
                if (lane == group)
                    mine = rank;
            }
            unsigned keep = 0;
            for (int round = 0; round < task.kept; ++round) {
                long long best = mine;
                int at = mine == kRemoved ? INT_MAX : lane;
                warp_best(best, at);
                if (at != INT_MAX)
                    keep |= 1u << at;
                if (lane == at)
                    mine = kRemoved;
            }
#pragma unroll
            for (int i = 0; i < PerLane; ++i) {
                const int e = i * 32 + lane;
                if (e < task.experts && !((keep >> (e / size)) & 1))
                    key[i] = kRemoved;
            }
        }
        int my_choice = 0;
        double my_score = 0;
        for (int round = 0; round < task.choices; ++round) {
            long long best = kRemoved;
            int index = INT_MAX;
            double held = 0;
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                if (key[i] > best)
                    best = key[i], index = i * 32 + lane, held = score[i];
            warp_best(best, index);
            held = __shfl_sync(0xffffffffu, held, index & 31);
            if (lane == round)
                my_choice = index, my_score = held;
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                if (index == i * 32 + lane)
                    key[i] = kRemoved;
        }
        double total = my_score;
        if (task.renormalise) {
#pragma unroll
            for (int offset = 16; offset > 0; offset /= 2)
                total += shuffle_xor(total, offset);
            my_score = total != 0 ? my_score / total : 0.0;
        }
        if (lane < task.choices) {
            const long long at = (long long)token * task.choices + lane;
            task.chosen[at] = my_choice;
            task.weights[at] = float(my_score * double(task.scale));
        }
    }
}

template <typename T> void launch(camblas_cuda_context *context, const ScoreTask &task)
{
    const long long blocks = (task.tokens + 3ll) / 4;
    const unsigned grid = unsigned(blocks < 65536 ? blocks : 65536);
    const int per_lane = (task.experts + 31) / 32;
    if (per_lane <= 1)
        score_kernel<1, T><<<grid, 128, 0, context->stream>>>(task);
    else if (per_lane <= 2)
        score_kernel<2, T><<<grid, 128, 0, context->stream>>>(task);
    else if (per_lane <= 4)
        score_kernel<4, T><<<grid, 128, 0, context->stream>>>(task);
    else if (per_lane <= 8)
        score_kernel<8, T><<<grid, 128, 0, context->stream>>>(task);
    else if (per_lane <= 16)
        score_kernel<16, T><<<grid, 128, 0, context->stream>>>(task);
    else
        score_kernel<32, T><<<grid, 128, 0, context->stream>>>(task);
}

} // namespace routing

extern "C" int camblas_cuda_route_experts(camblas_cuda_context *context, int dtype, int tokens,
                                          int experts, int choices, int sigmoid, int groups,
                                          int kept_groups, int renormalise, float scale,
                                          const void *logits, long long ld_logits,
                                          const float *bias, void *chosen, float *weights)
{
    return host::guarded(context, [&] {
        if ((dtype != 0 && dtype != 2) || tokens < 0 || experts < 1 ||
            experts > routing::kMostExperts || choices < 1 || choices > routing::kMostChoices ||
            groups < 1 || groups > 32 || experts % groups || kept_groups < 1 ||
            kept_groups > groups || choices > kept_groups * (experts / groups) ||
            (sigmoid != 0 && sigmoid != 1) || (renormalise != 0 && renormalise != 1) ||
            !std::isfinite(scale) || (tokens > 1 && ld_logits < experts))
            return host::fail(context, "invalid expert scoring dimensions", 1);
        if (tokens == 0)
            return 0;
        if (!logits || !chosen || !weights ||
            (reinterpret_cast<uintptr_t>(logits) & (dtype == 0 ? 3 : 1)) ||
            (reinterpret_cast<uintptr_t>(bias) & 3) || (reinterpret_cast<uintptr_t>(chosen) & 7) ||
            (reinterpret_cast<uintptr_t>(weights) & 3) || chosen == logits || weights == logits ||
            chosen == static_cast<void *>(weights) || weights == bias || chosen == bias)
            return host::fail(context, "invalid expert scoring operands", 1);
        const routing::ScoreTask task{tokens,      experts, choices, groups,    kept_groups,
                                      sigmoid,     renormalise, scale, logits,  ld_logits,
                                      bias,        static_cast<int64_t *>(chosen), weights};
        if (dtype == 0)
            routing::launch<float>(context, task);
        else
            routing::launch<__nv_bfloat16>(context, task);
        return host::launched(context, "expert scoring");
    });
}
