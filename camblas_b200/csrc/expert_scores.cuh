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
 * Equal ranks go to the lower index, and a NaN ranks behind every number.
 *
 * Which expert is chosen is a whole number that no tolerance covers, and ranks
 * may lie closer than FP32 can tell: they are compared in FP64. Without bias and
 * groups the choice is made on the logits themselves, with which both scores grow;
 * otherwise on FP32 ranks, whose error is bounded. It is made again on FP64 ranks
 * for a token where two ranks that decide anything lie within that bound (a few
 * tokens in a thousand; every FP64 exponential costs some forty instructions of a
 * rate of one in two), or where distinct logits that decide anything may have one
 * FP64 score (saturated sigmoids, exponentials that underflow). The weights are
 * FP64 throughout, which is cheap for the chosen few: renormalised softmax weights
 * do not need the sum over all.
 *
 * One warp per token, expert e on lane e % 32; a round of the choice is a local
 * maximum and two warp reductions of 32-bit keys that are ordered like the ranks.
 * Issue bounds the kernel, not its few bytes per token: some 700 instructions for
 * a token's eight of 128 experts, 16384 tokens in 14.9 us (28 with FP64 ranks for
 * all), 62 us with a bias and eight of 256 experts in eight groups; one token among
 * those takes 7.0 us, the latency of its chain of reductions.
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

/* The key and index of the largest key of the warp, the lowest index among
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

/* exp(x) for x <= 0, rounded to nearest among FP64's subnormal numbers too, where exp may be off by a unit,
 * which there can be all of it: 2^64 times as large first. */
__device__ __forceinline__ double falling_exponential(double x)
{
    return x < -700.0 ? exp(x + 44.361419555836498) * 0x1p-64 : exp(x);
}

/* Lane j < choices: the j-th expert by FP64 ranks. */
template <int PerLane>
__device__ __noinline__ int choose_exactly(const ScoreTask &task, const float (&x)[PerLane], float top)
{
    const int lane = threadIdx.x & 31;
    double score[PerLane], sum = 0;
    long long key[PerLane];
#pragma unroll
    for (int i = 0; i < PerLane; ++i) {
        score[i] = task.sigmoid ? 1.0 / (1.0 + exp(-double(x[i]))) : falling_exponential(double(x[i]) - top);
        sum += score[i];
    }
    if (!task.sigmoid) {
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
        key[i] = e < task.experts ? order_of(score[i] + (task.bias ? double(task.bias[e]) : 0.0)) : kRemoved;
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
                return k <= kNan ? double(NAN) : __longlong_as_double(k < 0 ? k ^ 0x7fffffffffffffffll : k);
            };
            const long long rank = order_of(size > 1 ? value(first) + value(second) : value(first));
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
    int mine = 0;
    for (int round = 0; round < task.choices; ++round) {
        long long best = kRemoved;
        int index = INT_MAX;
#pragma unroll
        for (int i = 0; i < PerLane; ++i)
            if (key[i] > best)
                best = key[i], index = i * 32 + lane;
        warp_best(best, index);
        if (lane == round)
            mine = index;
#pragma unroll
        for (int i = 0; i < PerLane; ++i)
            if (index == i * 32 + lane)
                key[i] = kRemoved;
    }
    return mine;
}

/* 32-bit keys ordered like FP32 numbers: 0 what was taken out, 1 a NaN. */
__device__ __forceinline__ unsigned key_of(float x)
{
    if (x != x)
        return 1;
    const int bits = __float_as_int(x + 0.f);
    return bits < 0 ? ~unsigned(bits) : unsigned(bits) | 0x80000000u;
}

__device__ __forceinline__ float rank_of(unsigned key)
{
    return key <= 1 ? NAN : __int_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

/* The largest of the warp's keys, the lowest index that has it; taken out. */
template <int PerLane> __device__ __forceinline__ unsigned take_best(unsigned (&key)[PerLane], int &index)
{
    const int lane = threadIdx.x & 31;
    unsigned best = key[0];
#pragma unroll
    for (int i = 1; i < PerLane; ++i)
        best = max(best, key[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    unsigned first = INT_MAX;
#pragma unroll
    for (int i = PerLane - 1; i >= 0; --i)
        if (key[i] == best)
            first = i * 32 + lane;
    first = __reduce_min_sync(0xffffffffu, first);
    index = int(first);
#pragma unroll
    for (int i = 0; i < PerLane; ++i)
        if (first == unsigned(i * 32 + lane))
            key[i] = 0;
    return best;
}

/* Whether a rank that was computed in FP32 is surely larger than another. An FP32 score, at most 1, is
 * off by less than 2^-18 (an exponential, up to 37 additions of a sum, a division), and its sum with a
 * bias by a rounding more. */
__device__ __forceinline__ bool surely_larger(float a, float b)
{
    return a - b > 0x1p-17f * (1.f + fabsf(a)); /* false for a NaN and for infinities */
}

/* How far the sum of a group's two largest ranks may be off, the larger of which has this magnitude: 2^-18
 * for either score, 2^-24 of the magnitude for either sum with a bias and twice that for the sum of the
 * two, which may be far smaller than they, and for taking the doubt from it: together below this. */
__device__ __forceinline__ float group_doubt(float magnitude) { return 0x1p-17f + 0x1p-20f * magnitude; }

/* Whether the scores of two logits, the larger first, are in the same order in FP64, and equal only where
 * the logits are. From 2^-25 apart the exponentials differ by that relative to them, and by far more than
 * FP64 rounds off, as long as the larger score is a normal number (`base` is the largest logit, for a sigmoid
 * 0) and the 1 that a sigmoid adds to its exponential does not cover the difference. */
__device__ __forceinline__ bool scores_ordered(float larger, float smaller, float base, bool sigmoid)
{
    return larger == smaller || (larger - smaller > 0x1p-25f && larger - base > -700.f && !(sigmoid && larger > 16.f));
}

template <int PerLane, typename T>
__global__ void __launch_bounds__(128) score_kernel(const __grid_constant__ ScoreTask task)
{
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (blockDim.x / 32);
    const int size = task.experts / task.groups;
    int group_of[PerLane]; /* exact: (e + 1/2) / size is no nearer than 1 / 2048 to a whole number */
    const float inverse = 1.f / size;
#pragma unroll
    for (int i = 0; i < PerLane; ++i)
        group_of[i] = int((i * 32 + lane + 0.5f) * inverse);
    /* 64 bits: the step behind the last token may leave 32 */
    for (long long token = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; token < task.tokens; token += warps) {
        const T *row = static_cast<const T *>(task.logits) + token * task.ld_logits;
        float x[PerLane];
        float top = -INFINITY;
        bool broken = false; /* a NaN or +infinity makes every softmax score NaN */
#pragma unroll
        for (int i = 0; i < PerLane; ++i) {
            const int e = i * 32 + lane;
            x[i] = e < task.experts ? load_logit(row + e) : -INFINITY;
            top = fmaxf(top, x[i]);
            broken = broken || !(x[i] < INFINITY);
        }
        if (!task.sigmoid) {
            top = rank_of(__reduce_max_sync(0xffffffffu, key_of(top)));
            if (!(top > -INFINITY)) /* no expert is open: all scores are zero */
                top = 0.f;
            broken = __any_sync(0xffffffffu, broken);
        }
        unsigned key[PerLane];
        bool certain = true;
        const bool by_logits = !task.bias && task.groups == 1;
        if (by_logits) {
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                key[i] = i * 32 + lane < task.experts ? (!task.sigmoid && broken ? 1 : key_of(x[i])) : 0;
        } else {
            float score[PerLane], sum = 0.f;
#pragma unroll
            for (int i = 0; i < PerLane; ++i) {
                score[i] = task.sigmoid ? 1.f / (1.f + expf(-x[i])) : expf(x[i] - top);
                sum += score[i];
            }
            if (!task.sigmoid) {
#pragma unroll
                for (int offset = 16; offset > 0; offset /= 2)
                    sum += __shfl_xor_sync(0xffffffffu, sum, offset);
                sum = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
                for (int i = 0; i < PerLane; ++i)
                    score[i] *= sum;
            }
#pragma unroll
            for (int i = 0; i < PerLane; ++i) {
                const int e = i * 32 + lane;
                key[i] = e < task.experts ? key_of(score[i] + (task.bias ? task.bias[e] : 0.f)) : 0;
            }
            if (task.groups > 1) {
                float mine = NAN; /* lane g: the rank of group g, and how far it may be off */
                float doubt = 0.f;
#pragma unroll 1
                for (int group = 0; group < task.groups; ++group) {
                    unsigned first = 0, second = 0;
#pragma unroll
                    for (int i = 0; i < PerLane; ++i) {
                        const unsigned k = group_of[i] == group ? key[i] : 0;
                        second = max(second, min(first, k));
                        first = max(first, k);
                    }
                    const unsigned best = __reduce_max_sync(0xffffffffu, first);
                    float rank = rank_of(best), magnitude = fabsf(rank);
                    if (size > 1) {
                        /* the lane of the largest offers its next, the others their first */
                        const unsigned owners = __ballot_sync(0xffffffffu, first == best);
                        const unsigned offer = lane == __ffs(owners) - 1 ? second : first;
                        const float next = rank_of(__reduce_max_sync(0xffffffffu, offer));
                        magnitude = fmaxf(magnitude, fabsf(next)), rank += next;
                    }
                    if (lane == group)
                        mine = rank, doubt = group_doubt(magnitude);
                }
                unsigned keep = 0;
                unsigned one[1] = {lane < task.groups ? key_of(mine) : 0};
#pragma unroll 1
                for (int round = 0; round < task.kept; ++round) {
                    int at;
                    take_best(one, at);
                    keep |= 1u << (at & 31);
                }
                if (task.kept < task.groups) {
                    const bool kept = (keep >> lane) & 1;
                    const unsigned least = __reduce_min_sync(0xffffffffu, kept ? key_of(mine - doubt) : ~0u);
                    const unsigned most =
                        __reduce_max_sync(0xffffffffu, !kept && lane < task.groups ? key_of(mine + doubt) : 0);
                    certain = rank_of(least) > rank_of(most); /* false for a NaN */
                }
#pragma unroll
                for (int i = 0; i < PerLane; ++i)
                    if (!((keep >> (group_of[i] & 31)) & 1))
                        key[i] = 0;
            }
        }
        int mine = 0;
        if (certain) {
            float before = INFINITY;
            unsigned taken = 0; /* lane j: the key of its choice */
#pragma unroll 1
            for (int round = 0; round < task.choices; ++round) {
                int index;
                const unsigned best = take_best(key, index);
                if (!by_logits) {
                    const float rank = rank_of(best);
                    certain = certain && (round == 0 ? rank == rank : surely_larger(before, rank));
                    before = rank;
                }
                if (lane == round)
                    mine = index, taken = best;
            }
            /* the first that was not chosen */
            unsigned next = 0;
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                next = max(next, key[i]);
            next = __reduce_max_sync(0xffffffffu, next);
            if (!by_logits) {
                certain = certain && (next == 0 || surely_larger(before, rank_of(next)));
            } else { /* lane j: its choice after the one before it; lane 0: the first not chosen after the last */
                const unsigned larger = __shfl_sync(0xffffffffu, taken, lane == 0 ? task.choices - 1 : lane - 1);
                const unsigned smaller = lane == 0 ? next : taken;
                certain = __all_sync(0xffffffffu, lane >= task.choices || smaller == 0 ||
                                                      scores_ordered(rank_of(larger), rank_of(smaller),
                                                                     task.sigmoid ? 0.f : top, task.sigmoid));
            }
        }
        if (!certain)
            mine = choose_exactly<PerLane>(task, x, top);
        /* the weights of the chosen, lane j the j-th */
        const bool chosen = lane < task.choices;
        const double logit = chosen ? double(load_logit(row + mine)) : -INFINITY;
        double score = task.sigmoid ? 1.0 / (1.0 + exp(-logit)) : exp(logit - top);
        if (!task.sigmoid && broken)
            score = NAN;
        double total = 1.0;
        if (task.renormalise) {
            total = chosen ? score : 0.0;
#pragma unroll
            for (int offset = 16; offset > 0; offset /= 2)
                total += shuffle_xor(total, offset);
        } else if (!task.sigmoid) {
            total = 0.0;
#pragma unroll
            for (int i = 0; i < PerLane; ++i)
                total += exp(double(x[i]) - top);
#pragma unroll
            for (int offset = 16; offset > 0; offset /= 2)
                total += shuffle_xor(total, offset);
        }
        if (chosen) {
            const long long at = token * task.choices + lane;
            task.chosen[at] = mine;
            task.weights[at] = float((total != 0 ? score / total : 0.0) * double(task.scale));
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
