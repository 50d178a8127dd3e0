// The choice of experts for every token: scores, a bias for the choice, groups, top-k, renormalised weights.
//
//   score_e  = softmax over the open experts, or sigmoid, of the logits; closed are those whose logit is NaN or -inf
//   choice_e = score_e + bias_e (closed, too, where that is NaN or -inf)
//   rank_g   = the sum of the group's group_scores (1 or 2) largest choices; a group without an open expert is closed
//   ids      = the top_k largest choices within the chosen_groups best groups, the lower number first among equals;
//              -1 where open experts run out
//   weights  = their scores (0 for -1), over the sum of the chosen ones' where renormalised, times scale
// All of it is held in 64 bits: experts next to one another are told apart as the definition does, not by what the last bit
// of an exponential made of them.
//
// One warp per token, expert e with thread e % 32.  (No pointer is __restrict__: loads through those may move in front of the wait
// for the kernel that writes the logits.)
#include "common.cuh"
#include "kernels.cuh"
#include "launch.cuh"

namespace nerve {

namespace {

__device__ __forceinline__ float logit_of(const float *logits, size_t at) { return logits[at]; }
__device__ __forceinline__ float logit_of(const uint16_t *logits, size_t at) { return bf16_bits_to_f32(logits[at]); }

// Unsigned numbers in the order of the values; above 0 for all but NaN and -inf, which are 0.
__device__ __forceinline__ uint64_t key_of(double value) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(value + 0.0));  // -0 ties with 0
    if (!(value > -__longlong_as_double(0x7ff0000000000000ll))) return 0;
    return (bits >> 63) ? ~bits : bits | 0x8000000000000000ull;
}
__device__ __forceinline__ uint64_t warp_max_key(uint64_t key) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
    const uint32_t low = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32) == high ? static_cast<uint32_t>(key) : 0u);
    return (static_cast<uint64_t>(high) << 32) | low;
}
__device__ __forceinline__ double value_of(uint64_t key) {  // of a key above 0
    return __longlong_as_double(static_cast<long long>((key >> 63) ? key & 0x7fffffffffffffffull : ~key));
}

constexpr int TOKENS_PER_CTA = 4;

template <typename T, int PER_THREAD>
__global__ void __launch_bounds__(32 * TOKENS_PER_CTA) route_experts_kernel(const T *logits, const float *bias, int *ids,
                                                                            float *weights, int tokens, Routing routing) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int token = blockIdx.x * TOKENS_PER_CTA + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (token >= tokens) return;
    const int experts = routing.experts;
    const float infinity = __uint_as_float(0x7f800000u);
    float logit[PER_THREAD];
    float top = -infinity;
#pragma unroll
    for (int j = 0; j < PER_THREAD; j++) {
        const int expert = lane + 32 * j;
        logit[j] = expert < experts ? logit_of(logits, static_cast<size_t>(token) * experts + expert) : -infinity;
        if (!(logit[j] > -infinity)) logit[j] = -infinity;
        top = fmaxf(top, logit[j]);
    }
    double score[PER_THREAD];
    if (routing.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) score[j] = logit[j] > -infinity ? 1.0 / (1.0 + exp(-static_cast<double>(logit[j]))) : 0.0;
    } else {
        top = warp_max(top);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) {
            score[j] = logit[j] > -infinity ? (logit[j] == top ? 1.0 : exp(static_cast<double>(logit[j]) - static_cast<double>(top))) : 0.0;
            sum += score[j];
        }
#pragma unroll
        for (int offset = 16; offset > 0; offset >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) score[j] = sum > 0.0 ? score[j] / sum : 0.0;
    }
    uint64_t key[PER_THREAD];
#pragma unroll
    for (int j = 0; j < PER_THREAD; j++) {
        const int expert = lane + 32 * j;
        key[j] = 0;
        if (logit[j] > -infinity) key[j] = key_of(bias != nullptr ? score[j] + static_cast<double>(bias[expert]) : score[j]);
    }
    if (routing.groups > 1) {
        const int size = experts / routing.groups;
        uint64_t rank = 0;  // of group `lane`
        for (int group = 0; group < routing.groups; group++) {
            uint64_t best = 0, next = 0;  // of this thread's experts in the group
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) {
                const int expert = lane + 32 * j;
                if (expert < group * size || expert >= (group + 1) * size) continue;
                if (key[j] > best) next = best, best = key[j];
                else if (key[j] > next) next = key[j];
            }
            const uint64_t first = warp_max_key(best);
            if (first == 0) continue;
            double value = value_of(first);
            if (routing.group_scores > 1) {
                const int holder = __ffs(__ballot_sync(0xffffffffu, best == first)) - 1;  // one of those that hold the largest
                const uint64_t second = warp_max_key(lane == holder ? next : best);
                if (second != 0) value += value_of(second);
            }
            if (lane == group) rank = key_of(value);
        }
        int before = 0;  // groups in front of group `lane`
        for (int group = 0; group < routing.groups; group++) {
            const uint64_t other = __shfl_sync(0xffffffffu, rank, group);
            before += other > rank || (other == rank && group < lane);
        }
        const uint32_t kept = __ballot_sync(0xffffffffu, lane < routing.groups && before < routing.chosen_groups);
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) {
            const int expert = lane + 32 * j;
            if (expert < experts && !((kept >> (expert / size)) & 1u)) key[j] = 0;
        }
    }
    // the largest key of the thread, the lower expert among equals
    uint64_t best;
    int best_at;
    auto find_best = [&] {
        best = 0;
        best_at = 0;
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++)
            if (key[j] > best) best = key[j], best_at = j;
    };
    find_best();
    int own_id[2] = {-1, -1};  // routes lane and lane + 32
    double own_score[2] = {0.0, 0.0}, total = 0.0;
    for (int route = 0; route < routing.top_k; route++) {
        const uint64_t most = warp_max_key(best);
        if (most == 0) break;
        const int expert = static_cast<int>(__reduce_min_sync(0xffffffffu, best == most ? static_cast<uint32_t>(lane + 32 * best_at) : 0xffffffffu));
        double chosen = 0.0;
        if ((expert & 31) == lane) {
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++)
                if (j == best_at) chosen = score[j], key[j] = 0;
            find_best();
        }
        chosen = __shfl_sync(0xffffffffu, chosen, expert & 31);
        total += chosen;
        if ((route & 31) == lane) {
            own_id[route >> 5] = expert;
            own_score[route >> 5] = chosen;
        }
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const int route = lane + 32 * half;
        if (route >= routing.top_k) break;
        double weight = own_score[half];
        if (routing.renormalise) weight = total > 0.0 ? weight / total : 0.0;
        ids[static_cast<size_t>(token) * routing.top_k + route] = own_id[half];
        weights[static_cast<size_t>(token) * routing.top_k + route] = static_cast<float>(weight * static_cast<double>(routing.scale));
    }
}

template <typename T>
cudaError_t launch(const T *logits, const float *bias, int *ids, float *weights, int tokens, const Routing &routing, cudaStream_t stream) {
    const dim3 grid((tokens + TOKENS_PER_CTA - 1) / TOKENS_PER_CTA), block(32 * TOKENS_PER_CTA);
    auto with = [&](auto kernel) { return launch_dependent(kernel, grid, block, 0, 1, stream, logits, bias, ids, weights, tokens, routing); };
    const int per_thread = (routing.experts + 31) / 32;
    if (per_thread <= 1) return with(route_experts_kernel<T, 1>);
    if (per_thread <= 2) return with(route_experts_kernel<T, 2>);
    if (per_thread <= 4) return with(route_experts_kernel<T, 4>);
    if (per_thread <= 8) return with(route_experts_kernel<T, 8>);
    if (per_thread <= 16) return with(route_experts_kernel<T, 16>);
    return with(route_experts_kernel<T, 32>);
}

}  // namespace

cudaError_t launch_route_experts(const void *logits, bool logits_f32, const float *bias, int *ids, float *weights, int tokens, const Routing &routing, cudaStream_t stream) {
    return logits_f32 ? launch(static_cast<const float *>(logits), bias, ids, weights, tokens, routing, stream)
                      : launch(static_cast<const uint16_t *>(logits), bias, ids, weights, tokens, routing, stream);
}

}  // namespace nerve
