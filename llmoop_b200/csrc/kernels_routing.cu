// The choice of experts for every token: scores, a bias for the choice, groups, top-k, renormalised weights.
//
//   score_e  = softmax over the open experts, or sigmoid, of the logits; closed are those whose logit is NaN or -inf
//   choice_e = score_e + bias_e (closed, too, where that is NaN or -inf)
//   rank_g   = the sum of the group's group_scores (1 or 2) largest choices; a group without an open expert is closed
//   ids      = the top_k largest choices within the chosen_groups best groups, the lower number first among equals;
//              -1 where open experts run out
//   weights  = their scores (0 for -1), over the sum of the chosen ones' where renormalised, times scale
// The definition holds all of it in 64 bits: experts next to one another are told apart as it does, not by what the last bit of an
// exponential made of them.  64-bit exponentials and keys are also what such a kernel spends its time on (16384 tokens of 256
// experts in 8 groups: 81 us), so that 32 bits, with a bound on the error, find the few candidates, which alone are scored and ranked
// in 64.  Groups closer than the error are ranked in 64 bits where they stand, if each is a run of threads.  Tokens that cannot be
// decided so are done by the definition: more than 31 candidates (top_k 32 to 64, and often from 20 on), sigmoids of logits above 20, logits of +inf, scores
// below 1e-250, and groups next to one another that are no runs of threads, have no scores or hold choices from 1e30 on.
//
// One warp per token, of which the chip holds enough to cover the loads.  Bound by the instructions that it issues, some 1080 a token, of which
// some 200 go by the experts and the others are a whole warp's steps for one token (groups, limit, candidates, ranks, weights):
// 16384 tokens of 256 experts in 8 groups, 23.0 us, of which the logits' bytes are 2.8.  One token of 128 experts takes 2.7 us, a launch and the
// chain of reductions.  (No pointer is __restrict__: loads through those may move in front of the wait
// for the kernel that writes the logits.)
#include <algorithm>

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

// One token by the definition.  Expert e with thread e % 32.
template <typename T, int PER_THREAD>
__device__ __noinline__ void route_in_64_bits(const T *logits, const float *bias, int *ids, float *weights, int token, const Routing &routing) {
    const int lane = threadIdx.x & 31;
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

// Unsigned numbers in the order of the values, above 0.  (-0 lies in front of 0.)
__device__ __forceinline__ uint32_t key_of(float value) {
    const uint32_t bits = __float_as_uint(value);
    return bits ^ (static_cast<uint32_t>(static_cast<int>(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key); }  // of a key above 0

// Scores in 32 bits, by 2^x and 1 / x as the chip has them: off by less than 1.5e-6 (the error of the exponential grows with the
// distance from the largest, which the score's smallness outweighs).
__device__ __forceinline__ float fast_exp(float x) {
    float out;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(out) : "f"(x * 1.4426950408889634f));
    return out;
}
__device__ __forceinline__ float fast_inverse(float x) {
    float out;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(out) : "f"(x));
    return out;
}
// How far two choices about `value`, or sums of two choices each of up to that magnitude, have to lie apart to be in that order in truth.
__device__ __forceinline__ float margin(float value) { return 1.6e-5f * (1.0f + fabsf(value)); }
constexpr float LARGEST = 3.402823466e+38f;

// PER_THREAD successive values, in sixteen bytes where they lie so.
template <int PER_THREAD>
__device__ __forceinline__ void load_run(const float *from, float (&to)[PER_THREAD]) {
    if constexpr (PER_THREAD % 4 == 0) {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j += 4) {
            const float4 four = *reinterpret_cast<const float4 *>(from + j);
            to[j] = four.x, to[j + 1] = four.y, to[j + 2] = four.z, to[j + 3] = four.w;
        }
    }
}
template <int PER_THREAD>
__device__ __forceinline__ void load_run(const uint16_t *from, float (&to)[PER_THREAD]) {
    if constexpr (PER_THREAD % 4 == 0) {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j += 4) {
            const uint2 four = *reinterpret_cast<const uint2 *>(from + j);
            to[j] = bf16_lo(four.x), to[j + 1] = bf16_hi(four.x), to[j + 2] = bf16_lo(four.y), to[j + 3] = bf16_hi(four.y);
        }
    }
}

struct Plan {
    Routing routing;
    int per;      // experts of a thread
    int threads;  // of a group whose threads hold runs of experts; 0: experts lie 32 apart
    int wide;     // runs of PER_THREAD logits and biases on boundaries of sixteen (bf16: eight) bytes
};
struct Candidates {
    uint32_t expert[32];
    float logit[32];
    double choice[32];
    uint32_t sorted_expert[32];
    double sorted_score[32];
};

// A token whose candidates are found in 32 bits, with a bound on the error, and ranked in 64; false where that is not certain to
// choose what the definition does.  Without a bias experts are in the order of their logits, which needs no arithmetic; groups of
// ranks closer than the error are decided here where a group is a run of threads (20 of 16384 tokens of 256 experts in 8 groups by
// sigmoids; by the definition they took 5 of 27 us, the last of them alone on the chip).  Thread l holds the `per` experts from l * per on, where that makes every group a
// run of threads and leaves few of them idle; else those 32 apart.
template <typename T, int PER_THREAD>
__device__ __forceinline__ bool route_in_32_bits(const T *logits, const float *bias, int *ids, float *weights, int token, const Plan &plan, Candidates &found) {
    const Routing &routing = plan.routing;
    const int lane = threadIdx.x & 31, experts = routing.experts, per = plan.per, base = plan.threads > 0 ? lane * per : lane, step = plan.threads > 0 ? 1 : 32;
    const T *row = logits + static_cast<size_t>(token) * experts;
    const float infinity = __uint_as_float(0x7f800000u);
    float logit[PER_THREAD], score[PER_THREAD];
    if (plan.wide) {
        load_run<PER_THREAD>(row + base, logit);
    } else {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) logit[j] = j < per && base + j * step < experts ? logit_of(row, base + j * step) : -infinity;
    }
    float top = -infinity;
#pragma unroll
    for (int j = 0; j < PER_THREAD; j++) top = fmaxf(top, logit[j]);
    top = value_of(__reduce_max_sync(0xffffffffu, key_of(top)));
    // (the sigmoids of larger logits next to one another meet in 64 bits)
    if (top == infinity || (routing.sigmoid && top > 20.0f)) return false;
    const bool scored = bias != nullptr || (routing.groups > 1 && routing.group_scores > 1);
    if (scored && routing.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) score[j] = fast_inverse(1.0f + fast_exp(-logit[j]));
    } else if (scored) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) {
            score[j] = fast_exp(fmaxf(logit[j], -infinity) - top);  // (NaN counts as -infinity)
            sum += score[j];
        }
        const float inverse = fast_inverse(warp_sum(sum));
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) score[j] *= inverse;
    }
    uint32_t key[PER_THREAD];  // of the choice, or of the logit; 0: closed
    if (bias != nullptr) {
        float own[PER_THREAD];
        if (plan.wide) {
            load_run<PER_THREAD>(bias + base, own);
        } else {
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) own[j] = j < per && base + j * step < experts ? bias[base + j * step] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) {
            const float value = score[j] + own[j];
            key[j] = logit[j] > -infinity && value > -infinity ? key_of(value) : 0u;
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) key[j] = logit[j] > -infinity ? key_of(logit[j] + 0.0f) : 0u;
    }
    if (routing.groups > 1) {
        const bool by_score = bias == nullptr && scored;
        auto value_at = [&](int j) { return by_score && key[j] != 0 ? key_of(score[j]) : key[j]; };
        const int threads = plan.threads, size = experts / routing.groups;
        uint32_t group_best = 0, group_next = 0;  // of the group of number own_group
        int own_group = lane;
        if (threads > 0) {
            own_group = lane / threads;
            const int first = own_group * threads;
            uint32_t best = 0, next = 0;
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) {
                const uint32_t value = value_at(j);
                next = max(next, min(best, value));
                best = max(best, value);
            }
            if ((threads & (threads - 1)) == 0) {
                group_best = best, group_next = next;
#pragma unroll
                for (int offset = 1; offset < 32; offset *= 2) {
                    if (offset >= threads) break;
                    const uint32_t b = __shfl_xor_sync(0xffffffffu, group_best, offset), n = __shfl_xor_sync(0xffffffffu, group_next, offset);
                    group_next = max(max(group_next, n), min(group_best, b));
                    group_best = max(group_best, b);
                }
            } else {
                for (int other = 0; other < threads; other++) {
                    const uint32_t b = __shfl_sync(0xffffffffu, best, first + other), n = __shfl_sync(0xffffffffu, next, first + other);
                    group_next = max(max(group_next, n), min(group_best, b));
                    group_best = max(group_best, b);
                }
            }
        } else {
            for (int group = 0; group < routing.groups; group++) {
                uint32_t best = 0, next = 0;
#pragma unroll
                for (int j = 0; j < PER_THREAD; j++) {
                    const int expert = base + j * step;
                    const uint32_t value = expert >= group * size && expert < (group + 1) * size ? value_at(j) : 0u;
                    next = max(next, min(best, value));
                    best = max(best, value);
                }
                const uint32_t most = __reduce_max_sync(0xffffffffu, best);
                const int holder = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
                const uint32_t second = __reduce_max_sync(0xffffffffu, lane == holder ? next : best);
                if (lane == group) group_best = most, group_next = second;
            }
        }
        const bool open = own_group < routing.groups && group_best != 0;
        float rank = open ? value_of(group_best) : -infinity, largest = fabsf(rank);
        if (routing.group_scores > 1 && open && group_next != 0) {
            rank += value_of(group_next);
            largest = fmaxf(largest, fabsf(value_of(group_next)));
        }
        if (open) rank = fminf(fmaxf(rank, -LARGEST), LARGEST);  // (two of the lowest values are no closed group's -infinity)
        // Where the rank lies in truth: it is off by its summands' errors, which may be more than all of it where biases of both signs
        // cancel.  (An infinite one lies anywhere.)
        const float error = scored ? 0.5f * margin(largest) : 0.0f, low = rank - error, high = rank + error;
        // the groups in front of this thread's: each of a group's threads compares some
        const int team = max(threads, 1), team_first = own_group * team;
        int before = 0;
        for (int from = 0; from < routing.groups; from += team) {
            const int group = from + lane - team_first;
            const float other = __shfl_sync(0xffffffffu, rank, min(group, routing.groups - 1) * team);
            const uint32_t in_front = __ballot_sync(0xffffffffu, group < routing.groups && (other > rank || (other == rank && group < own_group)));
            before += __popc((in_front >> team_first) & ((1u << team) - 1u));
        }
        bool kept = open && before < routing.chosen_groups;
        const uint32_t first_left = __reduce_max_sync(0xffffffffu, open && !kept ? key_of(high) : 0u), last_kept = __reduce_min_sync(0xffffffffu, kept ? key_of(low) : 0xffffffffu);
        if (first_left != 0) {  // (logits as close as 1e-12 may be one score in 64 bits)
            const float in = value_of(last_kept), out = value_of(first_left);
            if (!(scored ? in > out : in - out > 1e-12f)) {
                if (!scored || threads == 0) return false;
                // those in doubt are ranked in 64 bits; a group that lies above all that were left, or below all that were kept, is not
                const bool sure = open && low > out, doubt = open && !sure && high >= in;
                if (__any_sync(0xffffffffu, doubt && !(largest < 1e30f))) return false;
                const int places = routing.chosen_groups - __popc(__ballot_sync(0xffffffffu, sure && lane == team_first));
                const uint32_t least = routing.group_scores > 1 ? group_next : group_best;  // candidates for the group's largest: what is not further below
                uint32_t some = 0;
                if (doubt) {
                    const uint32_t from = least != 0 ? key_of(value_of(least) - margin(value_of(least))) : 1u;
#pragma unroll
                    for (int j = 0; j < PER_THREAD; j++) some |= value_at(j) >= from ? 1u << j : 0u;
                }
                double all = 0.0;  // the softmax's terms
                if (!routing.sigmoid) {
#pragma unroll 1
                    for (int j = 0; j < per; j++) {
                        const float at = base + j < experts ? logit_of(row, base + j) : -infinity;
                        if (at > -infinity) all += exp(static_cast<double>(at) - static_cast<double>(top));
                    }
#pragma unroll
                    for (int offset = 16; offset > 0; offset >>= 1) all += __shfl_xor_sync(0xffffffffu, all, offset);
                }
                double exact_best = -static_cast<double>(infinity), exact_next = exact_best;
                while (__any_sync(0xffffffffu, some != 0)) {
                    if (some == 0) continue;
                    const int expert = base + __ffs(some) - 1;
                    some &= some - 1;
                    const double at = static_cast<double>(logit_of(row, expert)), power = exp(routing.sigmoid ? -at : at - static_cast<double>(top));
                    double value = (routing.sigmoid ? 1.0 : power) / (routing.sigmoid ? 1.0 + power : all);
                    if (bias != nullptr) value += static_cast<double>(bias[expert]);
                    exact_next = fmax(exact_next, fmin(exact_best, value));
                    exact_best = fmax(exact_best, value);
                }
                double best_of_all = -static_cast<double>(infinity), next_of_all = best_of_all;
                for (int other = 0; other < threads; other++) {
                    const int from = min(team_first + other, 31);
                    const double b = __shfl_sync(0xffffffffu, exact_best, from), n = __shfl_sync(0xffffffffu, exact_next, from);
                    next_of_all = fmax(fmax(next_of_all, n), fmin(best_of_all, b));
                    best_of_all = fmax(best_of_all, b);
                }
                double exact = best_of_all;
                if (routing.group_scores > 1 && next_of_all > -static_cast<double>(infinity)) exact += next_of_all;
                const uint32_t doubtful = __ballot_sync(0xffffffffu, doubt);
                int ahead = 0;
                for (int group = 0; group < routing.groups; group++) {
                    const double other = __shfl_sync(0xffffffffu, exact, group * team);
                    ahead += ((doubtful >> (group * team)) & 1u) && (other > exact || (other == exact && group < own_group));
                }
                kept = sure || (doubt && ahead < places);
            }
        }
        if (threads > 0) {
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) key[j] = kept ? key[j] : 0u;
        } else {
            const uint32_t all_kept = __ballot_sync(0xffffffffu, kept);
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++)
                if (key[j] != 0 && !((all_kept >> ((base + j * step) / size)) & 1u)) key[j] = 0;
        }
    }
    // The top_k-th largest of the threads' own largest keys is no more than the top_k-th largest of all: what is not further below
    // it than the error is a candidate, few more than top_k.
    uint32_t own_best = 0, limit = 0;
#pragma unroll
    for (int j = 0; j < PER_THREAD; j++) own_best = max(own_best, key[j]);
    for (int route = 0; route < routing.top_k; route++) {
        limit = __reduce_max_sync(0xffffffffu, own_best);
        if (limit == 0) break;
        if (own_best == limit) own_best = 0;
    }
    if (limit == 0) limit = 1;  // all that are open
    else if (bias != nullptr && value_of(limit) < infinity) limit = key_of(value_of(limit) - margin(value_of(limit)));  // (infinite biases are equals, without an error)
    uint32_t left = 0, own = 0;  // the largest that is no candidate; bit j: one is
#pragma unroll
    for (int j = 0; j < PER_THREAD; j++) {
        const bool candidate = key[j] >= limit;
        left = max(left, candidate ? 0u : key[j]);
        own |= candidate ? 1u << j : 0u;
    }
    int count = 0, place = 0;  // of all, and of the threads before
    const int own_count = __popc(own);
#pragma unroll
    for (int bit = 0; (1 << bit) <= PER_THREAD; bit++) {
        const uint32_t set = __ballot_sync(0xffffffffu, (own_count >> bit) & 1);
        count += __popc(set) << bit;
        place += __popc(set & ((1u << lane) - 1u)) << bit;
    }
    if (count > 31) return false;
#pragma unroll
    for (int j = 0; j < PER_THREAD; j++)
        if ((own >> j) & 1u) {
            found.expert[place] = static_cast<uint32_t>(base + j * step);
            found.logit[place++] = logit[j];
        }
    left = bias == nullptr ? __reduce_max_sync(0xffffffffu, left) : 0u;  // (with a bias the margin keeps it apart)
    __syncwarp();
    // one candidate to a thread: its score in 64 bits, and the number of those in front of it; to the next thread the logit that is left
    double sum = 0.0;  // of the softmax's terms, where more than their order and ratios count
    if (!routing.sigmoid && (bias != nullptr || !routing.renormalise)) {
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++)
            if (logit[j] > -infinity) sum += exp(static_cast<double>(logit[j]) - static_cast<double>(top));
#pragma unroll
        for (int offset = 16; offset > 0; offset >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    }
    const uint32_t my_expert = lane < count ? found.expert[lane] : 0u;
    double own_score = 0.0, choice = 0.0;
    if (lane < count || (lane == count && left != 0)) {
        const double own_logit = static_cast<double>(lane < count ? found.logit[lane] : value_of(left));
        own_score = exp(routing.sigmoid ? -own_logit : own_logit - static_cast<double>(top));
        if (routing.sigmoid) own_score = 1.0 / (1.0 + own_score);
        else if (sum > 0.0) own_score /= sum;
        choice = bias != nullptr ? own_score + static_cast<double>(bias[my_expert]) : own_score;
        found.choice[lane] = choice;
    }
    if (__any_sync(0xffffffffu, lane < count && own_score < 1e-250)) return false;  // where scores run out of exponents
    // candidates whose scores, other than their logits, are no larger than one's that is left: the lower number may be that one's
    const double left_score = __shfl_sync(0xffffffffu, own_score, count);
    if (left != 0 && __any_sync(0xffffffffu, lane < count && own_score <= left_score)) return false;
    __syncwarp();
    // `width` threads for the candidates, as many of them to each as there are: every one of these compares some of the others
    const int width = count <= 8 ? 8 : count <= 16 ? 16 : 32, mine = lane & (width - 1);
    const double their_choice = found.choice[mine];
    const uint32_t their_expert = found.expert[mine];
    place = 0;
    for (int other = lane / width; other < count; other += 32 / width) {
        const double theirs = found.choice[other];
        place += theirs > their_choice || (theirs == their_choice && found.expert[other] < their_expert);
    }
    if (width <= 16) place += __shfl_xor_sync(0xffffffffu, place, 16);
    if (width <= 8) place += __shfl_xor_sync(0xffffffffu, place, 8);
    if (lane < count) {
        found.sorted_expert[place] = my_expert;
        found.sorted_score[place] = own_score;
    }
    __syncwarp();
    const bool chosen = lane < min(count, routing.top_k);
    double weight = chosen ? found.sorted_score[lane] : 0.0;
    if (routing.renormalise) {
        double total = weight;  // (those of threads from top_k on are 0)
#pragma unroll
        for (int offset = 16; offset > 0; offset >>= 1)
            if (offset < routing.top_k) total += __shfl_xor_sync(0xffffffffu, total, offset);
        weight = total > 0.0 ? weight / total : 0.0;
    }
    if (lane < routing.top_k) {
        ids[static_cast<size_t>(token) * routing.top_k + lane] = chosen ? static_cast<int>(found.sorted_expert[lane]) : -1;
        weights[static_cast<size_t>(token) * routing.top_k + lane] = static_cast<float>(weight * static_cast<double>(routing.scale));
    }
    return true;
}

template <typename T, int PER_THREAD>
__global__ void __launch_bounds__(32 * TOKENS_PER_CTA) route_experts_kernel(const T *logits, const float *bias, int *ids, float *weights, int tokens, Plan plan) {
    __shared__ Candidates found[TOKENS_PER_CTA];
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = static_cast<int>(threadIdx.x >> 5), token = blockIdx.x * TOKENS_PER_CTA + warp;
    if (token >= tokens) return;
    if (plan.routing.top_k <= 32 && route_in_32_bits<T, PER_THREAD>(logits, bias, ids, weights, token, plan, found[warp])) return;
    route_in_64_bits<T, PER_THREAD>(logits, bias, ids, weights, token, plan.routing);
}

template <typename T>
cudaError_t launch(const T *logits, const float *bias, int *ids, float *weights, int tokens, const Routing &routing, cudaStream_t stream) {
    const dim3 grid((tokens + TOKENS_PER_CTA - 1) / TOKENS_PER_CTA), block(32 * TOKENS_PER_CTA);
    Plan plan = {};
    plan.routing = routing;
    plan.per = (routing.experts + 31) / 32;
    const int size = routing.experts / routing.groups;
    for (int threads = std::min(size, 32 / routing.groups); threads * routing.groups > 16; threads--)  // (of a group, all of whose threads hold as many)
        if (size % threads == 0 && size / threads <= 32) {
            plan.threads = threads;
            plan.per = size / threads;
            break;
        }
    auto with = [&](auto kernel, int per_thread) {
        plan.wide = per_thread % 4 == 0 && routing.experts == 32 * per_thread && plan.threads > 0 && plan.per == per_thread && reinterpret_cast<uintptr_t>(logits) % (4 * sizeof(T)) == 0 &&
                    reinterpret_cast<uintptr_t>(bias) % 16 == 0;
        return launch_dependent(kernel, grid, block, 0, 1, stream, logits, bias, ids, weights, tokens, plan);
    };
    if (plan.per <= 1) return with(route_experts_kernel<T, 1>, 1);
    if (plan.per <= 2) return with(route_experts_kernel<T, 2>, 2);
    if (plan.per <= 4) return with(route_experts_kernel<T, 4>, 4);
    if (plan.per <= 8) return with(route_experts_kernel<T, 8>, 8);
    if (plan.per <= 16) return with(route_experts_kernel<T, 16>, 16);
    return with(route_experts_kernel<T, 32>, 32);
}

}  // namespace

cudaError_t launch_route_experts(const void *logits, bool logits_f32, const float *bias, int *ids, float *weights, int tokens, const Routing &routing, cudaStream_t stream) {
    return logits_f32 ? launch(static_cast<const float *>(logits), bias, ids, weights, tokens, routing, stream)
                      : launch(static_cast<const uint16_t *>(logits), bias, ids, weights, tokens, routing, stream);
}

}  // namespace nerve
