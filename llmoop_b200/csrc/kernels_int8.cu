// Linears of 8-bit integers on the fifth-generation tensor cores: y[m][n] = (sum_k q[m][k] w[n][k]) a[m] s[n], with int8
// weights w and one f32 scale s per output channel.  The activations are quantised per row on the way in: a = amax / 127,
// q = x / a to the nearest whole number, ties to even.  tcgen05.mma.kind::i8 adds the products in 32-bit integers, which
// hold every sum of up to 131072 columns (127 * 128 * 131072 < 2^31): the sums are exact, so that neither the shape of the
// tiles nor the company of a lane shows in its outputs, and the only roundings are those of q, of the scales' products
// and of the output.
//
// Kernels, and what bounds them (B200; us of one launch, or of the call where it says so):
//   quantise_rows_kernel  rows to whole numbers; DRAM and the issue of 134 warp instructions for sixteen values a thread (2048 x 14336 bf16
//                         from DRAM: 16 us, 5.4 TB/s)
//   int8_gemm_kernel      many lanes, experts of many tokens; the tensor pipe at the clock that the power limit leaves, 1.64 GHz
//                         (2048 x 4096 x 14336: 85 us, 2.8 POP/s; 8192 x 8192 x 8192: 3.0), or the weights' bytes (160 lanes of
//                         the 28672 x 8192 pair: 86 us a call, 5.6 TB/s), or the outputs where K is short
//   int8_stream_kernel    up to 128 lanes; the weights' bytes (4 x 128256 x 4096: 83 us, 6.3 TB/s) or the chain of its steps
//                         (1 x 4096 x 4096: 6.0 us a call from DRAM, 4.9 from L2)
//   expert_groups_kernel, experts_sum_kernel  around the experts' products; the chain of its barriers, DRAM
//
// The gate/up pair multiplies the same lanes by a tile of each matrix into sums that lie side by side, so that one thread holds both
// factors of an output.
//
// The experts' products are the same kernels over tiles that expert_groups_kernel, or few tokens themselves, make of the routes.
// Waits are bounded; a wait that expires sets the error word, and the CTA still frees its tensor memory.  In every role the unbounded
// wait for the kernel in front comes before the first of them that could last as long, so none counts that kernel's time.
//
// No pointer here is __restrict__: what the kernel in front writes may only be read behind the wait for it, and a load through a
// const __restrict__ pointer, which promises that nobody writes, is free to move in front of that (the routes of a replayed
// graph were read before they were there).
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "launch.cuh"

namespace nerve {

namespace {

constexpr int BLOCK_K = 128;  // columns per stage: one swizzled row of 128 bytes
constexpr int ROWS = 128;     // the MMA's M
constexpr int MAX_LANES = 256, MAX_STAGES = 32;
constexpr int OUTPUT_WARPS = 8, THREADS = 128 + 32 * OUTPUT_WARPS;
constexpr size_t SMEM_LIMIT = 226 * 1024, SMEM_HALF = 112 * 1024;
constexpr unsigned int SPIN_LIMIT = 1u << 22;  // tries of 1.5 us

constexpr int FEW = 8, STREAM_LANES = 128;         // lanes of which a CTA may quantise its own copy; the most of the few-lane kernel
constexpr int SPLIT_TILES = 32, SPLIT_K = 4096;    // the most tiles, of no fewer columns, whose columns are split
constexpr bool may_split(int lanes, int k) { return lanes > FEW && k >= SPLIT_K; }

enum Mode { LINEAR, PAIR, EXPERTS_PAIR, EXPERTS_DOWN };

__device__ __forceinline__ uint64_t swizzled_descriptor(uint32_t shared_address) {  // K-major, 128-byte swizzle, 1024 bytes between 8-row atoms
    return static_cast<uint64_t>((shared_address & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ bool wait_barrier(uint32_t barrier, uint32_t parity, int *error_flag) {
    unsigned int spins = 0;
    while (true) {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done)
            : "r"(barrier), "r"(parity)
            : "memory");
        if (done) return true;
        if (++spins > SPIN_LIMIT) {
            if (error_flag != nullptr) *static_cast<volatile int *>(error_flag) = 3;  // (mapped host memory)
            return false;
        }
    }
}
__device__ __forceinline__ bool elect_one() {
    uint32_t elected;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(elected));
    return elected != 0;
}
__device__ __forceinline__ void commit_to(uint32_t barrier) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t barrier, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_tile(uint32_t target, const CUtensorMap *map, int column, int row, uint32_t barrier) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(target), "l"(map), "r"(column), "r"(row),
                 "r"(barrier)
                 : "memory");
}

// Both on 16-byte boundaries, a multiple of sixteen bytes.
__device__ __forceinline__ void copy_bytes(uint32_t target, const uint8_t *from, uint32_t bytes, uint32_t barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(target), "l"(from), "r"(bytes), "r"(barrier) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---- of a pair of CTAs (cta_group::2)
__device__ __forceinline__ uint32_t of_rank(uint32_t address, int rank) {  // the same place in that CTA's shared memory
    uint32_t out;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(address), "r"(rank));
    return out;
}
__device__ __forceinline__ void copy_tile_of_pair(uint32_t target, const CUtensorMap *map, int column, int row, uint32_t barrier) {  // barrier: either CTA's
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(target), "l"(map), "r"(column),
                 "r"(row), "r"(barrier)
                 : "memory");
}
// The same for bytes that nobody reads again: the first to leave L2.
__device__ __forceinline__ void copy_tile_once(uint32_t target, const CUtensorMap *map, int column, int row, uint32_t barrier) {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(target), "l"(map),
                 "r"(column), "r"(row), "r"(barrier), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void commit_to_pair(uint32_t barrier) {  // that barrier of both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(barrier), "h"(static_cast<uint16_t>(3)) : "memory");
}
// Relaxed: a release to the other CTA would first wait for this thread's stores to global memory (12000 cycles a tile where
// the outputs took 500).  What it hands over are sums that have been read.
__device__ __forceinline__ void arrive_at(uint32_t barrier) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(barrier) : "memory"); }
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Into L2, which later writes to the tile reach: safe ahead of the wait for the kernel in front, whatever that writes.
__device__ __forceinline__ void prefetch_tile(const CUtensorMap *map, int column, int row) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(column), "r"(row) : "memory");
}

// Whether it holds for all COUNT threads of named barrier ID: they go on together or not at all.
template <int ID, int COUNT>
__device__ __forceinline__ bool all_of(bool mine) {
    uint32_t all;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %1, 0;\n"
        "bar.red.and.pred q, %2, %3, p;\n"
        "selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(all)
        : "r"(static_cast<uint32_t>(mine)), "n"(ID), "n"(COUNT)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ uint32_t shared_address(const void *pointer) { return static_cast<uint32_t>(__cvta_generic_to_shared(pointer)); }
__device__ __forceinline__ void arrive(uint32_t barrier) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory"); }
__device__ __forceinline__ void init_barrier(uint32_t barrier, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(count) : "memory"); }


// NaN stays NaN.
__device__ __forceinline__ uint16_t to_bf16(float value) { return __bfloat16_as_ushort(__float2bfloat16_rn(value)); }
__device__ __forceinline__ uint32_t two_bf16(float low, float high) {
    const __nv_bfloat162 both = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t *>(&both);
}

// ---- quantisation of activation rows

// Bytes from one quantised row to the next: a block of 128 columns is then one line of the cache, not two (1030
// lanes of 4096 x 12400: 61 us, 74 with rows of k bytes).
__host__ __device__ constexpr int pitch_of(int k) { return (k + BLOCK_K - 1) / BLOCK_K * BLOCK_K; }

// Sixteen values of a row, as they are read.
struct HeldBf16 {
    uint4 words[2];
    __device__ __forceinline__ void load(const uint16_t *row, int at, bool wide) {
        if (wide) {
            words[0] = reinterpret_cast<const uint4 *>(row + at)[0];
            words[1] = reinterpret_cast<const uint4 *>(row + at)[1];
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = row[at + 2 * i] | (static_cast<uint32_t>(row[at + 2 * i + 1]) << 16);
            words[0] = make_uint4(w[0], w[1], w[2], w[3]);
            words[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4 &four = words[i >> 2];
        return (i & 3) == 0 ? four.x : (i & 3) == 1 ? four.y : (i & 3) == 2 ? four.z : four.w;
    }
    // the largest magnitude, as the bits of an f32
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) most = __vmaxu2(most, word(i) & 0x7fff7fffu);
        return max(most & 0xffff0000u, most << 16);
    }
    __device__ __forceinline__ float value(int i) const { return i & 1 ? bf16_hi(word(i >> 1)) : bf16_lo(word(i >> 1)); }
    __device__ __forceinline__ void scale_up() {  // exact
        uint32_t *w = reinterpret_cast<uint32_t *>(words);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = (__float_as_uint(bf16_lo(w[i]) * 0x1p+90f) >> 16) | (__float_as_uint(bf16_hi(w[i]) * 0x1p+90f) & 0xffff0000u);
    }
};
struct HeldF32 {
    float4 words[4];
    __device__ __forceinline__ void load(const float *row, int at, bool) {
#pragma unroll
        for (int i = 0; i < 4; i++) words[i] = reinterpret_cast<const float4 *>(row + at)[i];
    }
    __device__ __forceinline__ float value(int i) const {
        const float4 &four = words[i >> 2];
        return (i & 3) == 0 ? four.x : (i & 3) == 1 ? four.y : (i & 3) == 2 ? four.z : four.w;
    }
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) most = max(most, __float_as_uint(fabsf(value(i))));
        return most;
    }
    __device__ __forceinline__ void scale_up() {
#pragma unroll
        for (int i = 0; i < 4; i++) words[i] = make_float4(words[i].x * 0x1p+90f, words[i].y * 0x1p+90f, words[i].z * 0x1p+90f, words[i].w * 0x1p+90f);
    }
};

// q = rint(x multiplier); rows of tiny values, whose 127 / amax is not finite, are taken times 2^90 (scale_up).  The multiplier is
// 127 / amax, or up to two steps more: a bf16 quotient 127 x / amax is 2^-16 of itself away from the nearest tie (both
// significands are whole numbers below 256) unless it is one; ties are x = amax / 2, whose 63.5 a multiplier too large sends to
// the even 64 as the true one does, and those of an amax of 254 powers of two, whose multiplier is a power of two and exact.
// (An approximate reciprocal, a step of Newton's and a look at the remainder: the division rounded up takes a kernel of
// microseconds 0.4 us.)  An f32 quotient (the experts' intermediate rows) may lie nearer to a tie than that and fall to its other side.
constexpr float UP = 0x1p+90f;
__device__ __forceinline__ bool is_tiny(uint32_t amax_bits) { return amax_bits < 0x12800000u; }  // 2^-90
__device__ __forceinline__ bool is_finite(uint32_t amax_bits) { return amax_bits < 0x7f800000u; }
__device__ __forceinline__ float row_multiplier(uint32_t amax_bits) {  // magnitudes compare as their bits do; infinities and NaN are the largest
    const float amax = __uint_as_float(amax_bits) * (is_tiny(amax_bits) ? UP : 1.0f);
    float inverse;
    asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(amax));
    const float first = 127.0f * inverse, second = __fmaf_rn(__fmaf_rn(-first, amax, 127.0f), inverse, first);
    const float up = __fmaf_rn(-second, amax, 127.0f) > 0.0f ? __uint_as_float(__float_as_uint(second) + 1u) : second;
    return amax_bits != 0 && is_finite(amax_bits) ? up : 0.0f;
}
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {  // a row with an infinity or a NaN is NaN throughout
    return is_finite(amax_bits) ? __uint_as_float(amax_bits) / 127.0f : __uint_as_float(0x7fffffffu);
}
// Sixteen whole numbers as bytes.
template <typename Held>
__device__ __forceinline__ uint4 quantise(const Held &held, float multiplier) {
    uint32_t out[4];
#pragma unroll
    for (int word = 0; word < 4; word++) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = __float_as_uint(__fmaf_rn(held.value(4 * word + i), multiplier, 12582912.0f));  // 1.5 * 2^23: one rounding, to even; two's complement in the low bits
        out[word] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// ---- the experts' routes: places in the order of the experts, tiles of them

// Routes by number, ids [pairs], and what is made of them: tiles {expert, first place, places}, counts {tiles, places}.
struct Grouping {
    const int *ids;
    int pairs, experts, tile_lanes;
    int4 *tiles;
    int *counts;
    __device__ __forceinline__ bool routed(int id) const { return static_cast<uint32_t>(id) < static_cast<uint32_t>(experts); }
};
// The most routes that every CTA of the rows' quantisation looks through, for that many routes a token and with that many threads at
// least: a launch less than with expert_groups_kernel in front.  Over 54 shapes of up to 512 routes 1.2 us less on average (14 tokens of 6 of
// 29 experts 20.0 us and 22.0, 24 of 8 of 128 experts 87.4 and 89.0, 250 of 2 of 8 17.4 and 18.7; at worst 1.5 more, 64 of 8 of 128
// experts 107.0 and 105.4).  A token's routes are looked up one after the other: 32 of 16 of 64 25.9 and 26.6, but 16 of 32 of 128 35.9 and
// 34.6, 9 of 56 of 64 29.7 and 26.2.  120 of 8 of 16, with twice as many routes allowed, 23.1 and 20.8.
constexpr int FEW_GROUPED = 512, FEW_GROUPED_TOP_K = 16, GROUPING_THREADS = 128;

// The routes of the table, some a thread; those to no expert behind all others.
constexpr int ROUTES_HELD = FEW_GROUPED / GROUPING_THREADS;
__device__ __forceinline__ void load_routes(const Grouping &g, int (&ids)[ROUTES_HELD]) {
#pragma unroll
    for (int i = 0; i < ROUTES_HELD; i++) {
        const int pair = threadIdx.x + i * blockDim.x;
        ids[i] = pair < g.pairs ? g.ids[pair] : -1;
        if (!g.routed(ids[i])) ids[i] = g.experts;
    }
}

// By a CTA: counts of every expert, then GROUPING_THREADS threads, of which each has a run of experts.
__device__ __forceinline__ void make_tiles(const Grouping &g) {
    __shared__ int count[EXPERTS_INT8_MAX + 1], warp_places[GROUPING_THREADS / 32], warp_tiles[GROUPING_THREADS / 32];
    int ids[ROUTES_HELD];
    load_routes(g, ids);
    const int thread = threadIdx.x;
    for (int expert = thread; expert < g.experts; expert += blockDim.x) count[expert] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUTES_HELD; i++) atomicAdd(&count[ids[i]], 1);
    __syncthreads();
    const int run = (g.experts + GROUPING_THREADS - 1) / GROUPING_THREADS, first = min(thread * run, g.experts), last = thread < GROUPING_THREADS ? min(first + run, g.experts) : first;
    int places = 0, tiles = 0;
    for (int expert = first; expert < last; expert++) places += count[expert], tiles += (count[expert] + g.tile_lanes - 1) / g.tile_lanes;
    const int own_places = places, own_tiles = tiles;
    for (int offset = 1; offset < 32; offset *= 2) {
        const int other_places = __shfl_up_sync(0xffffffffu, places, offset), other_tiles = __shfl_up_sync(0xffffffffu, tiles, offset);
        if ((thread & 31) >= offset) places += other_places, tiles += other_tiles;
    }
    if (thread < GROUPING_THREADS && (thread & 31) == 31) warp_places[thread >> 5] = places, warp_tiles[thread >> 5] = tiles;
    __syncthreads();
    if (thread >= GROUPING_THREADS) return;
    for (int warp = 0; warp < thread >> 5; warp++) places += warp_places[warp], tiles += warp_tiles[warp];
    if (thread == GROUPING_THREADS - 1) g.counts[0] = tiles, g.counts[1] = places;
    places -= own_places, tiles -= own_tiles;
    for (int expert = first; expert < last; expert++)
        for (int left = count[expert]; left > 0; left -= g.tile_lanes) {
            const int lanes = min(left, g.tile_lanes);
            g.tiles[tiles++] = make_int4(expert, places, lanes, 0);
            places += lanes;
        }
}

// By a CTA: the places of routes first ... first + count - 1, -1 for those to no expert; there behind the CTA's next barrier.
__device__ __forceinline__ void find_places(const Grouping &g, int first, int count, int *places) {
    int ids[ROUTES_HELD];
    load_routes(g, ids);
    __shared__ int own[FEW_GROUPED_TOP_K];
    for (int j = threadIdx.x; j < count; j += blockDim.x) {
        own[j] = g.ids[first + j];
        places[j] = g.routed(own[j]) ? 0 : -1;
    }
    __syncthreads();
    for (int j = 0; j < count; j++) {
        const int id = own[j];
        if (!g.routed(id)) continue;
        int before = 0;
#pragma unroll
        for (int i = 0; i < ROUTES_HELD; i++) before += ids[i] < id + (static_cast<int>(threadIdx.x + i * blockDim.x) < first + j ? 1 : 0);
        before = __reduce_add_sync(0xffffffffu, before);
        if ((threadIdx.x & 31) == 0 && before != 0) atomicAdd(&places[j], before);
    }
}

// A row of x is one CTA's, or one warp's (WARP), whose threads hold it in registers, HELD times sixteen values each; what is
// wider is read again, from the caches.  Without places the row goes to its own number; with them (the experts' inputs) once
// to the place of each of its top_k routes, where it has one, and leaves there which route that is (a store of its own for every
// route, which expert_groups_kernel's one CTA would take 8 us for).  With weights the scale is that of the row times its route's weight.
// Bound by DRAM and its instructions for large batches (2048 x 14336: 16 us, 5.4 TB/s), by the chain of loads, barrier and stores for small ones (2 us).
// wide: x rows start on 16-byte boundaries.  k is a multiple of 16.  width > 0: in the order of int8_stream_kernel's stages, blocks of
// 128 columns of that many rows, sixteen bytes of a row swizzled as TMA would.  zeroed: what the kernel behind wants to find at zero.
// GROUPS: places are not there yet.  Every CTA finds those of its own row's routes, as many as routes lie in front of them in the order
// of experts, then of numbers; the first CTA has no row and cuts the experts' places into tiles.
template <typename T, typename Held, int HELD, bool WARP, bool GROUPS>
__global__ void __launch_bounds__(512) quantise_rows_kernel(const T *x, int8_t *q, float *scales, const int *places,
                                                            const int *row_count, int *pair_of, const float *weights, int rows, int top_k,
                                                            int k, int wide, int width, uint4 *zeroed, int zeroed_count, Grouping groups) {
    __shared__ uint32_t warps[16];
    grid_launch_dependents();
    grid_dependency_wait();
    if (GROUPS && blockIdx.x == 0) {
        make_tiles(groups);
        return;
    }
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < zeroed_count; i += gridDim.x * blockDim.x) zeroed[i] = make_uint4(0, 0, 0, 0);
    const int at_row = WARP ? static_cast<int>(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) : static_cast<int>(blockIdx.x) - (GROUPS ? 1 : 0);
    if (row_count != nullptr) rows = *row_count;
    if (at_row >= rows) return;
    const T *row = x + static_cast<size_t>(at_row) * k;
    const int step = (WARP ? 32 : static_cast<int>(blockDim.x)) * 16, first = static_cast<int>(WARP ? threadIdx.x & 31 : threadIdx.x) * 16;
    Held held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (first + i * step < k) held[i].load(row, first + i * step, wide);
    __shared__ int found[GROUPS ? FEW_GROUPED_TOP_K : 1];
    if constexpr (GROUPS) find_places(groups, at_row * top_k, top_k, found);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (first + i * step < k) amax = max(amax, held[i].amax());
    for (int at = first + HELD * step; at < k; at += step) {
        Held more;
        more.load(row, at, wide);
        amax = max(amax, more.amax());
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (!WARP) {
        if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = amax;
        __syncthreads();
        amax = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < (blockDim.x >> 5) ? warps[threadIdx.x & 31] : 0u);
    }
    const float multiplier = row_multiplier(amax);
    const bool placed = GROUPS || places != nullptr;
    const int copies = placed ? top_k : 1;
    const int *const own_places = GROUPS ? found : places + (places != nullptr ? static_cast<size_t>(at_row) * top_k : 0);
    auto store = [&](int at, Held &values) {
        if (is_tiny(amax)) values.scale_up();
        const uint4 packed = quantise(values, multiplier);
        for (int copy = 0; copy < copies; copy++) {
            const int place = placed ? own_places[copy] : at_row;
            const size_t to = width > 0 ? (static_cast<size_t>(at >> 7) * width + place) * BLOCK_K + ((((at >> 4) ^ place) & 7) << 4) : static_cast<size_t>(place) * pitch_of(k) + at;
            if (place >= 0) *reinterpret_cast<uint4 *>(q + to) = packed;
        }
    };
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (first + i * step < k) store(first + i * step, held[i]);
    for (int at = first + HELD * step; at < k; at += step) {
        Held more;
        more.load(row, at, wide);
        store(at, more);
    }
    for (int copy = first / 16; copy < copies; copy += step / 16) {
        const int place = placed ? own_places[copy] : at_row;
        if (place < 0) continue;
        scales[place] = weights != nullptr ? __fmul_rn(row_scale(amax), weights[pair_of[place]]) : row_scale(amax);
        if (placed) pair_of[place] = at_row * top_k + copy;
    }
}

// Rows of up to 1024 columns of which there are more than the chip has warps to wait with are a warp's each (16384 rows of 768
// f32 values: 20 us with a CTA each, 12 with a warp).  Otherwise as many threads as sixteen columns each ask for up to 256, then
// more columns each; twice as many columns each where rows fill the chip, whose time is then the instructions around a thread's first
// load (2048 x 4096 x 14336: 97.9 us a call, 100.1 with half as many; 300 x 14336, where threads are few: 12.7 and 11.5).
template <typename T, typename Held, int MOST>
cudaError_t launch_quantise_rows(const T *x, int8_t *q, float *scales, const int *places, const int *row_count, int *pair_of, const float *weights, int rows, int top_k,
                                 int k, cudaStream_t stream, int width = 0, void *zeroed = nullptr, size_t zeroed_bytes = 0, const Grouping &groups = {}) {
    const int parts = k / 16, wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    const bool grouping = groups.ids != nullptr;
    auto with = [&](auto kernel, int held, int warp_rows) {
        int threads = warp_rows != 0 ? 32 * warp_rows : std::min(512, ((parts + held - 1) / held + 31) / 32 * 32);
        if (grouping) threads = std::max(threads, GROUPING_THREADS);
        return launch_dependent(kernel, dim3(warp_rows != 0 ? (rows + warp_rows - 1) / warp_rows : rows + grouping), dim3(threads), 0, 1, stream, x, q, scales, places, row_count,
                                pair_of, weights, rows, top_k, k, wide, width, static_cast<uint4 *>(zeroed), static_cast<int>(zeroed_bytes / sizeof(uint4)), groups);
    };
    if constexpr (MOST == 4)
        if (grouping) {
            if (parts <= 256) return with(quantise_rows_kernel<T, Held, 1, false, true>, 1, 0);
            if (parts <= 1024) return with(quantise_rows_kernel<T, Held, 2, false, true>, 2, 0);
            return with(quantise_rows_kernel<T, Held, 4, false, true>, 4, 0);
        }
    if (parts <= 64 && rows >= 1024) return with(quantise_rows_kernel<T, Held, 2, true, false>, 2, 8);
    const bool many = rows >= 512;
    if (parts <= 256 && (!many || parts <= 64)) return with(quantise_rows_kernel<T, Held, 1, false, false>, 1, 0);
    if (parts <= (many ? 256 : 1024) || MOST == 2) return with(quantise_rows_kernel<T, Held, 2, false, false>, 2, 0);
    return with(quantise_rows_kernel<T, Held, MOST, false, false>, MOST, 0);
}

// ---- the product

struct Int8Args {
    CUtensorMap weights, up, activations;  // boxes of 128 columns x rows weight rows, and x tile_lanes / 2 lanes
    const float *scales, *up_scales, *lane_scales;
    void *y;
    const uint16_t *residual;
    int lanes, n, k, to_f32;
    int *error_flag;
    int rows;  // output channels of a CTA's tile
    int tile_lanes, lane_tiles, row_tiles, stages, wide;  // wide: bf16 outputs and residual in sixteen bytes
    // splits > 1: as many items to a tile, each a run of its columns; their sums meet in partials (zero before), [tile][CTA][matrix][lane][ROWS],
    // and the last one, by a count per tile and CTA, writes the outputs
    int splits;
    int *partials, *arrived;
    // experts
    const int4 *tiles;
    const int *tile_count, *pair_of;
    int once;  // an expert's routes are one tile, mostly: its weights are read once
};

struct Tile {
    int row0;  // first output channel of this CTA
    int lane0, count, expert;
};
template <Mode MODE>
__device__ __forceinline__ Tile tile_at(const Int8Args &a, int index, int rank) {
    Tile tile;
    if (MODE == LINEAR || MODE == PAIR) {
        tile.row0 = (index / a.lane_tiles * 2 + rank) * a.rows;
        tile.lane0 = index % a.lane_tiles * a.tile_lanes;
        tile.count = min(a.tile_lanes, a.lanes - tile.lane0);
        tile.expert = 0;
    } else {
        const int4 group = a.tiles[index / a.row_tiles];
        tile.row0 = (index % a.row_tiles * 2 + rank) * a.rows;
        tile.expert = group.x;
        tile.lane0 = group.y;
        tile.count = group.z;
    }
    return tile;
}
// Gate's (or the only) weight rows of a tile, or up's: map and row of the matrix.
template <Mode MODE>
__device__ __forceinline__ const CUtensorMap *weights_of(const Int8Args &a, const Tile &tile, int up, int *row) {
    *row = MODE == EXPERTS_PAIR ? (tile.expert * 2 + up) * a.n + tile.row0 : tile.expert * a.n + tile.row0;
    return MODE == PAIR && up ? &a.up : &a.weights;
}

// The outputs' arithmetic, the same to the bit in every kernel (no contraction).
__device__ __forceinline__ float scaled(int sum, float factor, float lane_scale) { return __fmul_rn(__fmul_rn(static_cast<float>(sum), factor), lane_scale); }
__device__ __forceinline__ float silu_product(float gate, float up) { return __fmul_rn(__fdividef(gate, __fadd_rn(1.0f, __expf(-gate))), up); }

// What belongs to the lanes of a tile: the scale and where the row goes.
struct alignas(16) LaneInfo {
    float scale[MAX_LANES];
    int to[MAX_LANES];
};
struct GemmControl {
    LaneInfo lanes[2];
    int last;
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2];
    uint32_t tmem;
};
// bf16 outputs pass through shared memory: a warp's 32 channels of sixteen lanes, PITCH floats a lane (so that eight threads that
// read sixteen bytes each meet all banks), leave it as sixteen bytes a thread.
constexpr int PITCH = 36;
struct Transposed {
    float values[OUTPUT_WARPS][16 * PITCH];
};
template <Mode MODE>
constexpr size_t gemm_control() { return (sizeof(GemmControl) + (MODE == LINEAR || MODE == PAIR ? sizeof(Transposed) : 0) + 1023) / 1024 * 1024; }

__device__ __forceinline__ void load_eight(uint32_t address, int (&d)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void load_sums(uint32_t address, int (&d)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]), "=r"(d[8]), "=r"(d[9]), "=r"(d[10]), "=r"(d[11]),
                   "=r"(d[12]), "=r"(d[13]), "=r"(d[14]), "=r"(d[15])
                 : "r"(address)
                 : "memory");
}

// Persistent: a pair of CTAs (cta_group::2) walks output tiles of up to 256 weight rows (MMA M, half of them each CTA's) by up to
// 256 lanes (MMA N, of which each CTA holds half).  The pair's MMA reads both halves of the lanes, so that a multiprocessor
// copies and holds half of the activations that tiles of its own would take (37 x 1031 x 2032: 9.1 us a call with CTAs of their
// own, 7.0 in pairs; 2048 x 4096 x 14336: 127 and 126).
// Warps: 0 copies both operands with TMA (128-byte-swizzled rows of 128 columns) into a ring as deep as shared memory allows,
// straight on into the next tile; 1 of the first CTA issues the MMAs into one of two accumulators in tensor memory (one behind
// the other from its front and its back, as wide as the tile's lanes); 4-11 write the finished accumulator out while the other fills.
// A tile may have fewer than 256 weight rows: the rest of the MMA's A operand is then whatever lies behind in shared memory, and
// the rest of the accumulator is never read.  So the rows and lanes of a tile are chosen by the time that the whole matrix takes
// (plan_dense, plan_experts), not by the MMA's shape.
// bf16 outputs of even widths leave through shared memory, sixteen bytes a thread (2048 x 4096 x 14336 with a residual: 102 us a call, 105 one by one).
// SPLIT: the columns of a tile are cut into runs, an item each, for matrices of few tiles and many columns.  Their whole-number sums
// meet by atomic adds, in any order the same number, in a buffer that the quantisation has put at zero; whichever item comes last
// writes the outputs (143 x 405 x 18704: 15.5 us, 36.6 in one piece; the pair 20 and 68).
template <Mode MODE, bool SPLIT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) int8_gemm_kernel(const __grid_constant__ Int8Args a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr bool GROUPED = MODE == EXPERTS_PAIR || MODE == EXPERTS_DOWN, TWO = MODE == PAIR || MODE == EXPERTS_PAIR;
    constexpr int MATRICES = TWO ? 2 : 1;
    GemmControl &control = *reinterpret_cast<GemmControl *>(smem);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;         // rank: of the CTA in its pair
    const uint32_t a_bytes = static_cast<uint32_t>((a.rows + 7) / 8 * 8) * BLOCK_K, half_box = static_cast<uint32_t>(a.tile_lanes / 2) * BLOCK_K,
                   stage_bytes = MATRICES * a_bytes + half_box;
    const uint32_t base = shared_address(smem) + static_cast<uint32_t>(gemm_control<MODE>());
    const uint32_t full = shared_address(control.full), empty = shared_address(control.empty), acc_full = shared_address(control.acc_full),
                   acc_empty = shared_address(control.acc_empty);
    // the first CTA's barriers, which both CTAs' copies and outputs report to
    const uint32_t leader_full = of_rank(full, 0), leader_acc_empty = of_rank(acc_empty, 0);
    const int blocks = (a.k + BLOCK_K - 1) / BLOCK_K, splits = SPLIT ? a.splits : 1;
    // item `index`: a tile, or a run of a tile's blocks
    auto tile_of = [&](int index) { return tile_at<MODE>(a, SPLIT ? index / splits : index, rank); };
    auto first_block = [&](int index) { return SPLIT ? blocks * (index % splits) / splits : 0; };  // (1024 blocks at most)
    auto last_block = [&](int index) { return SPLIT ? blocks * (index % splits + 1) / splits : blocks; };
    if (threadIdx.x == 32) prefetch_map(&a.weights);
    if (threadIdx.x == 64) prefetch_map(&a.activations);
    if (MODE == PAIR && threadIdx.x == 96) prefetch_map(&a.up);
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; s++) {
            init_barrier(full + s * 8, 1);
            init_barrier(empty + s * 8, 1);
        }
        for (int s = 0; s < 2; s++) {
            init_barrier(acc_full + s * 8, 1);
            init_barrier(acc_empty + s * 8, 2 * OUTPUT_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // An accumulator: the sums of the tile's lanes, in steps of 32, gate's and then up's.  Those of the CTA's even tiles lie at the
    // front of tensor memory, of its odd ones at the back: where two successive ones have room beside one another, the outputs of
    // the one are written while the other fills.
    uint32_t columns = 32;
    while (columns < static_cast<uint32_t>(2 * MATRICES * a.tile_lanes) && columns < 512) columns *= 2;
    auto width_of = [&](int count) { return static_cast<uint32_t>(MATRICES * ((count + 31) / 32 * 32)); };
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&control.tmem)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    pair_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // not before the tensor memory is this pair's: one of the next kernel's that took it first would wait for this one
    grid_launch_dependents();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(shared_address(&control.tmem)) : "memory");
    tmem = __reduce_or_sync(0xffffffffu, tmem);  // a uniform register

    if (warp == 0) {  // ---- copies: this CTA's weight rows and its half of the lanes, one box each (a box takes some 65 cycles to issue)
        int stage = 0, issued = 0;
        uint32_t parity = 1;  // the first round waits for no release
        if (!GROUPED && lane < MATRICES) {
            int row;
            const CUtensorMap *map = weights_of<MODE>(a, tile_of(pair), lane, &row);
            for (int block = first_block(pair), s = 0; block < last_block(pair) && s < a.stages; block++, s++) prefetch_tile(map, block * BLOCK_K, row);
        }
        grid_dependency_wait();
        const int items = (GROUPED ? *a.tile_count : a.lane_tiles) * a.row_tiles * splits;
        const uint32_t bytes = 2 * (static_cast<uint32_t>(MATRICES * a.rows) * BLOCK_K + half_box);  // of both CTAs
        bool alive = true;
        Tile tile = pair < items ? tile_of(pair) : Tile{};
        for (int index = pair; index < items && alive; index += pairs) {
            const Tile next = index + pairs < items ? tile_of(index + pairs) : tile;
            int row;
            const CUtensorMap *map = lane < MATRICES ? weights_of<MODE>(a, tile, lane, &row) : &a.activations;
            const uint32_t offset = static_cast<uint32_t>(lane) * a_bytes;
            if (lane == MATRICES) row = tile.lane0 + rank * ((tile.count + 31) / 32 * 16);
            for (int block = first_block(index), end = last_block(index); block < end; block++) {
                if (!wait_barrier(empty + stage * 8, parity, a.error_flag)) {
                    for (int s = 0; rank == 0 && s < a.stages && s < issued; s++) {  // the copies in flight land before the CTAs give their memory up
                        const int which = (issued - 1 - s) % a.stages;
                        wait_barrier(full + which * 8, static_cast<uint32_t>(((issued - 1 - s) / a.stages) & 1), a.error_flag);
                    }
                    alive = false;
                    break;
                }
                if (rank == 0 && elect_one()) expect_bytes(full + stage * 8, bytes);
                __syncwarp();
                const uint32_t target = base + static_cast<uint32_t>(stage) * stage_bytes + offset;
                if (GROUPED && a.once && lane < MATRICES) copy_tile_once(target, map, block * BLOCK_K, row, leader_full + stage * 8);
                else if (lane <= MATRICES) copy_tile_of_pair(target, map, block * BLOCK_K, row, leader_full + stage * 8);
                __syncwarp();
                issued++;
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            tile = next;
        }
        // the MMAs' reports on the last stages are in before this CTA's barriers go
        for (int s = 0; alive && s < a.stages && s < issued; s++) {
            const int which = (issued - 1 - s) % a.stages;
            alive = wait_barrier(empty + which * 8, static_cast<uint32_t>(((issued - 1 - s) / a.stages) & 1), a.error_flag);
        }
    } else if (warp == 1) {  // ---- MMAs, by the first CTA for both
        const uint64_t first = swizzled_descriptor(base);
        int stage = 0, round = 0;
        uint32_t parity = 0, last_width = 0;
        bool alive = rank == 0;
        grid_dependency_wait();
        const int items = (GROUPED ? *a.tile_count : a.lane_tiles) * a.row_tiles * splits;
        int count = alive && pair < items ? tile_of(pair).count : 0;
        for (int index = pair; index < items && alive; index += pairs, round++) {
            const int next = index + pairs < items ? tile_of(index + pairs).count : 0;
            // instruction descriptor: s32 accumulator, A and B signed bytes, both K-major, N / 8 in bits 17-22, M / 16 in bits 24-28
            // (M = 256 with bytes: N in steps of 32)
            const uint32_t lanes = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>((count + 31) / 32 * 32)), width = MATRICES * lanes;
            const uint32_t instruction = (2u << 4) | (1u << 7) | (1u << 10) | (lanes / 8 << 17) | (16u << 24);
            const uint32_t accumulator = tmem + ((round & 1) != 0 ? columns - width : 0u);
            if (!wait_barrier(acc_empty + (round & 1) * 8, static_cast<uint32_t>((round / 2 + 1) & 1), a.error_flag)) break;
            if (width + last_width > columns && !wait_barrier(acc_empty + ((round - 1) & 1) * 8, static_cast<uint32_t>(((round - 1) / 2) & 1), a.error_flag)) break;
            last_width = width;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int begin = first_block(index), end = last_block(index);
            for (int block = begin; block < end; block++) {
                if (!wait_barrier(full + stage * 8, parity, a.error_flag)) {
                    alive = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    const uint64_t a_stage = first + static_cast<uint64_t>(stage) * (stage_bytes >> 4), b_stage = a_stage + MATRICES * (a_bytes >> 4);
#pragma unroll
                    for (int step = 0; step < 4 * MATRICES; step++) {  // K = 32 per instruction
                        const int matrix = step >> 2, part = step & 3;
                        const uint32_t accumulate = (block > begin || part > 0) ? 1u : 0u;
                        asm volatile(
                            "{\n"
                            ".reg .pred p;\n"
                            "setp.ne.b32 p, %4, 0;\n"
                            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
                            "}\n" ::"r"(accumulator + matrix * lanes),
                            "l"(a_stage + matrix * (a_bytes >> 4) + part * 2), "l"(b_stage + part * 2), "r"(instruction), "r"(accumulate)
                            : "memory");
                    }
                    commit_to_pair(empty + stage * 8);
                    if (block == end - 1) commit_to_pair(acc_full + (round & 1) * 8);
                }
                __syncwarp();
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            count = next;
        }
    } else if (warp >= 4) {  // ---- outputs: thread = row of the accumulator
        grid_dependency_wait();
        const int items = (GROUPED ? *a.tile_count : a.lane_tiles) * a.row_tiles * splits;
        const int quarter = warp & 3, part = (warp - 4) >> 2, thread = threadIdx.x - 128, row = quarter * 32 + lane;
        // what a tile's outputs take besides its sums; fetched a tile ahead
        struct Extra {
            float factor, up_factor, scale;
            int to;
        };
        auto fetch = [&](const Tile &tile) {
            Extra extra = {};
            const int channel = tile.row0 + row;
            if (row < a.rows && channel < a.n) {
                const size_t at = (GROUPED ? static_cast<size_t>(tile.expert) * MATRICES * a.n : 0) + channel;
                extra.factor = a.scales[at];
                if (TWO) extra.up_factor = MODE == PAIR ? a.up_scales[at] : a.scales[at + a.n];
            }
            if (thread < tile.count) {
                extra.scale = a.lane_scales[tile.lane0 + thread];
                extra.to = MODE == EXPERTS_DOWN ? a.pair_of[tile.lane0 + thread] : tile.lane0 + thread;
                if (MODE == LINEAR && a.residual != nullptr) {  // the tile's part of this lane's row, into L2
                    const char *from = reinterpret_cast<const char *>(a.residual + static_cast<size_t>(extra.to) * a.n + tile.row0);
                    for (int at = 0; at < 2 * min(a.rows, a.n - tile.row0); at += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + at));
                }
            }
            return extra;
        };
        int round = 0;
        Tile tile = {}, next = {};
        Extra extra = {};
        if (pair < items) {
            tile = tile_of(pair);
            if (pair + pairs < items) next = tile_of(pair + pairs);
            extra = fetch(tile);
        }
        for (int index = pair; index < items; index += pairs, round++) {
            LaneInfo &info = control.lanes[round & 1];  // (what stood there two tiles before is out: all threads have passed the last tile's barrier)
            info.scale[thread] = extra.scale;
            info.to[thread] = extra.to;
            const float factor = extra.factor, up_factor = extra.up_factor;
            if (!all_of<1, 32 * OUTPUT_WARPS>(wait_barrier(acc_full + (round & 1) * 8, static_cast<uint32_t>((round / 2) & 1), a.error_flag))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            Tile after = {};
            if (index + 2 * pairs < items) after = tile_of(index + 2 * pairs);
            if (index + pairs < items) extra = fetch(next);
            const uint32_t width = width_of(tile.count), accumulator = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + ((round & 1) != 0 ? columns - width : 0u);
            const int channel = tile.row0 + row;
            const bool in_range = row < a.rows && channel < a.n;
            int *const partials = SPLIT ? a.partials + static_cast<size_t>(index / splits * 2 + rank) * MATRICES * a.tile_lanes * ROWS + row : nullptr;
            bool writes = true;
            if (SPLIT) {
                if (quarter * 32 < a.rows)
                    for (int column = part * 16; column < tile.count; column += 32) {
#pragma unroll
                        for (int matrix = 0; matrix < MATRICES; matrix++) {
                            int sums[16];
                            load_sums(accumulator + matrix * (width / 2) + static_cast<uint32_t>(column), sums);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            int *const to = partials + static_cast<size_t>(matrix * a.tile_lanes + column) * ROWS;
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                atomicAdd(to + i * ROWS, sums[i]);  // (what lies behind the tile's rows and lanes is added too, and not read)
                        }
                    }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive_at(leader_acc_empty + (round & 1) * 8);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (thread == 0) {  // for all: a fence covers what the barrier has shown this thread
                    __threadfence();
                    control.last = atomicAdd(a.arrived + index / splits * 2 + rank, 1) == splits - 1;
                    __threadfence();
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                writes = control.last != 0;
            }
            if (quarter * 32 < a.rows && writes) {
                const uint16_t *residual = MODE == LINEAR ? a.residual : nullptr;
                // Wide outputs: thread = eight channels of lanes lane / 4 and lane / 4 + 8.  What is added to them is fetched a step ahead.
                const bool wide = (MODE == LINEAR || MODE == PAIR) && a.wide;
                const int eight = tile.row0 + quarter * 32 + (lane & 3) * 8;
                const bool eight_in_range = quarter * 32 + (lane & 3) * 8 < a.rows && eight < a.n;
                float *const transposed = reinterpret_cast<Transposed *>(smem + sizeof(GemmControl))->values[warp - 4];
                uint4 beside[2];
                auto fetch_beside = [&](int column) {
#pragma unroll
                    for (int half = 0; half < 2; half++)
                        if (eight_in_range && column + half * 8 + lane / 4 < tile.count)
                            beside[half] = *reinterpret_cast<const uint4 *>(residual + static_cast<size_t>(tile.lane0 + column + half * 8 + lane / 4) * a.n + eight);
                };
                uint16_t narrow[16];  // the same for outputs one by one: lane column + i
                auto fetch_narrow = [&](int column) {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (in_range && column + i < tile.count) narrow[i] = residual[static_cast<size_t>(tile.lane0 + column + i) * a.n + channel];
                };
                if (residual != nullptr) {
                    if (wide) fetch_beside(part * 16);
                    else fetch_narrow(part * 16);
                }
                for (int column = part * 16; column < tile.count; column += 32) {
                    int sums[16], up_sums[16];
                    if (SPLIT) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            sums[i] = __ldcg(partials + static_cast<size_t>(column + i) * ROWS);
                            if (TWO) up_sums[i] = __ldcg(partials + static_cast<size_t>(a.tile_lanes + column + i) * ROWS);
                        }
                    } else {
                        load_sums(accumulator + static_cast<uint32_t>(column), sums);
                        if (TWO) load_sums(accumulator + width / 2 + static_cast<uint32_t>(column), up_sums);
                    }
                    float scales[16];
                    int to[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        *reinterpret_cast<float4 *>(scales + i) = *reinterpret_cast<const float4 *>(info.scale + column + i);
                        if (GROUPED) *reinterpret_cast<int4 *>(to + i) = *reinterpret_cast<const int4 *>(info.to + column + i);
                    }
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    float values[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        values[i] = scaled(sums[i], factor, scales[i]);
                        if (TWO) values[i] = silu_product(values[i], scaled(up_sums[i], up_factor, scales[i]));
                    }
                    if (wide) {
#pragma unroll
                        for (int i = 0; i < 16; i++) transposed[i * PITCH + lane] = values[i];
                        __syncwarp();
                        uint4 out[2];
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const float4 *from = reinterpret_cast<const float4 *>(transposed + (half * 8 + lane / 4) * PITCH + (lane & 3) * 8);
                            const float4 low = from[0], high = from[1];
                            float v[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
                            if (residual != nullptr) {
                                const uint32_t words[4] = {beside[half].x, beside[half].y, beside[half].z, beside[half].w};
#pragma unroll
                                for (int i = 0; i < 8; i++) v[i] = __fadd_rn(v[i], i & 1 ? bf16_hi(words[i >> 1]) : bf16_lo(words[i >> 1]));
                            }
                            out[half] = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
                        }
                        if (residual != nullptr) fetch_beside(column + 32);
#pragma unroll
                        for (int half = 0; half < 2; half++)
                            if (eight_in_range && column + half * 8 + lane / 4 < tile.count)
                                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.y) + static_cast<size_t>(tile.lane0 + column + half * 8 + lane / 4) * a.n + eight) = out[half];
                        __syncwarp();
                        continue;
                    }
                    const int count = in_range ? tile.count - column : 0;
                    if (GROUPED) {
                        float *const out = static_cast<float *>(a.y) + channel;
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (i < count) out[static_cast<size_t>(to[i]) * a.n] = values[i];
                    } else {
                        const size_t at = static_cast<size_t>(tile.lane0 + column) * a.n + channel;
                        if (residual != nullptr) {
#pragma unroll
                            for (int i = 0; i < 16; i++) values[i] = __fadd_rn(values[i], bf16_bits_to_f32(narrow[i]));
                            fetch_narrow(column + 32);
                        }
                        if (MODE == LINEAR && a.to_f32) {
                            float *const out = static_cast<float *>(a.y) + at;
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (i < count) out[static_cast<size_t>(i) * a.n] = values[i];
                        } else {
                            uint16_t *const out = static_cast<uint16_t *>(a.y) + at;
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (i < count) out[static_cast<size_t>(i) * a.n] = to_bf16(values[i]);
                        }
                    }
                }
            }
            if (!SPLIT) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive_at(leader_acc_empty + (round & 1) * 8);
            }
            tile = next;
            next = after;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    pair_sync();  // neither CTA leaves while the other still reads its memory or reports to its barriers: the release waits for those reports
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// ---- few lanes: the weights stream by

// Up to 128 lanes: bound by the weights' bytes, or for small matrices by the chain of its steps.  A stage of the ring is the
// MMA's 128 rows; a tile with fewer weight rows puts `groups` successive blocks of 128 columns on top of one another there,
// 128 / groups rows to each, and multiplies them by as many blocks of the activations side by side (N = groups x width): of the
// products only those of a block with its own block count, the outputs add them up.  The tensor pipe takes some 70 cycles for
// an instruction of 128 rows whatever N up to 128, so that a tile of 28 rows costs a fourth of what one block after the
// other would.
// int8_gemm_kernel takes the same matrices; where the lanes come quantised, the lower of the two plans' estimates decides (32 x 4096 x
// 8192: 10.6 us here, 13.5 there; 100 x 1024 x 1040: 8.4 and 6.1; 100 x 64 x 14336: 20.8 and, with its columns split, 9.8; over 440 shapes of
// 12 to 128 lanes the choice costs 0.7 % of the better one's time on average).  For up to eight lanes that is almost always this one; wide pairs
// whose rows make a wave and a little here go there (4 lanes of a 9863 x 8304 pair: 43.8 us here, 33.9 there; 3 x 9853 x 36048: 160 and 116), and
// some linears of close estimates (8 x 19981 x 59648: 219 and 186).
// Activations, as blocks of 128 columns of `width` swizzled rows:
//   Up to eight lanes of few columns every CTA quantises itself while its first weights are on their way, and keeps them: one launch.
//   More are quantised by a kernel in front, which leaves them in this order (PREPARED), and come with every stage.
// Warps: 0 copies, 1 issues MMAs, 4-7 (PREPARED: 4-11) write outputs, 4-11 (the experts' down product: 8-11) quantise.
constexpr int STREAM_THREADS = 384, STREAM_MAX_STAGES = 12;
constexpr uint32_t ATOM = 1024, STREAM_STAGE = ROWS * BLOCK_K;
constexpr int FEW_ROUTES = 128;          // of the experts' form
constexpr int STREAM_SMALL_SHARE = 48;   // stages
// Values of which every CTA quantises its own copy (8 x 4096 lanes of a 4096 x 4096 matrix: 10.3 us so, 6.6 with a launch in front; 4 x 4096
// of a 14336 x 4096 pair: 21.3 so, 22.5 with one).
constexpr int STREAM_OWN = 16384;

struct StreamArgs {
    CUtensorMap weights, up;  // boxes of 128 columns x rows weight rows
    const void *x;            // bf16 rows; the down product: f32; on 16-byte boundaries.  PREPARED: blocks of 128 columns x width rows
    const float *scales, *up_scales, *lane_scales;
    void *y;
    const uint16_t *residual;
    int lanes, n, k, to_f32;
    int *error_flag;
    int rows, groups, row_tiles, stages;  // rows: output channels of a tile
    int width;                            // lanes of a block of the activations: 8, or a multiple of 16
    int span_log;                         // 32, 64 or 128 threads of the outputs, no fewer than rows, take a lane
    // experts
    const int *ids;
    const float *weights_of;
    int top_k, experts;
};

struct StreamControl {
    uint64_t full[STREAM_MAX_STAGES], empty[STREAM_MAX_STAGES], acc_full[2], acc_empty[2], b_full[2], b_empty[2];
    uint32_t tmem;
    int used;                                // experts with a route
    uint32_t amax[2][FEW];
    float lane_scales[2][FEW];
    float prepared_scales[STREAM_LANES];
};
// Routes by expert, for tables of up to FEW_ROUTES routes of FEW tokens.
struct StreamRoutes {
    int slot[EXPERTS_INT8_MAX];              // first route of an expert, then its number among the used ones
    int expert[FEW_ROUTES];
    int lead[FEW_ROUTES][FEW];               // a token's first route to the used expert; past all routes: none
    int ids[FEW_ROUTES];
    int before[FEW_ROUTES / 32];
};
constexpr int NO_ROUTE = 1 << 30;

// The first 128 threads, beside the others' quantisation.  The used experts are numbered in the order of their first routes, the
// same in every CTA.
__device__ __forceinline__ void find_routes(const StreamArgs &a, StreamControl &control, StreamRoutes &routes) {
    auto sync = [] { asm volatile("bar.sync 4, 128;" ::: "memory"); };
    const int thread = threadIdx.x, count = a.lanes * a.top_k;
    int expert = thread < count ? a.ids[thread] : -1;
    if (expert >= a.experts) expert = -1;
    for (int e = thread; e < a.experts; e += FEW_ROUTES) routes.slot[e] = NO_ROUTE;
#pragma unroll
    for (int i = 0; i < FEW; i++) routes.lead[thread][i] = NO_ROUTE;
    sync();
    routes.ids[thread] = expert;
    if (expert >= 0) atomicMin(&routes.slot[expert], thread);
    sync();
    const bool first = expert >= 0 && routes.slot[expert] == thread;
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    if ((thread & 31) == 0) routes.before[thread >> 5] = __popc(firsts);
    sync();
    int number = __popc(firsts & ((1u << (thread & 31)) - 1u)), used = 0;
    for (int warp = 0; warp < FEW_ROUTES / 32; warp++) {
        if (warp < thread >> 5) number += routes.before[warp];
        used += routes.before[warp];
    }
    if (first) {
        routes.slot[expert] = number;
        routes.expert[number] = expert;
    }
    if (thread == 0) control.used = used;
    sync();
    if (expert >= 0) atomicMin(&routes.lead[routes.slot[expert]][thread / a.top_k], thread);
    sync();
}

// Quantises rows into atoms at `atoms`, by WARPS warps of which this is number `warp`.  row_of(lane): where lane's row
// starts, NULL for a lane without one.  sync(): among those warps.  A warp takes thirty-two
// parts of sixteen columns at a time and requests BATCH such together (one after the other four lanes of 4096 columns took 6.4 us,
// each the latency of L2); where there are no more, it keeps them from the search for the largest to the quantisation.
template <int WARPS, int BATCH, typename T, typename Held, typename RowOf, typename Sync>
__device__ __forceinline__ void quantise_few(const StreamArgs &a, uint8_t *atoms, uint32_t *amax, float *scales, int warp, RowOf row_of, Sync sync) {
    const int parts = a.k / 16, runs = (parts + 31) / 32, thread = warp * 32 + static_cast<int>(threadIdx.x & 31);
    if (thread < FEW) amax[thread] = 0;
    struct Position {
        int lane, run;
    };
    auto advance = [&](Position at) {
        at.run += WARPS;
        while (at.run >= runs) at.run -= runs, at.lane++;
        return at;
    };
    auto start = [&] {
        Position at{0, warp};
        while (at.run >= runs) at.run -= runs, at.lane++;
        return at;
    };
    Held held[BATCH];
    auto load = [&](Position at) {
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            if (at.lane >= a.lanes) break;
            const T *row = row_of(at.lane);
            const int part = at.run * 32 + static_cast<int>(threadIdx.x & 31);
            if (row != nullptr && part < parts) held[j].load(row, part * 16, true);
            at = advance(at);
        }
        return at;
    };
    Position first = start(), next = load(first);
    const bool all_held = next.lane >= a.lanes;
    sync();  // amax is 0
    while (true) {
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            if (first.lane >= a.lanes) break;
            const int part = first.run * 32 + static_cast<int>(threadIdx.x & 31);
            const uint32_t most = __reduce_max_sync(0xffffffffu, row_of(first.lane) != nullptr && part < parts ? held[j].amax() : 0u);
            if ((threadIdx.x & 31) == 0) atomicMax(&amax[first.lane], most);
            first = advance(first);
        }
        if (first.lane >= a.lanes) break;
        load(first);
    }
    sync();
    // (rolled up: in a kernel of microseconds every instruction is fetched for the first time)
    first = start();
#pragma unroll 1
    while (first.lane < a.lanes) {
        if (!all_held) load(first);
#pragma unroll 1
        for (int j = 0; j < BATCH && first.lane < a.lanes; j++) {
            const int part = first.run * 32 + static_cast<int>(threadIdx.x & 31);
            if (is_tiny(amax[first.lane])) held[0].scale_up();
            if (row_of(first.lane) != nullptr && part < parts)
                *reinterpret_cast<uint4 *>(atoms + (part >> 3) * ATOM + first.lane * BLOCK_K + (((part & 7) ^ first.lane) << 4)) = quantise(held[0], row_multiplier(amax[first.lane]));
#pragma unroll
            for (int i = 0; i + 1 < BATCH; i++) held[i] = held[i + 1];
            first = advance(first);
        }
    }
    if (thread < FEW) scales[thread] = row_scale(amax[thread]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

constexpr size_t STREAM_CONTROL = (sizeof(StreamControl) + 1023) / 1024 * 1024, STREAM_ROUTES = (sizeof(StreamRoutes) + 1023) / 1024 * 1024;
// The sums of some lanes of a finished tile, per lane and row of the accumulator, for each team of four warps.
template <bool PREPARED>
constexpr int SUM_LANES = PREPARED ? 16 : FEW;
template <bool PREPARED>
constexpr size_t STREAM_SUMS = (PREPARED ? 2 : 1) * SUM_LANES<PREPARED> * ROWS * sizeof(int);

template <Mode MODE, bool PREPARED>
__global__ void __launch_bounds__(STREAM_THREADS, 2) int8_stream_kernel(const __grid_constant__ StreamArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr bool GROUPED = MODE == EXPERTS_PAIR || MODE == EXPERTS_DOWN, TWO = MODE == PAIR || MODE == EXPERTS_PAIR, DOWN = MODE == EXPERTS_DOWN;
    static_assert(!(GROUPED && PREPARED));
    StreamControl &control = *reinterpret_cast<StreamControl *>(smem);
    StreamRoutes &routes = *reinterpret_cast<StreamRoutes *>(smem + STREAM_CONTROL + STREAM_SUMS<PREPARED>);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform
    const int blocks = (a.k + BLOCK_K - 1) / BLOCK_K, steps = (blocks + a.groups - 1) / a.groups, slot_rows = ROWS / a.groups;
    const uint32_t block_bytes = static_cast<uint32_t>(a.width) * BLOCK_K;  // of activations
    const uint32_t products = static_cast<uint32_t>(max(16, a.groups * a.width));  // the MMA's N
    const uint32_t atom_bytes = PREPARED ? 0u : static_cast<uint32_t>(steps * a.groups) * ATOM, stage_bytes = STREAM_STAGE + (PREPARED ? products * BLOCK_K : 0u);
    uint8_t *const atoms = smem + STREAM_CONTROL + STREAM_SUMS<PREPARED> + (GROUPED ? STREAM_ROUTES : 0);
    const uint32_t ring = shared_address(atoms) + (DOWN ? 2 : 1) * atom_bytes;
    const uint32_t full = shared_address(control.full), empty = shared_address(control.empty), acc_full = shared_address(control.acc_full),
                   acc_empty = shared_address(control.acc_empty), b_full = shared_address(control.b_full), b_empty = shared_address(control.b_empty);
    constexpr int QUANTISING = DOWN ? 4 : 8;  // warps
    const int teams = PREPARED && a.lanes > SUM_LANES<PREPARED> ? 2 : 1;  // of four warps that write outputs
    if (threadIdx.x == 32) prefetch_map(&a.weights);
    if (MODE == PAIR && threadIdx.x == 96) prefetch_map(&a.up);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STREAM_MAX_STAGES; s++) {
            init_barrier(full + s * 8, 1);
            init_barrier(empty + s * 8, 1);
        }
        for (int s = 0; s < 2; s++) {
            init_barrier(acc_full + s * 8, 1);
            init_barrier(acc_empty + s * 8, 4 * teams);
            init_barrier(b_full + s * 8, QUANTISING);
            init_barrier(b_empty + s * 8, 2);  // the MMAs' commit and the outputs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const uint32_t acc_columns = (products + 31u) & ~31u;
    uint32_t columns = 64;
    while (columns < 2 * acc_columns + (a.width < SUM_LANES<PREPARED> ? 16u : 0u)) columns *= 2;  // (the outputs read SUM_LANES at a time)
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&control.tmem)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // not before the tensor memory is this CTA's: one of the next kernel's that took it first would wait for this one.  The experts'
    // gate/up product also waits for the kernel in front before: the down product, which may start then, reads the routes and the
    // weights while this one still runs, and waits for its rows alone.  (Its CTAs start where a multiprocessor has their shared memory left or
    // once this kernel's have gone: beside the 144 CTAs of one token of eight routes of 2048 x 768, which take all of it, on four.)
    if (MODE == EXPERTS_PAIR) grid_dependency_wait();
    grid_launch_dependents();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(shared_address(&control.tmem)) : "memory");
    tmem = __reduce_or_sync(0xffffffffu, tmem);  // a uniform register
    auto quantise_all = [&] {  // ---- the lanes, once, by warps 4-11
        auto sync = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        quantise_few<8, 4, uint16_t, HeldBf16>(a, atoms, control.amax[0], control.lane_scales[0], warp - 4,
                                               [&](int row) { return static_cast<const uint16_t *>(a.x) + static_cast<size_t>(row) * a.k; }, sync);
        __syncwarp();
        if (lane == 0) arrive(b_full);
        sync();  // the outputs read the scales
    };
    if (GROUPED && warp < 4) find_routes(a, control, routes);
    if (MODE == EXPERTS_PAIR && warp >= 4) quantise_all();
    if (GROUPED) __syncthreads();  // the routes are known (and the rows quantised)
    const int tiles = (GROUPED ? control.used : 1) * a.row_tiles;
    const int first_tile = static_cast<int>(static_cast<int64_t>(tiles) * blockIdx.x / gridDim.x), last_tile = static_cast<int>(static_cast<int64_t>(tiles) * (blockIdx.x + 1) / gridDim.x);

    if (warp == 0) {  // ---- copies
        const int copies = TWO ? 2 * a.groups : a.groups, group = TWO ? lane >> 1 : lane, up = TWO ? lane & 1 : 0;
        const CUtensorMap *const map = MODE == PAIR && up ? &a.up : &a.weights;
        if (!GROUPED) grid_dependency_wait();
        const uint32_t bytes = static_cast<uint32_t>(copies * a.rows) * BLOCK_K;
        int stage = 0, issued = 0;
        uint32_t parity = 1;  // the first round waits for no release
        bool alive = true;
        for (int tile = first_tile; tile < last_tile && alive; tile++) {
            const int row0 = tile % a.row_tiles * a.rows, expert = GROUPED ? routes.expert[tile / a.row_tiles] : 0;
            for (int step = 0; step < steps; step++) {
                if (DOWN && issued == a.stages) grid_dependency_wait();  // from here on the MMAs release the stages
                if (!wait_barrier(empty + stage * 8, parity, a.error_flag)) {
                    for (int s = 0; s < a.stages && s < issued; s++) {  // the copies in flight land before the CTA gives its memory up
                        const int which = (issued - 1 - s) % a.stages;
                        wait_barrier(full + which * 8, static_cast<uint32_t>(((issued - 1 - s) / a.stages) & 1), a.error_flag);
                    }
                    alive = false;
                    break;
                }
                const uint32_t stage_at = ring + static_cast<uint32_t>(stage) * stage_bytes;
                // (the last step's missing blocks are zeros among the weights, whatever the activations' part of the stage holds)
                const uint32_t prepared_bytes = PREPARED ? static_cast<uint32_t>(min(a.groups, blocks - step * a.groups)) * block_bytes : 0u;
                if (elect_one()) expect_bytes(full + stage * 8, bytes + prepared_bytes);
                __syncwarp();
                if (lane < copies) {
                    const uint32_t target = stage_at + static_cast<uint32_t>(group * slot_rows + up * (slot_rows / 2)) * BLOCK_K;
                    const int row = MODE == EXPERTS_PAIR ? (expert * 2 + up) * a.n + row0 : expert * a.n + row0;
                    copy_tile(target, map, (step * a.groups + group) * BLOCK_K, row, full + stage * 8);
                } else if (PREPARED && lane == copies) {
                    copy_bytes(stage_at + STREAM_STAGE, static_cast<const uint8_t *>(a.x) + static_cast<size_t>(step * a.groups) * block_bytes, prepared_bytes, full + stage * 8);
                }
                __syncwarp();
                issued++;
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp == 1) {  // ---- MMAs
        if (MODE != EXPERTS_PAIR) grid_dependency_wait();
        // instruction descriptor as in int8_gemm_kernel, M = 128
        const uint32_t instruction = __reduce_or_sync(0xffffffffu, (2u << 4) | (1u << 7) | (1u << 10) | (products / 8 << 17) | (8u << 24));
        const uint64_t a_first = swizzled_descriptor(ring), b_first = swizzled_descriptor(shared_address(atoms));
        int stage = 0, round = 0, builds = 0, expert = -1;
        uint32_t parity = 0;
        bool alive = true;
        for (int tile = first_tile; tile < last_tile && alive; tile++, round++) {
            const int which = DOWN ? tile / a.row_tiles : 0;
            if (!PREPARED && which != expert) {
                if (!wait_barrier(b_full + (builds & 1) * 8, static_cast<uint32_t>((builds >> 1) & 1), a.error_flag)) break;
                expert = which;
                builds++;
            }
            const bool last_of_build = DOWN && (tile + 1 == last_tile || (tile + 1) / a.row_tiles != which);
            const uint64_t b_base = b_first + static_cast<uint64_t>((builds - 1) & 1) * (DOWN ? atom_bytes >> 4 : 0);
            if (!wait_barrier(acc_empty + (round & 1) * 8, static_cast<uint32_t>((round / 2 + 1) & 1), a.error_flag)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t accumulator = tmem + (round & 1) * acc_columns;
            for (int step = 0; step < steps; step++) {
                if (!wait_barrier(full + stage * 8, parity, a.error_flag)) {
                    alive = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    const uint64_t a_stage = a_first + static_cast<uint64_t>(stage) * (stage_bytes >> 4),
                                   b_stage = PREPARED ? a_stage + (STREAM_STAGE >> 4) : b_base + static_cast<uint64_t>(step * a.groups) * (ATOM >> 4);
#pragma unroll
                    for (int part = 0; part < 4; part++) {  // K = 32 per instruction
                        const uint32_t accumulate = (step > 0 || part > 0) ? 1u : 0u;
                        asm volatile(
                            "{\n"
                            ".reg .pred p;\n"
                            "setp.ne.b32 p, %4, 0;\n"
                            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
                            "}\n" ::"r"(accumulator),
                            "l"(a_stage + part * 2), "l"(b_stage + part * 2), "r"(instruction), "r"(accumulate)
                            : "memory");
                    }
                    commit_to(empty + stage * 8);
                    if (step == steps - 1) {
                        commit_to(acc_full + (round & 1) * 8);
                        if (last_of_build) commit_to(b_empty + ((builds - 1) & 1) * 8);
                    }
                }
                __syncwarp();
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp >= 4) {
        if (MODE != EXPERTS_PAIR) grid_dependency_wait();
        if (PREPARED) {
            if (static_cast<int>(threadIdx.x) - 128 < a.lanes) control.prepared_scales[threadIdx.x - 128] = a.lane_scales[threadIdx.x - 128];
            asm volatile("bar.sync 1, 256;" ::: "memory");
        } else if (!GROUPED) {
            quantise_all();
        } else if (DOWN && warp >= 8) {  // ---- for every expert of this CTA's tiles, two at a time
            auto sync = [] { asm volatile("bar.sync 2, 128;" ::: "memory"); };
            int builds = 0, expert = -1;
            for (int tile = first_tile; tile < last_tile; tile++) {
                const int which = tile / a.row_tiles;
                if (which == expert) continue;
                expert = which;
                const int buffer = builds & 1;
                if (!all_of<2, 128>(wait_barrier(b_empty + buffer * 8, static_cast<uint32_t>((builds / 2 + 1) & 1), a.error_flag))) break;
                quantise_few<4, 2, float, HeldF32>(a, atoms + buffer * atom_bytes, control.amax[buffer], control.lane_scales[buffer], warp - 8,
                                                  [&](int token) -> const float * {
                                                      const int route = routes.lead[which][token];
                                                      return route == NO_ROUTE ? nullptr : static_cast<const float *>(a.x) + static_cast<size_t>(route) * a.k;
                                                  },
                                                  sync);
                __syncwarp();
                if (lane == 0) arrive(b_full + buffer * 8);
                builds++;
            }
        }
        const int team = (warp - 4) >> 2;
        if (team < teams) {  // ---- outputs, SUM_LANES lanes at a time
            constexpr int CHUNK = SUM_LANES<PREPARED>;
            const int quarter = warp & 3, group = quarter * a.groups / 4, thread = static_cast<int>(threadIdx.x & 127);
            const int span = 1 << a.span_log, row = thread & (span - 1), first_lane = thread >> a.span_log, lane_step = 128 >> a.span_log;
            int(*const sums)[ROWS] = reinterpret_cast<int(*)[ROWS]>(smem + STREAM_CONTROL) + team * CHUNK;
            auto team_sync = [&] {
                if (team == 0) asm volatile("bar.sync 3, 128;" ::: "memory");
                else asm volatile("bar.sync 5, 128;" ::: "memory");
            };
            int round = 0, builds = 0, expert = -1;
            for (int tile = first_tile; tile < last_tile; tile++, round++) {
                const int row0 = tile % a.row_tiles * a.rows, which = GROUPED ? tile / a.row_tiles : 0, channel = row0 + row;
                const bool in_range = row < a.rows && channel < a.n;
                bool alive = true;
                if (DOWN && which != expert) {
                    expert = which;
                    alive = wait_barrier(b_full + (builds & 1) * 8, static_cast<uint32_t>((builds >> 1) & 1), a.error_flag);
                    builds++;
                }
                const float *scales = PREPARED ? control.prepared_scales : control.lane_scales[DOWN ? (builds - 1) & 1 : 0];
                float factor = 0.0f, up_factor = 0.0f;
                if (in_range) {
                    const size_t at = (GROUPED ? static_cast<size_t>(routes.expert[which]) * (TWO ? 2 : 1) * a.n : 0) + channel;
                    factor = a.scales[at];
                    if (TWO) up_factor = MODE == PAIR ? a.up_scales[at] : a.scales[at + a.n];
                }
                uint16_t beside[4];  // four lanes of the residual ahead
                auto fetch_beside = [&](int from) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (in_range && from + i * lane_step < a.lanes) beside[i] = a.residual[static_cast<size_t>(from + i * lane_step) * a.n + channel];
                };
                if (MODE == LINEAR && a.residual != nullptr) fetch_beside(team * CHUNK + first_lane);
                alive = alive && wait_barrier(acc_full + (round & 1) * 8, static_cast<uint32_t>((round / 2) & 1), a.error_flag);
                // they go on together; and: the sums of the tile before have been read
                if (!(team == 0 ? all_of<3, 128>(alive) : all_of<5, 128>(alive))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int chunk = team * CHUNK; chunk < a.lanes; chunk += teams * CHUNK) {
                    const uint32_t address = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (round & 1) * acc_columns + static_cast<uint32_t>(group * a.width + chunk);
                    int d[CHUNK];
                    if constexpr (PREPARED) load_sums(address, d);
                    else load_eight(address, d);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (chunk != team * CHUNK) team_sync();
#pragma unroll
                    for (int i = 0; i < CHUNK; i++) sums[i][quarter * 32 + lane] = d[i];
                    if (chunk + teams * CHUNK >= a.lanes) {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) arrive(acc_empty + (round & 1) * 8);
                    }
                    team_sync();
                    if (!in_range) continue;
                    const int lanes = min(CHUNK, a.lanes - chunk);
                    auto value_of = [&](int token, float scale) {
                        int sum = 0, up_sum = 0;
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            if (g >= a.groups) break;
                            sum += sums[token][g * slot_rows + row];
                            if (TWO) up_sum += sums[token][g * slot_rows + slot_rows / 2 + row];
                        }
                        const float value = scaled(sum, factor, scale);
                        return TWO ? silu_product(value, scaled(up_sum, up_factor, scale)) : value;
                    };
                    if (DOWN) {
                        const int id = routes.expert[which];
                        for (int token = first_lane; token < lanes; token += lane_step) {
                            if (routes.lead[which][token] == NO_ROUTE) continue;
                            for (int route = token * a.top_k; route < (token + 1) * a.top_k; route++)
                                if (routes.ids[route] == id)
                                    static_cast<float *>(a.y)[static_cast<size_t>(route) * a.n + channel] = value_of(token, __fmul_rn(scales[token], a.weights_of[route]));
                        }
                    } else if (GROUPED) {
                        for (int token = first_lane; token < lanes; token += lane_step) {
                            const int route = routes.lead[which][token];
                            if (route != NO_ROUTE) static_cast<float *>(a.y)[static_cast<size_t>(route) * a.n + channel] = value_of(token, scales[token]);
                        }
                    } else {
                        for (int token = first_lane; token < lanes; token += 4 * lane_step) {
                            float value[4];  // four lanes side by side, past the last one the last one again
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int at = min(token + i * lane_step, lanes - 1);
                                value[i] = value_of(at, scales[chunk + at]);
                                if (MODE == LINEAR && a.residual != nullptr) value[i] = __fadd_rn(value[i], bf16_bits_to_f32(beside[i]));
                            }
                            if (MODE == LINEAR && a.residual != nullptr) fetch_beside(token + 4 * lane_step < lanes ? chunk + token + 4 * lane_step : chunk + teams * CHUNK + first_lane);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                if (token + i * lane_step >= lanes) continue;
                                const size_t out = static_cast<size_t>(chunk + token + i * lane_step) * a.n + channel;
                                if (MODE == LINEAR && a.to_f32) static_cast<float *>(a.y)[out] = value[i];
                                else static_cast<uint16_t *>(a.y)[out] = to_bf16(value[i]);
                            }
                        }
                    }
                }
                if (DOWN && (tile + 1 == last_tile || (tile + 1) / a.row_tiles != which)) {  // the scales may go
                    team_sync();
                    if (thread == 0) arrive(b_empty + ((builds - 1) & 1) * 8);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// ---- experts: routes grouped by expert

// For tables of more than FEW_GROUPED routes, or FEW_GROUPED_TOP_K a token.  Bound by the chain of its loads, shared-memory atomics and barriers: 16384 routes of
// 128 experts take 8 us, 1000 take 4.
// One CTA (several would have to wait for one another's counts) counts the routes of every expert, gives each a place behind those of the experts before it, and cuts every
// expert's places into tiles of tile_lanes.  Which of an expert's routes comes first is left to chance: a row's result does
// not depend on its place.  Routes to no expert (ids outside 0..experts-1) get place -1.  A thread holds GROUP_HELD routes and
// their ranks among their expert's.
constexpr int GROUP_THREADS = 1024, GROUP_HELD = 16;  // threads: and the most experts
__global__ void __launch_bounds__(GROUP_THREADS) expert_groups_kernel(const int *ids, int pairs, int experts, int tile_lanes, int4 *tiles, int *counts_out,
                                                                      int *place_of) {
    __shared__ int count[GROUP_THREADS], later[GROUP_THREADS], first[GROUP_THREADS], warp_places[32], warp_tiles[32];
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    count[thread] = 0;
    later[thread] = 0;
    grid_launch_dependents();
    __syncthreads();
    grid_dependency_wait();
    int held[GROUP_HELD], rank[GROUP_HELD];
#pragma unroll
    for (int i = 0; i < GROUP_HELD; i++) held[i] = thread + i * GROUP_THREADS < pairs ? ids[thread + i * GROUP_THREADS] : -1;
    auto routed = [&](int expert) { return static_cast<uint32_t>(expert) < static_cast<uint32_t>(experts); };
#pragma unroll
    for (int i = 0; i < GROUP_HELD; i++) rank[i] = routed(held[i]) ? atomicAdd(&count[held[i]], 1) : 0;
    for (int pair = thread + GROUP_HELD * GROUP_THREADS; pair < pairs; pair += GROUP_THREADS) {  // these are ranked behind the others
        const int expert = ids[pair];
        if (routed(expert)) atomicAdd(&later[expert], 1);
    }
    __syncthreads();
    // thread = expert: places and tiles in front of it
    const int own = count[thread] + later[thread], own_tiles = (own + tile_lanes - 1) / tile_lanes;
    int places = own, tile = own_tiles;
    auto scan = [&](int &p, int &t) {  // inclusive, of a warp
        for (int offset = 1; offset < 32; offset *= 2) {
            const int other_p = __shfl_up_sync(0xffffffffu, p, offset), other_t = __shfl_up_sync(0xffffffffu, t, offset);
            if (lane >= offset) p += other_p, t += other_t;
        }
    };
    scan(places, tile);
    if (lane == 31) warp_places[warp] = places, warp_tiles[warp] = tile;
    __syncthreads();
    int front_places = warp_places[lane], front_tiles = warp_tiles[lane];
    scan(front_places, front_tiles);
    if (warp > 0) {
        places += __shfl_sync(0xffffffffu, front_places, warp - 1);
        tile += __shfl_sync(0xffffffffu, front_tiles, warp - 1);
    }
    if (thread == GROUP_THREADS - 1) counts_out[0] = tile, counts_out[1] = places;
    places -= own, tile -= own_tiles;
    first[thread] = places;
    later[thread] = places + count[thread];
    for (int i = 0; i < own_tiles; i++) tiles[tile + i] = make_int4(thread, places + i * tile_lanes, min(tile_lanes, own - i * tile_lanes), 0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < GROUP_HELD; i++) {
        const int pair = thread + i * GROUP_THREADS;
        if (pair >= pairs) break;
        place_of[pair] = routed(held[i]) ? first[held[i]] + rank[i] : -1;
    }
    for (int pair = thread + GROUP_HELD * GROUP_THREADS; pair < pairs; pair += GROUP_THREADS) {
        const int expert = ids[pair];
        place_of[pair] = routed(expert) ? atomicAdd(&later[expert], 1) : -1;
    }
}

// y[token] = the sum of its routes' weighted rows, in their order (+ residual), rounded once.  Four columns to a thread, eight rows
// in flight.  Bound by DRAM: 2048 tokens of eight f32 rows of 2048, 28 us, 5.4 TB/s.  (The rows stay f32: rounding them to bf16 would
// halve this and add eight roundings to every output.  Columns in two to eight chunks, so that their rows would stay in L2, made
// the experts of 2048 tokens 210 to 247 us instead of 206: shorter products fill the chip worse than the cache saves.)
__global__ void experts_sum_kernel(const float *parts, const int *ids, const uint16_t *residual, uint16_t *y, int top_k, int experts, int hidden,
                                   int wide) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int column = (blockIdx.y * blockDim.x + threadIdx.x) * 4;
    if (column >= hidden) return;
    const size_t token = blockIdx.x, at = token * hidden + column;
    const float *part = parts + token * top_k * hidden + column;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int BATCH = 8;
    for (int first = 0; first < top_k; first += BATCH) {
        float4 values[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++)
            values[i] = first + i < top_k && static_cast<uint32_t>(ids[token * top_k + first + i]) < static_cast<uint32_t>(experts)
                            ? *reinterpret_cast<const float4 *>(part + static_cast<size_t>(first + i) * hidden)
                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < BATCH; i++) sum.x += values[i].x, sum.y += values[i].y, sum.z += values[i].z, sum.w += values[i].w;
    }
    if (wide) {  // residual and y on 8-byte boundaries
        if (residual != nullptr) {
            const uint2 r = *reinterpret_cast<const uint2 *>(residual + at);
            sum.x += bf16_lo(r.x), sum.y += bf16_hi(r.x), sum.z += bf16_lo(r.y), sum.w += bf16_hi(r.y);
        }
        *reinterpret_cast<uint2 *>(y + at) = make_uint2(to_bf16(sum.x) | (static_cast<uint32_t>(to_bf16(sum.y)) << 16), to_bf16(sum.z) | (static_cast<uint32_t>(to_bf16(sum.w)) << 16));
    } else {
        const float values[4] = {sum.x, sum.y, sum.z, sum.w};
        for (int i = 0; i < 4; i++) y[at + i] = to_bf16(values[i] + (residual != nullptr ? bf16_bits_to_f32(residual[at + i]) : 0.0f));
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {  // the driver's entry point, found through the runtime (the library does not link libcuda)
    static const EncodeTiled found = [] {
        void *pointer = nullptr;
        cudaDriverEntryPointQueryResult result;
        const cudaError_t status = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &pointer, cudaEnableDefault, &result);
        return status == cudaSuccess && result == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(pointer) : nullptr;
    }();
    return found;
}
bool encode(CUtensorMap *map, const int8_t *matrix, int64_t rows, int k, int pitch, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {BLOCK_K, static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
    const EncodeTiled function = encode_tiled();
    return function != nullptr && function(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(matrix), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// As many stages as fit, with room for an A operand of 128 rows at the last one's base.
template <Mode MODE>
size_t plan_stages(Int8Args &args) {
    constexpr int matrices = MODE == PAIR || MODE == EXPERTS_PAIR ? 2 : 1;
    const size_t a_bytes = static_cast<size_t>((args.rows + 7) / 8 * 8) * BLOCK_K, stage = matrices * a_bytes + static_cast<size_t>(args.tile_lanes / 2) * BLOCK_K;
    const size_t last = std::max(stage, (matrices - 1) * a_bytes + static_cast<size_t>(ROWS) * BLOCK_K);
    args.stages = static_cast<int>(std::min<size_t>(MAX_STAGES, 1 + (SMEM_LIMIT - gemm_control<MODE>() - last) / stage));
    return gemm_control<MODE>() + static_cast<size_t>(args.stages - 1) * stage + last;
}

template <Mode MODE, bool SPLIT>
cudaError_t launch_gemm(Int8Args &args, int most_items, cudaStream_t stream) {
    const size_t bytes = plan_stages<MODE>(args);
    const cudaError_t status = allow_shared_memory<int8_gemm_kernel<MODE, SPLIT>>(SMEM_LIMIT);
    if (status != cudaSuccess) return status;
    return launch_dependent(int8_gemm_kernel<MODE, SPLIT>, dim3(2 * std::min(most_items, multiprocessors() / 2)), dim3(THREADS), bytes, 1, stream, args);
}

// A tile's outputs, however many of the 128 rows it has.
int64_t output_cycles(int lanes, bool pair) { return lanes * (pair ? 34 : 18); }
// Tiles of a matrix of n output channels (`pair`: two weight rows each) for that many lanes, by an estimate of the cycles
// they take, which it returns: of a block of 128 columns the tensor pipe needs half the lanes' number for each of four instructions a matrix
// (the waits around them 330 at least), the copies arrive at some 56 bytes per cycle and multiprocessor (weights whose rows are no
// whole lines at two thirds of that), and the weights, which the first of a row's tiles brings in, at some 23; the outputs hide behind
// the next tile's sums, but for the last one's and all of a pair's whose two accumulators do not fit tensor memory; the first blocks
// come 200 cycles each later than the others, up to 3000.
// Columns are split where that comes out lower: to meet costs the sums 8500 cycles and what the atomic adds take, 400 a cycle, and
// their outputs hide behind nothing (143 x 1024 of 8192 columns: 14.4 us in one piece, 13.2 split; 256 x 4096 of 8192, where one
// piece is chosen: 17 and 20; over 480 shapes of 143 to 2048 lanes the choice costs 0.6 % of the better one's time on average).
int64_t plan_dense(Int8Args &args, bool pair) {
    const int pairs = multiprocessors() / 2, blocks = (args.k + BLOCK_K - 1) / BLOCK_K, matrices = pair ? 2 : 1;
    const int padded = (args.lanes + 31) / 32 * 32, least = (padded + MAX_LANES - 1) / MAX_LANES;
    int64_t best = 0;
    for (int split = least; split <= 2 * least + 2 && (split == least || padded / split >= 32); split++) {
        const int lanes = ((padded + split - 1) / split + 31) / 32 * 32, lane_tiles = (padded + lanes - 1) / lanes;
        for (int rows = ROWS; rows >= 8; rows -= 8) {  // (in steps of sixteen bytes of outputs)
            const int row_tiles = (args.n + 2 * rows - 1) / (2 * rows), waves = (row_tiles * lane_tiles + pairs - 1) / pairs;
            const int tensor = matrices * std::max(2 * lanes, 330), copies = (matrices * rows * (args.k % BLOCK_K == 0 ? 2 : 3) + lanes) * BLOCK_K / 112,
                      memory = matrices * rows * BLOCK_K / (23 * lane_tiles), block = std::max({tensor, copies, memory});
            const int64_t sums = static_cast<int64_t>(blocks) * block + 1000, outputs = output_cycles(lanes, pair);
            int64_t cost = waves * (2 * matrices * lanes <= 512 ? std::max(sums, outputs) : sums + outputs) + outputs + std::min(3000, 200 * blocks);
            int splits = 1;
            if (may_split(args.lanes, args.k) && row_tiles * lane_tiles <= SPLIT_TILES) {
                const int most = std::min(pairs / (row_tiles * lane_tiles), (blocks + 1) / 2);
                const int64_t added = static_cast<int64_t>(row_tiles * lane_tiles * most) * 2 * rows * lanes * matrices;
                const int64_t split_cost = static_cast<int64_t>((blocks + most - 1) / std::max(most, 1)) * block + 8500 + 3 * outputs + added / 400;
                if (most > 1 && split_cost < cost) cost = split_cost, splits = most;
            }
            if (best != 0 && cost >= best) continue;
            best = cost;
            args.rows = rows;
            args.row_tiles = row_tiles;
            args.tile_lanes = lanes;
            args.lane_tiles = lane_tiles;
            args.splits = splits;
        }
    }
    return best;
}

}  // namespace

namespace {

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Tiles of `matrices` matrices of n output channels for the few-lane kernel: as few rows for the busiest CTA as possible, a
// tile counted as the bytes of four rows more.  Returns an estimate of the cycles they take, as plan_dense does: a stage's four
// instructions take the tensor pipe 290 cycles or twice their N, its copies 340 and 70 a box to issue, and the outputs of a tile, lane by
// lane, are not hidden by much.
int64_t plan_stream(StreamArgs &args, int matrices, bool pair) {
    const int count = multiprocessors(), most = std::min(pair ? 64 : 128, args.n);
    int64_t best = 0;
    for (int waves = 1, tries = 0; tries < 8; waves++) {  // the fewest rows that many waves have room for
        const int tiles = static_cast<int>(static_cast<int64_t>(count) * waves / matrices);  // of a matrix
        const int rows = tiles > 0 ? (args.n + tiles - 1) / tiles : args.n;
        if (rows > most) {
            waves += std::max(0, static_cast<int>((static_cast<int64_t>(args.n) * matrices / most + count - 1) / count) - waves - 2);
            continue;
        }
        tries++;
        const int64_t cost = static_cast<int64_t>(waves) * (rows + 4);
        if (best == 0 || cost < best) best = cost, args.rows = rows;
    }
    args.row_tiles = (args.n + args.rows - 1) / args.rows;
    args.groups = args.rows * 4 <= (pair ? 64 : 128) ? 4 : args.rows * 2 <= (pair ? 64 : 128) ? 2 : 1;
    while (args.groups * args.width > MAX_LANES) args.groups /= 2;
    args.span_log = args.rows <= 32 ? 5 : args.rows <= 64 ? 6 : 7;
    const int blocks = (args.k + BLOCK_K - 1) / BLOCK_K, steps = (blocks + args.groups - 1) / args.groups, weight_rows = args.groups * args.rows * (pair ? 2 : 1);
    const int tensor = std::max(290, 2 * args.groups * args.width), copies = (weight_rows + args.groups * args.width) * BLOCK_K / 56, memory = weight_rows * BLOCK_K / 23,
              issue = 340 + 70 * args.groups * (pair ? 2 : 1);
    const int64_t waves = (static_cast<int64_t>(matrices) * args.row_tiles + count - 1) / count;
    return waves * (static_cast<int64_t>(steps) * std::max({tensor, copies, memory, issue}) + 900 + args.lanes * (30 + (57 << args.span_log) / 128));
}
// Stages in up to `most` bytes of shared memory, or in all of it where three do not fit into those.  False where three do not
// fit at all.
template <Mode MODE, bool PREPARED>
bool plan_stages(StreamArgs &args, size_t most, size_t *bytes) {
    constexpr bool GROUPED = MODE == EXPERTS_PAIR || MODE == EXPERTS_DOWN;
    const int blocks = (args.k + BLOCK_K - 1) / BLOCK_K, steps = (blocks + args.groups - 1) / args.groups;
    const size_t atoms = PREPARED ? 0 : static_cast<size_t>(steps * args.groups) * ATOM * (MODE == EXPERTS_DOWN ? 2 : 1);
    const size_t fixed = STREAM_CONTROL + STREAM_SUMS<PREPARED> + (GROUPED ? STREAM_ROUTES : 0) + atoms;
    const size_t stage = STREAM_STAGE + (PREPARED ? static_cast<size_t>(std::max(16, args.groups * args.width)) * BLOCK_K : 0);
    if (fixed + 3 * stage > most) most = SMEM_LIMIT;
    if (fixed + 3 * stage > most) return false;
    args.stages = static_cast<int>(std::min<size_t>(STREAM_MAX_STAGES, (most - fixed) / stage));
    *bytes = fixed + static_cast<size_t>(args.stages) * stage;
    return true;
}
// Where a CTA's share of the weights is small, half of a multiprocessor's shared memory does: a CTA of the next call can
// start on the other half while this one writes its outputs (one lane of 4096 x 4096 from L2: 5.0 us a call, 5.2 with all of it, from
// DRAM 6.0 and 5.9; four of a 14336 x 4096 pair: 25.6 with half, 22.0 with all of it).
size_t stream_share(const StreamArgs &args) {
    const int blocks = (args.k + BLOCK_K - 1) / BLOCK_K, count = multiprocessors(), steps = (args.row_tiles + count - 1) / count * ((blocks + args.groups - 1) / args.groups);
    return steps <= STREAM_SMALL_SHARE ? SMEM_HALF : SMEM_LIMIT;
}
template <Mode MODE, bool PREPARED>
cudaError_t launch_stream(const StreamArgs &args, int tiles, size_t bytes, cudaStream_t stream) {
    const cudaError_t status = allow_shared_memory<int8_stream_kernel<MODE, PREPARED>>(SMEM_LIMIT);
    if (status != cudaSuccess) return status;
    return launch_dependent(int8_stream_kernel<MODE, PREPARED>, dim3(std::min(tiles, multiprocessors())), dim3(STREAM_THREADS), bytes, 1, stream, args);
}

// Lanes of a block of the few-lane kernel's activations.
int stream_width(int lanes) { return lanes <= FEW ? FEW : (lanes + 15) / 16 * 16; }
// The scratch buffer of a linear: the activations' whole numbers, as rows or as blocks of 128 columns, one scale per lane, and the sums
// of tiles whose columns are split, where they may be.
size_t row_bytes(int lanes, int k) {
    return padded(lanes <= STREAM_LANES ? static_cast<size_t>((k + BLOCK_K - 1) / BLOCK_K) * BLOCK_K * stream_width(lanes) : static_cast<size_t>(lanes) * pitch_of(k));
}
struct Int8Rows {
    int8_t *values;
    float *scales;
    int *partials;
    size_t bytes;
    Int8Rows(void *scratch, int lanes, int k) {
        uint8_t *const base = static_cast<uint8_t *>(scratch);
        values = reinterpret_cast<int8_t *>(base);
        scales = reinterpret_cast<float *>(base + row_bytes(lanes, k));
        bytes = row_bytes(lanes, k) + padded(static_cast<size_t>(lanes) * sizeof(float));
        partials = reinterpret_cast<int *>(base + bytes);
        if (may_split(lanes, k)) bytes += partial_bytes(SPLIT_TILES, std::min(MAX_LANES, (lanes + 31) / 32 * 32), 2);
    }
    // sums of split tiles, and how many items of a tile have arrived in each CTA's place
    static size_t partial_bytes(int tiles, int tile_lanes, int matrices) {
        return static_cast<size_t>(tiles) * 2 * matrices * tile_lanes * ROWS * sizeof(int) + padded(static_cast<size_t>(tiles) * 2 * sizeof(int));
    }
};

// gate alone (up == nullptr) or the pair.
template <Mode MODE>
cudaError_t launch_dense(const uint16_t *x, const int8_t *w, const float *scales, const int8_t *up, const float *up_scales, void *y, const uint16_t *residual, void *scratch,
                         int lanes, int n, int k, int to_f32, int *error_flag, cudaStream_t stream) {
    constexpr bool TWO = MODE == PAIR;
    const Int8Rows rows(scratch, lanes, k);
    Int8Args args = {};
    args.lanes = lanes, args.n = n, args.k = k, args.to_f32 = to_f32, args.error_flag = error_flag;
    if (lanes <= STREAM_LANES) {
        // (no CTA writes onto a row that another one may still have to quantise)
        const uintptr_t x_at = reinterpret_cast<uintptr_t>(x), y_at = reinterpret_cast<uintptr_t>(y), x_bytes = static_cast<uintptr_t>(lanes) * k * 2,
                        y_bytes = static_cast<uintptr_t>(lanes) * n * (to_f32 ? 4 : 2);
        const bool apart = x_at >= y_at + y_bytes || y_at >= x_at + x_bytes;
        const bool own = lanes <= FEW && static_cast<int64_t>(lanes) * k <= STREAM_OWN && x_at % 16 == 0 && apart;
        StreamArgs few = {};
        few.x = x, few.scales = scales, few.up_scales = up_scales, few.lane_scales = rows.scales, few.y = y, few.residual = residual;
        few.lanes = lanes, few.n = n, few.k = k, few.to_f32 = to_f32, few.error_flag = error_flag;
        few.width = stream_width(lanes);
        size_t bytes;
        const int64_t cost = plan_stream(few, 1, TWO);
        if (own || cost <= plan_dense(args, TWO)) {
            if (!encode(&few.weights, w, n, k, k, few.rows) || (TWO && !encode(&few.up, up, n, k, k, few.rows))) return cudaErrorInvalidValue;
            if (own && plan_stages<MODE, false>(few, stream_share(few), &bytes)) return launch_stream<MODE, false>(few, few.row_tiles, bytes, stream);
            const cudaError_t status =
                launch_quantise_rows<uint16_t, HeldBf16, 4>(x, rows.values, rows.scales, nullptr, nullptr, nullptr, nullptr, lanes, 1, k, stream, few.width);
            if (status != cudaSuccess) return status;
            few.x = rows.values;
            if (!plan_stages<MODE, true>(few, stream_share(few), &bytes)) return cudaErrorInvalidValue;  // (three stages always fit)
            return launch_stream<MODE, true>(few, few.row_tiles, bytes, stream);
        }
    } else {
        plan_dense(args, TWO);
    }
    const int tiles = args.row_tiles * args.lane_tiles;
    size_t zeroed = 0;
    if (args.splits > 1) {
        zeroed = Int8Rows::partial_bytes(tiles, args.tile_lanes, TWO ? 2 : 1);
        args.partials = rows.partials;
        args.arrived = rows.partials + static_cast<size_t>(tiles) * 2 * (TWO ? 2 : 1) * args.tile_lanes * ROWS;
    }
    const cudaError_t status =
        launch_quantise_rows<uint16_t, HeldBf16, 4>(x, rows.values, rows.scales, nullptr, nullptr, nullptr, nullptr, lanes, 1, k, stream, 0, rows.partials, zeroed);
    if (status != cudaSuccess) return status;
    if (!encode(&args.weights, w, n, k, k, args.rows) || (TWO && !encode(&args.up, up, n, k, k, args.rows)) ||
        !encode(&args.activations, rows.values, lanes, k, pitch_of(k), args.tile_lanes / 2))
        return cudaErrorInvalidValue;
    args.scales = scales, args.up_scales = up_scales, args.lane_scales = rows.scales, args.y = y, args.residual = residual;
    args.wide = !to_f32 && n % 8 == 0 && (reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) % 16 == 0;
    return args.splits > 1 ? launch_gemm<MODE, true>(args, tiles * args.splits, stream) : launch_gemm<MODE, false>(args, tiles, stream);
}

}  // namespace

size_t linear_int8_scratch_bytes(int lanes, int k) { return Int8Rows(nullptr, lanes, k).bytes; }

cudaError_t launch_linear_int8(const uint16_t *x, const int8_t *w, const float *scales, void *y, const uint16_t *residual, void *scratch, int lanes, int n, int k, int to_f32,
                               int *error_flag, cudaStream_t stream) {
    return launch_dense<LINEAR>(x, w, scales, nullptr, nullptr, y, residual, scratch, lanes, n, k, to_f32, error_flag, stream);
}

cudaError_t launch_linear_int8_silu_pair(const uint16_t *x, const int8_t *gate, const float *gate_scales, const int8_t *up, const float *up_scales, uint16_t *y, void *scratch,
                                         int lanes, int n, int k, int *error_flag, cudaStream_t stream) {
    return launch_dense<PAIR>(x, gate, gate_scales, up, up_scales, y, nullptr, scratch, lanes, n, k, 0, error_flag, stream);
}

// ---- the experts

namespace {

// The scratch buffer of one call, in parts on 256-byte boundaries.  The weighted rows of the down product take the place of
// what the gate/up product read and wrote, but for calls of few tokens, whose down product reads the latter itself.
struct ExpertsScratch {
    int4 *tiles;
    int *counts, *place_of, *pair_of;
    float *x_scales, *h_scales, *h, *parts;
    int8_t *xq, *hq;
    size_t bytes;
    ExpertsScratch(void *base, int tokens, int top_k, int experts, int hidden, int inter) {
        const size_t pairs = static_cast<size_t>(tokens) * top_k;
        size_t used = 0;
        auto take = [&](size_t size) {
            uint8_t *at = static_cast<uint8_t *>(base) + used;
            used += padded(size);
            return at;
        };
        tiles = reinterpret_cast<int4 *>(take((pairs / 16 + std::min<size_t>(experts, pairs) + 1) * sizeof(int4)));
        counts = reinterpret_cast<int *>(take(2 * sizeof(int)));
        place_of = reinterpret_cast<int *>(take(pairs * sizeof(int)));
        pair_of = reinterpret_cast<int *>(take(pairs * sizeof(int)));
        x_scales = reinterpret_cast<float *>(take(pairs * sizeof(float)));
        h_scales = reinterpret_cast<float *>(take(pairs * sizeof(float)));
        hq = reinterpret_cast<int8_t *>(take(pairs * pitch_of(inter)));
        const size_t shared = used;
        xq = reinterpret_cast<int8_t *>(take(pairs * pitch_of(hidden)));
        h = reinterpret_cast<float *>(take(pairs * inter * sizeof(float)));
        const size_t product_end = used;
        if (tokens > FEW) used = shared;
        parts = reinterpret_cast<float *>(take(pairs * hidden * sizeof(float)));
        bytes = std::max(product_end, used);
    }
};

// Tiles of the experts' products.  pairs: routes of the call, the most there can be.
// Room for twice an expert's even share, so that most experts meet their weights once, as long as two accumulators of the pair fit
// into tensor memory (2048 tokens over 128 experts: gate/up 85 us, 91 with tiles of up to 256).
int expert_tile_lanes(int pairs, int experts) {
    const int share = (pairs + experts - 1) / experts;
    int lanes = 32;
    while (lanes < 2 * share && lanes < 128) lanes *= 2;
    return lanes;
}
// As plan_dense, for the tiles that experts with even shares have.
void plan_experts(Int8Args &args, int pairs, int experts, bool pair) {
    args.tile_lanes = expert_tile_lanes(pairs, experts);
    // (24 tokens over 128 experts: 75 us with the weights first to leave L2, 77.5 without; where experts have several tiles the
    // second finds them gone: 2048 tokens 224 and 210)
    args.once = 2 * ((pairs + experts - 1) / experts) <= args.tile_lanes;
    const int used = std::min(experts, pairs), share = (pairs + used - 1) / used, lane_tiles = (share + args.tile_lanes - 1) / args.tile_lanes;
    const int count = multiprocessors() / 2, blocks = (args.k + BLOCK_K - 1) / BLOCK_K, matrices = pair ? 2 : 1, lanes = std::min((share + 31) / 32 * 32, args.tile_lanes);
    int64_t best = 0;
    for (int rows = ROWS; rows >= 16; rows -= 8) {
        const int row_tiles = (args.n + 2 * rows - 1) / (2 * rows);
        const int64_t waves = (static_cast<int64_t>(row_tiles) * used * lane_tiles + count - 1) / count;
        const int tensor = matrices * std::max(2 * lanes, 330), copies = (matrices * rows + args.tile_lanes / 2) * BLOCK_K / 56, memory = matrices * rows * BLOCK_K / (23 * lane_tiles);
        const int64_t cost = waves * std::max(static_cast<int64_t>(blocks) * std::max({tensor, copies, memory}) + 1000, output_cycles(lanes, pair));
        if (best != 0 && cost >= best) continue;
        best = cost;
        args.rows = rows;
        args.row_tiles = row_tiles;
    }
}

}  // namespace

size_t experts_int8_scratch_bytes(int tokens, int top_k, int experts, int hidden, int inter) { return ExpertsScratch(nullptr, tokens, top_k, experts, hidden, inter).bytes; }

cudaError_t launch_experts_int8(const uint16_t *x, const int *ids, const float *weights, const int8_t *gate_up, const float *gate_up_scales, const int8_t *down,
                                const float *down_scales, uint16_t *y, const uint16_t *residual, void *scratch, int tokens, int top_k, int experts, int hidden, int inter,
                                int *error_flag, cudaStream_t stream) {
    const ExpertsScratch part(scratch, tokens, top_k, experts, hidden, inter);
    const int pairs = tokens * top_k;
    auto sum = [&] {
        const int wide = (reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) % 8 == 0;
        return launch_dependent(experts_sum_kernel, dim3(tokens, (hidden / 4 + 255) / 256), dim3(std::min(256, (hidden / 4 + 31) / 32 * 32)), 0, 1, stream, part.parts, ids,
                                residual, y, top_k, experts, hidden, wide);
    };
    if (tokens <= FEW && pairs <= FEW_ROUTES && reinterpret_cast<uintptr_t>(x) % 16 == 0) {
        StreamArgs first = {}, second = {};
        first.n = inter, first.k = hidden, first.x = x, first.scales = gate_up_scales, first.y = part.h;
        second.n = hidden, second.k = inter, second.x = part.h, second.scales = down_scales, second.y = part.parts;
        for (StreamArgs *args : {&first, &second}) {
            args->lanes = tokens, args->ids = ids, args->weights_of = weights, args->top_k = top_k, args->experts = experts, args->error_flag = error_flag;
            args->width = FEW;
            plan_stream(*args, std::min(experts, pairs), args == &first);
        }
        size_t first_bytes, second_bytes;
        if (plan_stages<EXPERTS_PAIR, false>(first, SMEM_LIMIT, &first_bytes) && plan_stages<EXPERTS_DOWN, false>(second, SMEM_HALF, &second_bytes)) {
            if (!encode(&first.weights, gate_up, static_cast<int64_t>(experts) * 2 * inter, hidden, hidden, first.rows) ||
                !encode(&second.weights, down, static_cast<int64_t>(experts) * hidden, inter, inter, second.rows))
                return cudaErrorInvalidValue;
            cudaError_t status = launch_stream<EXPERTS_PAIR, false>(first, std::min(experts, pairs) * first.row_tiles, first_bytes, stream);
            if (status != cudaSuccess) return status;
            status = launch_stream<EXPERTS_DOWN, false>(second, std::min(experts, pairs) * second.row_tiles, second_bytes, stream);
            return status != cudaSuccess ? status : sum();
        }
    }
    Int8Args first = {}, second = {};
    first.n = inter, first.k = hidden;
    second.n = hidden, second.k = inter;
    plan_experts(first, pairs, experts, true);
    plan_experts(second, pairs, experts, false);
    if (!encode(&first.weights, gate_up, static_cast<int64_t>(experts) * 2 * inter, hidden, hidden, first.rows) ||
        !encode(&first.activations, part.xq, pairs, hidden, pitch_of(hidden), first.tile_lanes / 2) ||
        !encode(&second.weights, down, static_cast<int64_t>(experts) * hidden, inter, inter, second.rows) ||
        !encode(&second.activations, part.hq, pairs, inter, pitch_of(inter), second.tile_lanes / 2))
        return cudaErrorInvalidValue;
    first.scales = gate_up_scales, second.scales = down_scales;
    first.lane_scales = part.x_scales, second.lane_scales = part.h_scales;
    first.y = part.h, second.y = part.parts;
    second.pair_of = part.pair_of;
    for (Int8Args *args : {&first, &second}) {
        args->tiles = part.tiles;
        args->tile_count = part.counts;
        args->error_flag = error_flag;
    }
    const int most_tiles = pairs / first.tile_lanes + std::min(experts, pairs);
    cudaError_t status;
    if (pairs <= FEW_GROUPED && top_k <= FEW_GROUPED_TOP_K) {
        status = launch_quantise_rows<uint16_t, HeldBf16, 4>(x, part.xq, part.x_scales, nullptr, nullptr, part.pair_of, nullptr, tokens, top_k, hidden, stream, 0, nullptr, 0,
                                                             Grouping{ids, pairs, experts, first.tile_lanes, part.tiles, part.counts});
    } else {
        status = launch_dependent(expert_groups_kernel, dim3(1), dim3(GROUP_THREADS), 0, 1, stream, ids, pairs, experts, first.tile_lanes, part.tiles, part.counts, part.place_of);
        if (status != cudaSuccess) return status;
        status = launch_quantise_rows<uint16_t, HeldBf16, 4>(x, part.xq, part.x_scales, part.place_of, nullptr, part.pair_of, nullptr, tokens, top_k, hidden, stream);
    }
    if (status != cudaSuccess) return status;
    status = launch_gemm<EXPERTS_PAIR, false>(first, most_tiles * first.row_tiles, stream);
    if (status != cudaSuccess) return status;
    status = launch_quantise_rows<float, HeldF32, 2>(part.h, part.hq, part.h_scales, nullptr, part.counts + 1, part.pair_of, weights, pairs, 1, inter, stream);
    if (status != cudaSuccess) return status;
    status = launch_gemm<EXPERTS_DOWN, false>(second, most_tiles * second.row_tiles, stream);
    return status != cudaSuccess ? status : sum();
}

}  // namespace nerve
