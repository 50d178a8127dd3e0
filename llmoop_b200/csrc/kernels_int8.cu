// Linears of 8-bit integers on the fifth-generation tensor cores: y[m][n] = (sum_k q[m][k] w[n][k]) a[m] s[n], with int8
// weights w and one f32 scale s per output channel.  The activations are quantised per row on the way in: a = amax / 127,
// q = x / a to the nearest whole number, ties to even.  tcgen05.mma.kind::i8 adds the products in 32-bit integers, which
// hold every sum of up to 131072 columns (127 * 128 * 131072 < 2^31): the sums are exact, so that neither the shape of the
// tiles nor the company of a lane shows in its outputs, and the only roundings are those of q, of the scales' products
// and of the output.
//
// int8_gemm_kernel, persistent: a CTA walks output tiles of up to 128 weight rows (MMA M) by up to 256 lanes (MMA N).  One
// warp copies both operands with TMA (128-byte-swizzled rows of 128 columns) into a ring as deep as shared memory allows,
// straight on into the next tile; one warp issues the MMAs into one of two accumulators in tensor memory; eight warps
// write the finished accumulator out while the other one fills.  A tile may have fewer than 128 weight rows: the rest of
// the MMA's A operand is then whatever lies behind in shared memory, and the rest of the accumulator is never read.  So a
// matrix is cut into as many row tiles as the chip has multiprocessors, and few lanes need no split of K.
//
// The gate/up pair takes both matrices in one tile: every 32 rows of A are sixteen of gate and the same sixteen of up, so
// that the two factors of an output meet by one exchange between the two halves of a warp.
//
// The experts' products are the same kernel over tiles that expert_groups_kernel makes of the routes.
// Waits are bounded; a wait that expires sets the error word, and the CTA still frees its tensor memory.  The unbounded wait
// for the kernel in front comes before them in every role, so none of them counts that kernel's time.
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
constexpr size_t SMEM_LIMIT = 226 * 1024, CONTROL_BYTES = 1024;
constexpr unsigned int SPIN_LIMIT = 1u << 22;  // tries of 1.5 us

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

// NaN stays NaN.
__device__ __forceinline__ uint16_t to_bf16(float value) { return __bfloat16_as_ushort(__float2bfloat16_rn(value)); }

// ---- quantisation of activation rows

// Largest magnitude of a block's values; NaN (as an infinity or a NaN among them makes it) spreads.
__device__ __forceinline__ float block_amax(float mine, float *warps) {
    // magnitudes compare as their bits do, and those of NaN and infinity are the largest
    const uint32_t best = __reduce_max_sync(0xffffffffu, __float_as_uint(mine));
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = __uint_as_float(best);
    __syncthreads();
    uint32_t all = 0;
    for (int warp = 0; warp < static_cast<int>(blockDim.x >> 5); warp++) all = max(all, __float_as_uint(warps[warp]));
    return __uint_as_float(all);
}

struct RowScale {
    float pre, multiplier, scale;
};
// q = rint((x pre) multiplier).  pre lifts rows of tiny values to where 127 / amax is finite.
__device__ __forceinline__ RowScale row_scale(float amax) {
    RowScale row;
    const bool finite = amax <= 3.4028234e38f;
    row.pre = amax < 0x1p-90f ? 0x1p+90f : 1.0f;
    row.multiplier = finite && amax > 0.0f ? 127.0f / (amax * row.pre) : 0.0f;
    row.scale = finite ? amax / 127.0f : __uint_as_float(0x7fffffffu);  // a row with an infinity or a NaN is NaN throughout
    return row;
}
// The whole number as the low byte.  x multiplier carries a relative error below 2^-22, which matters at ties alone: a bf16
// quotient 127 x / amax is either a tie, with at most eight significant bits, or 2^-16 of itself away from one (both
// significands are whole numbers below 256), so that rounding the product to nineteen bits first puts ties, and nothing
// else, back onto themselves.  f32 inputs go without.
template <bool TIES>
__device__ __forceinline__ uint32_t quantise(float x, const RowScale &row) {
    float t = (x * row.pre) * row.multiplier;
    if (TIES) t = __uint_as_float((__float_as_uint(t) + 0x10u) & ~0x1Fu);
    return __float_as_uint(t + 12582912.0f);  // 1.5 * 2^23: rounds to even, leaves two's complement in the low bits
}
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Eight values of a row from `at` on.
struct Eight {
    float v[8];
};
__device__ __forceinline__ Eight load_eight(const uint16_t *row, int at, bool wide) {
    Eight out;
    if (wide) {
        const uint4 words = *reinterpret_cast<const uint4 *>(row + at);
        const uint32_t w[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            out.v[2 * i] = bf16_lo(w[i]);
            out.v[2 * i + 1] = bf16_hi(w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) out.v[i] = bf16_bits_to_f32(row[at + i]);
    }
    return out;
}
__device__ __forceinline__ Eight load_eight(const float *row, int at, bool) {
    Eight out;
    const float4 low = *reinterpret_cast<const float4 *>(row + at), high = *reinterpret_cast<const float4 *>(row + at + 4);
    out.v[0] = low.x, out.v[1] = low.y, out.v[2] = low.z, out.v[3] = low.w;
    out.v[4] = high.x, out.v[5] = high.y, out.v[6] = high.z, out.v[7] = high.w;
    return out;
}

// One CTA per row of x.  Without places the row goes to its own number; with them (the experts' inputs) once to the place of
// each of its top_k routes, where it has one.  The second reading of the row comes from the caches.
// wide: x rows start on 16-byte boundaries.  k is a multiple of 16.
template <typename T>
__global__ void quantise_rows_kernel(const T *__restrict__ x, int8_t *__restrict__ q, float *__restrict__ scales, const int *__restrict__ places,
                                     const int *__restrict__ row_count, int top_k, int k, int wide) {
    __shared__ float warps[32];
    grid_launch_dependents();
    grid_dependency_wait();
    if (row_count != nullptr && static_cast<int>(blockIdx.x) >= *row_count) return;
    const T *row = x + static_cast<size_t>(blockIdx.x) * k;
    float amax = 0.0f;
    for (int at = threadIdx.x * 8; at < k; at += blockDim.x * 8) {
        const Eight eight = load_eight(row, at, wide);
#pragma unroll
        for (int i = 0; i < 8; i++) amax = __uint_as_float(max(__float_as_uint(amax), __float_as_uint(fabsf(eight.v[i]))));
    }
    const RowScale scale = row_scale(block_amax(amax, warps));
    const int copies = places != nullptr ? top_k : 1;
    for (int at = threadIdx.x * 8; at < k; at += blockDim.x * 8) {
        const Eight eight = load_eight(row, at, wide);
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; i++) b[i] = quantise<sizeof(T) == 2>(eight.v[i], scale);
        const uint2 packed = make_uint2(pack_bytes(b[0], b[1], b[2], b[3]), pack_bytes(b[4], b[5], b[6], b[7]));
        for (int copy = 0; copy < copies; copy++) {
            const int place = places != nullptr ? places[static_cast<size_t>(blockIdx.x) * top_k + copy] : static_cast<int>(blockIdx.x);
            if (place >= 0) *reinterpret_cast<uint2 *>(q + static_cast<size_t>(place) * k + at) = packed;
        }
    }
    if (static_cast<int>(threadIdx.x) < copies) {
        const int place = places != nullptr ? places[static_cast<size_t>(blockIdx.x) * top_k + threadIdx.x] : static_cast<int>(blockIdx.x);
        if (place >= 0) scales[place] = scale.scale;
    }
}

int quantise_threads(int k) { return std::min(512, std::max(64, (k / 8 + 31) / 32 * 32)); }

// ---- the product

struct Int8Args {
    CUtensorMap weights, up, activations;  // boxes of 128 columns x box_rows weight rows, and x box_lanes lanes
    const float *scales, *up_scales, *lane_scales;
    void *y;
    const uint16_t *residual;
    int lanes, n, k, to_f32;
    int *error_flag;
    int tile_rows, tile_lanes, box_lanes, lane_tiles, row_tiles, stages;
    // experts
    const int4 *tiles;
    const int *tile_count, *pair_of;
    const float *weights_of;
};

struct Tile {
    int row0;   // first output channel
    int lane0, count, expert;
};
template <Mode MODE>
__device__ __forceinline__ Tile tile_at(const Int8Args &a, int index) {
    Tile tile;
    const int outputs = MODE == PAIR || MODE == EXPERTS_PAIR ? a.tile_rows / 2 : a.tile_rows;
    if (MODE == LINEAR || MODE == PAIR) {
        tile.row0 = index / a.lane_tiles * outputs;
        tile.lane0 = index % a.lane_tiles * a.tile_lanes;
        tile.count = min(a.tile_lanes, a.lanes - tile.lane0);
        tile.expert = 0;
    } else {
        const int4 group = a.tiles[index / a.row_tiles];
        tile.row0 = index % a.row_tiles * outputs;
        tile.expert = group.x;
        tile.lane0 = group.y;
        tile.count = group.z;
    }
    return tile;
}
// The weight copies of one stage: box `which` of `boxes`.
template <Mode MODE>
__device__ __forceinline__ void copy_weights(const Int8Args &a, const Tile &tile, int which, int column, uint32_t target, uint32_t barrier) {
    if (MODE == LINEAR || MODE == EXPERTS_DOWN) {
        copy_tile(target, &a.weights, column, tile.expert * a.n + tile.row0, barrier);
    } else {  // sixteen rows each, by turns of gate and of up
        const bool up = which & 1;
        const int row = tile.row0 + (which >> 1) * 16;
        if (MODE == PAIR) copy_tile(target + which * 16 * BLOCK_K, up ? &a.up : &a.weights, column, row, barrier);
        else copy_tile(target + which * 16 * BLOCK_K, &a.weights, column, tile.expert * 2 * a.n + (up ? a.n : 0) + row, barrier);
    }
}

__device__ __forceinline__ float silu_product(float gate, float up) { return __fdividef(gate, 1.0f + __expf(-gate)) * up; }

template <Mode MODE>
__global__ void __launch_bounds__(THREADS, 1) int8_gemm_kernel(const __grid_constant__ Int8Args a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr bool GROUPED = MODE == EXPERTS_PAIR || MODE == EXPERTS_DOWN, TWO = MODE == PAIR || MODE == EXPERTS_PAIR;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform
    const uint32_t a_bytes = static_cast<uint32_t>(a.tile_rows) * BLOCK_K, stage_bytes = a_bytes + static_cast<uint32_t>(a.tile_lanes) * BLOCK_K;
    const uint32_t control = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), base = control + static_cast<uint32_t>(CONTROL_BYTES);
    const uint32_t full = control, empty = full + 8 * MAX_STAGES, acc_full = empty + 8 * MAX_STAGES, acc_empty = acc_full + 16, tmem_slot = acc_empty + 16;
    const int blocks = (a.k + BLOCK_K - 1) / BLOCK_K;
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; s++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + s * 8) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty + s * 8) : "memory");
        }
        for (int s = 0; s < 2; s++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(acc_full + s * 8) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(acc_empty + s * 8), "r"(OUTPUT_WARPS) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const uint32_t acc_columns = (static_cast<uint32_t>(a.tile_lanes) + 31u) & ~31u;
    uint32_t columns = 32;
    while (columns < 2 * acc_columns) columns *= 2;
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // not before the tensor memory is this CTA's: one of the next kernel's that took it first would wait for this one
    grid_launch_dependents();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");
    tmem = __reduce_or_sync(0xffffffffu, tmem);  // a uniform register

    if (warp == 0) {  // ---- copies
        const int weight_boxes = TWO ? a.tile_rows / 16 : 1;
        int stage = 0, issued = 0, ahead = 0;
        uint32_t parity = 1;  // the first round waits for no release
        if (!GROUPED && static_cast<int>(blockIdx.x) < a.row_tiles * a.lane_tiles) {
            // the weights of the first stages do not wait for the kernel in front, which is the quantisation
            const Tile tile = tile_at<MODE>(a, blockIdx.x);
            const uint32_t bytes = a_bytes + static_cast<uint32_t>((tile.count + a.box_lanes - 1) / a.box_lanes * a.box_lanes) * BLOCK_K;
            ahead = min(a.stages, blocks);
            for (int block = 0; block < ahead; block++) {
                if (elect_one()) expect_bytes(full + block * 8, bytes);
                __syncwarp();
                if (lane < weight_boxes) copy_weights<MODE>(a, tile, lane, block * BLOCK_K, base + static_cast<uint32_t>(block) * stage_bytes, full + block * 8);
            }
        }
        grid_dependency_wait();
        const int tiles = (GROUPED ? *a.tile_count : a.lane_tiles) * a.row_tiles;
        bool alive = true;
        for (int index = blockIdx.x; index < tiles && alive; index += gridDim.x) {
            const Tile tile = tile_at<MODE>(a, index);
            const int lane_boxes = (tile.count + a.box_lanes - 1) / a.box_lanes;
            const uint32_t bytes = a_bytes + static_cast<uint32_t>(lane_boxes * a.box_lanes) * BLOCK_K;
            for (int block = 0; block < blocks; block++) {
                const uint32_t target = base + static_cast<uint32_t>(stage) * stage_bytes, barrier = full + stage * 8;
                if (!wait_barrier(empty + stage * 8, parity, a.error_flag)) {
                    for (int s = 0; s < a.stages && s < issued; s++) {  // the copies in flight land before the CTA gives its memory up
                        const int which = (issued - 1 - s) % a.stages;
                        wait_barrier(full + which * 8, static_cast<uint32_t>(((issued - 1 - s) / a.stages) & 1), a.error_flag);
                    }
                    alive = false;
                    break;
                }
                if (issued >= ahead) {
                    if (elect_one()) expect_bytes(barrier, bytes);
                    __syncwarp();
                    if (lane < weight_boxes) copy_weights<MODE>(a, tile, lane, block * BLOCK_K, target, barrier);
                }
                if (lane < lane_boxes)
                    copy_tile(target + a_bytes + static_cast<uint32_t>(lane * a.box_lanes) * BLOCK_K, &a.activations, block * BLOCK_K, tile.lane0 + lane * a.box_lanes, barrier);
                __syncwarp();
                issued++;
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp == 1) {  // ---- MMAs
        const uint64_t first = swizzled_descriptor(base);
        int stage = 0, round = 0;
        uint32_t parity = 0;
        bool alive = true;
        grid_dependency_wait();
        const int tiles = (GROUPED ? *a.tile_count : a.lane_tiles) * a.row_tiles;
        for (int index = blockIdx.x; index < tiles && alive; index += gridDim.x, round++) {
            const Tile tile = tile_at<MODE>(a, index);
            // instruction descriptor: s32 accumulator, A and B signed bytes, both K-major, N / 8 in bits 17-22, M / 16 in bits 24-28
            const uint32_t instruction =
                __reduce_or_sync(0xffffffffu, (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>((tile.count + 15) / 16 * 2) << 17) | (8u << 24));
            const uint32_t accumulator = tmem + (round & 1) * acc_columns;
            if (!wait_barrier(acc_empty + (round & 1) * 8, static_cast<uint32_t>((round / 2 + 1) & 1), a.error_flag)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int block = 0; block < blocks; block++) {
                if (!wait_barrier(full + stage * 8, parity, a.error_flag)) {
                    alive = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    const uint64_t a_stage = first + static_cast<uint64_t>(stage) * (stage_bytes >> 4), b_stage = a_stage + (a_bytes >> 4);
#pragma unroll
                    for (int step = 0; step < 4; step++) {  // K = 32 per instruction
                        const uint32_t accumulate = (block > 0 || step > 0) ? 1u : 0u;
                        asm volatile(
                            "{\n"
                            ".reg .pred p;\n"
                            "setp.ne.b32 p, %4, 0;\n"
                            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
                            "}\n" ::"r"(accumulator),
                            "l"(a_stage + step * 2), "l"(b_stage + step * 2), "r"(instruction), "r"(accumulate)
                            : "memory");
                    }
                    commit_to(empty + stage * 8);
                    if (block == blocks - 1) commit_to(acc_full + (round & 1) * 8);
                }
                __syncwarp();
                if (++stage == a.stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp >= 4) {  // ---- outputs: thread = row of the accumulator
        grid_dependency_wait();
        const int tiles = (GROUPED ? *a.tile_count : a.lane_tiles) * a.row_tiles;
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        int round = 0;
        for (int index = blockIdx.x; index < tiles; index += gridDim.x, round++) {
            const Tile tile = tile_at<MODE>(a, index);
            const bool mine = quarter * 32 < a.tile_rows;
            // the output channel of this thread, and its factor: a lane of a pair's upper half holds up's row of the same channel
            const int channel = TWO ? tile.row0 + quarter * 16 + (lane & 15) : tile.row0 + quarter * 32 + lane;
            const bool in_range = channel < a.n && (TWO || quarter * 32 + lane < a.tile_rows);
            float factor = 0.0f;
            if (mine && in_range) {
                if (MODE == LINEAR) factor = a.scales[channel];
                else if (MODE == PAIR) factor = (lane < 16 ? a.scales : a.up_scales)[channel];
                else if (MODE == EXPERTS_PAIR) factor = a.scales[static_cast<size_t>(tile.expert) * 2 * a.n + (lane < 16 ? 0 : a.n) + channel];
                else factor = a.scales[static_cast<size_t>(tile.expert) * a.n + channel];
            }
            if (!wait_barrier(acc_full + (round & 1) * 8, static_cast<uint32_t>((round / 2) & 1), a.error_flag)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t accumulator = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (round & 1) * acc_columns;
            if (mine)
                for (int column = part * 16; column < tile.count; column += 32) {
                    uint32_t d[16];
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]), "=r"(d[8]), "=r"(d[9]),
                                   "=r"(d[10]), "=r"(d[11]), "=r"(d[12]), "=r"(d[13]), "=r"(d[14]), "=r"(d[15])
                                 : "r"(accumulator + static_cast<uint32_t>(column))
                                 : "memory");
                    const int count = min(16, tile.count - column), first_lane = tile.lane0 + column;
                    // thread i < 16 fetches what belongs to lane i of these sixteen
                    float lane_scale = 0.0f;
                    int pair = 0;
                    if (lane < count) {
                        lane_scale = a.lane_scales[first_lane + lane];
                        if (MODE == EXPERTS_DOWN) {
                            pair = a.pair_of[first_lane + lane];
                            lane_scale *= a.weights_of[pair];
                        }
                    }
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (TWO) {
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {  // the warp's lower half finishes lane i, its upper half lane i + 1
                            const float low = static_cast<float>(static_cast<int>(d[i])) * factor * __shfl_sync(0xffffffffu, lane_scale, i);
                            const float high = static_cast<float>(static_cast<int>(d[i + 1])) * factor * __shfl_sync(0xffffffffu, lane_scale, i + 1);
                            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? high : low, 16);
                            const float product = lane < 16 ? silu_product(low, other) : silu_product(other, high);
                            const int at = i + (lane >> 4);
                            if (in_range && at < count) {
                                const size_t out = static_cast<size_t>(first_lane + at) * a.n + channel;
                                if (MODE == PAIR) reinterpret_cast<uint16_t *>(a.y)[out] = to_bf16(product);
                                else reinterpret_cast<float *>(a.y)[out] = product;
                            }
                        }
                    } else {
                        float residual[16];
                        if (MODE == LINEAR && a.residual != nullptr)
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (in_range && i < count) residual[i] = bf16_bits_to_f32(a.residual[static_cast<size_t>(first_lane + i) * a.n + channel]);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            float value = static_cast<float>(static_cast<int>(d[i])) * factor * __shfl_sync(0xffffffffu, lane_scale, i);
                            const int to = MODE == EXPERTS_DOWN ? __shfl_sync(0xffffffffu, pair, i) : first_lane + i;
                            if (!in_range || i >= count) continue;
                            const size_t out = static_cast<size_t>(to) * a.n + channel;
                            if (MODE == EXPERTS_DOWN) {
                                reinterpret_cast<float *>(a.y)[out] = value;
                            } else {
                                if (a.residual != nullptr) value += residual[i];
                                if (a.to_f32) reinterpret_cast<float *>(a.y)[out] = value;
                                else reinterpret_cast<uint16_t *>(a.y)[out] = to_bf16(value);
                            }
                        }
                    }
                }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(acc_empty + (round & 1) * 8) : "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// ---- experts: routes grouped by expert

// One CTA counts the routes of every expert, gives each a place behind those of the experts before it, and cuts every
// expert's places into tiles of tile_lanes.  Which of an expert's routes comes first is left to chance: a row's result does
// not depend on its place.  Routes to no expert (ids outside 0..experts-1) get place -1.
constexpr int GROUP_THREADS = 1024;  // and the most experts
__global__ void __launch_bounds__(GROUP_THREADS) expert_groups_kernel(const int *__restrict__ ids, int pairs, int experts, int tile_lanes, int4 *tiles, int *counts_out,
                                                                      int *place_of, int *pair_of) {
    __shared__ int count[GROUP_THREADS], cursor[GROUP_THREADS], warp_places[32], warp_tiles[32];
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    count[thread] = 0;
    grid_launch_dependents();
    __syncthreads();
    grid_dependency_wait();
    for (int pair = thread; pair < pairs; pair += GROUP_THREADS) {
        const int expert = ids[pair];
        if (expert >= 0 && expert < experts) atomicAdd(&count[expert], 1);
    }
    __syncthreads();
    // thread = expert: places and tiles in front of it
    const int own = count[thread], own_tiles = (own + tile_lanes - 1) / tile_lanes;
    int places = own, tile = own_tiles;
    for (int offset = 1; offset < 32; offset *= 2) {
        const int p = __shfl_up_sync(0xffffffffu, places, offset), t = __shfl_up_sync(0xffffffffu, tile, offset);
        if (lane >= offset) places += p, tile += t;
    }
    if (lane == 31) warp_places[warp] = places, warp_tiles[warp] = tile;
    __syncthreads();
    for (int before = 0; before < warp; before++) places += warp_places[before], tile += warp_tiles[before];
    if (thread == GROUP_THREADS - 1) counts_out[0] = tile, counts_out[1] = places;
    places -= own, tile -= own_tiles;
    cursor[thread] = places;
    for (int i = 0; i < own_tiles; i++) tiles[tile + i] = make_int4(thread, places + i * tile_lanes, min(tile_lanes, own - i * tile_lanes), 0);
    __syncthreads();
    for (int pair = thread; pair < pairs; pair += GROUP_THREADS) {
        const int expert = ids[pair];
        int place = -1;
        if (expert >= 0 && expert < experts) {
            place = atomicAdd(&cursor[expert], 1);
            pair_of[place] = pair;
        }
        place_of[pair] = place;
    }
}

// y[token] = the sum of its routes' weighted rows, in their order (+ residual), rounded once.  Four columns to a thread.
__global__ void experts_sum_kernel(const float *__restrict__ parts, const int *__restrict__ place_of, const uint16_t *residual, uint16_t *y, int top_k, int hidden,
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
            if (first + i < top_k && place_of[token * top_k + first + i] >= 0) values[i] = *reinterpret_cast<const float4 *>(part + static_cast<size_t>(first + i) * hidden);
            else values[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
bool encode(CUtensorMap *map, const int8_t *matrix, int64_t rows, int k, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(k)};
    const cuuint32_t box[2] = {BLOCK_K, static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
    const EncodeTiled function = encode_tiled();
    return function != nullptr && function(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(matrix), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// As many stages as fit, with room for an A operand of 128 rows at the last one's base.
void plan_stages(Int8Args &args) {
    const size_t stage = static_cast<size_t>(args.tile_rows + args.tile_lanes) * BLOCK_K, last = std::max(stage, static_cast<size_t>(ROWS) * BLOCK_K);
    args.stages = static_cast<int>(std::min<size_t>(MAX_STAGES, 1 + (SMEM_LIMIT - CONTROL_BYTES - last) / stage));
}
size_t shared_bytes(const Int8Args &args) {
    const size_t stage = static_cast<size_t>(args.tile_rows + args.tile_lanes) * BLOCK_K;
    return CONTROL_BYTES + static_cast<size_t>(args.stages - 1) * stage + std::max(stage, static_cast<size_t>(ROWS) * BLOCK_K);
}

template <Mode MODE>
cudaError_t launch_gemm(const Int8Args &args, int most_tiles, cudaStream_t stream) {
    const cudaError_t status = cudaFuncSetAttribute(int8_gemm_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM_LIMIT));
    if (status != cudaSuccess) return status;
    return launch_dependent(int8_gemm_kernel<MODE>, dim3(std::min(most_tiles, multiprocessors())), dim3(THREADS), shared_bytes(args), 1, stream, args);
}

// Tiles of a matrix of n output channels (`pair`: two weight rows each) for that many lanes.
void plan_dense(Int8Args &args, bool pair) {
    const int padded = (args.lanes + 15) / 16 * 16, count = multiprocessors();
    args.lane_tiles = (padded + MAX_LANES - 1) / MAX_LANES;
    args.tile_lanes = ((padded + args.lane_tiles - 1) / args.lane_tiles + 15) / 16 * 16;
    args.lane_tiles = (padded + args.tile_lanes - 1) / args.tile_lanes;
    args.box_lanes = args.tile_lanes;
    // as few waves of the chip as 128 rows allow, and then as few rows as make that many waves
    const int step = pair ? 16 : 8, most = pair ? 64 : 128;
    const int waves = ((args.n + most - 1) / most * args.lane_tiles + count - 1) / count;
    int rows = step;
    while (rows < most && ((args.n + rows - 1) / rows * args.lane_tiles + count - 1) / count > waves) rows += step;
    args.row_tiles = (args.n + rows - 1) / rows;
    args.tile_rows = pair ? 2 * rows : rows;
    plan_stages(args);
}

}  // namespace

cudaError_t launch_quantise_int8(const uint16_t *x, int8_t *q, float *scales, int lanes, int k, cudaStream_t stream) {
    const int wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    return launch_dependent(quantise_rows_kernel<uint16_t>, dim3(lanes), dim3(quantise_threads(k)), 0, 1, stream, x, q, scales, nullptr, nullptr, 1, k, wide);
}

cudaError_t launch_linear_int8(const int8_t *q, const float *lane_scales, const int8_t *w, const float *scales, void *y, const uint16_t *residual, int lanes, int n,
                               int k, int to_f32, int *error_flag, cudaStream_t stream) {
    Int8Args args = {};
    args.lanes = lanes;
    args.n = n;
    args.k = k;
    plan_dense(args, false);
    if (!encode(&args.weights, w, n, k, args.tile_rows) || !encode(&args.activations, q, lanes, k, args.box_lanes)) return cudaErrorInvalidValue;
    args.scales = scales;
    args.lane_scales = lane_scales;
    args.y = y;
    args.residual = residual;
    args.to_f32 = to_f32;
    args.error_flag = error_flag;
    return launch_gemm<LINEAR>(args, args.row_tiles * args.lane_tiles, stream);
}

cudaError_t launch_linear_int8_silu_pair(const int8_t *q, const float *lane_scales, const int8_t *gate, const float *gate_scales, const int8_t *up,
                                         const float *up_scales, uint16_t *y, int lanes, int n, int k, int *error_flag, cudaStream_t stream) {
    Int8Args args = {};
    args.lanes = lanes;
    args.n = n;
    args.k = k;
    plan_dense(args, true);
    if (!encode(&args.weights, gate, n, k, 16) || !encode(&args.up, up, n, k, 16) || !encode(&args.activations, q, lanes, k, args.box_lanes)) return cudaErrorInvalidValue;
    args.scales = gate_scales;
    args.up_scales = up_scales;
    args.lane_scales = lane_scales;
    args.y = y;
    args.error_flag = error_flag;
    return launch_gemm<PAIR>(args, args.row_tiles * args.lane_tiles, stream);
}

// ---- the experts

namespace {

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// The scratch buffer of one call, in parts on 256-byte boundaries; the weighted rows of the down product take the place of
// what the gate/up product read and wrote.
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
        hq = reinterpret_cast<int8_t *>(take(pairs * inter));
        const size_t shared = used;
        xq = reinterpret_cast<int8_t *>(take(pairs * hidden));
        h = reinterpret_cast<float *>(take(pairs * inter * sizeof(float)));
        const size_t product_end = used;
        used = shared;
        parts = reinterpret_cast<float *>(take(pairs * hidden * sizeof(float)));
        bytes = std::max(product_end, used);
    }
};

// Tiles of the experts' products.  pairs: routes of the call, the most there can be.
void plan_experts(Int8Args &args, int pairs, int experts, bool pair) {
    // room for twice an expert's even share, so that most experts meet their weights once
    const int share = (pairs + experts - 1) / experts;
    int lanes = 16;
    while (lanes < 2 * share && lanes < MAX_LANES) lanes *= 2;
    args.tile_lanes = lanes;
    args.box_lanes = std::min(lanes, 32);
    args.tile_rows = 128;
    const int outputs = pair ? 64 : 128;
    args.row_tiles = (args.n + outputs - 1) / outputs;
    plan_stages(args);
}

}  // namespace

size_t experts_int8_scratch_bytes(int tokens, int top_k, int experts, int hidden, int inter) { return ExpertsScratch(nullptr, tokens, top_k, experts, hidden, inter).bytes; }

cudaError_t launch_experts_int8(const uint16_t *x, const int *ids, const float *weights, const int8_t *gate_up, const float *gate_up_scales, const int8_t *down,
                                const float *down_scales, uint16_t *y, const uint16_t *residual, void *scratch, int tokens, int top_k, int experts, int hidden, int inter,
                                int *error_flag, cudaStream_t stream) {
    const ExpertsScratch part(scratch, tokens, top_k, experts, hidden, inter);
    const int pairs = tokens * top_k;
    Int8Args first = {}, second = {};
    first.n = inter, first.k = hidden;
    second.n = hidden, second.k = inter;
    plan_experts(first, pairs, experts, true);
    plan_experts(second, pairs, experts, false);
    if (!encode(&first.weights, gate_up, static_cast<int64_t>(experts) * 2 * inter, hidden, 16) || !encode(&first.activations, part.xq, pairs, hidden, first.box_lanes) ||
        !encode(&second.weights, down, static_cast<int64_t>(experts) * hidden, inter, second.tile_rows) || !encode(&second.activations, part.hq, pairs, inter, second.box_lanes))
        return cudaErrorInvalidValue;
    first.scales = gate_up_scales, second.scales = down_scales;
    first.lane_scales = part.x_scales, second.lane_scales = part.h_scales;
    first.y = part.h, second.y = part.parts;
    second.pair_of = part.pair_of, second.weights_of = weights;
    for (Int8Args *args : {&first, &second}) {
        args->tiles = part.tiles;
        args->tile_count = part.counts;
        args->error_flag = error_flag;
    }
    const int most_tiles = pairs / first.tile_lanes + std::min(experts, pairs);
    cudaError_t status = launch_dependent(expert_groups_kernel, dim3(1), dim3(GROUP_THREADS), 0, 1, stream, ids, pairs, experts, first.tile_lanes, part.tiles, part.counts,
                                          part.place_of, part.pair_of);
    if (status != cudaSuccess) return status;
    const int wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    status = launch_dependent(quantise_rows_kernel<uint16_t>, dim3(tokens), dim3(quantise_threads(hidden)), 0, 1, stream, x, part.xq, part.x_scales, part.place_of, nullptr,
                              top_k, hidden, wide);
    if (status != cudaSuccess) return status;
    status = launch_gemm<EXPERTS_PAIR>(first, most_tiles * first.row_tiles, stream);
    if (status != cudaSuccess) return status;
    status = launch_dependent(quantise_rows_kernel<float>, dim3(pairs), dim3(quantise_threads(inter)), 0, 1, stream, part.h, part.hq, part.h_scales, nullptr, part.counts + 1, 1,
                              inter, 1);
    if (status != cudaSuccess) return status;
    status = launch_gemm<EXPERTS_DOWN>(second, most_tiles * second.row_tiles, stream);
    if (status != cudaSuccess) return status;
    const int narrow = (reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) % 8 == 0;
    return launch_dependent(experts_sum_kernel, dim3(tokens, (hidden / 4 + 255) / 256), dim3(std::min(256, (hidden / 4 + 31) / 32 * 32)), 0, 1, stream, part.parts,
                            part.place_of, residual, y, top_k, hidden, narrow);
}

}  // namespace nerve
