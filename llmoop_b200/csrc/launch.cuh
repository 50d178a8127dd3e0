// Host-side launch with the programmatic-dependent-launch attribute: the kernel may start while its predecessor in the
// stream drains, and waits for it (grid_dependency_wait) before it touches anything the predecessor reads or writes.
#pragma once

#include <cuda_runtime.h>

#include <stdint.h>

#include <atomic>

namespace nerve {

constexpr int MAX_DEVICES = 64;  // whose properties are remembered

// Multiprocessors of the current device, for grids and plans that go by waves of them.
inline int multiprocessors() {
    static std::atomic<int> known[MAX_DEVICES];
    int device = 0, count = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 1;
    if (device < MAX_DEVICES && (count = known[device].load(std::memory_order_relaxed)) > 0) return count;
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || count < 1) return 1;
    if (device < MAX_DEVICES) known[device].store(count, std::memory_order_relaxed);
    return count;
}

// Lets `kernel` take that much dynamic shared memory; asked of the runtime once per kernel and device.
template <auto KERNEL>
cudaError_t allow_shared_memory(size_t bytes) {
    static std::atomic<uint64_t> allowed;
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess) return status;
    const uint64_t bit = device < MAX_DEVICES ? uint64_t(1) << device : 0;
    if (allowed.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    status = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (status == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
    return status;
}

template <typename... Parameters, typename... Arguments>
cudaError_t launch_dependent(void (*kernel)(Parameters...), dim3 grid, dim3 block, size_t smem, int cluster_z, cudaStream_t stream, Arguments... arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = 1;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = static_cast<unsigned int>(cluster_z);
    config.attrs = attributes;
    config.numAttrs = cluster_z > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
}

}  // namespace nerve
