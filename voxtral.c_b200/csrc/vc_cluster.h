// vc_cluster.h - launches whose CTAs share a row tile as one cluster along x:
// per-device opt-ins, how many clusters of each size the device runs at once,
// and the launch.
#pragma once

#include "vc_internal.h"

#include <algorithm>
#include <atomic>

namespace vc {

constexpr int kMaxCluster = 16;

// One per kernel (a function-local static of its launch).
struct ClusterKernel {
    std::atomic<uint64_t> ready{0};                        // devices with the opt-ins set
    std::atomic<int> active[16][kMaxCluster + 1] = {};     // by device (of 16) and size: clusters at once, 0: not known yet, -1: none
};

inline cudaLaunchConfig_t cluster_config(dim3 grid, int threads, size_t smem, int size, cudaLaunchAttribute *attr,
                                         cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = size;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

// Sets the current device's opt-ins: dynamic shared memory, clusters of 16.
template <typename K>
cudaError_t cluster_prepare(ClusterKernel &ck, K kernel, size_t smem, int *dev) {
    cudaError_t e = cudaGetDevice(dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (*dev & 63);
    if (ck.ready.load() & bit) return cudaSuccess;
    if (smem) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) ck.ready.fetch_or(bit);
    return e;
}

// The most keys that a tile of `packed` rows can see.
inline long long most_keys(const RowsAttnParams &p, int packed) {
    if (p.window <= 0) return p.c.cap;
    const long long rows = p.r.parent ? p.r.max_rows : std::min<long long>(p.r.max_rows, (packed - 1) / p.group + 2);
    return std::min<long long>(p.c.cap, p.window + rows + p.c.n_sink);
}

// A count that the device is asked for once.  Only an answer is kept - a failed
// question would else change the share counts, and with them a result's last
// bits, for the rest of the process - and the error goes to the caller.  A size
// that the device does not have counts as an answer: none.
template <typename Query>
cudaError_t ask_once(std::atomic<int> &known, int *n, Query query) {
    *n = known.load();
    if (*n != 0) return cudaSuccess;
    int answer = 0;
    const cudaError_t e = query(&answer);
    if (e == cudaErrorInvalidClusterSize) answer = 0;
    else if (e != cudaSuccess) return e;
    *n = answer > 0 ? answer : -1;
    known.store(*n);
    return cudaSuccess;
}

// Clusters of `size` CTAs that run at once (a cluster lies within one GPC, so
// this falls off in steps: with one CTA per SM a B200 runs 148, 74, ... 15 of
// 9, 11 of 10 and 7 of 11 to 16).
template <typename K>
cudaError_t cluster_active(ClusterKernel &ck, K kernel, int dev, int threads, size_t smem, int size, int *n) {
    return ask_once(ck.active[dev & 15][size], n, [&](int *answer) {
        cudaLaunchAttribute a;
        const cudaLaunchConfig_t cfg = cluster_config(dim3(size), threads, smem, size, &a, nullptr);
        const cudaError_t e = cudaOccupancyMaxActiveClusters(answer, kernel, &cfg);
        if (e != cudaSuccess) cudaGetLastError();   // reported here
        return e;
    });
}

}  // namespace vc
