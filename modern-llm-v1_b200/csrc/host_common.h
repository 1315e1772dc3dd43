// What the host sides of the C ABI share: argument checks, launches, and the per-device state that b200attn_api.cu owns.
#pragma once

#include "../../include/b200attn.h"

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200attn {

constexpr int kMaxDevices = 64;

// Device address of the status word of the current device, and the word behind it, the epoch (see decode_count); nullptr and *err
// when there is no such device.
int* status_ptr(int* err);
// SM count of the current device (cached per device).
int sm_count();
// What tells a decode launch's counters from those of every other launch (see decode_count).
unsigned long long next_decode_tag();

struct Strides {
    long long t, h, b;  // element strides
};

inline Strides strides_for(int layout, int H, int T, int D) {
    Strides s;
    if (layout == B200ATTN_LAYOUT_BHTD) {
        s.t = D;
        s.h = (long long)T * D;
        s.b = (long long)H * T * D;
    } else {
        s.t = (long long)H * D;
        s.h = D;
        s.b = (long long)T * H * D;
    }
    return s;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int check_common(int B, int T, int Hq, int Hkv, int D, int layout) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return B200ATTN_ERR_INVALID_ARG;
    if (Hq % Hkv != 0) return B200ATTN_ERR_INVALID_ARG;
    if (layout != B200ATTN_LAYOUT_BHTD && layout != B200ATTN_LAYOUT_BTHD) return B200ATTN_ERR_INVALID_ARG;
    if (D != 64 && D != 128) return B200ATTN_ERR_UNSUPPORTED;
    return B200ATTN_OK;
}

// Launch with programmatic stream serialization: the kernel may become resident while the
// previous kernel of the stream drains; it calls griddepcontrol.wait before touching global memory.
// cluster > 1: in thread-block clusters of that many blocks.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, int cluster,
                           Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, Args&&... args) {
    return launch_cluster(kernel, grid, block, smem, st, 1, args...);
}

template <typename K>
int set_smem_once(K kernel, int bytes, bool* done) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (!done[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
            cudaGetLastError();
            return B200ATTN_ERR_CUDA;
        }
        done[dev] = true;
    }
    return B200ATTN_OK;
}

}  // namespace b200attn
