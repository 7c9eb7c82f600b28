// ops_common.cuh -- what the device-buffer operators of include/czg_ops.h share:
// element types, launches and the reasons of refused calls.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <utility>

#include "czg_ops.h"

namespace czg {

// Sets the text of czg_ops_last_error for this thread and returns `status`.
int ops_fail(int status, const char *why);
int ops_cuda(cudaError_t e);   // CZG_OK, or CZG_E_DEVICE with CUDA's text

int kv4_timeouts(int *bits);   // take_timeouts of ops_kv4.cu

namespace {

__device__ int g_ops_timeout;   // a bounded wait of this file's kernels ran out on this device

// Waits of this file's kernels that ran out since the last call (the device is idle).
inline int take_timeouts(int *bits) {
    const int zero = 0;
    *bits = 0;
    if (int st = ops_cuda(cudaMemcpyFromSymbol(bits, g_ops_timeout, sizeof(*bits)))) return st;
    return *bits ? ops_cuda(cudaMemcpyToSymbol(g_ops_timeout, &zero, sizeof(zero))) : CZG_OK;
}

template <typename T> struct DType;
template <> struct DType<float> { static constexpr int kCode = CZG_F32; };
template <> struct DType<__nv_bfloat16> { static constexpr int kCode = CZG_BF16; };
template <> struct DType<__half> { static constexpr int kCode = CZG_F16; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

inline bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool dtype_ok(int d) { return d == CZG_F32 || d == CZG_BF16 || d == CZG_F16; }
inline int elem_bytes(int d) { return d == CZG_F32 ? 4 : 2; }

// One launch.  pdl: the kernel may begin while the one before it on the stream still
// runs: it calls griddepcontrol.wait before it touches memory that another kernel may
// write, in every CTA, and lets the next one begin (launch_dependents) only after that, so
// whatever is older than the kernel before it is complete too.  Such a kernel has begun while
// that memory may still change, so it reads it by plain loads, never by the read-only path
// (__ldg, const __restrict__ parameters).  cluster: CTAs of x.
template <typename... KArgs, typename... Args>
inline cudaError_t ops_launch(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t st, bool pdl,
                              int cluster, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace
}  // namespace czg
