// Declarations shared by the dense operators' files (gated feed-forward, 8-bit linear, sampling).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include "glmx.h"
#include "glmx_internal.h"

namespace glmx {

inline int dense_fail(int code, const char* msg)
{
    set_error(msg);
    return code;
}

inline int dense_cuda_fail(cudaError_t e, const char* what)
{
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return GLMX_E_CUDA;
}

inline bool dense_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What is found out once a device. Threads whose first calls meet: one runs fill(value), the others wait for it; a value is seen whole or
// not at all. After an error the next call tries again.
template <typename T>
class PerDevice
{
    std::mutex m;
    std::atomic<bool> ready[64] = {};
    T value[64] = {};

public:
    template <typename F>
    cudaError_t get(int device, const T** out, F fill)
    {
        if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
        if (!ready[device].load(std::memory_order_acquire))
        {
            std::lock_guard<std::mutex> lock(m);
            if (!ready[device].load(std::memory_order_relaxed))
            {
                T v{};
                const cudaError_t e = fill(v);
                if (e != cudaSuccess) return e;
                value[device] = v;
                ready[device].store(true, std::memory_order_release);
            }
        }
        *out = &value[device];
        return cudaSuccess;
    }
};

// A launch that returns its own error: cudaGetLastError after <<<>>> would also report one that an earlier call of the thread has
// returned already.
template <typename... P, typename... A>
cudaError_t dense_launch(void (*kernel)(P...), unsigned grid, unsigned block, cudaStream_t st, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// the dynamic shared memory that a kernel's launches may ask for, set once
inline cudaError_t dense_smem(PerDevice<int>& set, int device, const void* kernel, int bytes)
{
    const int* done;
    return set.get(device, &done, [&](int&) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

int dense_device();                          // the current device, or -1
int dense_sms(int device);

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

}  // namespace glmx
