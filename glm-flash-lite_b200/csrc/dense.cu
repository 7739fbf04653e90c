// Error word of the dense operators (glmx_dense_check): one per device, sticky, set by a kernel whose bounded wait expired.
#include "dense.h"

namespace glmx {

static __device__ int g_dense_err;

cudaError_t dense_err_ptr(int** p) { return cudaGetSymbolAddress(reinterpret_cast<void**>(p), g_dense_err); }

}  // namespace glmx

using namespace glmx;

extern "C" int glmx_dense_check(void* stream, int* flags)
{
    int* p = nullptr;
    int v = 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = dense_err_ptr(&p);
    if (e == cudaSuccess) e = cudaMemcpyAsync(&v, p, sizeof(int), cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, sizeof(int), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return dense_cuda_fail(e, "glmx_dense_check");
    if (flags) *flags = v;
    return v ? dense_fail(GLMX_E_DEVICE, "glmx_dense_check: a bounded wait expired in a dense operator") : GLMX_OK;
}
