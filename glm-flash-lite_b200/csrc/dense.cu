// What the dense operators' launches share: tensor maps, device facts, and the error word (glmx_dense_check): one per device, for the
// kernels of all streams; sticky, set by a kernel whose bounded wait expired.
#include "gemm_tc.cuh"

namespace glmx {

static __device__ int g_dense_err;

static __global__ void clear_kernel(int* p, int bits) { atomicAnd(p, ~bits); }

int dense_device()
{
    int d = -1;
    if (cudaGetDevice(&d) != cudaSuccess) return -1;
    // the tensor-map encoder is a driver call and needs the device's context current in this thread, which a thread's first
    // runtime calls (an autograd worker's, say) need not have made it
    static thread_local int bound = -1;
    if (bound != d)
    {
        if (cudaSetDevice(d) != cudaSuccess) return -1;
        bound = d;
    }
    return d;
}

cudaError_t dense_err_ptr(int** p)
{
    static PerDevice<int*> ptr;
    int* const* v;
    const cudaError_t e = ptr.get(dense_device(), &v, [](int*& q) { return cudaGetSymbolAddress(reinterpret_cast<void**>(&q), g_dense_err); });
    if (e == cudaSuccess) *p = *v;
    return e;
}

int dense_sms(int device)
{
    static PerDevice<int> sms;
    const int* n;
    const cudaError_t e = sms.get(device, &n, [&](int& v) { return cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device); });
    return e == cudaSuccess && *n >= 2 ? *n : 2;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t dense_map(CUtensorMap* m, int dtype, const Mat& t, int box_inner, int box_rows)
{
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
    }();
    if (!fn) return cudaErrorNotSupported;
    const int size = dtype == GLMX_F32 ? 4 : dtype == GLMX_F16 || dtype == GLMX_BF16 ? 2 : 1;
    const cuuint64_t dims[2] = { (cuuint64_t) t.inner, (cuuint64_t) t.rows };
    const cuuint64_t strides[1] = { (cuuint64_t) t.pitch * size };
    const cuuint32_t box[2] = { (cuuint32_t) box_inner, (cuuint32_t) box_rows };
    const cuuint32_t es[2] = { 1, 1 };
    const CUtensorMapDataType type = size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == GLMX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = fn(m, type, 2, const_cast<void*>(t.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace glmx

using namespace glmx;

extern "C" int glmx_dense_check(void* stream, int* flags)
{
    int* p = nullptr;
    int v = 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = dense_err_ptr(&p);
    if (e == cudaSuccess) e = cudaMemcpyAsync(&v, p, sizeof(int), cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && v)
    {
        // the bits that are reported, no others: a kernel of another stream may have set one since
        e = dense_launch(clear_kernel, 1, 1, st, p, v);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    }
    if (e != cudaSuccess) return dense_cuda_fail(e, "glmx_dense_check");
    if (flags) *flags = v;
    return v ? dense_fail(GLMX_E_DEVICE, "glmx_dense_check: a bounded wait expired in a dense operator") : GLMX_OK;
}
