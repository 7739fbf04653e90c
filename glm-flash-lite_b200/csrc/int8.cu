// 8-bit linear (glmx_quantize_rows, glmx_linear_i8): rows to int8 with one scale each, and the product of two int8
// matrices with a scale per token and per output channel.
#include "gemm_tc.cuh"

namespace glmx {

namespace {

// One CTA per row: the row's largest magnitude, then its quotients (the second read comes from cache). Bound by the read
// of x. Quotients and the scale are IEEE divisions, so that the integers follow from the definition alone.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* x, long long ldx, int K, signed char* q, long long ldq, float* scale)
{
    const T* xr = x + (size_t) blockIdx.x * ldx;
    float m = 0.0f;
    bool nan = false;
    for (int k = threadIdx.x; k < K; k += 256)
    {
        const float v = to_f32(xr[k]);
        nan |= v != v;
        m = fmaxf(m, fabsf(v));
    }
    __shared__ float sm[8];
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    nan = __syncthreads_or(nan);
    for (int w = 0; w < 8; ++w) m = fmaxf(m, sm[w]);
    // a NaN in the row shows in its scale, and so in every output of the row
    const float s = nan ? __int_as_float(0x7fc00000) : __fdiv_rn(m, 127.0f);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    signed char* qr = q + (size_t) blockIdx.x * ldq;
    for (int k = threadIdx.x; k < K; k += 256)
        qr[k] = (signed char) (s > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(to_f32(xr[k]), s)))) : 0);
}

}  // namespace

}  // namespace glmx

using namespace glmx;

extern "C" int glmx_quantize_rows(const void* x, int x_dtype, long long ldx, int rows, int K, signed char* q, long long ldq,
                                  float* scale, void* stream)
{
    if (rows < 0 || K < 1 || ldx < K || ldq < K) return dense_fail(GLMX_E_ARG, "glmx_quantize_rows: rows >= 0, K >= 1, ldx >= K and ldq >= K required");
    if (x_dtype != GLMX_F16 && x_dtype != GLMX_BF16 && x_dtype != GLMX_F32)
        return dense_fail(GLMX_E_ARG, "glmx_quantize_rows: x must be fp16, bf16 or fp32");
    if (rows == 0) return GLMX_OK;
    if (!x || !q || !scale) return dense_fail(GLMX_E_ARG, "glmx_quantize_rows: null argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (x_dtype == GLMX_F32) quantize_kernel<<<rows, 256, 0, st>>>(static_cast<const float*>(x), ldx, K, q, ldq, scale);
    else if (x_dtype == GLMX_F16) quantize_kernel<<<rows, 256, 0, st>>>(static_cast<const __half*>(x), ldx, K, q, ldq, scale);
    else quantize_kernel<<<rows, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(x), ldx, K, q, ldq, scale);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_quantize_rows: launch");
}

extern "C" int glmx_linear_i8(const signed char* xq, long long ldxq, const float* x_scale, int ntok, int K, int N,
                              const signed char* wq, long long ldwq, const float* w_scale, const float* bias, void* y,
                              long long ldy, int y_dtype, void* stream)
{
    if (ntok < 0 || N < 1 || K < 1 || K > GLMX_I8_MAX_K)
        return dense_fail(GLMX_E_ARG, "glmx_linear_i8: ntok >= 0, N >= 1 and 1 <= K <= GLMX_I8_MAX_K required");
    if (ldxq < K || ldwq < K || ldxq % 16 || ldwq % 16 || ldy < N)
        return dense_fail(GLMX_E_ARG, "glmx_linear_i8: ldxq and ldwq must be multiples of 16, at least K, and ldy at least N");
    if (y_dtype != GLMX_F16 && y_dtype != GLMX_BF16 && y_dtype != GLMX_F32)
        return dense_fail(GLMX_E_ARG, "glmx_linear_i8: y must be fp16, bf16 or fp32");
    if (ntok == 0) return GLMX_OK;
    if (!xq || !x_scale || !wq || !w_scale || !y) return dense_fail(GLMX_E_ARG, "glmx_linear_i8: null argument");
    if (!dense_aligned(xq) || !dense_aligned(wq)) return dense_fail(GLMX_E_ARG, "glmx_linear_i8: xq and wq must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Product p{};
    p.a[0] = { xq, ntok, K, ldxq };
    p.b[0] = { wq, N, K, ldwq };
    p.e.M = ntok; p.e.N = N; p.e.y = y; p.e.ldy = ldy; p.e.y_dtype = y_dtype;
    p.e.xs = x_scale; p.e.ws = w_scale; p.e.bias = bias;
    p.e.vec = dense_aligned(y) && ldy * (y_dtype == GLMX_F32 ? 4 : 2) % 16 == 0;
    const cudaError_t e = launch_product<true, false, EPI_I8>(GLMX_I32, p, 1, K, false, st);
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_linear_i8: launch");
}
