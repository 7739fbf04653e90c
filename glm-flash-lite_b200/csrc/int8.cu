// 8-bit linear (glmx_quantize_rows, glmx_linear_i8): rows to int8 with one scale each, and the product of two int8
// matrices with a scale per token and per output channel.
#include <type_traits>

#include "gemm_tc.cuh"

namespace glmx {

namespace {

constexpr int QT = 256;

// The block's largest magnitude, of fp32 bit patterns without sign: as integers they are in order, infinity next to last and NaN
// above it, so that a NaN anywhere is the result and shows in the row's scale and so in every output of the row.
__device__ __forceinline__ float block_amax(uint32_t m)
{
    __shared__ uint32_t sm[QT / 32];
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < QT / 32; ++w) m = max(m, sm[w]);
    return __uint_as_float(m);
}

__device__ __forceinline__ int quantise(float x, float s)
{
    return s > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x, s)))) : 0;
}

// two fp32 values in one register pair, and a * b + c of both, each rounded once
__device__ __forceinline__ uint64_t pair_of(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// the values 2 p and 2 p + 1 of a 16-byte group
template <typename T>
__device__ __forceinline__ float2 values_of(const uint4& v, int p)
{
    const uint32_t w[4] = { v.x, v.y, v.z, v.w };
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * p]), __uint_as_float(w[2 * p + 1]));
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(reinterpret_cast<const __half2&>(w[p]));
    else return make_float2(__uint_as_float(w[p] << 16), __uint_as_float(w[p] & 0xffff0000u));
}

// Rows of whole 16-byte groups: a CTA holds its row in registers (NV groups a thread), so that x is read once. The quotients come from the
// scale's reciprocal y, rounded once, by Markstein's theorem: where q is within one unit in the last place of x / s, q + y (x - q s), the
// remainder exact, is x / s rounded once. x y may be 1.5 units off; after one such step it is within one, after two it is the quotient.
// Adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low byte. Two values an instruction, magnitudes of
// 16-bit types as pairs of integers. Bound by the reads: 4096 rows of 6144 in bf16 15.6 us (75 MB, 4.8 TB/s; 30 us by the kernel below), one
// row 2 us.
template <typename T, int NV>
__global__ void __launch_bounds__(QT) quantize_kernel(const T* x, long long ldx, int K, signed char* q, long long ldq, float* scale)
{
    constexpr int G = 16 / sizeof(T);
    grid_release();
    const uint4* xr = reinterpret_cast<const uint4*>(x + (size_t) blockIdx.x * ldx);
    const int ng = K / G;
    uint4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        const int g = threadIdx.x + i * QT;
        v[i] = g < ng ? __ldcs(xr + g) : make_uint4(0, 0, 0, 0);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        constexpr uint32_t ABS = G == 4 ? 0x7fffffffu : 0x7fff7fffu;
        const uint32_t a = v[i].x & ABS, b = v[i].y & ABS, c = v[i].z & ABS, d = v[i].w & ABS;
        if constexpr (G == 4) m = max(max(m, a), max(max(b, c), d));
        else m = __vimax3_u16x2(__vimax3_u16x2(m, a, b), c, d);
    }
    if constexpr (G == 8)
    {
        const float2 f = values_of<T>(make_uint4(m, 0, 0, 0), 0);
        m = max(__float_as_uint(f.x), __float_as_uint(f.y));
    }
    const float s = __fdiv_rn(block_amax(m), 127.0f);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    const float inv = 1.0f / s;
    const bool plain = s > 0x1p-100f && s < 0x1p100f;      // 1 / s is a normal number
    const uint64_t inv2 = pair_of(inv, inv), minus_s = pair_of(-s, -s), zero = 0, one = pair_of(1.0f, 1.0f), magic = pair_of(12582912.0f, 12582912.0f);
    signed char* qr = q + (size_t) blockIdx.x * ldq;
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        const int g = threadIdx.x + i * QT;
        if (g >= ng) break;
        uint32_t n[G];
#pragma unroll
        for (int p = 0; p < G / 2; ++p)
        {
            const float2 e = values_of<T>(v[i], p);
            if (plain)
            {
                const uint64_t x2 = pair_of(e.x, e.y);
                uint64_t f = fma2(x2, inv2, zero);
                f = fma2(fma2(f, minus_s, x2), inv2, f);
                f = fma2(fma2(f, minus_s, x2), inv2, f);
                f = fma2(f, one, magic);
                n[2 * p] = (uint32_t) f;
                n[2 * p + 1] = (uint32_t) (f >> 32);
            }
            else
            {
                n[2 * p] = (uint32_t) quantise(e.x, s);
                n[2 * p + 1] = (uint32_t) quantise(e.y, s);
            }
        }
        uint32_t w[G / 4];
#pragma unroll
        for (int j = 0; j < G / 4; ++j)
            w[j] = __byte_perm(__byte_perm(n[4 * j], n[4 * j + 1], 0x0040), __byte_perm(n[4 * j + 2], n[4 * j + 3], 0x0040), 0x5410);
        if constexpr (G == 8) reinterpret_cast<uint2*>(qr)[g] = make_uint2(w[0], w[1]);
        else reinterpret_cast<uint32_t*>(qr)[g] = w[0];
    }
}

// rows of any length, alignment and distance: two passes over the row, the second from cache
template <typename T>
__global__ void __launch_bounds__(QT) quantize_any_kernel(const T* x, long long ldx, int K, signed char* q, long long ldq, float* scale)
{
    grid_release();
    const T* xr = x + (size_t) blockIdx.x * ldx;
    uint32_t m = 0;
    for (int k = threadIdx.x; k < K; k += QT) m = max(m, __float_as_uint(to_f32(xr[k])) & 0x7fffffffu);
    const float s = __fdiv_rn(block_amax(m), 127.0f);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    signed char* qr = q + (size_t) blockIdx.x * ldq;
    for (int k = threadIdx.x; k < K; k += QT) qr[k] = (signed char) quantise(to_f32(xr[k]), s);
}

template <typename T>
cudaError_t launch_quantize(const void* xv, long long ldx, int rows, int K, signed char* q, long long ldq, float* scale, cudaStream_t st)
{
    constexpr int G = 16 / sizeof(T);
    const T* x = static_cast<const T*>(xv);
    const int nv = (K / G + QT - 1) / QT;
    auto kernel = quantize_kernel<T, 8>;
    if (K % G || ldx % G || !dense_aligned(x) || ldq % 8 || reinterpret_cast<uintptr_t>(q) % 8 || nv > 8) kernel = quantize_any_kernel<T>;
    else if (nv == 1) kernel = quantize_kernel<T, 1>;
    else if (nv == 2) kernel = quantize_kernel<T, 2>;
    else if (nv == 3) kernel = quantize_kernel<T, 3>;
    else if (nv == 4) kernel = quantize_kernel<T, 4>;
    return dense_launch(kernel, (unsigned) rows, QT, st, x, ldx, K, q, ldq, scale);
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
    const cudaError_t e = x_dtype == GLMX_F32 ? launch_quantize<float>(x, ldx, rows, K, q, ldq, scale, st)
                        : x_dtype == GLMX_F16 ? launch_quantize<__half>(x, ldx, rows, K, q, ldq, scale, st)
                                              : launch_quantize<__nv_bfloat16>(x, ldx, rows, K, q, ldq, scale, st);
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
