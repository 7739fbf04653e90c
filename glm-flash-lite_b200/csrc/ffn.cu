// Gated feed-forward block (glmx_ffn_forward / glmx_ffn_backward), simple form: one tiled product kernel on the CUDA
// cores, fp32 sums, 64 x 64 outputs per CTA.
//   forward:  g = x Wg^T, u = x Wu^T, h = min(silu(g), L) * clamp(u, -L, L), y = h Wd^T
//   backward: dh = dy Wd, du = dh * p, dg = dh * q, dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// with p = min(silu(g), L) [|u| <= L] and q = clamp(u) silu'(g) [silu(g) <= L] kept in fp32 by the forward pass: rounded
// to 16 bits they would add their rounding to that of dg and du.
#include "dense.h"

namespace glmx {

namespace {

// strided operand: element (row, k) at p + row * sr + k * sk
struct Op
{
    const void* p;
    long long sr, sk;
};

enum { EPI_GATED, EPI_STORE, EPI_DACT };

struct FfnArgs
{
    Op a[2], b[2];              // GATED: b[0] gate, b[1] up over one a; STORE: the sum of a[s] b[s] over nseg segments
    int nseg;
    int M, N, K;
    void* y; long long ldy; int y_f32, accumulate;
    void* o0; void* o1;         // GATED: o0 = h; DACT: o0 = dg, o1 = du  ([M][N])
    float* p; float* q;
    float limit;
};

constexpr int TS = 64, TKS = 16;

template <typename T, int EPI>
__global__ void __launch_bounds__(256) simple_kernel(FfnArgs a)
{
    __shared__ float sa[TKS][TS + 1], sb[2][TKS][TS + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int m0 = blockIdx.y * TS, n0 = blockIdx.x * TS;
    constexpr int NB = EPI == EPI_GATED ? 2 : 1;
    float acc[NB][4][4] = {};
    for (int s = 0; s < a.nseg; ++s)
        for (int k0 = 0; k0 < a.K; k0 += TKS)
        {
            for (int i = threadIdx.x; i < TS * TKS; i += 256)
            {
                const int r = i / TKS, k = i % TKS;
                const bool kin = k0 + k < a.K;
                sa[k][r] = kin && m0 + r < a.M ? to_f32(static_cast<const T*>(a.a[s].p)[(m0 + r) * a.a[s].sr + (k0 + k) * a.a[s].sk]) : 0.0f;
                for (int b = 0; b < NB; ++b)
                {
                    const Op& o = a.b[NB == 2 ? b : s];
                    sb[b][k][r] = kin && n0 + r < a.N ? to_f32(static_cast<const T*>(o.p)[(n0 + r) * o.sr + (k0 + k) * o.sk]) : 0.0f;
                }
            }
            __syncthreads();
            for (int k = 0; k < TKS; ++k)
                for (int b = 0; b < NB; ++b)
                    for (int i = 0; i < 4; ++i)
                        for (int j = 0; j < 4; ++j) acc[b][i][j] = fmaf(sa[k][ty * 4 + i], sb[b][k][tx * 4 + j], acc[b][i][j]);
            __syncthreads();
        }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
        {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= a.M || n >= a.N) continue;
            const size_t o = (size_t) m * a.N + n;
            float v = acc[0][i][j];
            if constexpr (EPI == EPI_GATED)
            {
                const float g = v, u = acc[1][i][j], L = a.limit;
                const float s = 1.0f / (1.0f + expf(-g));
                float act = g * s, up = u;
                const bool kg = L == 0.0f || act <= L, ku = L == 0.0f || fabsf(u) <= L;
                if (L != 0.0f) { act = fminf(act, L); up = fminf(fmaxf(u, -L), L); }
                static_cast<T*>(a.o0)[o] = from_f32<T>(act * up);
                if (a.p) { a.p[o] = ku ? act : 0.0f; a.q[o] = kg ? up * (s * (1.0f + g * (1.0f - s))) : 0.0f; }
            }
            else if constexpr (EPI == EPI_DACT)
            {
                static_cast<T*>(a.o0)[o] = from_f32<T>(v * a.q[o]);
                static_cast<T*>(a.o1)[o] = from_f32<T>(v * a.p[o]);
            }
            else if (a.y_f32)
            {
                float* d = static_cast<float*>(a.y) + m * a.ldy + n;
                *d = a.accumulate ? *d + v : v;
            }
            else
            {
                T* d = static_cast<T*>(a.y) + m * a.ldy + n;
                *d = from_f32<T>(a.accumulate ? to_f32(*d) + v : v);
            }
        }
}

template <int EPI>
cudaError_t launch(int dtype, const FfnArgs& a, cudaStream_t st)
{
    const dim3 grid((a.N + TS - 1) / TS, (a.M + TS - 1) / TS);
    if (dtype == GLMX_BF16) simple_kernel<__nv_bfloat16, EPI><<<grid, 256, 0, st>>>(a);
    else simple_kernel<__half, EPI><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
}

int check_ffn(const glmx_ffn* f)
{
    if (!f) return dense_fail(GLMX_E_ARG, "glmx_ffn: null block");
    if (f->hidden <= 0 || f->intermediate <= 0 || f->hidden % 8 || f->intermediate % 8)
        return dense_fail(GLMX_E_ARG, "glmx_ffn: hidden and intermediate must be positive multiples of 8");
    if (f->dtype != GLMX_BF16 && f->dtype != GLMX_F16) return dense_fail(GLMX_E_ARG, "glmx_ffn: dtype must be bf16 or fp16");
    if (!(f->act_limit >= 0.0f)) return dense_fail(GLMX_E_ARG, "glmx_ffn: act_limit must be 0 (none) or positive");
    if (!f->w_gate || !f->w_up || !f->w_down) return dense_fail(GLMX_E_ARG, "glmx_ffn: null weight");
    if (!dense_aligned(f->w_gate) || !dense_aligned(f->w_up) || !dense_aligned(f->w_down))
        return dense_fail(GLMX_E_ARG, "glmx_ffn: weights must be 16-byte aligned");
    return GLMX_OK;
}

}  // namespace

}  // namespace glmx

using namespace glmx;

extern "C" int glmx_ffn_forward(const glmx_ffn* f, const void* x, long long ldx, int ntok, void* y, long long ldy, int y_dtype,
                                int accumulate, void* h, float* p, float* q, void* stream)
{
    int rc = check_ffn(f);
    if (rc) return rc;
    const int H = f->hidden, I = f->intermediate;
    if (ntok < 0) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: ntok >= 0 required");
    if (y_dtype != f->dtype && y_dtype != GLMX_F32) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: y must have the block's dtype or fp32");
    if (ldx < H || ldx % 8 || ldy < H) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: ldx must be a multiple of 8 and ldx, ldy >= hidden");
    if ((p == nullptr) != (q == nullptr)) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: p and q come together");
    if (ntok == 0) return GLMX_OK;
    if (!x || !y || !h) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: null x / y / h");
    if (!dense_aligned(x) || !dense_aligned(y) || !dense_aligned(h) || !dense_aligned(p) || !dense_aligned(q))
        return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: x, y, h, p and q must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    FfnArgs a{};
    a.a[0] = { x, ldx, 1 }; a.b[0] = { f->w_gate, H, 1 }; a.b[1] = { f->w_up, H, 1 };
    a.nseg = 1; a.M = ntok; a.N = I; a.K = H; a.o0 = h; a.p = p; a.q = q; a.limit = f->act_limit;
    cudaError_t e = launch<EPI_GATED>(f->dtype, a, st);
    if (e == cudaSuccess)
    {
        FfnArgs d{};
        d.a[0] = { h, I, 1 }; d.b[0] = { f->w_down, I, 1 };
        d.nseg = 1; d.M = ntok; d.N = H; d.K = I; d.y = y; d.ldy = ldy; d.y_f32 = y_dtype == GLMX_F32; d.accumulate = accumulate;
        e = launch<EPI_STORE>(f->dtype, d, st);
    }
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_ffn_forward: launch");
}

extern "C" int glmx_ffn_backward(const glmx_ffn* f, const void* dy, long long lddy, const void* x, long long ldx, int ntok,
                                 const void* h, const float* p, const float* q, void* dg, void* du, void* dx, void* dw_gate,
                                 void* dw_up, void* dw_down, void* stream)
{
    int rc = check_ffn(f);
    if (rc) return rc;
    const int H = f->hidden, I = f->intermediate;
    if (ntok < 0) return dense_fail(GLMX_E_ARG, "glmx_ffn_backward: ntok >= 0 required");
    if (lddy < H || lddy % 8 || ldx < H || ldx % 8)
        return dense_fail(GLMX_E_ARG, "glmx_ffn_backward: lddy and ldx must be multiples of 8, at least hidden");
    const bool inner = dx || dw_gate || dw_up;
    if (ntok > 0 && (!dy || (inner && (!p || !q || !dg || !du)) || ((dw_gate || dw_up) && !x) || (dw_down && !h)))
        return dense_fail(GLMX_E_ARG, "glmx_ffn_backward: null argument");
    if (!dense_aligned(dy) || !dense_aligned(x) || !dense_aligned(h) || !dense_aligned(p) || !dense_aligned(q) || !dense_aligned(dg) ||
        !dense_aligned(du) || !dense_aligned(dx) || !dense_aligned(dw_gate) || !dense_aligned(dw_up) || !dense_aligned(dw_down))
        return dense_fail(GLMX_E_ARG, "glmx_ffn_backward: pointers must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (ntok == 0)
    {
        // no rows: the weights' gradients are sums over nothing
        if (dw_gate) e = cudaMemsetAsync(dw_gate, 0, (size_t) H * I * 2, st);
        if (e == cudaSuccess && dw_up) e = cudaMemsetAsync(dw_up, 0, (size_t) H * I * 2, st);
        if (e == cudaSuccess && dw_down) e = cudaMemsetAsync(dw_down, 0, (size_t) H * I * 2, st);
        return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_ffn_backward: memset");
    }
    auto product = [&](Op a0, Op b0, int M, int N, int K, void* out) {
        FfnArgs a{};
        a.a[0] = a0; a.b[0] = b0; a.nseg = 1; a.M = M; a.N = N; a.K = K; a.y = out; a.ldy = N;
        return launch<EPI_STORE>(f->dtype, a, st);
    };
    if (inner)
    {
        FfnArgs a{};
        a.a[0] = { dy, lddy, 1 }; a.b[0] = { f->w_down, 1, I };
        a.nseg = 1; a.M = ntok; a.N = I; a.K = H; a.o0 = dg; a.o1 = du; a.p = const_cast<float*>(p); a.q = const_cast<float*>(q);
        e = launch<EPI_DACT>(f->dtype, a, st);
    }
    if (e == cudaSuccess && dx)
    {
        FfnArgs a{};
        a.a[0] = { dg, I, 1 }; a.b[0] = { f->w_gate, 1, H }; a.a[1] = { du, I, 1 }; a.b[1] = { f->w_up, 1, H };
        a.nseg = 2; a.M = ntok; a.N = H; a.K = I; a.y = dx; a.ldy = H;
        e = launch<EPI_STORE>(f->dtype, a, st);
    }
    if (e == cudaSuccess && dw_gate) e = product({ dg, 1, I }, { x, 1, ldx }, I, H, ntok, dw_gate);
    if (e == cudaSuccess && dw_up) e = product({ du, 1, I }, { x, 1, ldx }, I, H, ntok, dw_up);
    if (e == cudaSuccess && dw_down) e = product({ dy, 1, lddy }, { h, 1, I }, H, I, ntok, dw_down);
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_ffn_backward: launch");
}
