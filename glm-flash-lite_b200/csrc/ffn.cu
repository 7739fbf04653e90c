// Gated feed-forward block (glmx_ffn_forward / glmx_ffn_backward).
//   forward:  g = x Wg^T, u = x Wu^T, h = min(silu(g), L) * clamp(u, -L, L), y = h Wd^T
//   backward: dh = dy Wd, du = dh * p, dg = dh * q, dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// with p = min(silu(g), L) [|u| <= L] and q = clamp(u) silu'(g) [silu(g) <= L] kept in fp32 by the forward pass: rounded
// to 16 bits they would add their rounding to that of dg and du.
//
// Gate and up are one product whose tiles hold the same columns of both, so that the activation is its epilogue; dg and du are
// the epilogue of dh; dx is one sum over both of its products; the weights' gradients are one launch.
#include <cmath>

#include "gemm_tc.cuh"

namespace glmx {

namespace {

// rows of h, dg and du: 128-byte lines, which a copy of 128-byte boxes from rows between lines would read twice
long long hidden_pitch(const glmx_ffn* f) { return (f->intermediate + 63) / 64 * 64; }

Epi epi(const glmx_ffn* f, int M, int N)
{
    Epi e{};
    e.M = M; e.N = N; e.bf16 = f->dtype == GLMX_BF16; e.vec = 1; e.limit = std::isinf(f->act_limit) ? 0.0f : f->act_limit; e.y_dtype = f->dtype; e.ldy = N;
    return e;
}

// Norms of rows of K 16-bit values, rounded up to bf16, a warp a row: those of a, then of b (both packed), then of x. Squares that overflow make
// a norm infinite, those that vanish (below 2^-75 of a value) are covered by 2^-50. Bound by the reads: 4096 x 6144 inputs
// and 2 x 1536 x 6144 weights (88 MB) 17 us.
constexpr int NORM_WARPS = 8;
__global__ void __launch_bounds__(NORM_WARPS * 32) norms_kernel(const void* a, const void* b, int ab_rows, const void* x, long long ldx, int x_rows, int K,
                                                                int bf16, __nv_bfloat16* norms)
{
    grid_release();
    const long long row = (long long) blockIdx.x * NORM_WARPS + (threadIdx.x >> 5);
    if (row >= 2ll * ab_rows + x_rows) return;
    const uint16_t* r = row < ab_rows ? static_cast<const uint16_t*>(a) + row * K
                      : row < 2ll * ab_rows ? static_cast<const uint16_t*>(b) + (row - ab_rows) * K
                      : static_cast<const uint16_t*>(x) + (row - 2ll * ab_rows) * ldx;
    float s[8] = {};
#pragma unroll 4
    for (int k = (threadIdx.x & 31) * 8; k < K; k += 256)
    {
        const uint4 v = *reinterpret_cast<const uint4*>(r + k);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const float e = load16(&v, i, bf16);
            s[i] = fmaf(e, e, s[i]);
        }
    }
    float d = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    // 2^-10: the sum's own roundings, K / 256 + 8 of 2^-24 each (H is below 2^22 where a weight fits the device), and the root's
    if ((threadIdx.x & 31) == 0) norms[row] = __float2bfloat16_ru(sqrtf(d) * (1.0f + 0x1p-10f) + 0x1p-50f);
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
    const long long P = hidden_pitch(f);
    if (ntok < 0) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: ntok >= 0 required");
    if (y_dtype != f->dtype && y_dtype != GLMX_F32) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: y must have the block's dtype or fp32");
    if (ldx < H || ldx % 8 || ldy < H) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: ldx must be a multiple of 8 and ldx, ldy >= hidden");
    if ((p == nullptr) != (q == nullptr)) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: p and q come together");
    if (ntok == 0) return GLMX_OK;
    if (!x || !y || !h) return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: null x / y / h");
    if (!dense_aligned(x) || !dense_aligned(y) || !dense_aligned(h) || !dense_aligned(p) || !dense_aligned(q))
        return dense_fail(GLMX_E_ARG, "glmx_ffn_forward: x, y, h, p and q must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Product g{};
    g.a[0] = { x, ntok, H, ldx };
    g.b[0] = { f->w_gate, I, H, H };
    g.b[1] = { f->w_up, I, H, H };
    g.e = epi(f, ntok, I);
    g.e.o0 = h; g.e.ldo = P; g.e.p = p; g.e.q = q; g.e.x = x; g.e.wg = f->w_gate; g.e.wu = f->w_up; g.e.ldx = ldx; g.e.K = H;
    cudaError_t e = cudaSuccess;
    // y takes the norms of the operands' rows until the second product writes it, where it is large enough, packed and not read by this call
    const long long rows = 2ll * I + ntok, y_bytes = (long long) ntok * H * (y_dtype == GLMX_F32 ? 4 : 2);
    const uint8_t *yb = static_cast<const uint8_t*>(y), *xb = static_cast<const uint8_t*>(x);
    const bool apart = yb >= xb + ((ntok - 1) * ldx + H) * 2 || xb >= yb + y_bytes;
    if (p && g.e.limit != 0.0f && !accumulate && ldy == H && y_bytes >= 2 * rows && apart)
    {
        __nv_bfloat16* norms = static_cast<__nv_bfloat16*>(y);
        e = dense_launch(norms_kernel, (unsigned) ((rows + NORM_WARPS - 1) / NORM_WARPS), NORM_WARPS * 32, st, f->w_gate, f->w_up, I, x, ldx, ntok, H,
                         g.e.bf16, norms);
        g.e.norms = norms;
    }
    if (e == cudaSuccess) e = launch_product<false, false, EPI_GATED>(f->dtype, g, 1, H, false, st);
    if (e == cudaSuccess)
    {
        Product d{};
        d.a[0] = { h, ntok, I, P };
        d.b[0] = { f->w_down, H, I, I };
        d.e = epi(f, ntok, H);
        d.e.y = y; d.e.ldy = ldy; d.e.y_dtype = y_dtype; d.e.accumulate = accumulate;
        d.e.vec = ldy * (y_dtype == GLMX_F32 ? 4 : 2) % 16 == 0;
        // the kernel in front is this call's own and writes no weights: they may be read while it runs
        e = launch_product<false, false, EPI_STORE>(f->dtype, d, 1, I, true, st);
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
    const long long P = hidden_pitch(f);
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
    if (inner)
    {
        Product d{};
        d.a[0] = { dy, ntok, H, lddy };
        d.b[0] = { f->w_down, H, I, I };
        d.e = epi(f, ntok, I);
        d.e.o0 = dg; d.e.o1 = du; d.e.ldo = P; d.e.p = const_cast<float*>(p); d.e.q = const_cast<float*>(q);
        e = launch_product<false, true, EPI_DACT>(f->dtype, d, 1, H, false, st);
    }
    if (e == cudaSuccess && dx)
    {
        Product d{};
        d.a[0] = { dg, ntok, I, P }; d.b[0] = { f->w_gate, I, H, H };
        d.a[1] = { du, ntok, I, P }; d.b[1] = { f->w_up, I, H, H };
        d.e = epi(f, ntok, H);
        d.e.y = dx;
        e = launch_product<false, true, EPI_STORE>(f->dtype, d, 2, I, true, st);
    }
    Product w[3] = {};
    int n = 0;
    auto add = [&](const void* rows, long long width, long long pitch, const void* cols, int N, long long cpitch, void* out) {
        w[n].a[0] = { rows, ntok, width, pitch };
        w[n].b[0] = { cols, ntok, N, cpitch };
        w[n].e = epi(f, (int) width, N);
        w[n++].e.y = out;
    };
    if (dw_gate) add(dg, I, P, x, H, ldx, dw_gate);
    if (dw_up) add(du, I, P, x, H, ldx, dw_up);
    if (dw_down) add(dy, H, lddy, h, I, P, dw_down);
    if (e == cudaSuccess && n)
    {
        const Epi es[3] = { w[0].e, w[1].e, w[2].e };
        e = launch_pair<false, true, true, EPI_STORE>(f->dtype, n, w, 1, ntok, pair_plan(n, es, false, false, (ntok + 63) / 64, dense_sms(dense_device())).BN, st);
    }
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_ffn_backward: launch");
}
