// Matrix products of the dense operators on the 5th-generation tensor cores (tcgen05, accumulators in tensor memory), with
// their epilogues. Two kernels:
//
//   pair_kernel: many rows. Persistent CTA pairs (cta_group::2), 256 tokens x 64 to 256 columns per tile, each CTA holding half of
//     the rows of A and half of the columns of B, so that a byte of shared memory feeds 256 products' worth of either side. Bound by
//     the tensor cores: a bf16 feed-forward of 4096 rows, H = 2048, I = 8192, 278 us, 1.48 PFLOP/s where a large library
//     product reaches 1.61; 8-bit, 4096 x 6144 x 12288, 194 us, 3.19 POP/s. What is lost is the last round of tiles, the
//     start and the last epilogue.
//   cols_kernel: few rows. The weights are the M operand (128 of their rows per tile), the tokens the N operand (16 .. 256),
//     and K is split over the CTAs of a cluster, whose partial tiles are added in rank order over distributed shared memory:
//     enough CTAs to stream the weights at full bandwidth, one launch, no scratch, the same bits in every run. Bound by that
//     stream, 5.3 to 7 TB/s, and 5 us around it (the first weights' arrival, the join): 6144 x 6144 bytes 11.4 us for one row,
//     a feed-forward of 56.6 MB 17.8 us; 65536 x 4096 bytes for 48 rows 55 us.
//
// Operands are row-major matrices read by TMA with the 128-byte swizzle: K-major ones [rows][K] in boxes of 128 bytes of K,
// MN-major ones [K][rows] in boxes of 64 rows x 64 K. Boxes past an edge are zero-filled; stores are predicated.
#pragma once
#include <cuda.h>

#include "dense.h"
#include "glmx_common.cuh"

namespace glmx {

enum { EPI_GATED, EPI_STORE, EPI_DACT, EPI_I8 };

// What becomes of the sums: element (t, n) of an [M tokens][N] result.
struct Epi
{
    int M, N;
    int bf16;                   // 16-bit type: bf16 or fp16
    int vec;                    // rows of every output can take 16-byte stores (always but for I8 with an odd width)
    void* y; long long ldy; int y_dtype;                 // STORE, I8
    int accumulate;             // STORE
    void* o0; void* o1;         // GATED: o0 = h; DACT: o0 = dg, o1 = du; [M] rows of N, ldo apart
    long long ldo;
    float* p; float* q;         // [M][N]
    float limit;
    const void* x; const void* wg; const void* wu; long long ldx; int K;   // GATED with p: the operands, for the sums next to the limit,
    const __nv_bfloat16* norms; // and their rows' norms, rounded up: [N] gate, [N] up, [M] tokens (NULL: every sum counts as next to it)
    const float* xs; const float* ws; const float* bias; // I8
};

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int bf16)
{
    if (bf16)
    {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store16(void* base, size_t off, const float (&v)[4], int bf16)
{
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(base) + off * 2) = make_uint2(pack16(v[0], v[1], bf16), pack16(v[2], v[3], bf16));
}

__device__ __forceinline__ float load16(const void* base, size_t off, int bf16)
{
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[off]) : __half2float(static_cast<const __half*>(base)[off]);
}

__device__ __forceinline__ void store_f32(float* d, const float (&v)[4]) { *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]); }

// the two values of a 32-bit word, as a pair of fp32 registers
template <bool BF16>
__device__ __forceinline__ uint64_t unpack16(uint32_t w)
{
    float2 f;
    if constexpr (BF16) f = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(f.x), "f"(f.y));
    return r;
}

// Whether v = sum_k x[k] w[k], as silu(v) or |v|, is at most L in 64 bits; by a warp (K a multiple of 8, both rows 16-byte aligned). most: a bound
// of |x| |w|. The sum is first formed in fp32, 256 chains of K / 256 fused products: it is within (K / 256 + 9) 2^-24 of the bound, and few of the
// values that come here need the second one.
template <bool BF16>
static __device__ __noinline__ bool warp_within(const void* x, const void* w, int K, bool silu, float L, float most)
{
    const int k0 = (threadIdx.x & 31) * 8;
    constexpr int U = 2;                                   // (more would have the kernel around spill)
    // 2^-100: products that vanish
    const float e = most * (float) (K / 256 + 12) * 0x1p-24f + 0x1p-100f;
    if (e < 3e38f)
    {
        // two sets of U pieces of either row: one on its way while the other is added (volatile: fetched as written, not next to their use)
        uint4 a[2][U], b[2][U];
        uint64_t s[4] = {};
        auto fetch = [&](int h, int k) {
#pragma unroll
            for (int j = 0; j < U; ++j)
            {
                a[h][j] = b[h][j] = make_uint4(0, 0, 0, 0);
                if (k + 256 * j < K)
                {
                    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(a[h][j].x), "=r"(a[h][j].y), "=r"(a[h][j].z), "=r"(a[h][j].w) : "l"(static_cast<const uint16_t*>(x) + k + 256 * j));
                    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(b[h][j].x), "=r"(b[h][j].y), "=r"(b[h][j].z), "=r"(b[h][j].w) : "l"(static_cast<const uint16_t*>(w) + k + 256 * j));
                }
            }
        };
        auto add = [&](int h) {
#pragma unroll
            for (int j = 0; j < U; ++j)
            {
                const uint32_t aw[4] = { a[h][j].x, a[h][j].y, a[h][j].z, a[h][j].w }, bw[4] = { b[h][j].x, b[h][j].y, b[h][j].z, b[h][j].w };
#pragma unroll
                for (int i = 0; i < 4; ++i) asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(s[i]) : "l"(unpack16<BF16>(aw[i])), "l"(unpack16<BF16>(bw[i])));
            }
        };
        fetch(0, k0);
        for (int k = k0; k - k0 < K; k += 512 * U)
        {
            fetch(1, k + 256 * U);
            add(0);
            fetch(0, k + 512 * U);
            add(1);
        }
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) v += __uint_as_float((uint32_t) s[i]) + __uint_as_float((uint32_t) (s[i] >> 32));
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        // (|silu'| < 1.1; the exponential and the division: some ulp)
        const float y = silu ? v / (1.0f + expf(-v)) : fabsf(v), room = silu ? 1.1f * e + 0x1p-20f * L : e;
        if (fabsf(y - L) > room) return y <= L;
    }
    double d = 0.0;
    for (int k = k0; k < K; k += 256)
    {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + k);
        const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + k);
#pragma unroll
        for (int i = 0; i < 8; ++i) d += (double) load16(&a, i, BF16) * (double) load16(&b, i, BF16);
    }
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    return (silu ? d / (1.0 + exp(-d)) : fabs(d)) <= (double) L;
}

// h (and p, q) of 4 consecutive columns n .. n + 3 of token t, a multiple of 4; called by whole warps. acc, acc2: the sums of gate and up.
// Which side of the limit a value falls on decides whether its gradient passes, and so must not hang on the last bits of the tensor cores'
// truncated sums: within their error's bound the sum is formed again. An MMA of 16 inputs cuts each of its 17 addends to 2^-25 of
// the largest one's power of two (measured: two bits below fp32's) and the sum to 2^-23: 5 2^-23 of the largest. The products' part in this is at
// most |x| |w| (Cauchy-Schwarz) over all of K; the running sum v_k is at most |x_1..k| |w_1..k| and |v| + |x_k+1..| |w_k+1..|, hence
// (|x| |w| + |v|) / 2 in each of the K / 16 steps, and less in a split's own sum. In all 5 2^-28 (K + 32) (|x| |w| + |v|); 96 for the splits' additions.
__device__ __forceinline__ void emit_gated(const Epi& e, int t, int n, const uint32_t (&acc)[4], const uint32_t (&acc2)[4])
{
    // N is a multiple of 8: all columns are inside, or none
    const bool in = t < e.M && n < e.N;
    const float L = e.limit;
    float g[4], u[4], s[4], act[4];
    bool kg[4], ku[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        g[i] = __uint_as_float(acc[i]);
        u[i] = __uint_as_float(acc2[i]);
        s[i] = __fdividef(1.0f, 1.0f + __expf(-g[i]));
        act[i] = g[i] < -100.0f ? 0.0f : g[i] * s[i];      // silu(-inf) = 0 (not -inf * 0)
        kg[i] = L == 0.0f || act[i] <= L;
        ku[i] = L == 0.0f || fabsf(u[i]) <= L;
    }
    if (e.p && L != 0.0f)
    {
        uint32_t near = 0;
        if (in)
        {
            const float inf = __int_as_float(0x7f800000);
            float ng[4] = { inf, inf, inf, inf }, nu[4] = { inf, inf, inf, inf };
            if (e.norms)
            {
                const uint2 a = *reinterpret_cast<const uint2*>(e.norms + n), b = *reinterpret_cast<const uint2*>(e.norms + e.N + n);
#pragma unroll
                for (int i = 0; i < 4; ++i) { ng[i] = load16(&a, i, 1); nu[i] = load16(&b, i, 1); }
            }
            const float nx = e.norms ? load16(e.norms, 2 * (size_t) e.N + t, 1) : 1.0f, c = (float) (e.K + 96) * 0x1.4p-26f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                // |silu'| < 1.1; 2^-18: the exponential and the division
                const float wg = 1.1f * c * (nx * ng[i] + fabsf(g[i])) + L * 0x1p-18f, wu = c * (nx * nu[i] + fabsf(u[i]));
                near |= (fabsf(act[i] - L) <= wg ? 1u : 0u) << i | (fabsf(fabsf(u[i]) - L) <= wu ? 16u : 0u) << i;
            }
        }
        uint32_t lanes = __ballot_sync(0xffffffffu, near != 0);
        while (lanes)
        {
            const int src = __ffs(lanes) - 1;
            lanes &= lanes - 1;
            uint32_t bits = __shfl_sync(0xffffffffu, near, src);
            const int tt = __shfl_sync(0xffffffffu, t, src), nn = __shfl_sync(0xffffffffu, n, src);
            while (bits)
            {
                const int b = __ffs(bits) - 1, c = nn + (b & 3);
                bits &= bits - 1;
                const void* xr = static_cast<const uint16_t*>(e.x) + (size_t) tt * e.ldx;
                const void* wr = static_cast<const uint16_t*>(b < 4 ? e.wg : e.wu) + (size_t) c * e.K;
                const float bound = e.norms ? load16(e.norms, 2 * (size_t) e.N + tt, 1) * load16(e.norms, (size_t) (b < 4 ? 0 : e.N) + c, 1) : __int_as_float(0x7f800000);
                const bool keep = e.bf16 ? warp_within<true>(xr, wr, e.K, b < 4, L, bound) : warp_within<false>(xr, wr, e.K, b < 4, L, bound);
                if ((threadIdx.x & 31) == src)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        if (b == i) kg[i] = keep;
                        if (b == i + 4) ku[i] = keep;
                    }
            }
        }
    }
    if (!in) return;
    float hh[4], pp[4], qq[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float ac = act[i], up = u[i];
        if (L != 0.0f)
        {
            ac = fminf(ac, L);
            up = fminf(fmaxf(up, -L), L);
            if (u[i] != u[i]) up = u[i];                   // NaN stays NaN
            if (g[i] != g[i]) ac = g[i];
        }
        hh[i] = ac * up;
        pp[i] = ku[i] ? ac : 0.0f;
        qq[i] = kg[i] ? up * (s[i] + act[i] * (1.0f - s[i])) : 0.0f;
    }
    store16(e.o0, (size_t) t * e.ldo + n, hh, e.bf16);
    const size_t o = (size_t) t * e.N + n;
    if (e.p) { store_f32(e.p + o, pp); store_f32(e.q + o, qq); }
}

// W (4, or 1 where rows cannot take wide stores) consecutive columns n .. n + W - 1 of token t; n is a multiple of W. acc: the sums (I8: int32).
template <int EPI, int W>
__device__ __forceinline__ void emit(const Epi& e, int t, int n, const uint32_t (&acc)[W])
{
    if (t >= e.M || n >= e.N) return;
    float v[W];
    if constexpr (EPI == EPI_DACT)
    {
        const size_t o = (size_t) t * e.N + n;
        const float4 p = *reinterpret_cast<const float4*>(e.p + o), q = *reinterpret_cast<const float4*>(e.q + o);
        const float pv[4] = { p.x, p.y, p.z, p.w }, qv[4] = { q.x, q.y, q.z, q.w };
        float dg[4], du[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float d = __uint_as_float(acc[i]);
            dg[i] = d * qv[i];
            du[i] = d * pv[i];
        }
        store16(e.o0, (size_t) t * e.ldo + n, dg, e.bf16);
        store16(e.o1, (size_t) t * e.ldo + n, du, e.bf16);
        return;
    }
    if constexpr (EPI == EPI_I8)
    {
        const float xs = e.xs[t];
#pragma unroll
        for (int i = 0; i < W; ++i)
        {
            const int c = n + i < e.N ? n + i : e.N - 1;
            v[i] = (float) (int) acc[i] * (xs * e.ws[c]);
            if (e.bias) v[i] += e.bias[c];
        }
    }
    else
    {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = __uint_as_float(acc[i]);
    }
    const size_t o = (size_t) t * e.ldy + n;
    const bool f32 = e.y_dtype == GLMX_F32, bf = e.y_dtype == GLMX_BF16;
    const bool held = EPI == EPI_STORE && e.accumulate;
    if constexpr (W == 4)
        if (e.vec && n + W <= e.N)
        {
            if (held)
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] += f32 ? static_cast<const float*>(e.y)[o + i] : load16(e.y, o + i, bf);
            if (f32) store_f32(static_cast<float*>(e.y) + o, v);
            else store16(e.y, o, v, bf);
            return;
        }
#pragma unroll
    for (int i = 0; i < W; ++i)
    {
        if (n + i >= e.N) break;
        if (f32)
        {
            float* d = static_cast<float*>(e.y) + o + i;
            *d = held ? *d + v[i] : v[i];
        }
        else
        {
            const float w = held ? load16(e.y, o + i, bf) + v[i] : v[i];
            if (bf) static_cast<__nv_bfloat16*>(e.y)[o + i] = __float2bfloat16_rn(w);
            else static_cast<__half*>(e.y)[o + i] = __float2half_rn(w);
        }
    }
}

// ---- tcgen05 / TMA / cluster primitives ------------------------------------------------------------------------------

// shared-memory matrix descriptor with the 128-byte swizzle. K-major: 8-row groups 1024 bytes apart (leading offset
// unused). MN-major: 64-row blocks `lbo` apart, 8-K groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo)
{
    return (uint64_t) ((saddr & 0x3FFFFu) >> 4) | ((uint64_t) (lbo >> 4) << 16) | ((uint64_t) (1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// instruction descriptor: 16-bit floats to fp32, or signed bytes to int32; bits 15 / 16 for MN-major A / B
__host__ __device__ constexpr uint32_t tc_idesc(bool i8, bool bf16, bool a_mn, bool b_mn, int m, int n)
{
    return ((i8 ? 2u : 1u) << 4) | ((i8 || bf16 ? 1u : 0u) << 7) | ((i8 || bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
           ((b_mn ? 1u : 0u) << 16) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (m >> 4) << 24);
}

template <bool I8, int CG>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc)
{
    const uint32_t en = acc;
    if constexpr (I8 && CG == 1)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(en));
    else if constexpr (I8)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(en));
    else if constexpr (CG == 1)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(en));
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(en));
}

// arrive on `bar` (CG 2: on both CTAs' barrier at that offset) once this thread's earlier MMAs are complete
template <int CG>
__device__ __forceinline__ void tc_commit(uint64_t* bar)
{
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t) 3) : "memory");
}

template <int CG>
__device__ __forceinline__ void tc_alloc(uint32_t* slot, uint32_t cols)
{
    if constexpr (CG == 1)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    else
    {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}

template <int CG>
__device__ __forceinline__ void tc_dealloc(uint32_t tmem, uint32_t cols)
{
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 16 consecutive 32-bit columns of this thread's tensor-memory lane (valid after tc_wait_ld)
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}

// one lane of a converged warp: issuing instructions under it, with the loops around them run by the whole warp, keeps
// descriptors and addresses in uniform registers
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// address of rank's copy of a shared-memory address
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// a CTA pair's load: into this CTA's shared memory, counted on a barrier that may be the other CTA's
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// a tile of shared memory (128-byte swizzle) to global memory; rows and columns past the edges are left out
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n cp.async.bulk.commit_group;" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// a box into L2 only: also before the kernels in front have finished, since L2 takes their writes, too
__device__ __forceinline__ void prefetch_2d(const CUtensorMap* map, int x, int y)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y) : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Bounded wait for a stage. The clock is first read after many tries: reading it takes longer than a stage does.
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity)
{
    for (int i = 0; i < 256; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait_bounded(bar, parity);
}

// The same for a whole warp that waits long: one lane asks, with pauses. (256 threads that ask without one keep the shared-memory
// pipe so busy that the loads' and MMAs' threads take twice as long for a stage.) False where the wait expired.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity)
{
    bool ok = true;
    if ((threadIdx.x & 31) == 0)
    {
        ok = false;
        for (int i = 0; i < 256 && !(ok = mbar_try_wait(bar, parity)); ++i) __nanosleep(64);
        if (!ok) ok = mbar_wait_bounded(bar, parity);
    }
    return __shfl_sync(0xffffffffu, (int) ok, 0) != 0;
}

// place in a ring of stages and the parity of its round
struct Ring
{
    int s = 0, n;
    uint32_t ph = 0;
    __device__ __forceinline__ explicit Ring(int stages) : n(stages) {}
    __device__ __forceinline__ void next()
    {
        if (++s == n) { s = 0; ph ^= 1u; }
    }
};

// wait for asynchronous copies that nobody will wait for any more (only after a bounded wait has expired)
__device__ __forceinline__ void drain_pause()
{
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 1000000) __nanosleep(10000);
}

// A warp copies its staging tile (32 rows of 128 bytes, 16-byte piece i of row r at place i ^ (r & 7)) to rows of any alignment: fp32 by single
// elements, 16-bit ones by words, which in rows that start between two words are made of neighbours' halves.
__device__ __forceinline__ void copy_rows(const Epi& e, const uint4* stg, int row0, int n0, int wide, int lane)
{
    const uint32_t* w = reinterpret_cast<const uint32_t*>(stg);
    const int rows = min(32, e.M - row0), cols = min(wide, e.N - n0);
    if (cols <= 0) return;
    const size_t first = (size_t) row0 * e.ldy + n0;
    // eight rows at a time, their loads and exchanges before their stores
    for (int r0 = 0; r0 < rows; r0 += 8)
    {
        uint32_t v[8], next[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = w[((r0 + i) * 8 + ((lane >> 2) ^ i)) * 4 + (lane & 3)];
        if (wide == 32)
        {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r0 + i < rows && lane < cols) static_cast<uint32_t*>(e.y)[first + (size_t) (r0 + i) * e.ldy + lane] = v[i];
            continue;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) next[i] = __shfl_down_sync(0xffffffffu, v[i], 1);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            uint16_t* d = static_cast<uint16_t*>(e.y) + first + (size_t) (r0 + i) * e.ldy;
            const bool odd = (reinterpret_cast<uintptr_t>(d) & 2) != 0, in = r0 + i < rows;
            const uint32_t word = odd ? __funnelshift_r(v[i], next[i], 16) : v[i];
            const int c = 2 * lane + odd;                  // the word's first column
            if (in && c + 1 < cols) *reinterpret_cast<uint32_t*>(d + c) = word;
            if (in && c + 1 == cols) d[c] = (uint16_t) word;
            if (in && odd && lane == 0) d[0] = (uint16_t) v[i];
        }
    }
}

// Shared memory of a CTA that allocates `cols` columns of tensor memory: at least the same share of the SM's, so that CTAs which fit
// an SM together, of whatever launches and streams, never want more than its 512 columns. Allocation waits for columns without limit, and CTAs
// of a cluster wait for one another: two clusters that each held columns that the other's CTAs wait for would hang.
constexpr int tmem_smem(int cols, int bytes) { return bytes > cols * 452 ? bytes : cols * 452; }
static_assert((512 + 32) * 452 > 228 * 1024, "one allocation more than 512 columns does not fit an SM's 228 KB");

// ---- pair_kernel -------------------------------------------------------------------------------------------------------

constexpr int MAXPROB = 3;

struct PairMaps
{
    CUtensorMap a[MAXPROB], b[MAXPROB];
    CUtensorMap y[MAXPROB];     // STORE, I8 with Epi.tma: boxes of 32 rows x 128 bytes
};

struct PairArgs
{
    int nprob;                  // products in the launch (the weights' gradients: three); problem p has maps a[p], b[p], epilogue e[p]
    int nseg;                   // 1; 2: one product whose sum runs over a[0] b[0] and a[1] b[1]
    int K, bk;                  // inputs per segment, and per stage (128 bytes)
    int BN;                     // columns per tile: 128 or 256; with K-major weights also 64 or 192
    int mt[MAXPROB], nt[MAXPROB], tile0[MAXPROB + 1];    // tiles along M and N, and the first tile of each problem
    uint32_t idesc;
    int* err;
    Epi e[MAXPROB];
};

constexpr int PAIR_BM = 128;                             // rows per CTA, 256 per pair
constexpr int PAIR_EPI = 8;                              // epilogue warps: two per tensor-memory lane quarter
constexpr int PAIR_THREADS = (2 + PAIR_EPI) * 32;
constexpr int PAIR_STAGES_MAX = 8;
constexpr int PAIR_SMEM = 227 * 1024;
constexpr int PAIR_STG = PAIR_EPI * 4096;                // the epilogue warps' staging
constexpr int pair_stage(int bn) { return PAIR_BM * 128 + bn / 2 * 128; }
constexpr int pair_stages(int bn)
{
    const int n = (PAIR_SMEM - 1024 - 1024 - PAIR_STG) / pair_stage(bn);   // 1 KB of static shared memory, 1 KB of alignment
    return n > PAIR_STAGES_MAX ? PAIR_STAGES_MAX : n;
}
constexpr int pair_smem(int bn) { return tmem_smem(512, 1024 + pair_stages(bn) * pair_stage(bn) + PAIR_STG); }
static_assert(pair_smem(64) <= PAIR_SMEM - 1024 && pair_smem(128) <= PAIR_SMEM - 1024 && pair_smem(192) <= PAIR_SMEM - 1024 && pair_smem(256) <= PAIR_SMEM - 1024, "");

// I8: signed bytes; A_MN / B_MN: operand stored [K][rows]; EPI
template <bool I8, bool A_MN, bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairArgs a)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[PAIR_STAGES_MAX], empty[PAIR_STAGES_MAX], tfull[2], tempty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_abort;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int BN = a.BN, NST = pair_stages(BN), STAGE = pair_stage(BN);
    if (warp == 0)
    {
        if (lane < NST) { mbar_init(&full[lane], 1); mbar_init(&empty[lane], 1); }
        if (lane < 2) { mbar_init(&tfull[lane], 1); mbar_init(&tempty[lane], 2 * PAIR_EPI); }
        if (lane == 0) s_abort = 0;
        fence_barrier_init();
    }
    else if (warp == 2 && lane == 0)
    {
        prefetch_map(&maps.a[0]);
        prefetch_map(&maps.b[EPI == EPI_GATED ? (int) rank : 0]);
    }
    if (warp == 1) tc_alloc<2>(&tmem_slot, 512);
    tc_before();
    __syncthreads();
    cluster_sync();
    tc_after();
    const uint32_t tmem = tmem_slot;
    // the next kernel may start once the ones in front of this one are complete: it may read weights before its own wait
    grid_wait();
    grid_release();

    const int pairs = gridDim.x >> 1, first = blockIdx.x >> 1, ntiles = a.tile0[a.nprob];
    const int ksteps = (a.K + a.bk - 1) / a.bk, nk = ksteps * a.nseg;
    auto find = [&](int t, int& p, int& m, int& n) {
        p = 0;
        while (p + 1 < a.nprob && t >= a.tile0[p + 1]) ++p;
        t -= a.tile0[p];
        m = t % a.mt[p];
        n = t / a.mt[p];
    };

    if (warp == 0)
    {
        // (this loop and the MMA's run a stage in few instructions, without divisions: at 256 columns a stage takes about 500 cycles)
        Ring r(NST);
        const uint32_t full0 = map_rank(smem_u32(&full[0]), 0), smem0 = smem_u32(smem), bytes = (uint32_t) (2 * STAGE);
        const int bk = a.bk, nseg = a.nseg;
        for (int t = first; t < ntiles && !s_abort; t += pairs)
        {
            int p, m, n;
            find(t, p, m, n);
            const int m0 = m * 2 * PAIR_BM + (int) rank * PAIR_BM;
            const int n0 = EPI == EPI_GATED ? n * (BN / 2) : n * BN + (int) rank * (BN / 2);
            for (int seg = 0; seg < nseg && !s_abort; ++seg)
            {
                const int mp = nseg > 1 ? seg : p;
                const CUtensorMap* ma = &maps.a[mp];
                // GATED: gate columns from CTA 0, the same up columns from CTA 1
                const CUtensorMap* mb = &maps.b[EPI == EPI_GATED ? (int) rank : mp];
                for (int k = 0, kc = 0; k < ksteps; ++k, kc += bk)
                {
                    if (!ring_wait(&empty[r.s], r.ph ^ 1u)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_EMPTY); s_abort = 1; break; }
                    const uint32_t sa = smem0 + (uint32_t) (r.s * STAGE), sb = sa + PAIR_BM * 128, bar = full0 + 8u * r.s;
                    if (elect_one())
                    {
                        // the pair's four half tiles are counted on the leader's barrier
                        if (rank == 0) mbar_arrive_expect_tx(&full[r.s], bytes);
                        if constexpr (A_MN)
                        {
                            tma_load_pair(sa, ma, m0, kc, bar);
                            tma_load_pair(sa + 8192, ma, m0 + 64, kc, bar);
                        }
                        else
                            tma_load_pair(sa, ma, kc, m0, bar);
                        if constexpr (B_MN)
                        {
                            tma_load_pair(sb, mb, n0, kc, bar);
                            if (BN > 128) tma_load_pair(sb + 8192, mb, n0 + 64, kc, bar);
                        }
                        else
                            tma_load_pair(sb, mb, kc, n0, bar);
                    }
                    __syncwarp();
                    r.next();
                }
            }
        }
        // the last arrivals on this CTA's barriers come from the pair's leader: they are in before it may exit
        for (int i = 0; i < NST && !s_abort; ++i, r.next())
            if (!ring_wait(&empty[r.s], r.ph ^ 1u)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_EMPTY); s_abort = 1; }
    }
    else if (warp == 1)
    {
        if (rank == 0)
        {
            Ring r(NST);
            int lt = 0;
            const uint64_t da0 = desc_sw128(smem_u32(smem), 8192), db0 = desc_sw128(smem_u32(smem) + PAIR_BM * 128, 8192);
            const uint32_t idesc = a.idesc;
            for (int t = first; t < ntiles && !s_abort; t += pairs, ++lt)
            {
                const int acc = lt & 1;
                const uint32_t d = tmem + (uint32_t) (acc * 256);
                if (!ring_wait(&tempty[acc], (uint32_t) ((lt >> 1) & 1) ^ 1u)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_EMPTY); s_abort = 1; break; }
                tc_after();
                for (int k = 0; k < nk; ++k)
                {
                    if (!ring_wait(&full[r.s], r.ph)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_FULL); s_abort = 1; break; }
                    tc_after();
                    // descriptors count 16-byte units: a stage, and 32 bytes of K (16 rows of an MN-major tile) per instruction
                    const uint64_t off = (uint64_t) (uint32_t) (r.s * STAGE >> 4);
                    if (elect_one())
                    {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            tc_mma<I8, 2>(d, da0 + off + kk * (A_MN ? 128 : 2), db0 + off + kk * (B_MN ? 128 : 2), idesc, (k | kk) != 0);
                        tc_commit<2>(&empty[r.s]);
                        if (k == nk - 1) tc_commit<2>(&tfull[acc]);
                    }
                    __syncwarp();
                    r.next();
                }
            }
        }
    }
    else
    {
        const int q = warp & 3, half = (warp - 2) >> 2;
        uint4* stg = reinterpret_cast<uint4*>(smem + (size_t) NST * STAGE) + (warp - 2) * 256;   // 4 KB: 32 rows of 128 bytes
        int lt = 0;
        for (int t = first; t < ntiles && !s_abort; t += pairs, ++lt)
        {
            const int acc = lt & 1;
            int p, m, n;
            find(t, p, m, n);
            if (!warp_wait(&tfull[acc], (uint32_t) ((lt >> 1) & 1))) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_FULL); s_abort = 1; break; }
            tc_after();
            const Epi e = a.e[p];       // in registers: the stores in between would have it read again
            const uint32_t tq = tmem + ((uint32_t) (32 * q) << 16) + (uint32_t) (acc * 256);
            const bool staged = EPI == EPI_I8 || (EPI == EPI_STORE && !e.accumulate);
            if (staged)
            {
                // whole rows of 128 bytes (64 or 32 columns) into the staging tile, from there by TMA, or row by row where the
                // output's rows are not 16-byte aligned
                const int row0 = m * 2 * PAIR_BM + (int) rank * PAIR_BM + 32 * q;
                const bool f32 = e.y_dtype == GLMX_F32, bf = e.y_dtype == GLMX_BF16;
                const float xs = EPI == EPI_I8 && row0 + lane < e.M ? e.xs[row0 + lane] : 0.0f;
                const int wide = f32 ? 32 : 64;
                for (int c = half * wide; c < BN; c += 2 * wide)
                {
                    const int n0 = n * BN + c;
                    if (lane == 0) tma_store_read();                   // the tile before has been read
                    __syncwarp();
                    // 32 columns a wait: all 64 at once take the registers that the 8-bit epilogue needs
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        if (f32 && h) break;
                        uint32_t v[2][16];
                        tc_ld16(tq + (uint32_t) (c + 32 * h), v[0]);
                        tc_ld16(tq + (uint32_t) (c + 32 * h + 16), v[1]);
                        tc_wait_ld();
#pragma unroll
                        for (int d = 0; d < 2; ++d)
                        {
                            if constexpr (EPI == EPI_I8)
                            {
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                {
                                    const int col = min(n0 + 32 * h + 16 * d + i, e.N - 1);
                                    float f = (float) (int) v[d][i] * (xs * __ldg(e.ws + col));
                                    if (e.bias) f += __ldg(e.bias + col);
                                    v[d][i] = __float_as_uint(f);
                                }
                            }
                            if (f32)
                            {
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    stg[lane * 8 + ((4 * d + i) ^ (lane & 7))] = make_uint4(v[d][4 * i], v[d][4 * i + 1], v[d][4 * i + 2], v[d][4 * i + 3]);
                            }
                            else
                            {
                                uint32_t w[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) w[i] = pack16(__uint_as_float(v[d][2 * i]), __uint_as_float(v[d][2 * i + 1]), bf);
#pragma unroll
                                for (int i = 0; i < 2; ++i) stg[lane * 8 + ((4 * h + 2 * d + i) ^ (lane & 7))] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (!e.vec)
                    {
                        copy_rows(e, stg, row0, n0, wide, lane);
                        __syncwarp();
                    }
                    else if (lane == 0 && row0 < e.M && n0 < e.N) tma_store_2d(&maps.y[p], n0, row0, smem_u32(stg));
                }
            }
            if constexpr (EPI != EPI_I8)
                if (!staged)
                {
                    // this warp's half of the tile's columns, 32 at a time (GATED: 16 of gate and of up): a lane holds a row, and through shared memory
                    // each 8 (4) lanes get 4 columns each of one row, so that global accesses run along rows
                    const int cols = EPI == EPI_GATED ? BN / 4 : BN / 2, c0 = half * cols;
                    constexpr int CC = EPI == EPI_GATED ? 16 : 32, LPR = CC / 4;
                    for (int c = c0; c < c0 + cols; c += CC)
                    {
                        uint32_t v[16], u[16];
                        tc_ld16(tq + (uint32_t) c, v);
                        tc_ld16(tq + (uint32_t) (EPI == EPI_GATED ? BN / 2 + c : c + 16), u);
                        tc_wait_ld();
                        // 16-byte piece i of row r sits at place i ^ (r & 7)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                        {
                            stg[lane * 8 + (i ^ (lane & 7))] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                            stg[lane * 8 + ((i + 4) ^ (lane & 7))] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
                        }
                        __syncwarp();
                        const int nn = n * (EPI == EPI_GATED ? BN / 2 : BN) + c, row0 = m * 2 * PAIR_BM + (int) rank * PAIR_BM + 32 * q;
#pragma unroll
                        for (int i = 0; i < LPR; ++i)
                        {
                            const int r = i * (32 / LPR) + lane / LPR, pc = lane % LPR;
                            const uint4 x = stg[r * 8 + (pc ^ (r & 7))], y = EPI == EPI_GATED ? stg[r * 8 + ((pc + 4) ^ (r & 7))] : x;
                            const uint32_t x4[4] = { x.x, x.y, x.z, x.w }, y4[4] = { y.x, y.y, y.z, y.w };
                            if constexpr (EPI == EPI_GATED) emit_gated(e, row0 + r, nn + 4 * pc, x4, y4);
                            else emit<EPI, 4>(e, row0 + r, nn + 4 * pc, x4);
                        }
                        __syncwarp();
                    }
                }
            tc_before();
            __syncwarp();
            if (lane == 0) arrive_remote(map_rank(smem_u32(&tempty[acc]), 0));
        }
        if (lane == 0) tma_store_done();
    }
    __syncwarp();
    if (s_abort) drain_pause();
    tc_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1)
    {
        tc_after();
        tc_dealloc<2>(tmem, 512);
    }
}

// ---- cols_kernel -------------------------------------------------------------------------------------------------------

template <int N> struct Int { static constexpr int value = N; };

struct ColsMaps
{
    CUtensorMap w[2], x[2];     // weights (GATED: gate, up; two segments: one each) and tokens
};

struct ColsArgs
{
    int nseg, K, bk;
    int NT;                     // tokens per tile: a multiple of 16, at most 256
    int xrows;                  // rows of a token box: NT, or all tokens where there are fewer (the MMA's other columns are not read, and
                                // rows outside of the matrix would cost the copy more than others do)
    int stages;
    int mtiles;                 // weight-row tiles; the grid is [splits][mtiles * token tiles]
    int tcols;                  // tensor-memory columns: a power of 2 >= NT, at least 32
    int prefetch;               // weights may be read before the kernels in front have finished
    uint32_t idesc;
    int* err;
    Epi e;
};

constexpr int COLS_THREADS = 192;
constexpr int COLS_STAGES_MAX = 12;
constexpr int COLS_L2_AHEAD = 16;                        // stages: 37 MB from 144 CTAs

template <bool I8, bool W_MN, int EPI>
__global__ void __launch_bounds__(COLS_THREADS, 2) cols_kernel(const __grid_constant__ ColsMaps maps, const __grid_constant__ ColsArgs a)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[COLS_STAGES_MAX], empty[COLS_STAGES_MAX], tfull;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_abort;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int splits = gridDim.x, split = blockIdx.x;      // one cluster along x
    const int mtile = blockIdx.y % a.mtiles, ttile = blockIdx.y / a.mtiles;
    const int NT = a.NT, NST = a.stages, STAGE = 16384 + NT * 128;
    const int ksteps = (a.K + a.bk - 1) / a.bk, nk_all = ksteps * a.nseg;
    const int k0 = (int) ((long long) nk_all * split / splits), nk = (int) ((long long) nk_all * (split + 1) / splits) - k0;
    const int rows = EPI == EPI_GATED ? 64 : 128;          // output columns (weight rows of one matrix) per tile
    const uint32_t tx = 16384u + (uint32_t) a.xrows * 128;
    // next stage to load: segment and place in it
    int seg = k0 / ksteps, kc = (k0 - seg * ksteps) * a.bk;
    const int kend = ksteps * a.bk;
    auto step = [&](int& sg, int& c) {
        c += a.bk;
        if (c == kend) { c = 0; ++sg; }
    };
    auto load_w = [&](int s, int sg, int c) {
        uint8_t* sw = smem + (size_t) s * STAGE;
        mbar_arrive_expect_tx(&full[s], tx);
        if constexpr (EPI == EPI_GATED)
            for (int j = 0; j < 2; ++j) tma_load_2d(sw + j * 8192, &maps.w[j], c, mtile * 64, &full[s]);
        else if constexpr (W_MN)
            for (int j = 0; j < 2; ++j) tma_load_2d(sw + j * 8192, &maps.w[sg], mtile * 128 + 64 * j, c, &full[s]);
        else
            tma_load_2d(sw, &maps.w[sg], c, mtile * 128, &full[s]);
    };
    auto load_x = [&](int s, int sg, int c) { tma_load_2d(smem + (size_t) s * STAGE + 16384, &maps.x[sg], c, ttile * NT, &full[s]); };
    const int ahead = nk < NST ? nk : NST;                 // stages that need no wait
    if (warp == 0)
    {
        if (lane < NST) { mbar_init(&full[lane], 1); mbar_init(&empty[lane], 1); }
        if (lane == COLS_STAGES_MAX) { mbar_init(&tfull, 1); s_abort = 0; }
        fence_barrier_init();
        __syncwarp();
    }
    else if (warp == 2 && lane == 0)
    {
        prefetch_map(&maps.w[0]);
        prefetch_map(&maps.x[0]);
        if (EPI == EPI_GATED) prefetch_map(&maps.w[1]);
        // the weights that this CTA has to wait with go to L2 meanwhile: their stream runs while the kernels in front finish (one token
        // through H = 6144, I = 1536 19.2 -> 17.9 us; a chain of 8-bit products lost by it, 11.3 -> 12.6 us)
        const int from = a.prefetch ? ahead : 0, to = I8 ? 0 : min(nk, from + COLS_L2_AHEAD);
        int sg = seg, c = kc;
        for (int i = 0; i < to; ++i, step(sg, c))
        {
            if (i < from) continue;
            if constexpr (EPI == EPI_GATED)
                for (int j = 0; j < 2; ++j) prefetch_2d(&maps.w[j], c, mtile * 64);
            else if constexpr (W_MN)
                for (int j = 0; j < 2; ++j) prefetch_2d(&maps.w[sg], mtile * 128 + 64 * j, c);
            else
                prefetch_2d(&maps.w[sg], c, mtile * 128);
        }
    }
    if (tid == 0)
    {
        // the first loads do not wait for the rest of the CTA
        if (!a.prefetch) grid_wait();
        for (int i = 0, sg = seg, c = kc; i < ahead; ++i, step(sg, c)) load_w(i, sg, c);
        if (a.prefetch) grid_wait();
        for (int i = 0; i < ahead; ++i, step(seg, kc)) load_x(i, seg, kc);
    }
    if (warp == 1) tc_alloc<1>(&tmem_slot, (uint32_t) a.tcols);
    __syncwarp();
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_slot;
    grid_release();                                        // (thread 0 has waited for the kernels in front)

    if (warp == 0)
    {
        // lane 0's segment and place after the first loads
        seg = __shfl_sync(0xffffffffu, seg, 0);
        kc = __shfl_sync(0xffffffffu, kc, 0);
        Ring r(NST);
        r.ph = 1;                                          // the ring's second round
        for (int i = ahead; i < nk; ++i, step(seg, kc), r.next())
        {
            if (!ring_wait(&empty[r.s], r.ph ^ 1u)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_EMPTY); s_abort = 1; break; }
            if (elect_one())
            {
                load_w(r.s, seg, kc);
                load_x(r.s, seg, kc);
            }
            __syncwarp();
        }
    }
    else if (warp == 1)
    {
        grid_wait();
        Ring r(NST);
        const uint64_t dw0 = desc_sw128(smem_u32(smem), 8192), dx0 = desc_sw128(smem_u32(smem) + 16384, 8192);
        const uint32_t idesc = a.idesc;
        for (int i = 0; i < nk; ++i, r.next())
        {
            if (!ring_wait(&full[r.s], r.ph)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_FULL); s_abort = 1; break; }
            tc_after();
            const uint64_t off = (uint64_t) (uint32_t) (r.s * STAGE >> 4);
            if (elect_one())
            {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) tc_mma<I8, 1>(tmem, dw0 + off + kk * (W_MN ? 128 : 2), dx0 + off + kk * 2, idesc, (i | kk) != 0);
                tc_commit<1>(&empty[r.s]);
                if (i == nk - 1) tc_commit<1>(&tfull);
            }
            __syncwarp();
        }
    }
    __syncwarp();
    grid_wait();
    // every load has been multiplied: the partial tile [token][weight row] takes the ring's place
    if (warp >= 2 && !warp_wait(&tfull, 0)) { if (lane == 0) atomicOr(a.err, ERR_TIMEOUT_FULL); s_abort = 1; }
    if (s_abort) drain_pause();
    __syncthreads();
    tc_after();
    float* part = reinterpret_cast<float*>(smem);
    const int ncols = min(NT, a.e.M - ttile * NT);         // tokens of the tile that exist
    if (warp >= 2 && !s_abort)
    {
        const int q = warp & 3;
        const uint32_t tq = tmem + ((uint32_t) (32 * q) << 16);
        for (int c = 0; c < ncols; c += 16)
        {
            uint32_t v[16];
            tc_ld16(tq + (uint32_t) c, v);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) part[(c + i) * 128 + 32 * q + lane] = __uint_as_float(v[i]);
        }
    }
    tc_before();
    if (splits > 1) cluster_sync(); else __syncthreads();
    if (warp == 1)
    {
        tc_after();
        tc_dealloc<1>(tmem, (uint32_t) a.tcols);
    }
    // Spread over the cluster's CTAs: units of 4 weight rows of one token (or, where the output's rows take no wide stores, of single ones).
    // A unit's partials are fetched from all CTAs at once and added in rank order.
    const uint32_t base = smem_u32(part);
    auto join = [&](auto wide) {
        constexpr int W = decltype(wide)::value;
        const int per = rows / W, units = ncols * per;
        const int u0 = (int) ((long long) units * split / splits), u1 = (int) ((long long) units * (split + 1) / splits);
        // consecutive units in consecutive lanes; in different warps where a warp's units may have sums to form again, one after the other
        const int place = EPI == EPI_GATED && a.e.p && a.e.limit != 0.0f ? lane * (COLS_THREADS / 32) + warp : tid;
        for (int ub = u0; ub < u1; ub += COLS_THREADS)
        {
            // (whole warps stay together: the last ones' lanes past the end work on the last unit and drop it)
            const int u = min(ub + place, u1 - 1);
            const bool mine = ub + place < u1;
            const int c = u / per, r = (u - c * per) * W;
            uint32_t v[W];
            auto sum = [&](uint32_t (&d)[W], uint32_t off) {
                uint32_t x[8][W];
#pragma unroll
                for (int rk = 0; rk < 8; ++rk)
                    if (rk < splits)
                    {
                        const uint32_t at = map_rank(base + off, (uint32_t) rk);
                        if constexpr (W == 4) asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[rk][0]), "=r"(x[rk][1]), "=r"(x[rk][2]), "=r"(x[rk][3]) : "r"(at));
                        else asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x[rk][0]) : "r"(at));
                    }
#pragma unroll
                for (int i = 0; i < W; ++i) d[i] = x[0][i];
#pragma unroll
                for (int rk = 1; rk < 8; ++rk)
                    if (rk < splits)
#pragma unroll
                        for (int i = 0; i < W; ++i) d[i] = I8 ? d[i] + x[rk][i] : __float_as_uint(__fadd_rn(__uint_as_float(d[i]), __uint_as_float(x[rk][i])));
            };
            sum(v, (uint32_t) (c * 128 + r) * 4);
            const int t = mine ? ttile * NT + c : a.e.M;
            if constexpr (EPI == EPI_GATED)
            {
                uint32_t w[W];
                sum(w, (uint32_t) (c * 128 + 64 + r) * 4);
                emit_gated(a.e, t, mtile * rows + r, v, w);
            }
            else
                emit<EPI, W>(a.e, t, mtile * rows + r, v);
        }
    };
    if (!s_abort)
    {
        if constexpr (EPI == EPI_I8)
        {
            if (a.e.vec) join(Int<4>()); else join(Int<1>());
        }
        else
            join(Int<4>());
    }
    __syncwarp();
    if (splits > 1) cluster_sync();                        // nobody leaves while its partial tile is read
}

// ---- host ----------------------------------------------------------------------------------------------------------------

// a row-major matrix operand: [rows][inner], rows `pitch` elements apart
struct Mat
{
    const void* p;
    long long rows, inner, pitch;
};

// tensor map of boxes of box_inner x box_rows elements with the 128-byte swizzle
cudaError_t dense_map(CUtensorMap* m, int dtype, const Mat& t, int box_inner, int box_rows);
cudaError_t dense_err_ptr(int** p);          // the current device's error word

// One product of the launch: sums over segs (A: tokens, B: weights; GATED: B of seg 0 and 1 are gate and up)
struct Product
{
    Mat a[2], b[2];
    Epi e;
};

template <bool I8, bool A_MN, bool B_MN, int EPI>
cudaError_t launch_pair(int dtype, int nprob, const Product* pr, int nseg, int K, int BN, cudaStream_t st)
{
    auto kernel = pair_kernel<I8, A_MN, B_MN, EPI>;
    const int dev = dense_device();
    static PerDevice<int> smem;
    cudaError_t err = dense_smem(smem, dev, reinterpret_cast<const void*>(kernel), PAIR_SMEM - 1024);
    if (err != cudaSuccess) return err;
    PairMaps maps;
    PairArgs a{};
    a.nprob = nprob; a.nseg = nseg; a.K = K; a.bk = I8 ? 128 : 64; a.BN = BN;
    a.idesc = tc_idesc(I8, dtype == GLMX_BF16, A_MN, B_MN, 256, BN);
    if ((err = dense_err_ptr(&a.err)) != cudaSuccess) return err;
    const int width = EPI == EPI_GATED ? BN / 2 : BN;
    for (int i = 0; i < nprob; ++i)
    {
        a.e[i] = pr[i].e;
        const Epi& e = pr[i].e;
        if (EPI == EPI_STORE || EPI == EPI_I8)
        {
            if (e.vec && !e.accumulate)
                if ((err = dense_map(&maps.y[i], e.y_dtype, Mat{ e.y, e.M, e.N, e.ldy }, e.y_dtype == GLMX_F32 ? 32 : 64, 32)) != cudaSuccess) return err;
        }
        a.mt[i] = (pr[i].e.M + 255) / 256;
        a.nt[i] = (pr[i].e.N + width - 1) / width;
        a.tile0[i + 1] = a.tile0[i] + a.mt[i] * a.nt[i];
    }
    for (int i = 0; i < (nprob > 1 ? nprob : nseg); ++i)
    {
        const Mat& ma = nprob > 1 ? pr[i].a[0] : pr[0].a[i];
        if ((err = dense_map(&maps.a[i], dtype, ma, A_MN ? 64 : a.bk, A_MN ? 64 : PAIR_BM)) != cudaSuccess) return err;
    }
    for (int i = 0; i < (EPI == EPI_GATED ? 2 : nprob > 1 ? nprob : nseg); ++i)
    {
        const Mat& mb = nprob > 1 ? pr[i].b[0] : pr[0].b[i];
        if ((err = dense_map(&maps.b[i], dtype, mb, B_MN ? 64 : a.bk, B_MN ? 64 : BN / 2)) != cudaSuccess) return err;
    }
    const int tiles = a.tile0[nprob], pairs = dense_sms(dev) / 2;
    return launch_chained(kernel, dim3(2 * (tiles < pairs ? tiles : pairs)), dim3(PAIR_THREADS), (size_t) pair_smem(BN), st, maps, a);
}

// Microseconds of a launch by a simple model of what was measured on a B200; the kernel and its tiling are those of the least.
//   pair_kernel: rounds of tiles over the pairs, each stage (128 bytes of K) 0.345 us at 256 columns, 0.27 at 192, 0.20 at 128, 0.16 at 64
//     (the loads of A then bind) or its share of the weights' stream from memory, a round at least the epilogue of a tile, plus the
//     start and the last tile's epilogue.
//   cols_kernel: rounds of clusters, each CTA 3.4 us and 0.018 per token column (start, join) plus its stages on the tensor
//     cores; or the stream of all tiles' weights from memory (5.9 TB/s from 130 CTAs on), or of all stages from L2 (9 TB/s).
// E.g. (measured, us, cols / pair 64 / 128 / 256): feed-forward at H = 6144, I = 1536 of 1 row 18 / 54 / 38 / 45, of 200 rows 29 / 33
// / 31 / 48, of 512 48 / 53 / 37 / 49, of 4096 263 / 272 / 184 / 163; int8 1024 x 1024 of 48 rows 4.6 / 5.8 / 6.4 / 8.8, of 512 9.5
// / 5.8 / 6.7 / 9.3.
struct PairPlan
{
    int BN;
    double us;
};

inline PairPlan pair_plan(int nprob, const Epi* e, bool gated, bool kmajor, int nk, int sms)
{
    PairPlan best{ 256, 1e30 };
    for (int BN = 256; BN >= 64; BN -= 64)
    {
        if (BN % 128 && !kmajor) continue;                 // MN-major boxes are 64 columns, two halves of a tile
        long long tiles = 0;
        const int width = gated ? BN / 2 : BN;
        for (int i = 0; i < nprob; ++i) tiles += (long long) ((e[i].M + 255) / 256) * ((e[i].N + width - 1) / width);
        const double rounds = (double) ((tiles + sms / 2 - 1) / (sms / 2));
        double step = BN == 256 ? 0.345 : BN == 192 ? 0.27 : BN == 128 ? 0.20 : 0.16;
        const double active = (double) (tiles < sms / 2 ? tiles : sms / 2), stream = active * BN * 128 / ((e[0].M + 255) / 256) / 5.4e6;
        if (nprob == 1 && stream > step) step = stream;
        const double main = nk * step, drain = BN == 256 ? 2.6 : BN == 192 ? 2.4 : BN == 128 ? 2.0 : 1.2;
        const double us = (BN == 256 ? 6.6 : BN == 192 ? 6.0 : BN == 128 ? 5.2 : 4.4) + rounds * (main > drain ? main : drain);
        if (us < best.us - 1e-9) best = { BN, us };
    }
    return best;
}

struct ColsPlan
{
    int NT, ttiles, mtiles, splits, stages;
    double us;
};

constexpr int COLS_SMEM2 = 112 * 1024, COLS_SMEM1 = 224 * 1024;   // two CTAs an SM (tiles of up to 64 tokens), or one

// clusters of each size that the device holds at once, for either shared memory size
struct ColsCapacity
{
    int n[2][9];
};

// Tokens per tile: all of them up to 256, else equal tiles. Splits of K: at most 8 (the portable cluster size), each CTA with at least
// two stages.
inline ColsPlan cols_plan(int M, int N, bool gated, int nk, const ColsCapacity& cap)
{
    ColsPlan p;
    p.ttiles = (M + 255) / 256;
    p.NT = ((M + p.ttiles - 1) / p.ttiles + 15) / 16 * 16;
    p.mtiles = (N + (gated ? 63 : 127)) / (gated ? 64 : 128);
    const int stage = 16384 + p.NT * 128, one = p.NT <= 64 ? 0 : 1;
    const long long tiles = (long long) p.ttiles * p.mtiles;
    p.splits = 1;
    p.us = 1e30;
    for (int s = 1; s <= 8 && (s == 1 || 2 * s <= nk) && tiles <= 65535; ++s)   // (tiles are the grid's y dimension)
    {
        const int room = cap.n[one][s];
        if (room < 1) continue;
        const double ctas = (double) (tiles < room ? tiles : room) * s;              // at once
        const double rounds = (double) ((tiles + room - 1) / room), own = 3.4 + 0.018 * p.NT;
        const double tc = rounds * (own + (double) ((nk + s - 1) / s) * (0.2 + 0.0016 * p.NT));
        const double hbm = own + (double) p.mtiles * nk * 16384 / (5.9e6 * (ctas < 130 ? ctas / 130 : 1.0)), l2 = own + (double) tiles * nk * stage / 9.0e6;
        const double most = tc > hbm ? tc : hbm, us = (most > l2 ? most : l2) + 0.02 * s;
        if (us < p.us - 1e-9) { p.us = us; p.splits = s; }
    }
    const int room = one ? COLS_SMEM1 : COLS_SMEM2, per = (nk + p.splits - 1) / p.splits;
    p.stages = (room - 2048) / stage;
    if (p.stages > COLS_STAGES_MAX) p.stages = COLS_STAGES_MAX;
    const int part = (p.NT * 512 + stage - 1) / stage;     // the partial tile takes the ring's place
    if (p.stages > per) p.stages = per;
    if (p.stages < part) p.stages = part;
    return p;
}

inline int cols_tmem(const ColsPlan& p)
{
    int n = 32;
    while (n < p.NT) n *= 2;
    return n;
}

inline int cols_smem(const ColsPlan& p) { return tmem_smem(cols_tmem(p), 1024 + p.stages * (16384 + p.NT * 128)); }

template <bool I8, bool W_MN, int EPI>
cudaError_t cols_capacity(int dev, const ColsCapacity** out)
{
    static PerDevice<ColsCapacity> capacity;
    return capacity.get(dev, out, [](ColsCapacity& cap) {
        auto kernel = cols_kernel<I8, W_MN, EPI>;
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, COLS_SMEM1);
        if (err == cudaSuccess)
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        for (int s = 1; s <= 8 && err == cudaSuccess; ++s)
        {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(s, 1024);
            cfg.blockDim = dim3(COLS_THREADS);
            cfg.dynamicSmemBytes = COLS_SMEM1;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = s; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            err = cudaOccupancyMaxActiveClusters(&cap.n[1][s], kernel, &cfg);
            // the occupancy calculator counts one CTA an SM for every kernel that allocates tensor memory; two of the smaller kind do
            // run at once (seen by their clocks and SM numbers)
            cap.n[0][s] = 2 * cap.n[1][s];
        }
        return err;
    });
}

template <bool I8, bool W_MN, int EPI>
cudaError_t launch_cols(int dtype, const Product& pr, int nseg, int K, const ColsPlan& p, bool prefetch, cudaStream_t st)
{
    auto kernel = cols_kernel<I8, W_MN, EPI>;
    cudaError_t err;
    ColsMaps maps;
    ColsArgs a{};
    a.nseg = nseg; a.K = K; a.bk = I8 ? 128 : 64;
    a.NT = p.NT; a.xrows = pr.e.M < p.NT ? pr.e.M : p.NT; a.stages = p.stages; a.mtiles = p.mtiles; a.prefetch = prefetch;
    a.tcols = cols_tmem(p);
    a.idesc = tc_idesc(I8, dtype == GLMX_BF16, W_MN, false, 128, p.NT);
    if ((err = dense_err_ptr(&a.err)) != cudaSuccess) return err;
    a.e = pr.e;
    for (int i = 0; i < (EPI == EPI_GATED ? 2 : nseg); ++i)
        if ((err = dense_map(&maps.w[i], dtype, pr.b[i], W_MN ? 64 : a.bk, W_MN || EPI == EPI_GATED ? 64 : 128)) != cudaSuccess) return err;
    for (int i = 0; i < nseg; ++i)
        if ((err = dense_map(&maps.x[i], dtype, pr.a[i], a.bk, a.xrows)) != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits, p.mtiles * p.ttiles);
    cfg.blockDim = dim3(COLS_THREADS);
    cfg.dynamicSmemBytes = cols_smem(p);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, maps, a);
}

// One product by the kernel and tiling of the least modelled time.
template <bool I8, bool W_MN, int EPI>
cudaError_t launch_product(int dtype, const Product& pr, int nseg, int K, bool prefetch, cudaStream_t st)
{
    const int dev = dense_device();
    const int nk = nseg * ((K + (I8 ? 127 : 63)) / (I8 ? 128 : 64)), sms = dense_sms(dev);
    const ColsCapacity* cap;
    const cudaError_t err = cols_capacity<I8, W_MN, EPI>(dev, &cap);
    if (err != cudaSuccess) return err;
    const ColsPlan c = cols_plan(pr.e.M, pr.e.N, EPI == EPI_GATED, nk, *cap);
    const PairPlan p = pair_plan(1, &pr.e, EPI == EPI_GATED, !W_MN, nk, sms);
    if (c.us <= p.us) return launch_cols<I8, W_MN, EPI>(dtype, pr, nseg, K, c, prefetch, st);
    return launch_pair<I8, false, W_MN, EPI>(dtype, 1, &pr, nseg, K, p.BN, st);
}

}  // namespace glmx
