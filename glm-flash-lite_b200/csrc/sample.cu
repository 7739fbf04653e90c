// Sampling (glmx_sample), simple form: one CTA per row, the row read again in each pass.
//
// A weight is w = exp((l - m) / T) <= 1 in fp32, held as the integer floor(w * 2^44): sums of up to 2^19 weights fit 64 bits
// and do not depend on their order. Equal logits have equal weights, so each filter is a threshold on the logits' order-preserving
// 32-bit key plus a number of kept ties, the lowest ids first:
//   top-k: the key with count(>) < k <= count(>=), by four 8-bit digits of a radix selection;
//   top-p: the key with mass(>) < top_p * S <= mass(>=), the same with sums of weights;
// then the pick is the lowest id at which the running sum of kept weights exceeds floor(u * S).
#include "dense.h"

namespace glmx {

namespace {

struct SampleArgs
{
    const void* logits; long long ld; int V;
    const float* u; const float* temperature; float temperature0; const int* top_k; int top_k0;
    const float* top_p; float top_p0; const float* min_p; float min_p0;
    void* ids; int ids64;
};

constexpr int ST = 1024;
constexpr uint32_t KEY_NONE = 0x007fffffu;                 // key of -inf, and of NaN: never picked

__device__ __forceinline__ uint32_t key_of(float l)
{
    if (l != l) return KEY_NONE;
    const uint32_t b = __float_as_uint(l + 0.0f);          // -0 counts as +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Weight
{
    float m, ch, cl;                                       // row maximum, log2(e) / T as hi + lo
    __device__ __forceinline__ void init(float max, float T)
    {
        m = max;
        const double c = 1.4426950408889634 / (double) T;
        ch = (float) fmin(c, 3e38);
        cl = c < 3e38 ? (float) (c - (double) ch) : 0.0f;
    }
    // floor(2^44 exp((l - m) / T)): l - m with its rounding error (two-sum), scaled to a power of 2 in hi + lo, the power
    // split into an integer and |f| <= 1/2, 2^f by its Taylor series in f ln 2 (0.347^8 / 8! = 5e-9)
    __device__ __forceinline__ unsigned long long operator()(uint32_t key) const
    {
        if (key <= KEY_NONE) return 0;
        const float l = of_key(key);
        if (l == m) return 1ull << 44;
        const float d = l - m, bb = d - l, derr = (l - (d - bb)) + (-m - bb);
        const float x = d * ch;
        if (!(x > -46.0f)) return 0;
        const float lo = fmaf(d, ch, -x) + fmaf(d, cl, derr * ch);
        const float n = rintf(x), f = ((x - n) + lo) * 0.693147180559945f;
        float e = fmaf(f, 1.0f / 5040, 1.0f / 720);
        e = fmaf(e, f, 1.0f / 120); e = fmaf(e, f, 1.0f / 24); e = fmaf(e, f, 1.0f / 6); e = fmaf(e, f, 0.5f);
        e = fmaf(e, f, 1.0f); e = fmaf(e, f, 1.0f);
        const unsigned long long w = (unsigned long long) __float2uint_rd(e * 16777216.0f);
        const int sh = 20 + (int) n;
        return sh >= 0 ? w << sh : w >> -sh;
    }
};

template <typename V>
__device__ V block_sum(V v, V* s)                          // over ST threads; s: 33 entries
{
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    V t = 0;
    for (int i = 0; i < ST / 32; ++i) t += s[i];
    __syncthreads();
    return t;
}

// lowest index whose running sum of weight(index) exceeds target; V where none does. Each warp sums a run of the row, the warp
// in whose run the target falls walks it again.
template <typename F>
__device__ int ordered_find(int V, unsigned long long target, F weight, unsigned long long* s, int* found)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int run = ((V + ST - 1) / ST) * 32, lo = min(V, warp * run), hi = min(V, lo + run);
    unsigned long long mine = 0;
    for (int i = lo + lane; i < hi; i += 32) mine += weight(i);
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) s[warp] = mine;
    if (threadIdx.x == 0) *found = V;
    __syncthreads();
    unsigned long long before = 0;
    for (int i = 0; i < warp; ++i) before += s[i];
    if (before <= target && before + mine > target)
        for (int i0 = lo; i0 < hi; i0 += 32)
        {
            unsigned long long c = i0 + lane < hi ? weight(i0 + lane) : 0;
            for (int o = 1; o < 32; o <<= 1)
            {
                const unsigned long long t = __shfl_up_sync(0xffffffffu, c, o);
                if (lane >= o) c += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, before + c > target);
            if (hit)
            {
                if (lane == 0) *found = i0 + __ffs(hit) - 1;
                break;
            }
            before += __shfl_sync(0xffffffffu, c, 31);
        }
    __syncthreads();
    return *found;
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_kernel(SampleArgs a)
{
    __shared__ unsigned long long hist[256], s64[33];
    __shared__ uint32_t s_key;
    __shared__ unsigned long long s_above;
    __shared__ int s_idx, s_found;
    const int b = blockIdx.x;
    const T* row = static_cast<const T*>(a.logits) + (size_t) b * a.ld;
    auto key = [&](int i) { return key_of(to_f32(row[i])); };
    auto put = [&](int id) {
        if (a.ids64) static_cast<long long*>(a.ids)[b] = id; else static_cast<int*>(a.ids)[b] = id;
    };
    // the largest key, then its lowest id
    uint32_t kmax = 0;
    for (int i = threadIdx.x; i < a.V; i += ST) kmax = max(kmax, key(i));
    if (threadIdx.x == 0) { s_key = 0; s_idx = a.V; }
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_key, kmax);
    __syncthreads();
    kmax = s_key;
    const float T0 = a.temperature ? a.temperature[b] : a.temperature0;
    if (kmax <= KEY_NONE)
    {
        if (threadIdx.x == 0) put(-1);
        return;
    }
    if (!(T0 > 0.0f))
    {
        for (int i = threadIdx.x; i < a.V; i += ST)
            if (key(i) == kmax) { atomicMin(&s_idx, i); break; }
        __syncthreads();
        if (threadIdx.x == 0) put(s_idx);
        return;
    }
    Weight weight;
    weight.init(of_key(kmax), T0);
    const int k = a.top_k ? a.top_k[b] : a.top_k0;
    const float top_p = a.top_p ? a.top_p[b] : a.top_p0;
    const float min_p = a.min_p ? a.min_p[b] : a.min_p0;
    // kept: key > thr, or key == thr and id <= cut
    uint32_t thr = KEY_NONE;
    int cut = a.V;
    auto kept = [&](uint32_t ky, int i) { return ky > thr || (ky == thr && i <= cut); };
    // the key at which the running sum (from the largest key) of f(key) over kept ids first reaches `need`; the sum above it in s_above
    auto select = [&](unsigned long long need, auto f) {
        uint32_t pre = 0;
        unsigned long long above = 0;
        for (int sh = 24; sh >= 0; sh -= 8)
        {
            for (int i = threadIdx.x; i < 256; i += ST) hist[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < a.V; i += ST)
            {
                const uint32_t ky = key(i);
                if ((sh == 24 || (ky >> (sh + 8)) == pre) && kept(ky, i)) atomicAdd(&hist[(ky >> sh) & 255], f(ky));
            }
            __syncthreads();
            if (threadIdx.x == 0)
            {
                int d = 255;
                unsigned long long c = above;
                while (d > 0 && c + hist[d] < need) c += hist[d--];
                s_key = (pre << 8) | d;
                s_above = c;
            }
            __syncthreads();
            pre = s_key;
            above = s_above;
            __syncthreads();
        }
        return pre;
    };
    // the first m ties at key t stay
    auto limit = [&](uint32_t t, unsigned long long m) {
        const int c = ordered_find(a.V, m - 1, [&](int i) { const uint32_t ky = key(i); return (unsigned long long) (ky == t && kept(ky, i)); }, s64, &s_found);
        thr = t;
        cut = c;
    };
    if (k > 0 && k < a.V)
    {
        const uint32_t t = select((unsigned long long) k, [](uint32_t) { return 1ull; });
        if (t > KEY_NONE) limit(t, (unsigned long long) k - s_above);
        __syncthreads();
    }
    if (top_p < 1.0f)
    {
        unsigned long long mine = 0;
        for (int i = threadIdx.x; i < a.V; i += ST)
        {
            const uint32_t ky = key(i);
            if (kept(ky, i)) mine += weight(ky);
        }
        const unsigned long long S = block_sum(mine, s64);
        // an id stays while the mass before it is below top_p * S: the first always
        unsigned long long need = top_p > 0.0f ? (unsigned long long) ceil((double) top_p * (double) S) : 1ull;
        if (need < 1) need = 1;
        const uint32_t t = select(need, weight);
        const unsigned long long w = weight(t);
        const unsigned long long m = w ? (need - s_above + w - 1) / w : 1ull;
        __syncthreads();
        limit(t, m);
    }
    const double mp = fmin((double) min_p, 1.0);
    const unsigned long long least = mp > 0.0 ? (unsigned long long) ceil(mp * 17592186044416.0) : 0ull;
    auto final_weight = [&](int i) {
        const uint32_t ky = key(i);
        const unsigned long long w = kept(ky, i) ? weight(ky) : 0ull;
        return w >= least ? w : 0ull;
    };
    unsigned long long mine = 0;
    for (int i = threadIdx.x; i < a.V; i += ST) mine += final_weight(i);
    const unsigned long long S = block_sum(mine, s64);
    const double u = fmin(fmax((double) a.u[b], 0.0), 1.0);
    unsigned long long target = (unsigned long long) (u * (double) S);
    if (target >= S) target = S - 1;
    const int id = ordered_find(a.V, target, final_weight, s64, &s_found);
    if (threadIdx.x == 0) put(id);
}

}  // namespace

}  // namespace glmx

using namespace glmx;

extern "C" int glmx_sample(const void* logits, int dtype, long long ld, int B, int V, const float* u, const float* temperature,
                           float temperature0, const int* top_k, int top_k0, const float* top_p, float top_p0,
                           const float* min_p, float min_p0, void* ids, int ids_dtype, void* stream)
{
    if (B < 0 || V < 1 || V > GLMX_SAMPLE_MAX_VOCAB || ld < V)
        return dense_fail(GLMX_E_ARG, "glmx_sample: B >= 0, 1 <= V <= GLMX_SAMPLE_MAX_VOCAB and ld >= V required");
    if (dtype != GLMX_F16 && dtype != GLMX_BF16 && dtype != GLMX_F32) return dense_fail(GLMX_E_ARG, "glmx_sample: logits must be fp16, bf16 or fp32");
    if (ids_dtype != GLMX_I32 && ids_dtype != GLMX_I64) return dense_fail(GLMX_E_ARG, "glmx_sample: ids must be int32 or int64");
    if (B == 0) return GLMX_OK;
    if (!logits || !u || !ids) return dense_fail(GLMX_E_ARG, "glmx_sample: null argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const SampleArgs a{ logits, ld, V, u, temperature, temperature0, top_k, top_k0, top_p, top_p0, min_p, min_p0, ids, ids_dtype == GLMX_I64 };
    if (dtype == GLMX_F32) sample_kernel<float><<<B, ST, 0, st>>>(a);
    else if (dtype == GLMX_F16) sample_kernel<__half><<<B, ST, 0, st>>>(a);
    else sample_kernel<__nv_bfloat16><<<B, ST, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_sample: launch");
}
