// Sampling (glmx_sample): one cluster of up to 8 CTAs per row, the row's logits held in their shared memory, so that global memory is
// read once and every further pass runs on chip. One row of 131072 logits is bound by the passes' latency (cluster barriers,
// block scans): 13 us in bf16 with all filters. A batch is bound by the passes over the rows that keep many tokens, about 35 us each:
// 64 rows of 150001 in fp32, some with each filter, 54 us (512 CTAs, of which 296 run at a time).
//
// A weight is w = exp((l - m) / T) <= 1 in fp32, held as the integer floor(w * 2^44): sums of up to 2^19 weights fit 64 bits
// and do not depend on their order. Equal logits have equal weights, so each filter is a threshold on the logits plus a
// number of kept ties, the lowest ids first:
//   top-k: the value with count(>) < k <= count(>=);  top-p: the value with mass(>) < top_p * S <= mass(>=);  min-p: a least weight.
// Few logits matter as a rule. The largest logit of each thread's share is known from the load: where k of these lie above a bin's
// edge, the top k logits do. What lies above is gathered (at most 512 logits, else the general way) and sorted in one
// CTA, which finishes the row; without a top-k the same is done where the gathered weights reach top_p.
// Otherwise the threshold is found by a histogram of 512 bins of m - l (for top-p of the interval of exponents in which it
// falls, known from the pass that sums the weights), whose bin is gathered and sorted or, where it holds more than 512 logits, narrowed by histograms over
// keys (order-preserving integers); and the pick by running sums over the row: the CTA, the warp, then the lane in whose
// run the target falls.
#include "dense.h"
#include "glmx_common.cuh"

#include <cstddef>

namespace glmx {

namespace {

typedef unsigned long long u64;

struct SampleArgs
{
    const void* logits; long long ld; int V, per;          // per: logits of a CTA's slice (a multiple of 8)
    const float* u; const float* temperature; float temperature0; const int* top_k; int top_k0;
    const float* top_p; float top_p0; const float* min_p; float min_p0;
    void* ids; int ids64;
    int ordered;                                           // the rows that may take long first
};

constexpr int ST = 512, SBINS = ST, SLIST = 512, SRANKS = 8;
constexpr int SLICE_MAX = GLMX_SAMPLE_MAX_VOCAB / SRANKS;  // 49152 logits: 192 KB
constexpr int NPV = 4;                                     // weights are also summed down to these exponents: a histogram then covers one interval
__device__ constexpr float PV[NPV + 1] = { 4.0f, 6.5f, 9.0f, 12.0f, 30.6f };   // (exp(-30.5) = 2^-44: what lies further down weighs nothing)
constexpr int TRY = 320;                                   // without a top-k: thread maxima above the gathered logits' edge

// order-preserving key of a logit that is not NaN; TS bits are the same in all values of the type
template <typename T> struct KeyShift { static constexpr int v = 0; };
template <> struct KeyShift<__nv_bfloat16> { static constexpr int v = 16; };
template <> struct KeyShift<__half> { static constexpr int v = 13; };
template <typename T>
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __float_as_uint(l);
    return (b & 0x80000000u ? ~b : b | 0x80000000u) >> KeyShift<T>::v;
}

// the logit of a key: the dropped bits are 0, in negative ones 1
template <typename T>
__device__ __forceinline__ float of_key(uint32_t k)
{
    const uint32_t full = k << KeyShift<T>::v;
    return __uint_as_float(full & 0x80000000u ? full & 0x7fffffffu : ~(full | ((1u << KeyShift<T>::v) - 1)));
}

struct Weight
{
    float h, c;                                            // -(row maximum) / 2, 2 log2(e) / T
    __device__ __forceinline__ void init(float max, float T)
    {
        h = -0.5f * max;
        // never 0, also where T is infinite: -inf * 0 would be NaN
        c = (float) fmax(fmin(2.8853900817779268 / (double) T, 3e38), 0x1p-149);
    }
    // floor(2^44 2^((l - m) / T log2(e))), of half the difference, which no two finite logits overflow. The exponent's three roundings
    // (the difference, the scale, their product) move a weight of 2^-x by x 2^-23 of itself, the exponential by 2^-22: no more than the last bits of
    // fp32 logits of that distance do. -inf gives 0 at every temperature
    __device__ __forceinline__ u64 operator()(float l) const
    {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(l, 0.5f, h) * c));
        return __float2ull_rd(e * 17592186044416.0f);
    }
};

struct alignas(16) Hist                                    // (cleared in 16-byte pieces)
{
    uint32_t lo[4][SBINS], hi[SBINS], cnt[SBINS];          // masses in two words (or counts in the low one), counts. Four copies of
                                                           // the low word: lanes that hit one bin meet less often
};

struct Found                                               // the bin in which a running sum reaches its need
{
    int bin;                                               // -1: nowhere
    u64 above, in;                                         // the sum above it and its own
    uint32_t cnt_in;
};

struct Shared
{
    u64 mail[2][NPV + 1][SRANKS];
    u64 part[NPV + 1][ST / 32];
    u64 warp[ST / 32], result;
    uint32_t warp32[ST / 32];
    u64 list[SLIST];                                       // (logit, id) of the gathered logits, in CTA 0
    uint32_t maxima[SBINS];                                // histogram of the threads' maxima
    union alignas(16)
    {
        Hist hist;
        struct { u64 sorted[SLIST]; uint32_t order[SLIST]; };
    };
    Found found;
    int n_list, id;
};

__device__ __forceinline__ uint32_t dsmem_map(const void* p, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
// the word at p in each of nc CTAs, all loads in flight at once
__device__ __forceinline__ void dsmem_ld_all(const uint32_t* p, int nc, uint32_t (&v)[SRANKS])
{
#pragma unroll
    for (int r = 0; r < SRANKS; ++r)
    {
        v[r] = 0;
        if (r < nc) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[r]) : "r"(dsmem_map(p, r)) : "memory");
    }
}
__device__ __forceinline__ uint32_t dsmem_add(const void* p, uint32_t rank, uint32_t v)
{
    uint32_t old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(dsmem_map(p, rank)), "r"(v) : "memory");
    return old;
}
__device__ __forceinline__ void dsmem_st(const void* p, uint32_t rank, u64 v)
{
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_map(p, rank)), "l"(v) : "memory");
}

template <typename V>
__device__ __forceinline__ V warp_scan(V v, int lane)      // inclusive
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const V t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// inclusive sum over the block's threads in order; total in `all`. s: one entry a warp
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* s, V& all)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    v = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) s[warp] = v;
    __syncthreads();
    V before = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < ST / 32; ++i)
    {
        const V t = s[i];
        if (i < warp) before += t;
        all += t;
    }
    return before + v;
}

// sorts N keys, one a thread of threads 0 .. N - 1, in descending order: a bitonic network, exchanges within a warp by shuffles
template <int N, typename V>
__device__ __forceinline__ V block_sort(V v, V* s)
{
    const int t = threadIdx.x;
#pragma unroll
    for (int size = 2; size <= N; size <<= 1)
#pragma unroll
        for (int st = size >> 1; st > 0; st >>= 1)
        {
            V o;
            if (st >= 32)
            {
                asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
                s[t] = v;
                asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
                o = s[t ^ st];
            }
            else
                o = __shfl_xor_sync(0xffffffffu, v, st);
            const bool larger = ((t & st) == 0) == ((t & size) == 0);
            v = larger == (v > o) ? v : o;
        }
    return v;
}

// the same for n <= ST keys; threads from n on bring 0, which no key is
template <typename V>
__device__ __forceinline__ V sort_n(V v, int n, V* s)
{
    const int t = threadIdx.x;
    if (n <= 64) { if (t < 64) v = block_sort<64>(v, s); }
    else if (n <= 128) { if (t < 128) v = block_sort<128>(v, s); }
    else if (n <= 256) { if (t < 256) v = block_sort<256>(v, s); }
    else v = block_sort<ST>(v, s);
    return v;
}

static_assert(offsetof(Shared, hist) % 16 == 0 && sizeof(Hist) % 16 == 0, "the histogram is cleared in 16-byte pieces");

template <typename T>
__global__ void __launch_bounds__(ST, 2) sample_kernel(const __grid_constant__ SampleArgs a)
{
    extern __shared__ float4 smem4[];
    __shared__ Shared sh;
    float* lg = reinterpret_cast<float*>(smem4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int NC = gridDim.x;
    int b = blockIdx.y;
    const uint32_t rank = blockIdx.x;
    const float INF = __int_as_float(0x7f800000), NONE = -INF;   // NONE: never picked; NaN and what is outside the slice become it
    int slot = 0;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;");
    if (a.ordered)
    {
        // the row of this cluster: those with a top-p but no small top-k first, then those without either, then the others: a row of the
        // first kind that starts when others have ended is what the call waits for (64 rows of 150001, 13 of them of that kind: 54 us, 66 in
        // the rows' order). A thread sorts a row: with more rows than threads they are taken in order, and what a row of the first kind
        // takes is then a smaller part of the call
        int c = 3;
        if (tid < (int) gridDim.y)
        {
            const int k = a.top_k ? a.top_k[tid] : a.top_k0;
            const float p = a.top_p ? a.top_p[tid] : a.top_p0, t = a.temperature ? a.temperature[tid] : a.temperature0;
            c = !(t > 0.0f) || (k > 0 && k <= SLIST) ? 2 : p < 1.0f || (k > 0 && k < a.V) ? 0 : 1;
        }
        const uint32_t in0 = __ballot_sync(0xffffffffu, c == 0), in1 = __ballot_sync(0xffffffffu, c == 1), in2 = __ballot_sync(0xffffffffu, c == 2);
        if (lane == 0) sh.part[0][warp] = (u64) __popc(in0) | (u64) __popc(in1) << 20 | (u64) __popc(in2) << 40;
        __syncthreads();
        u64 below = 0, all = 0;
        for (int w = 0; w < ST / 32; ++w) { if (w < warp) below += sh.part[0][w]; all += sh.part[0][w]; }
        const int n0 = (int) (all & 0xfffff), n1 = (int) (all >> 20 & 0xfffff);
        const uint32_t same = c == 0 ? in0 : c == 1 ? in1 : in2;
        const int at = (c > 0 ? n0 : 0) + (c > 1 ? n1 : 0) + (int) (below >> (20 * c) & 0xfffff) + __popc(same & ((1u << lane) - 1));
        if (c < 3 && at == b) sh.id = tid;
        __syncthreads();
        b = sh.id;
    }

    auto sync = [&]() {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    };
    // every CTA's values, by rank, in sh.mail[the returned slot] (valid until the next exchange but one)
    auto exchange = [&](u64 v0, u64 v1 = 0, u64 v2 = 0) {
        const int sl = slot;
        slot ^= 1;
        if (tid < NC)
        {
            dsmem_st(&sh.mail[sl][0][rank], tid, v0);
            dsmem_st(&sh.mail[sl][1][rank], tid, v1);
            dsmem_st(&sh.mail[sl][2][rank], tid, v2);
        }
        sync();
        return sl;
    };
    // the block's sums of up to NPV + 1 values, from every CTA, in the same way
    auto exchange_sums = [&](auto... values) {
        constexpr int N = sizeof...(values);
        u64 v[N] = { (u64) values... };
        const int sl = slot;
        slot ^= 1;
#pragma unroll
        for (int i = 0; i < N; ++i)
            for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane == i) sh.part[i][warp] = v[i];
        __syncthreads();
        if (tid < N * NC)
        {
            const int i = tid / NC;
            u64 t = 0;
            for (int w = 0; w < ST / 32; ++w) t += sh.part[i][w];
            dsmem_st(&sh.mail[sl][i][rank], tid - i * NC, t);
        }
        sync();
        return sl;
    };
    auto total_of = [&](int sl, int i) {
        u64 t = 0;
        for (int r = 0; r < NC; ++r) t += sh.mail[sl][i][r];
        return t;
    };
    auto put = [&](int id) {
        if (a.ids64) static_cast<long long*>(a.ids)[b] = id; else static_cast<int*>(a.ids)[b] = id;
    };

    // the slice [s0, s1) of the row into shared memory, in 16-byte loads of whole groups, four in flight; lg[0] is logit g0, the
    // first of the aligned group that holds s0
    constexpr int G = 16 / sizeof(T);
    const T* row = static_cast<const T*>(a.logits) + (size_t) b * a.ld;
    const int s0 = min(a.V, (int) rank * a.per), s1 = min(a.V, s0 + a.per);
    const int head = (int) ((reinterpret_cast<uintptr_t>(row + s0) & 15) / sizeof(T));
    const int g0 = s0 - head, n = (s1 - g0 + G - 1) / G * G * (s1 > s0);
    float mine_max = NONE;
    auto take = [&](int j, const float (&v0)[G]) {
        float v[G];
#pragma unroll
        for (int q = 0; q < G; ++q)
        {
            v[q] = v0[q] == v0[q] ? v0[q] + 0.0f : NONE;   // -0 counts as +0
            mine_max = fmaxf(mine_max, v[q]);
        }
#pragma unroll
        for (int q = 0; q < G / 4; ++q) reinterpret_cast<float4*>(lg + j)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    };
    for (int jj = tid * G; jj < n; jj += 4 * ST * G)
    {
        uint4 w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            const int j = jj + r * ST * G, i = g0 + j;
            if (j < n && i >= s0 && i + G <= s1) w[r] = __ldcs(reinterpret_cast<const uint4*>(row + i));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            const int j = jj + r * ST * G, i = g0 + j;
            if (j >= n) break;
            float v[G];
            if (i >= s0 && i + G <= s1)
            {
                const T* e = reinterpret_cast<const T*>(&w[r]);
#pragma unroll
                for (int q = 0; q < G; ++q) v[q] = to_f32(e[q]);
            }
            else
            {
#pragma unroll
                for (int q = 0; q < G; ++q) v[q] = i + q >= s0 && i + q < s1 ? to_f32(row[i + q]) : NONE;
            }
            take(j, v);
        }
    }
    for (int i = tid; i < SBINS; i += ST) sh.maxima[i] = 0;
    // the largest logit, and the smallest of the threads' largest ones
    float mx = mine_max, mn = mine_max == NONE ? INF : mine_max;
    {
        for (int o = 16; o; o >>= 1)
        {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        }
        if (lane == 0) { sh.warp32[warp] = __float_as_uint(mx); sh.warp[warp] = __float_as_uint(mn); }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ST / 32; ++i)
        {
            mx = fmaxf(mx, __uint_as_float(sh.warp32[i]));
            mn = fminf(mn, __uint_as_float((uint32_t) sh.warp[i]));
        }
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every CTA of the cluster has started
        const int sl = exchange(__float_as_uint(mx), __float_as_uint(mn));
        for (int r = 0; r < NC; ++r)
        {
            mx = fmaxf(mx, __uint_as_float((uint32_t) sh.mail[sl][0][r]));
            mn = fminf(mn, __uint_as_float((uint32_t) sh.mail[sl][1][r]));
        }
    }
    const float T0 = a.temperature ? a.temperature[b] : a.temperature0;
    if (mx == NONE || !(T0 > 0.0f))
    {
        // nothing to pick, or the largest logit: its lowest id
        int id = a.V;
        if (mx != NONE && mine_max == mx)
            for (int j = tid * G; j < n && id == a.V; j += ST * G)
                for (int q = G - 1; q >= 0; --q)
                    if (lg[j + q] == mx) id = g0 + j + q;
        if (tid == 0) sh.id = a.V;
        __syncthreads();
        id = __reduce_min_sync(0xffffffffu, id);
        if (lane == 0) atomicMin(&sh.id, id);
        __syncthreads();
        const int sl = exchange((u64) sh.id);
        if (rank == 0 && tid == 0)
        {
            for (int r = 0; r < NC; ++r) id = min(id, (int) sh.mail[sl][0][r]);
            put(mx == NONE ? -1 : id);
        }
        return;
    }
    if (mx == INF)
    {
        // equal shares of the infinite logits: as if they were 0 and the others masked
        for (int j = tid; j < n; j += ST) lg[j] = lg[j] == INF ? 0.0f : NONE;
        mine_max = mine_max == INF ? 0.0f : NONE;
        mx = mn = 0.0f;
        __syncthreads();
    }
    Weight weight;
    weight.init(mx, T0);
    const int k = a.top_k ? a.top_k[b] : a.top_k0;
    const float top_p = a.top_p ? a.top_p[b] : a.top_p0;
    const double mp = fmin((double) (a.min_p ? a.min_p[b] : a.min_p0), 1.0);
    const u64 least = mp > 0.0 ? (u64) ceil(mp * 17592186044416.0) : 0ull;
    const double u = fmin(fmax((double) a.u[b], 0.0), 1.0);
    const bool by_k = k > 0 && k < a.V, by_p = top_p < 1.0f;
    auto need_of = [&](u64 S) {                            // the mass before which a logit stays: at least the first does
        const u64 v = top_p > 0.0f ? (u64) ceil((double) top_p * (double) S) : 1ull;
        return v < 1 ? 1ull : v;
    };
    auto target_of = [&](u64 S) {
        const u64 t = (u64) (u * (double) S);
        return t >= S ? S - 1 : t;
    };
    // bins of m - l (monotone in l); what lies beyond the span is in the last one
    auto bin_scale = [&](float span) { return span > 0.0f ? (SBINS - 0.1f) / span : 0.0f; };
    auto bin_at = [&](float l, float scale) { return l == mx ? 0 : (int) fminf((mx - l) * scale, SBINS - 1.0f); };
    // f(logit, place in the slice) of this thread's share, the groups that it loaded
    auto each = [&](auto f) {
        for (int j = tid * G; j < n; j += ST * G)
#pragma unroll
            for (int q = 0; q < G / 4; ++q)
            {
                const int at = j + 4 * q;
                const float4 v = *reinterpret_cast<const float4*>(lg + at);
                f(v.x, at); f(v.y, at + 1); f(v.z, at + 2); f(v.w, at + 3);
            }
    };
    // at most the smallest logit whose bin is `bin` or less: what is below it lies in a later bin
    auto bin_floor = [&](int bin, float scale) {
        return scale > 0.0f && bin < SBINS - 1 ? mx - (float) (bin + 1) / scale * (1.0f + 0x1p-18f) - fabsf(mx) * 0x1p-20f : NONE;
    };
    auto block_sum = [&](u64 v) {
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) sh.warp[warp] = v;
        __syncthreads();
        u64 all = 0;
#pragma unroll
        for (int i = 0; i < ST / 32; ++i) all += sh.warp[i];
        return all;
    };
    // the bin (a thread's each) in which the running sum of v reaches need
    auto crossing = [&](u64 v, u64 upto, u64 need, uint32_t cnt) {
        if (upto - v < need && upto >= need) sh.found = Found{ tid, upto - v, v, cnt };
        __syncthreads();
        return sh.found;
    };

    u64 S = 0;                                             // the weights' sum, where top-p needs it
    // a logit into CTA 0's list
    auto push = [&](float l, int j) {
        const uint32_t at = dsmem_add(&sh.n_list, 0, 1u);
        if (at < SLIST) dsmem_st(&sh.list[at], 0, (u64) __float_as_uint(l) << 32 | (uint32_t) (g0 + j));
    };
    // element tid of the list's n (at most SLIST) by descending logit, then by id; it is in any order: the sort fixes it. Keys are those of
    // fp32, from which the logit comes back
    auto sorted_list = [&](int n_list, float& l, uint32_t& id) {
        const bool in = tid < n_list;
        const u64 e = in ? sh.list[tid] : 0ull;
        u64 s = in ? (u64) key_of<float>(__uint_as_float((uint32_t) (e >> 32))) << 32 | (uint32_t) ~(uint32_t) e : 0ull;
        s = sort_n(s, n_list, sh.sorted);
        l = of_key<float>((uint32_t) (s >> 32));
        id = ~(uint32_t) s;
        return in;
    };
    if (by_k || by_p)
    {
        // the edge: the bin at which k of the threads' maxima are reached (without a top-k, TRY of them or all)
        const float scale = bin_scale(mx - mn);
        if (mine_max != NONE) atomicAdd(&sh.maxima[bin_at(mine_max, scale)], 1u);
        if (tid == 0) { sh.n_list = 0; sh.found.bin = -1; }
        sync();
        uint32_t cnt = 0, all32, c[SRANKS];
        dsmem_ld_all(&sh.maxima[tid], NC, c);
#pragma unroll
        for (int r = 0; r < SRANKS; ++r) cnt += c[r];
        const uint32_t upto32 = block_scan(cnt, sh.warp32, all32);
        const uint32_t want = by_k ? (uint32_t) k : min(all32, (uint32_t) TRY);
        const int edge = crossing(cnt, upto32, want, cnt).bin;   // -1: fewer maxima than k
        // gathered: what lies up to the edge (and a rounding more), straight into CTA 0's list, so that the others are done once their
        // shares are in; with top-p alone, all weights are summed as well
        const float floor_l = edge >= 0 ? bin_floor(edge, scale) : INF;
        int got = 0, total;
        u64 listed = 0;
        if (by_k)
        {
            if (mine_max >= floor_l)
                each([&](float l, int j) { if (l >= floor_l && l != NONE) { push(l, j); ++got; } });
            total = (int) total_of(exchange_sums(got), 0);
        }
        else
        {
            u64 sum = 0;
            each([&](float l, int j) {
                const u64 w = weight(l);
                sum += w;
                if (l >= floor_l && l != NONE) { push(l, j); ++got; listed += w; }
            });
            const int sl = exchange_sums(got, listed, sum);
            total = (int) total_of(sl, 0);
            listed = total_of(sl, 1);
            S = total_of(sl, 2);
        }
        if (edge >= 0 && total <= SLIST && (by_k || listed >= need_of(S)))
        {
            if (rank == 0)
            {
                float l;
                uint32_t id;
                const bool in = sorted_list(total, l, id);
                u64 w = in && (!by_k || tid < k) ? weight(l) : 0ull, all;
                u64 upto = block_scan(w, sh.warp, all);
                if (by_p && tid > 0 && upto - w >= need_of(by_k ? all : S)) w = 0;
                if (w < least) w = 0;
                // the pick, in id order
                uint32_t o = w ? ((0x3fffffu - id) << 9 | (uint32_t) tid) : 0u;
                __syncthreads();
                sh.sorted[tid] = w;
                o = sort_n(o, total, sh.order);
                __syncthreads();
                const u64 wo = o ? sh.sorted[o & 511] : 0ull;
                upto = block_scan(wo, sh.warp, all);
                const u64 target = target_of(all);
                if (wo && upto - wo <= target && upto > target) put((int) (0x3fffffu - (o >> 9)));
            }
            return;
        }
    }

    // ---- the general way: many logits are kept ----
    // kept: l > thr, or l == thr and id <= cut
    float thr = NONE;
    int cut = a.V;
    auto kept = [&](float l, int j) { return l > thr || (l == thr && g0 + j <= cut); };

    // A histogram over the cluster of the kept logits for which bin(l) >= 0, and the bin at which the running sum of counts (mass: of
    // weights, with the counts too where wanted) reaches `need`
    auto histogram = [&](bool mass, bool counts, u64 need, auto bin) {
        Hist& h = sh.hist;
        sync();                                            // nobody reads an earlier one
        for (int i = tid; i < (int) (sizeof(Hist) / 16); i += ST) reinterpret_cast<uint4*>(&h)[i] = make_uint4(0, 0, 0, 0);
        if (tid == 0) { sh.found.bin = -1; sh.n_list = 0; }
        __syncthreads();
        each([&](float l, int j) {
            const int q = l != NONE && kept(l, j) ? bin(l) : -1;
            if (q < 0) return;
            if (!mass) { atomicAdd(&h.lo[lane & 3][q], 1u); return; }
            if (counts) atomicAdd(&h.cnt[q], 1u);
            const u64 w = weight(l);
            const uint32_t wl = (uint32_t) w;
            uint32_t up = (uint32_t) (w >> 32);
            if (wl) up += atomicAdd(&h.lo[lane & 3][q], wl) > ~wl;   // the carry of the low word
            if (up) atomicAdd(&h.hi[q], up);
        });
        __syncthreads();
        // the copies into one
        {
            const u64 t = (u64) h.lo[0][tid] + h.lo[1][tid] + h.lo[2][tid] + h.lo[3][tid];
            h.lo[0][tid] = (uint32_t) t;
            h.hi[tid] += (uint32_t) (t >> 32);
        }
        sync();
        // bin tid of all CTAs
        u64 v = 0, all;
        uint32_t cnt = 0, c[SRANKS], hi[SRANKS];
        dsmem_ld_all(&h.lo[0][tid], NC, c);
        dsmem_ld_all(&h.hi[tid], NC, hi);
#pragma unroll
        for (int r = 0; r < SRANKS; ++r) v += (u64) hi[r] << 32 | c[r];
        if (counts)
        {
            dsmem_ld_all(&h.cnt[tid], NC, c);
#pragma unroll
            for (int r = 0; r < SRANKS; ++r) cnt += c[r];
        }
        const u64 upto = block_scan(v, sh.warp, all);
        return crossing(v, upto, need, mass ? cnt : (uint32_t) v);
    };
    // id order over the cluster: this CTA's share of a sum, the sums before it and of all
    auto spread = [&](u64 mine, u64& before, u64& all) {
        const int sl = exchange(mine);
        before = all = 0;
        for (int r = 0; r < NC; ++r)
        {
            const u64 v = sh.mail[sl][0][r];
            if (r < (int) rank) before += v;
            all += v;
        }
    };
    // this warp's run of the slice, in rows of 128: four a lane
    const int run = (n + ST * 4 - 1) / (ST * 4) * 128, j0 = min(n, warp * run), j1 = min(n, j0 + run);
    // sum of f over the slice; `mine` gets this warp's part
    auto slice_sum = [&](auto f, u64& mine) {
        mine = 0;
#pragma unroll 4
        for (int j = j0 + lane * 4; j < j1; j += 128)
        {
            const float4 v = *reinterpret_cast<const float4*>(lg + j);
            mine += f(v.x, j) + f(v.y, j + 1) + f(v.z, j + 2) + f(v.w, j + 3);
        }
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        return block_sum(lane == 0 ? mine : 0ull);
    };
    // lowest id whose running sum exceeds target (the sum before this CTA given), after slice_sum: put_id is called by the lane that
    // holds it, if it is in this CTA
    auto find = [&](auto f, u64 mine, u64 before, u64 target, auto put_id) {
        for (int i = 0; i < warp; ++i) before += sh.warp[i];
        if (before <= target && before + mine > target)
            for (int q = j0; q < j1; q += 128)
            {
                const int j = q + lane * 4;
                u64 w[4] = {};
                if (j < j1)
                {
                    const float4 v = *reinterpret_cast<const float4*>(lg + j);
                    w[0] = f(v.x, j); w[1] = f(v.y, j + 1); w[2] = f(v.z, j + 2); w[3] = f(v.w, j + 3);
                }
                const u64 own = w[0] + w[1] + w[2] + w[3], c = warp_scan(own, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, before + c > target);
                if (hit)
                {
                    if (lane == __ffs(hit) - 1)
                    {
                        u64 at = before + c - own;
                        int i = 0;
                        while (at + w[i] <= target) at += w[i++];
                        put_id(g0 + j + i);
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, c, 31);
            }
    };

    // from a bin, gathered and sorted in CTA 0, to the exact threshold, in thr and cut; false where it holds too many
    auto resolve = [&](bool mass, u64 need, const Found& f, auto in_bin) {
        int got = 0;
        each([&](float l, int j) { if (in_bin(l, j)) { push(l, j); ++got; } });
        const int total = (int) total_of(exchange_sums(got), 0);
        if (total > SLIST) return false;
        if (rank == 0)
        {
            float l;
            uint32_t id;
            const bool in = sorted_list(total, l, id);
            const u64 w = in ? mass ? weight(l) : 1ull : 0ull, rest = need - f.above;
            u64 all;
            const u64 upto = block_scan(w, sh.warp, all);
            if (upto - w < rest && upto >= rest)
                for (int r = 0; r < NC; ++r) dsmem_st(&sh.result, r, (u64) __float_as_uint(l) << 32 | id);
        }
        sync();
        thr = __uint_as_float((uint32_t) (sh.result >> 32));
        cut = (int) (uint32_t) sh.result;
        return true;
    };
    // the same by histograms over the keys of the bin's logits
    auto narrow = [&](bool mass, u64 need, Found f, auto in_bin) {
        u64 above = f.above;
        uint32_t lo = 0xffffffffu, hi = 0, cnt = 0;
        each([&](float l, int j) {
            if (!in_bin(l, j)) return;
            const uint32_t ky = key_of<T>(l);
            lo = min(lo, ky);
            hi = max(hi, ky);
            ++cnt;
        });
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        cnt = __reduce_add_sync(0xffffffffu, cnt);
        __syncthreads();
        if (lane == 0) { sh.warp32[warp] = lo; sh.warp[warp] = (u64) cnt << 32 | hi; }
        __syncthreads();
        cnt = 0;
        for (int i = 0; i < ST / 32; ++i)
        {
            lo = min(lo, sh.warp32[i]);
            hi = max(hi, (uint32_t) sh.warp[i]);
            cnt += (uint32_t) (sh.warp[i] >> 32);
        }
        const int sl = exchange(lo, hi, cnt);
        cnt = 0;
        for (int r = 0; r < NC; ++r)
        {
            lo = min(lo, (uint32_t) sh.mail[sl][0][r]);
            hi = max(hi, (uint32_t) sh.mail[sl][1][r]);
            cnt += (uint32_t) sh.mail[sl][2][r];
        }
        f.cnt_in = cnt;
        while (lo < hi)
        {
            const int s = max(0, 32 - __clz(hi - lo) - 9);       // 512 bins
            const float lo_l = of_key<T>(lo), hi_l = of_key<T>(hi);
            f = histogram(mass, true, need - above, [&](float l) { return l >= lo_l && l <= hi_l ? (int) ((hi - key_of<T>(l)) >> s) : -1; });
            above += f.above;
            hi -= (uint32_t) f.bin << s;
            lo = max(lo, hi - ((1u << s) - 1));
        }
        // ties at key hi: the first m of them stay
        const u64 w = mass ? f.in / f.cnt_in : 1ull;
        const u64 m = w ? (need - above + w - 1) / w : (u64) f.cnt_in;
        int c = a.V;
        const float t = of_key<T>(hi);
        if (m < f.cnt_in)
        {
            auto tie = [&](float l, int j) { return (u64) (l == t && kept(l, j)); };
            u64 mine, before, all;
            if (tid == 0) sh.id = 0;
            const u64 sum = slice_sum(tie, mine);
            spread(sum, before, all);
            find(tie, mine, before, m - 1, [&](int id) { sh.id = id + 1; });
            __syncthreads();
            const int sl2 = exchange((u64) sh.id);
            for (int r = 0; r < NC; ++r)
                if (sh.mail[sl2][0][r]) c = (int) sh.mail[sl2][0][r] - 1;
        }
        else if (t == thr)
            c = cut;
        thr = t;
        cut = c;
    };

    if (by_k)
    {
        // bins over the whole row, from a pass for its smallest logit
        float least_l = mx;
        each([&](float l, int) { if (l != NONE) least_l = fminf(least_l, l); });
        // order-preserving, so that the block's minimum is an integer one
        uint32_t kl = key_of<float>(least_l);
        kl = __reduce_min_sync(0xffffffffu, kl);
        __syncthreads();
        if (lane == 0) sh.warp32[warp] = kl;
        __syncthreads();
        for (int i = 0; i < ST / 32; ++i) kl = min(kl, sh.warp32[i]);
        const int sl = exchange(kl);
        for (int r = 0; r < NC; ++r) kl = min(kl, (uint32_t) sh.mail[sl][0][r]);
        const float scale = bin_scale(mx - of_key<float>(kl));
        const Found f = histogram(false, false, (u64) k, [&](float l) { return bin_at(l, scale); });
        if (f.bin >= 0)                                    // else: fewer than k logits may be picked at all
        {
            const float floor_l = bin_floor(f.bin, scale);
            auto in_bin = [&](float l, int) { return l >= floor_l && l != NONE && bin_at(l, scale) == f.bin; };
            if (!resolve(false, (u64) k, f, in_bin)) narrow(false, (u64) k, f, in_bin);
        }
    }
    if (by_p)
    {
        // the kept weights' sum S and M, the sums from each pv up; the interval of exponents in which top_p * S is reached
        float pv[NPV];
        u64 M[NPV] = {};
        S = 0;
#pragma unroll
        for (int i = 0; i < NPV; ++i) pv[i] = mx - PV[i] * T0;
        each([&](float l, int j) {
            const u64 w = kept(l, j) ? weight(l) : 0ull;
            S += w;
#pragma unroll
            for (int i = 0; i < NPV; ++i) M[i] += l >= pv[i] ? w : 0ull;
        });
        const int sl = exchange_sums(S, M[0], M[1], M[2], M[3]);
        S = total_of(sl, 0);
#pragma unroll
        for (int i = 0; i < NPV; ++i) M[i] = total_of(sl, 1 + i);
        u64 need = need_of(S), above = 0;
        float top = mx, low = NONE, below = INF, width = PV[NPV] - PV[NPV - 1];
        bool open = true;
#pragma unroll
        for (int i = 0; i < NPV; ++i)
            if (open)
            {
                if (M[i] >= need) { low = pv[i]; width = PV[i] - (i ? PV[i - 1] : 0.0f); open = false; }
                else { above = M[i]; top = below = pv[i]; }
            }
        need -= above;
        const float scale = bin_scale(width * T0);
        auto bin = [&](float l) { return l >= low && l < below ? (int) fminf((top - l) * scale, SBINS - 1.0f) : -1; };
        const Found f = histogram(true, false, need, bin);
        auto in_bin = [&](float l, int j) { return l != NONE && bin(l) == f.bin && kept(l, j); };
        if (!resolve(true, need, f, in_bin)) narrow(true, need, f, in_bin);
    }
    u64 mine, before, all;
    auto pick = [&](auto final_weight) {
        const u64 sum = slice_sum(final_weight, mine);
        spread(sum, before, all);
        find(final_weight, mine, before, target_of(all), put);
    };
    if (thr == NONE && !least) pick([&](float l, int) { return weight(l); });
    else
        pick([&](float l, int j) {
            if (!kept(l, j)) return 0ull;
            const u64 w = weight(l);
            return w >= least ? w : 0ull;
        });
}

template <typename T>
cudaError_t launch_sample(const SampleArgs& a0, int B, cudaStream_t st)
{
    auto kernel = sample_kernel<T>;
    int dev = -1;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    static PerDevice<int> smem;
    if ((err = dense_smem(smem, dev, reinterpret_cast<const void*>(kernel), SLICE_MAX * 4 + 64)) != cudaSuccess) return err;
    SampleArgs a = a0;
    // CTAs per row: all 8 from 16384 logits on; a slice below 2048 logits would wait more than it works
    int nc = 1;
    while (nc < SRANKS && a.V > 2048 * nc) nc *= 2;
    a.per = ((a.V + nc - 1) / nc + 7) / 8 * 8;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nc; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(ST);
    cfg.dynamicSmemBytes = (size_t) a.per * 4 + 64;        // 64: up to 7 logits of the first group in front of the slice
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // rows are the grid's y dimension, at most 65535 a launch
    for (long long r = 0; r < B; r += 65535)
    {
        SampleArgs c = a;
        const int rows = (int) (B - r < 65535 ? B - r : 65535);
        c.logits = static_cast<const T*>(a.logits) + (size_t) r * a.ld;
        c.u += r;
        if (c.temperature) c.temperature += r;
        if (c.top_k) c.top_k += r;
        if (c.top_p) c.top_p += r;
        if (c.min_p) c.min_p += r;
        c.ids = static_cast<uint8_t*>(a.ids) + (size_t) r * (a.ids64 ? 8 : 4);
        cfg.gridDim = dim3(nc, rows);
        c.ordered = (a.top_k || a.top_p) && rows <= ST && (long long) rows * nc > 2 * dense_sms(dev);
        if ((err = cudaLaunchKernelEx(&cfg, kernel, c)) != cudaSuccess) return err;
    }
    return cudaSuccess;
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
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == GLMX_F32 ? 4 : 2)) return dense_fail(GLMX_E_ARG, "glmx_sample: logits must be aligned to their type");
    const SampleArgs a{ logits, ld, V, 0, u, temperature, temperature0, top_k, top_k0, top_p, top_p0, min_p, min_p0, ids, ids_dtype == GLMX_I64, 0 };
    const cudaError_t e = dtype == GLMX_F32 ? launch_sample<float>(a, B, st)
                        : dtype == GLMX_F16 ? launch_sample<__half>(a, B, st) : launch_sample<__nv_bfloat16>(a, B, st);
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_sample: launch");
}
