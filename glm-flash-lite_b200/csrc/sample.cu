// Sampling (glmx_sample): one cluster of up to 8 CTAs per row, the row's logits held in their shared memory, so that global memory is
// read once and every further pass runs on chip. One row of 131072 logits is bound by the passes' latency (cluster barriers,
// block scans), a batch by the exponentials of the rows that keep many tokens.
//
// A weight is w = exp((l - m) / T) <= 1 in fp32, held as the integer floor(w * 2^44): sums of up to 2^19 weights fit 64 bits
// and do not depend on their order. Equal logits have equal weights, so each filter is a threshold on the logits'
// order-preserving integer key plus a number of kept ties, the lowest ids first:
//   top-k: the key with count(>) < k <= count(>=);  top-p: the key with mass(>) < top_p * S <= mass(>=);  min-p: a least weight.
// The first histogram (1024 bins of m - l, as wide as 2^-44 reaches) finds the bin in which the first active filter ends. Where
// the bins up to it hold at most 512 logits, these are gathered and sorted in one CTA, which finishes the row. Otherwise the
// threshold is narrowed by further histograms of 1024 bins over the keys of that bin, and the pick is found by
// running sums over the row: the CTA, the warp, then the lane in whose run the target falls.
#include "dense.h"
#include "glmx_common.cuh"

namespace glmx {

namespace {

typedef unsigned long long u64;

struct SampleArgs
{
    const void* logits; long long ld; int V, per;          // per: logits of a CTA's slice (a multiple of 8)
    const float* u; const float* temperature; float temperature0; const int* top_k; int top_k0;
    const float* top_p; float top_p0; const float* min_p; float min_p0;
    void* ids; int ids64;
};

constexpr int ST = 512, SBINS = 1024, SLIST = 512, SRANKS = 8;
constexpr int SLICE_MAX = GLMX_SAMPLE_MAX_VOCAB / SRANKS;  // 49152 logits: 192 KB
constexpr float SPAN = 30.6f;                              // exp(-30.5) = 2^-44: weights further down are 0

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
    __device__ __forceinline__ u64 operator()(float l) const
    {
        if (l == m) return 1ull << 44;
        const float d = l - m, bb = d - l, derr = (l - (d - bb)) + (-m - bb);
        const float x = d * ch;
        if (!(x > -46.0f)) return 0;
        const float lo = fmaf(d, ch, -x) + fmaf(d, cl, derr * ch);
        const float n = rintf(x), f = ((x - n) + lo) * 0.693147180559945f;
        float e = fmaf(f, 1.0f / 5040, 1.0f / 720);
        e = fmaf(e, f, 1.0f / 120); e = fmaf(e, f, 1.0f / 24); e = fmaf(e, f, 1.0f / 6); e = fmaf(e, f, 0.5f);
        e = fmaf(e, f, 1.0f); e = fmaf(e, f, 1.0f);
        const u64 w = (u64) __float2uint_rd(e * 16777216.0f);
        const int sh = 20 + (int) n;
        return sh >= 0 ? w << sh : w >> -sh;
    }
};

struct Hist
{
    uint32_t cnt[SBINS], lo[SBINS], hi[SBINS];             // counts, and 64-bit masses in two words
};

struct Found                                               // the bin in which a running sum reaches its need
{
    int bin;
    u64 above, in;                                         // the sum above it and its own
    uint32_t cnt_above, cnt_in;
};

struct Shared
{
    Hist hist[2];
    u64 mail[2][2][SRANKS];
    u64 warp[ST / 32];
    uint32_t warp32[ST / 32];
    u64 list[SLIST];                                       // (key, ~id) of this CTA's gathered logits
    u64 sorted[SLIST];
    uint32_t order[SLIST];
    Found found;
    int n_list, id;
};

__device__ __forceinline__ uint32_t dsmem_map(const void* p, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ u64 dsmem_ld(const void* p, uint32_t rank)
{
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(dsmem_map(p, rank)) : "memory");
    return v;
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

// sorts n <= N keys (N a power of 2 from 32 to ST, one a thread) in descending order
template <typename V>
__device__ __forceinline__ V block_sort(V v, int N, V* s)
{
    const int t = threadIdx.x;
    for (int size = 2; size <= N; size <<= 1)
        for (int st = size >> 1; st > 0; st >>= 1)
        {
            V o;
            if (st >= 32)
            {
                __syncthreads();
                s[t] = v;
                __syncthreads();
                o = s[t ^ st];
            }
            else
                o = __shfl_xor_sync(0xffffffffu, v, st);
            const bool larger = ((t & st) == 0) == ((t & size) == 0);
            v = larger ? (v > o ? v : o) : (v < o ? v : o);
        }
    return v;
}

template <typename T>
__global__ void __launch_bounds__(ST, 2) sample_kernel(const __grid_constant__ SampleArgs a)
{
    extern __shared__ float4 smem4[];
    __shared__ Shared sh;
    float* lg = reinterpret_cast<float*>(smem4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int NC = gridDim.x, b = blockIdx.y;
    const uint32_t rank = blockIdx.x;
    const float NONE = __int_as_float(0xff800000);         // -inf: never picked; NaN and what is outside the slice become it
    int slot = 0, hslot = 0;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;");

    auto sync = [&]() {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    };
    // every CTA's pair of values, by rank, in sh.mail[the returned slot] (valid until the next exchange but one)
    auto exchange = [&](u64 v0, u64 v1) {
        const int sl = slot;
        slot ^= 1;
        if (tid < NC)
        {
            dsmem_st(&sh.mail[sl][0][rank], tid, v0);
            dsmem_st(&sh.mail[sl][1][rank], tid, v1);
        }
        sync();
        return sl;
    };
    auto put = [&](int id) {
        if (a.ids64) static_cast<long long*>(a.ids)[b] = id; else static_cast<int*>(a.ids)[b] = id;
    };

    // the slice [s0, s1) of the row into shared memory, in 16-byte loads of whole groups; lg[0] is logit g0, the first of the
    // aligned group that holds s0
    constexpr int G = 16 / sizeof(T);
    const T* row = static_cast<const T*>(a.logits) + (size_t) b * a.ld;
    const int s0 = min(a.V, (int) rank * a.per), s1 = min(a.V, s0 + a.per);
    const int head = (int) ((reinterpret_cast<uintptr_t>(row + s0) & 15) / sizeof(T));
    const int g0 = s0 - head, n = (s1 - g0 + G - 1) / G * G * (s1 > s0);
    float mx = NONE, mn = __int_as_float(0x7f800000);
    for (int j = tid * G; j < n; j += ST * G)
    {
        const int i = g0 + j;
        float v[G];
        if (i >= s0 && i + G <= s1)
        {
            const uint4 w = __ldcs(reinterpret_cast<const uint4*>(row + i));
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int q = 0; q < G; ++q) v[q] = to_f32(e[q]);
        }
        else
        {
#pragma unroll
            for (int q = 0; q < G; ++q) v[q] = i + q >= s0 && i + q < s1 ? to_f32(row[i + q]) : NONE;
        }
#pragma unroll
        for (int q = 0; q < G; ++q)
        {
            v[q] = v[q] == v[q] ? v[q] + 0.0f : NONE;      // -0 counts as +0
            mx = fmaxf(mx, v[q]);
            if (v[q] != NONE) mn = fminf(mn, v[q]);
        }
#pragma unroll
        for (int q = 0; q < G / 4; ++q) reinterpret_cast<float4*>(lg + j)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
    {
        // maximum and minimum over the block, then the cluster
        for (int o = 16; o; o >>= 1)
        {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        }
        if (lane == 0) { sh.warp32[warp] = __float_as_uint(mx); sh.warp[warp] = __float_as_uint(mn); }
        __syncthreads();
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
        if (mx != NONE)
            for (int j = tid; j < n; j += ST)
                if (lg[j] == mx) { id = g0 + j; break; }
        if (tid == 0) sh.id = a.V;
        __syncthreads();
        id = __reduce_min_sync(0xffffffffu, id);
        if (lane == 0) atomicMin(&sh.id, id);
        __syncthreads();
        const int sl = exchange((u64) sh.id, 0);
        if (rank == 0 && tid == 0)
        {
            for (int r = 0; r < NC; ++r) id = min(id, (int) sh.mail[sl][0][r]);
            put(mx == NONE ? -1 : id);
        }
        return;
    }
    Weight weight;
    weight.init(mx, T0);
    const int k = a.top_k ? a.top_k[b] : a.top_k0;
    const float top_p = a.top_p ? a.top_p[b] : a.top_p0;
    const double mp = fmin((double) (a.min_p ? a.min_p[b] : a.min_p0), 1.0);
    const u64 least = mp > 0.0 ? (u64) ceil(mp * 17592186044416.0) : 0ull;
    const double u = fmin(fmax((double) a.u[b], 0.0), 1.0);
    const bool by_k = k > 0 && k < a.V, by_p = top_p < 1.0f;
    // bins of m - l (monotone in l); what lies beyond the span is in the last one
    const float span = fminf(SPAN * T0, mx - mn), bscale = span > 0.0f ? 1023.9f / span : 0.0f;
    auto bin_of = [&](float l) { return l == mx ? 0 : (int) fminf((mx - l) * bscale, 1023.0f); };
    auto need_of = [&](u64 S) {                            // the mass before which a logit stays: at least the first does
        const u64 v = top_p > 0.0f ? (u64) ceil((double) top_p * (double) S) : 1ull;
        return v < 1 ? 1ull : v;
    };
    auto target_of = [&](u64 S) {
        const u64 t = (u64) (u * (double) S);
        return t >= S ? S - 1 : t;
    };

    // kept: key > thr, or key == thr and id <= cut
    uint32_t thr = 0;
    int cut = a.V;
    auto kept = [&](uint32_t ky, int i) { return ky > thr || (ky == thr && i <= cut); };

    // A histogram over the cluster of the kept logits for which bin(l, key) >= 0, and the bin at which the running sum of
    // counts (mass: of weights) reaches `need` (frac: need_of the whole sum). total: the whole sum
    auto histogram = [&](bool mass, bool frac, u64& need, u64& total, auto bin) {
        Hist& h = sh.hist[hslot];
        for (int i = tid; i < (int) (sizeof(Hist) / 4); i += ST) reinterpret_cast<uint32_t*>(&h)[i] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += ST)
        {
            const float l = lg[j];
            if (l == NONE) continue;
            const uint32_t ky = key_of<T>(l);
            const int q = kept(ky, g0 + j) ? bin(l, ky) : -1;
            if (q < 0) continue;
            atomicAdd(&h.cnt[q], 1u);
            if (mass)
            {
                const u64 w = weight(l);
                const uint32_t wl = (uint32_t) w, wh = (uint32_t) (w >> 32);
                if (wl)
                {
                    const uint32_t old = atomicAdd(&h.lo[q], wl);
                    if (wh + (old + wl < old)) atomicAdd(&h.hi[q], wh + (old + wl < old));
                }
                else if (wh)
                    atomicAdd(&h.hi[q], wh);
            }
        }
        sync();
        // bins 2 tid and 2 tid + 1 of all CTAs
        u64 v0 = 0, v1 = 0;
        uint32_t c0 = 0, c1 = 0;
        for (int r = 0; r < NC; ++r)
        {
            const u64 c = dsmem_ld(&h.cnt[2 * tid], r);
            c0 += (uint32_t) c;
            c1 += (uint32_t) (c >> 32);
            if (mass)
            {
                const u64 l = dsmem_ld(&h.lo[2 * tid], r), hi = dsmem_ld(&h.hi[2 * tid], r);
                v0 += (l & 0xffffffffu) + (hi << 32);
                v1 += (l >> 32) + (hi >> 32 << 32);
            }
        }
        hslot ^= 1;
        uint32_t call;
        const uint32_t cs = block_scan(c0 + c1, sh.warp32, call);
        if (!mass) { v0 = c0; v1 = c1; }
        u64 vs = cs;
        total = call;
        if (mass) vs = block_scan(v0 + v1, sh.warp, total);
        if (frac) need = need_of(total);
        const u64 before = vs - v0 - v1;
        if (before < need && vs >= need)
        {
            const bool second = before + v0 < need;
            Found f;
            f.bin = 2 * tid + second;
            f.above = before + (second ? v0 : 0);
            f.in = second ? v1 : v0;
            f.cnt_above = cs - c0 - c1 + (second ? c0 : 0);
            f.cnt_in = second ? c1 : c0;
            sh.found = f;
        }
        __syncthreads();
        return sh.found;
    };

    // id order over the cluster: this CTA's share of a sum, the sums before it and of all
    auto spread = [&](u64 mine, u64& before, u64& all) {
        const int sl = exchange(mine, 0);
        before = all = 0;
        for (int r = 0; r < NC; ++r)
        {
            const u64 v = sh.mail[sl][0][r];
            if (r < (int) rank) before += v;
            all += v;
        }
    };
    // this warp's run of the slice, in rows of 32
    const int run = (n + ST - 1) / ST * 32, j0 = min(n, warp * run), j1 = min(n, j0 + run);
    // sum of f over the slice; `mine` gets this warp's part
    auto slice_sum = [&](auto f, u64& mine) {
        mine = 0;
        for (int j = j0 + lane; j < j1; j += 32) mine += f(lg[j], g0 + j);
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        u64 all;
        const u64 s = block_scan(lane == 0 ? mine : 0ull, sh.warp, all);
        (void) s;
        return all;
    };
    // lowest id whose running sum exceeds target (the sums before this CTA given); only the warp that holds it calls put_id
    auto find = [&](auto f, u64 mine, u64 before, u64 target, auto put_id) {
        for (int i = 0; i < warp; ++i) before += sh.warp[i];
        if (before <= target && before + mine > target)
            for (int q = j0; q < j1; q += 32)
            {
                const u64 c = warp_scan(q + lane < j1 ? f(lg[q + lane], g0 + q + lane) : 0ull, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, before + c > target);
                if (hit)
                {
                    if (lane == 0) put_id(g0 + q + __ffs(hit) - 1);
                    break;
                }
                before += __shfl_sync(0xffffffffu, c, 31);
            }
    };

    // from the first histogram's bin to the exact threshold, in thr and cut
    auto narrow = [&](bool mass, u64 need, Found f) {
        const int b0 = f.bin;
        u64 above = f.above;
        uint32_t lo = 0xffffffffu, hi = 0;
        for (int j = tid; j < n; j += ST)
        {
            const float l = lg[j];
            if (l == NONE || bin_of(l) != b0) continue;
            const uint32_t ky = key_of<T>(l);
            if (kept(ky, g0 + j)) { lo = min(lo, ky); hi = max(hi, ky); }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        __syncthreads();
        if (lane == 0) { sh.warp32[warp] = lo; sh.warp[warp] = hi; }
        __syncthreads();
        for (int i = 0; i < ST / 32; ++i) { lo = min(lo, sh.warp32[i]); hi = max(hi, (uint32_t) sh.warp[i]); }
        const int sl = exchange(lo, hi);
        for (int r = 0; r < NC; ++r) { lo = min(lo, (uint32_t) sh.mail[sl][0][r]); hi = max(hi, (uint32_t) sh.mail[sl][1][r]); }
        while (lo < hi)
        {
            const int s = max(0, 32 - __clz(hi - lo) - 10);
            u64 left = need - above, total;
            f = histogram(mass, false, left, total, [&](float, uint32_t ky) { return ky >= lo && ky <= hi ? (int) ((hi - ky) >> s) : -1; });
            above += f.above;
            hi -= (uint32_t) f.bin << s;
            lo = max(lo, hi - ((1u << s) - 1));
        }
        // ties at key hi: the first m of them stay
        const u64 w = mass ? f.in / f.cnt_in : 1ull;
        const u64 m = w ? (need - above + w - 1) / w : (u64) f.cnt_in;
        int c = a.V;
        if (m < f.cnt_in)
        {
            auto tie = [&](float l, int i) { const uint32_t ky = key_of<T>(l); return (u64) (l != NONE && ky == hi && kept(ky, i)); };
            u64 mine, before, all;
            if (tid == 0) sh.id = 0;
            const u64 sum = slice_sum(tie, mine);
            spread(sum, before, all);
            find(tie, mine, before, m - 1, [&](int id) { sh.id = id + 1; });
            __syncthreads();
            const int sl2 = exchange((u64) sh.id, 0);
            for (int r = 0; r < NC; ++r)
                if (sh.mail[sl2][0][r]) c = (int) sh.mail[sl2][0][r] - 1;
        }
        thr = hi;
        cut = c;
    };

    if (by_k || by_p)
    {
        u64 need = by_k ? (u64) k : 0, S;
        auto first = [&](float l, uint32_t) { return bin_of(l); };
        // fewer logits than k that may be picked at all: top-k keeps them
        Found f;
        bool done_k = !by_k;
        if (tid == 0) sh.found.bin = -1;
        if (by_k)
        {
            f = histogram(false, false, need, S, first);
            if (f.bin < 0) done_k = true;
        }
        if (done_k && by_p) f = histogram(true, true, need, S, first);
        if (!(done_k && !by_p) && f.cnt_above + f.cnt_in <= SLIST)
        {
            // few logits: gathered, sorted and finished in CTA 0
            const int total = (int) (f.cnt_above + f.cnt_in);
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            for (int j = tid; j < n; j += ST)
            {
                const float l = lg[j];
                if (l == NONE || bin_of(l) > f.bin) continue;
                sh.list[atomicAdd(&sh.n_list, 1)] = (u64) __float_as_uint(l) << 32 | (uint32_t) (g0 + j);
            }
            __syncthreads();
            const int sl = exchange((u64) sh.n_list, 0);
            if (rank == 0)
            {
                // element tid of the CTAs' lists, in any order: the sort fixes it
                u64 e = 0;
                int at = tid;
                for (int r = 0; r < NC; ++r)
                {
                    const int c = (int) sh.mail[sl][0][r];
                    if (at >= 0 && at < c) { e = dsmem_ld(&sh.list[at], r); at = -1; }
                    else if (at >= 0) at -= c;
                }
                int N = 32;
                while (N < total) N <<= 1;
                const bool in = tid < total;
                // by key, then by id: descending (key, ~id); with the key of fp32, from which the logit comes back
                u64 s = in ? (u64) key_of<float>(__uint_as_float((uint32_t) (e >> 32))) << 32 | (uint32_t) ~(uint32_t) e : 0ull;
                s = block_sort(s, N, sh.sorted);
                const uint32_t ky = (uint32_t) (s >> 32), id = ~(uint32_t) s;
                const float l = __uint_as_float(ky & 0x80000000u ? ky & 0x7fffffffu : ~ky);
                u64 w = in && (!by_k || done_k || tid < k) ? weight(l) : 0ull, all;
                u64 upto = block_scan(w, sh.warp, all);
                if (by_p && tid > 0 && upto - w >= need_of(done_k ? S : all)) w = 0;
                if (w < least) w = 0;
                // the pick, in id order
                uint32_t o = w ? ((0x3fffffu - id) << 9 | (uint32_t) tid) : 0u;
                sh.order[tid] = 0;
                __syncthreads();
                sh.sorted[tid] = w;
                o = block_sort(o, N, sh.order);
                __syncthreads();
                const u64 wo = o ? sh.sorted[o & 511] : 0ull;
                upto = block_scan(wo, sh.warp, all);
                const u64 target = target_of(all);
                if (wo && upto - wo <= target && upto > target) put((int) (0x3fffffu - (o >> 9)));
            }
            sync();                                        // the lists are read
            return;
        }
        if (!done_k)
        {
            narrow(false, need, f);
            if (by_p)
            {
                f = histogram(true, true, need, S, first);
                narrow(true, need, f);
            }
        }
        else if (by_p)
            narrow(true, need, f);
    }
    auto final_weight = [&](float l, int i) {
        if (l == NONE || !kept(key_of<T>(l), i)) return 0ull;
        const u64 w = weight(l);
        return w >= least ? w : 0ull;
    };
    u64 mine, before, all;
    const u64 sum = slice_sum(final_weight, mine);
    spread(sum, before, all);
    find(final_weight, mine, before, target_of(all), put);
}

template <typename T>
cudaError_t launch_sample(const SampleArgs& a0, int B, cudaStream_t st)
{
    auto kernel = sample_kernel<T>;
    int dev = -1;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64) return cudaErrorInvalidDevice;
    static bool ready[64] = {};
    if (!ready[dev])
    {
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SLICE_MAX * 4 + 64)) != cudaSuccess) return err;
        ready[dev] = true;
    }
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
    for (int r = 0; r < B; r += 65535)
    {
        SampleArgs c = a;
        const int rows = B - r < 65535 ? B - r : 65535;
        c.logits = static_cast<const T*>(a.logits) + (size_t) r * a.ld;
        c.u += r;
        if (c.temperature) c.temperature += r;
        if (c.top_k) c.top_k += r;
        if (c.top_p) c.top_p += r;
        if (c.min_p) c.min_p += r;
        c.ids = static_cast<uint8_t*>(a.ids) + (size_t) r * (a.ids64 ? 8 : 4);
        cfg.gridDim = dim3(nc, rows);
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
    const SampleArgs a{ logits, ld, V, 0, u, temperature, temperature0, top_k, top_k0, top_p, top_p0, min_p, min_p0, ids, ids_dtype == GLMX_I64 };
    const cudaError_t e = dtype == GLMX_F32 ? launch_sample<float>(a, B, st)
                        : dtype == GLMX_F16 ? launch_sample<__half>(a, B, st) : launch_sample<__nv_bfloat16>(a, B, st);
    return e == cudaSuccess ? GLMX_OK : dense_cuda_fail(e, "glmx_sample: launch");
}
