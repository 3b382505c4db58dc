// One token for each row of logits: temperature, top-k, top-p, min-p, and the draw from a given
// uniform number.
//
// Weights w = 2^shift exp((x - max) / T) are rounded to whole numbers (shift so that V of them fit
// 62 bits: 46 at 50257 logits), so sums are exact in any order and a threshold found by adding
// bins is the one found by adding values one by one.  The order by falling value, lowest index first
// among equals, is that of a whole-number key of the value; the kept set is always "keys above K,
// and the first `ties` at K".
//
// Three launches.  sample_max_kernel: the first maximum of each of C chunks of a row (C so that the
// chip is full).  sample_hist_kernel: each chunk's histogram over bins of d = max - x, 64 to each
// doubling of d, so that rows of any spread fit: of counts where top_k is small, of weights
// otherwise.  sample_finish_kernel, a workgroup a row: the bins say where the cut falls; only that
// bin's values are gathered from the row and sorted, the chunk that holds u follows from the
// chunks' histograms, and only that chunk is walked.  Rows whose cut falls into a crowded bin
// (thousands of values within 2 %), with top_k above 1024, or with an infinite maximum or
// temperature take sample_row_general, which finds K digit by digit.
//
// 128 rows of 128000 bf16 logits, top-p: 72 us (7.6, 22.8 and 41.9 alone), of which one read of the logits
// would be 6.4.  The histogram is bound by the 64-bit exponentials of the weights (about 25 instructions
// of a logit); the last step by one workgroup's latencies: 9 us until the bins are there, 11 to
// gather 256 KB, 3 for K, 4 for the chunks' sums, 8 for the walk.  One row of 50257, every filter: 25 us,
// 18 of them the last step.  Loads of it moved before the row's parameters (72.7 us), twice as many
// chunks (71.7, for twice the workspace) and two batches of the gather in flight (72.7) did not help.
#include "jas_common.hpp"

#include <algorithm>
#include <cmath>

namespace jas {

struct SampleArgs {
    const void *x;
    int n, V, shift;
    long ld;
    const float *temp, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *ids;
    float *logp;
    int C, chunk, vec;    // chunks of a row, logits of one (a multiple of 1024); rows start on 16 bytes
    uint32_t *chunk_key;  // [n][C] largest key of a chunk
    int32_t *chunk_idx;   // and its first index
    unsigned long long *hist;  // [n][C][NB]
};

// Keys grow with the value: -inf and NaN have the least, 0
__device__ __forceinline__ uint32_t sample_key(float x)
{
    if (!(x > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);  // (-0 and 0 are equals)
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k)
{
    return k == 0u ? -INFINITY : __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
template <typename T>
__device__ __forceinline__ uint32_t logit_key(const T *x, long i)
{
    if constexpr (sizeof(T) == 4) return sample_key(x[i]);
    else return sample_key(bf16_to_f32(x[i]));
}

// How a row's weights are formed
struct SampleScale {
    double mx, inv_t;
    double unit;  // 2^shift
    bool inf;     // the maximum is +inf: weight 1 for its equals, 0 for the rest
};
__device__ __forceinline__ double sample_z(const SampleScale &sc, float x)
{
    if (sc.inf) return x == INFINITY ? 0.0 : -INFINITY;
    if (x == -INFINITY) return -INFINITY;
    return ((double)x - sc.mx) / sc.inv_t;
}
__device__ __forceinline__ double sample_w(const SampleScale &sc, uint32_t key)
{
    return exp(sample_z(sc, key_value(key)));
}
__device__ __forceinline__ unsigned long long sample_mass(const SampleScale &sc, uint32_t key)
{
    return (unsigned long long)rint(sample_w(sc, key) * sc.unit);
}

constexpr int ST = 1024;      // threads of a row
constexpr int NB = 1536;      // bins
constexpr int SMALL_K = 1024; // largest top_k whose kept logits are sorted whole
constexpr int CAP = 4096;     // logits that a row's cut may gather
constexpr int MAX_CHUNKS = 1024;

// Sums and extremes over a wave without LDS: rows of 16 lanes by DPP shifts, the rows by scalars
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x, uint32_t none)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ unsigned long long dpp_u64(unsigned long long x)
{
    return (unsigned long long)dpp_u32<CTRL>((uint32_t)(x >> 32), 0u) << 32 | dpp_u32<CTRL>((uint32_t)x, 0u);
}
__device__ __forceinline__ unsigned long long lane_u64(unsigned long long x, int lane)
{
    return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ unsigned long long row_scan(unsigned long long v)  // lanes up to one's own, of its 16
{
    v += dpp_u64<0x111>(v);  // row_shr
    v += dpp_u64<0x112>(v);
    v += dpp_u64<0x114>(v);
    return v + dpp_u64<0x118>(v);
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v)
{
    v = row_scan(v);
    const int row = (threadIdx.x & 63) >> 4;
    const unsigned long long a = lane_u64(v, 15), b = a + lane_u64(v, 31), c = b + lane_u64(v, 47);
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
    v = max(v, dpp_u32<0x111>(v, 0u));
    v = max(v, dpp_u32<0x112>(v, 0u));
    v = max(v, dpp_u32<0x114>(v, 0u));
    v = max(v, dpp_u32<0x118>(v, 0u));
    const auto at = [&](int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); };
    return max(max(at(15), at(31)), max(at(47), at(63)));
}

// Bin of d = max - x >= 0: below 2^-6 the first, then 64 to a doubling, the last from 2^17.9 up.
// It does not fall as x falls.
__device__ __forceinline__ int sample_bin(float d)
{
    const int t = (int)(__float_as_uint(fmaxf(d, 0x1p-7f)) >> 17) - (int)(0x3c800000u >> 17) + 1;
    return max(0, min(t, NB - 1));
}

// d from which bin b starts, for b up to NB (the last bin has no end)
__device__ __forceinline__ float bin_edge(int b)
{
    return b <= 0 ? 0.f : b >= NB ? INFINITY : __uint_as_float((uint32_t)(b - 1 + (0x3c800000 >> 17)) << 17);
}

// Values that no logit of a bin lies above, or below: mx less the bin's edge, and 2^-20 of each more
// than the subtractions' roundings
__device__ __forceinline__ float bin_top(float mx, int b)
{
    const float t = mx - bin_edge(b) * (1 - 0x1p-20f);
    return t + fabsf(t) * 0x1p-20f;
}
__device__ __forceinline__ float bin_bottom(float mx, int b)
{
    const float t = mx - bin_edge(b + 1) * (1 + 0x1p-20f);
    return t - fabsf(t) * 0x1p-20f;
}

// Weight 2^shift e^((x - max) / T) as a whole number: c = log2(e) / T; 2^f by its series, |f| <= 1/2
// (to 2^-47), and rounded by an addition of 2^52 (shift <= 51)
__device__ __forceinline__ unsigned long long sample_weight(float x, double mx, double c, int shift)
{
    const double y = fmax(((double)x - mx) * c, -2000.0), n = rint(y), f = y - n;
    double r = 4.4455382718708116e-10;  // ln(2)^k / k!, k = 11 .. 0
    r = fma(r, f, 7.054911620801123e-09);
    r = fma(r, f, 1.01780860092397e-07);
    r = fma(r, f, 1.321548679014431e-06);
    r = fma(r, f, 1.5252733804059841e-05);
    r = fma(r, f, 0.0001540353039338161);
    r = fma(r, f, 0.0013333558146428443);
    r = fma(r, f, 0.009618129107628477);
    r = fma(r, f, 0.05550410866482158);
    r = fma(r, f, 0.24022650695910072);
    r = fma(r, f, 0.6931471805599453);
    r = fma(r, f, 1.0);
    const double v = ldexp(r, (int)n + shift) + 0x1p52;
    return (unsigned long long)__double_as_longlong(v) & 0xfffffffffffffull;
}

// How a row is drawn
struct SampleRow {
    float temp;
    int top_k;      // 0: all
    float top_p;    // 1: all
    double min_p, u;
    bool greedy, plain;  // the first maximum; 1 / T is finite
    double c;       // log2(e) / T
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs &p, int row)
{
    // (five loads in flight: an absent array's is one of u)
    const float u = p.u[row], temp = *(p.temp ? p.temp + row : p.u), top_p = *(p.top_p ? p.top_p + row : p.u),
                min_p = *(p.min_p ? p.min_p + row : p.u);
    const int32_t top_k = *(p.top_k ? p.top_k + row : (const int32_t *)p.u);
    SampleRow r;
    r.temp = p.temp ? temp : 1.f;
    r.top_k = p.top_k ? top_k : 0;
    if (r.top_k <= 0 || r.top_k >= p.V) r.top_k = 0;
    r.greedy = !(r.temp > 0.f) || r.top_k == 1;
    r.top_p = p.top_p && top_p < 1.f ? top_p : 1.f;
    r.min_p = p.min_p && min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
    r.u = !(u > 0.f) ? 0.f : fminf(u, 0x1.fffffep-1f);
    r.c = 1.4426950408889634074 / (double)r.temp;
    r.plain = r.c > 0.0 && r.c < 1e300;
    return r;
}

// Logits of a row before the first on 16 bytes
template <typename T>
__device__ __forceinline__ int logits_before_16(const T *x)
{
    return (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
}

// Calls f(x, index) for logits [i0, i1) of a row, by NT threads, each with rising indexes.  CLEAN: a
// NaN as -inf.
template <typename T, int NT, bool CLEAN = true, typename F>
__device__ __forceinline__ void each_logit(const T *x, int i0, int i1, F f)
{
    constexpr int E = 16 / sizeof(T), U = 8;
    const auto clean = [](float v) { return CLEAN ? fmaxf(v, -INFINITY) : v; };
    const auto one = [&](int at) {
        float v;
        if constexpr (sizeof(T) == 4) v = x[at];
        else v = bf16_to_f32(x[at]);
        f(clean(v), at);
    };
    const int head = min(i1, i0 + logits_before_16(x + i0)), whole = head + (i1 - head) / E * E;
    if (i0 + (int)threadIdx.x < head) one(i0 + (int)threadIdx.x);
    for (int at0 = head + (int)threadIdx.x * E; at0 < whole; at0 += U * NT * E) {  // eight loads in flight
        u32x4 v[U];
#pragma unroll
        for (int k = 0; k < U; ++k) v[k] = *(const u32x4 *)(x + min(at0 + k * NT * E, whole - E));
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int at = at0 + k * NT * E;
            if (at >= whole) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) f(clean(__uint_as_float(v[k][e])), at + e);
                else {
                    f(clean(__uint_as_float(v[k][e] << 16)), at + 2 * e);
                    f(clean(__uint_as_float(v[k][e] & 0xffff0000u)), at + 2 * e + 1);
                }
            }
        }
    }
    if (whole + (int)threadIdx.x < i1) one(whole + (int)threadIdx.x);
}

__device__ __forceinline__ void key_combine(uint32_t &k, int &i, uint32_t ok, int oi)
{
    if (ok > k || (ok == k && oi < i)) k = ok, i = oi;
}

template <typename T>
__global__ void __launch_bounds__(256) sample_max_kernel(const SampleArgs p)
{
    __shared__ uint32_t sk[4];
    __shared__ int si[4];
    const int row = blockIdx.y, c = blockIdx.x;
    const T *x = (const T *)p.x + (long)row * p.ld;
    float best = -INFINITY;
    int i = 0x7fffffff;  // (a thread's indexes rise: a later equal is not larger, and neither is a NaN)
    each_logit<T, 256, false>(x, c * p.chunk, min(p.V, (c + 1) * p.chunk), [&](float v, int at) {
        const bool more = v > best;
        best = more ? v : best, i = more ? at : i;
    });
    uint32_t k = sample_key(best);
    for (int o = 32; o; o >>= 1) key_combine(k, i, (uint32_t)__shfl_xor((int)k, o, WAVE), __shfl_xor(i, o, WAVE));
    if ((threadIdx.x & 63) == 0) sk[threadIdx.x >> 6] = k, si[threadIdx.x >> 6] = i;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) key_combine(k, i, sk[w], si[w]);
        p.chunk_key[(long)row * p.C + c] = k;
        p.chunk_idx[(long)row * p.C + c] = i;
    }
}

// The row's first maximum from its chunks', by every wave for itself
__device__ __forceinline__ void row_max_key(const SampleArgs &p, int row, uint32_t &k, int &i)
{
    k = 0, i = 0x7fffffff;
    for (int c = threadIdx.x & 63; c < p.C; c += 64) key_combine(k, i, p.chunk_key[(long)row * p.C + c], p.chunk_idx[(long)row * p.C + c]);
    const uint32_t own = k;
    k = wave_max_u32(k);
    i = (int)~wave_max_u32(own == k ? ~(uint32_t)i : 0u);  // the least index among the largest
}

template <typename T>
__global__ void __launch_bounds__(256) sample_hist_kernel(const SampleArgs p)
{
    __shared__ unsigned long long bins[NB];
    const int row = blockIdx.y, c = blockIdx.x;
    const SampleRow r = sample_row(p, row);
    uint32_t kmax;
    int imax;
    row_max_key(p, row, kmax, imax);
    const float mx = key_value(kmax);
    if (kmax == 0u || mx == INFINITY || r.greedy || !r.plain || r.top_k > SMALL_K) return;
    for (int b = threadIdx.x; b < NB; b += 256) bins[b] = 0;
    __syncthreads();
    const T *x = (const T *)p.x + (long)row * p.ld;
    const int i0 = c * p.chunk, i1 = min(p.V, (c + 1) * p.chunk);
    if (r.top_k) each_logit<T, 256>(x, i0, i1, [&](float v, int) { atomicAdd((unsigned *)&bins[sample_bin(mx - v)], 1u); });
    else each_logit<T, 256>(x, i0, i1, [&](float v, int) {
        const unsigned long long w = sample_weight(v, mx, r.c, p.shift);
        if (w) atomicAdd(&bins[sample_bin(mx - v)], w);
    });
    __syncthreads();
    unsigned long long *out = p.hist + ((long)row * p.C + c) * NB;
    for (int b = threadIdx.x; b < NB; b += 256) out[b] = bins[b];
}

// The ST threads' 64-bit sums in thread order: exclusive prefix and total
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long *red, unsigned long long &total)
{
    static_assert(ST == 1024, "a wave's sum in each of 16 lanes");
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned long long inc = wave_scan(v);
    __syncthreads();
    if (lane == 63) red[w] = inc;
    __syncthreads();
    const unsigned long long sums = row_scan(red[lane & 15]);
    total = lane_u64(sums, 15);
    return (w ? lane_u64(sums, w - 1) : 0) + inc - v;
}

// A row by one workgroup, whatever it holds: K by four passes of eight bits over the keys, each for
// top-k and top-p
template <typename T>
__device__ __attribute__((noinline)) void sample_row_general(const SampleArgs &p, int row, unsigned long long *red)
{
    __shared__ unsigned cnt[256];
    __shared__ unsigned long long mass[256];
    __shared__ unsigned s_key, s_ties;
    __shared__ unsigned long long s_mass;
    __shared__ float s_max[16];
    const int tid = threadIdx.x, lane = tid & 63;
    const T *x = (const T *)p.x + (long)row * p.ld;
    const int V = p.V;
    uint32_t kmax = 0;
    for (int i = tid; i < V; i += ST) kmax = max(kmax, logit_key(x, i));
    for (int o = 32; o; o >>= 1) kmax = max(kmax, (uint32_t)__shfl_xor((int)kmax, o, WAVE));
    if (lane == 0) s_max[tid >> 6] = __uint_as_float(kmax);
    __syncthreads();
    for (int i = 0; i < ST / 64; ++i) kmax = max(kmax, __float_as_uint(s_max[i]));
    if (kmax == 0u) {  // nothing above -inf
        if (tid == 0) {
            p.ids[row] = -1;
            if (p.logp) p.logp[row] = -INFINITY;
        }
        return;
    }
    const float temp = p.temp ? p.temp[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    SampleScale sc;
    sc.mx = key_value(kmax), sc.inf = key_value(kmax) == INFINITY, sc.unit = ldexp(1.0, p.shift), sc.inv_t = greedy ? 1.0 : temp;
    const int top_k = greedy ? 1 : p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.f;

    // kept: keys above K, and the first `ties` at K (in index order)
    uint32_t K = 1;  // (every key of a value above -inf)
    unsigned ties = 0xffffffffu;
    unsigned long long total = 0;
    // pass 0 finds K of top-k, pass 1 of top-p among those
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 0 && (top_k <= 0 || top_k >= V)) continue;
        double want = 0.0;
        if (pass == 1) {
            if (!(top_p < 1.f)) continue;
            // sum of what top-k keeps
            unsigned long long m = 0;
            unsigned eq = 0;
            for (int i = tid; i < V; i += ST) {
                const uint32_t k = logit_key(x, i);
                if (k > K) m += sample_mass(sc, k);
                else if (k == K) ++eq;
            }
            unsigned long long all, all_eq;
            block_scan(m, red, all);
            block_scan(eq, red, all_eq);
            all += min((unsigned long long)ties, all_eq) * sample_mass(sc, K);
            want = (double)top_p * (double)all;
        }
        uint32_t prefix = 0;                  // digits found so far
        unsigned long long above_m = 0;       // weight, count above the prefix's keys
        unsigned above_c = 0;
        for (int d = 24; d >= 0; d -= 8) {
            for (int i = tid; i < 256; i += ST) cnt[i] = 0, mass[i] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += ST) {
                const uint32_t k = logit_key(x, i);
                if (k < K || (d < 24 && (k >> (d + 8)) != (prefix >> (d + 8)))) continue;
                atomicAdd(&cnt[k >> d & 255], 1u);
                if (pass == 1) atomicAdd(&mass[k >> d & 255], sample_mass(sc, k));
            }
            __syncthreads();
            if (tid == 0) {
                // the highest digit whose keys and those above reach what is wanted; the weight of
                // K's own ties that top-k leaves out is not there
                int v = 255, last = -1;
                unsigned c = above_c;
                unsigned long long m = above_m;
                for (; v >= 0; --v) {
                    if (!cnt[v]) continue;
                    last = v;
                    if (pass == 0 ? c + cnt[v] >= (unsigned)top_k : (double)(m + mass[v]) >= want) break;
                    if (v == 0) break;
                    c += cnt[v], m += mass[v];
                }
                if (v < 0) {  // all of them: the lowest digit present
                    v = last;
                    c -= cnt[v], m -= mass[v];
                }
                s_key = prefix | (uint32_t)v << d, s_ties = c, s_mass = m;
            }
            __syncthreads();
            prefix = s_key, above_c = s_ties, above_m = s_mass;
            __syncthreads();
        }
        if (pass == 0) K = prefix, ties = (unsigned)top_k - above_c;
        else {
            // of the ties at the new K, as many as start below what is wanted (one at least if
            // nothing lies above)
            const unsigned long long each = sample_mass(sc, prefix);
            unsigned lim = prefix == K ? ties : 0xffffffffu;
            unsigned need = 0;
            if (each == 0) need = lim;
            else {
                const double q = ceil((want - (double)above_m) / (double)each);
                need = q >= 4294967295.0 ? 0xffffffffu : q < 1.0 ? 0u : (unsigned)q;
                while (need && (double)(above_m + (need - 1) * each) >= want) --need;
                while (need < 0xffffffffu && (double)(above_m + need * each) < want) ++need;
            }
            if (need == 0 && above_m == 0) need = 1;
            K = prefix, ties = min(lim, need);
        }
        __syncthreads();
    }
    const double min_p = p.min_p && p.min_p[row] > 0.f ? fmin((double)p.min_p[row], 1.0) : 0.0;

    // sums of contiguous ranges, one a wave; then the range that holds the target again
    const int w = tid >> 6, per = ((V + ST / 64 - 1) / (ST / 64) + 63) / 64 * 64;
    const int i0 = min(V, w * per), i1 = min(V, i0 + per);
    const bool tie_in = sample_w(sc, K) >= min_p;
    const unsigned long long each = tie_in ? sample_mass(sc, K) : 0;
    unsigned long long m = 0;
    unsigned eq = 0;
    for (int i = i0 + lane; i < i1; i += 64) {
        const uint32_t k = logit_key(x, i);
        if (k > K) {
            if (sample_w(sc, k) >= min_p) m += sample_mass(sc, k);
        } else if (k == K && k) ++eq;
    }
    for (int o = 32; o; o >>= 1) {
        m += __shfl_xor(m, o, WAVE);
        eq += __shfl_xor(eq, o, WAVE);
    }
    __shared__ unsigned long long wm[ST / 64];
    __shared__ unsigned we[ST / 64];
    if (lane == 0) wm[w] = m, we[w] = eq;
    __syncthreads();
    unsigned long long before = 0;
    unsigned eq_before = 0;
    for (int i = 0; i < ST / 64; ++i) {
        const unsigned in = eq_before >= ties ? 0 : min(ties - eq_before, we[i]);
        const unsigned long long t = wm[i] + in * each;
        if (i < w) before += t;
        total += t;
        if (i == w) m = t, eq = eq_before;
        eq_before += we[i];
    }
    float u = p.u[row];
    u = !(u > 0.f) ? 0.f : fminf(u, 0x1.fffffep-1f);
    const double target = (double)u * (double)total;
    if (!((double)before <= target && (double)(before + m) > target)) return;
    // one wave is left
    unsigned long long run = before;
    unsigned seen = eq;
    for (int i = i0; i < i1; i += 64) {
        const int at = i + lane;
        const uint32_t k = at < i1 ? logit_key(x, at) : 0u;
        const bool tie = k == K && k;
        const unsigned long long tied = __builtin_amdgcn_ballot_w64(tie);
        const unsigned rank = seen + __popcll(tied & ((1ull << lane) - 1));
        unsigned long long v = 0;
        if (k > K) v = sample_w(sc, k) >= min_p ? sample_mass(sc, k) : 0;
        else if (tie && rank < ties) v = each;
        unsigned long long inc = v;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long t = __shfl_up(inc, o, WAVE);
            if (lane >= o) inc += t;
        }
        const bool past = v && (double)(run + inc) > target;
        const unsigned long long hit = __builtin_amdgcn_ballot_w64(past);
        if (hit) {
            if (lane == __ffsll((long long)hit) - 1) {
                p.ids[row] = at;
                if (p.logp) p.logp[row] = (float)(sample_z(sc, key_value(k)) - log((double)total / sc.unit));
            }
            return;
        }
        run += __shfl(inc, 63, WAVE);
        seen += __popcll(tied);
    }
}

// Sorts the n <= CAP different entries of s to fall, by the whole workgroup: few by counting the
// larger ones of each, more by bitonic exchanges (s has room for the next power of two)
__device__ __forceinline__ void sort_falling(unsigned long long *s, int n)
{
    if (n <= 256) {  // a wave counts for 64 entries, over a quarter of the list
        const int i = threadIdx.x & 255, part = threadIdx.x >> 8;
        const unsigned long long e = i < n ? s[i] : 0;
        int rank = 0;
        if ((i & ~63) < n)
#pragma unroll 8
            for (int j = part; j < n; j += 4) rank += s[j] > e;
        __shared__ int ranks[256];
        if (part == 0) ranks[i] = rank;
        __syncthreads();
        if (part && rank) atomicAdd(&ranks[i], rank);
        __syncthreads();
        if (part == 0 && i < n) s[ranks[i]] = e;
        __syncthreads();
        return;
    }
    const int m = 1 << (32 - __builtin_clz(n - 1));
    for (int i = n + threadIdx.x; i < m; i += ST) s[i] = 0;
    for (int k = 2; k <= m; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < m / 2; i += ST) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const unsigned long long u = s[a], v = s[b];
                if ((u < v) == ((a & k) == 0)) s[a] = v, s[b] = u;
            }
        }
    __syncthreads();
}

// Entries of a list of logits: key and index, falling by key, then rising by index
__device__ __forceinline__ unsigned long long list_entry(uint32_t key, int i) { return (unsigned long long)key << 32 | (uint32_t)~i; }
__device__ __forceinline__ uint32_t entry_key(unsigned long long e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ int entry_index(unsigned long long e) { return (int)~(uint32_t)e; }

struct FinishShared {
    unsigned long long list[CAP];
    unsigned long long sums[NB];
    unsigned long long red[ST / 64], sum[2];
    unsigned tie[MAX_CHUNKS], n;
    int at[4];
};
static_assert(NB >= ST && NB <= 2 * ST && MAX_CHUNKS <= ST, "a bin or two, and a chunk, a thread");

// False: the row is one for sample_row_general
template <typename T>
__device__ __forceinline__ bool sample_finish(const SampleArgs &p, int row, FinishShared &sh)
{
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const T *x = (const T *)p.x + (long)row * p.ld;
    const SampleRow r = sample_row(p, row);
    uint32_t kmax;
    int imax;
    row_max_key(p, row, kmax, imax);
    if (kmax == 0u) {  // nothing above -inf
        if (tid == 0) {
            p.ids[row] = -1;
            if (p.logp) p.logp[row] = -INFINITY;
        }
        return true;
    }
    const float mx = key_value(kmax);
    if (r.greedy) {
        if (tid == 0) {
            p.ids[row] = imax;
            if (p.logp) p.logp[row] = 0.f;
        }
        return true;
    }
    if (mx == INFINITY || !r.plain || r.top_k > SMALL_K) return false;
    const SampleScale sc = {(double)mx, (double)r.temp, ldexp(1.0, p.shift), false};
    const unsigned long long *hist = p.hist + (long)row * p.C * NB;
    auto logit = [&](int i) {
        float v;
        if constexpr (sizeof(T) == 4) v = x[i];
        else v = bf16_to_f32(x[i]);
        return fmaxf(v, -INFINITY);
    };
    // The logits of bins lo .. hi, in any order (false: too many).  A thread marks its logits by two
    // comparisons each (a little outside the bins' edges) and looks again at the few it marked.
    int n = 0;
    auto gather = [&](int lo, int hi) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        const float vtop = bin_top(mx, lo), vbottom = bin_bottom(mx, hi);
        auto look = [&](int at) {
            const float v = logit(at);
            const int b = sample_bin(mx - v);
            if (b >= lo && b <= hi && v > -INFINITY) {
                const unsigned k = atomicAdd(&sh.n, 1u);
                if (k < CAP) sh.list[k] = list_entry(sample_key(v), at);
            }
        };
        constexpr int E = 16 / sizeof(T), U = 32 / E;  // 32 logits a thread and batch
        const int head = min(p.V, logits_before_16(x)), whole = head + (p.V - head) / E * E;
        if (tid < head) look(tid);
        for (int at0 = head + tid * E; at0 < whole; at0 += U * ST * E) {
            u32x4 v[U];
#pragma unroll
            for (int k = 0; k < U; ++k) v[k] = *(const u32x4 *)(x + min(at0 + k * ST * E, whole - E));
            unsigned marks = 0;
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float f;
                    if constexpr (sizeof(T) == 4) f = __uint_as_float(v[k][e]);
                    else f = __uint_as_float(e % 2 ? v[k][e / 2] & 0xffff0000u : v[k][e / 2] << 16);
                    marks |= (unsigned)(f >= vbottom && f <= vtop) << (k * E + e);
                }
            for (; marks; marks &= marks - 1) {
                const int bit = __builtin_ctz(marks), at = at0 + bit / E * (ST * E) + bit % E;
                if (at < whole) look(at);  // (past the end the last vector was read again)
            }
        }
        if (whole + tid < p.V) look(whole + tid);
        __syncthreads();
        n = (int)sh.n;
        return n <= CAP;
    };
    // the chunks' bins together, and the bin where their sum reaches what is wanted
    unsigned long long total = 0;
    if (tid == 0) sh.at[0] = -1;
    {
        typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
        unsigned long long a = 0, b = 0;  // bins 2 tid, 2 tid + 1
        if (2 * tid < NB)
            for (int c = 0; c < p.C; c += 8) {
                u64x2 h[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) h[k] = c + k < p.C ? *(const u64x2 *)(hist + (long)(c + k) * NB + 2 * tid) : u64x2{0, 0};
#pragma unroll
                for (int k = 0; k < 8; ++k) a += h[k][0], b += h[k][1];
            }
        const unsigned long long before = block_scan(a + b, sh.red, total);
        const double want = r.top_k ? (double)r.top_k : (double)r.top_p * (double)total;
        if (r.top_k || r.top_p < 1.f) {  // (one thread finds it)
            if (a && ((double)before < want || before == 0) && (double)(before + a) >= want) sh.at[0] = 2 * tid, sh.sum[0] = before;
            else if (b && ((double)(before + a) < want || before + a == 0) && (double)(before + a + b) >= want) sh.at[0] = 2 * tid + 1, sh.sum[0] = before + a;
        }
        __syncthreads();
    }
    if (r.top_k) {  // few: all that top-k keeps, in LDS
        // (fewer logits above -inf than top_k: all of them)
        if (!gather(0, sh.at[0] < 0 ? NB - 1 : sh.at[0])) return false;
        sort_falling(sh.list, n);
        const int kept = min(n, r.top_k);
        const unsigned long long e = tid < kept ? sh.list[tid] : 0;
        const float v = key_value(entry_key(e));
        unsigned long long wt = tid < kept ? sample_weight(v, mx, r.c, p.shift) : 0, all;
        const unsigned long long before = block_scan(wt, sh.red, all);
        if (r.top_p < 1.f && tid > 0 && !((double)before < (double)r.top_p * (double)all)) wt = 0;
        if (r.min_p > 0.0 && tid < kept && !(exp(sample_z(sc, v)) >= r.min_p)) wt = 0;
        // in index order
        if (tid < kept) sh.list[tid] = (unsigned long long)(uint32_t)~entry_index(e) << 32 | (uint32_t)tid;
        sh.sums[tid] = wt;
        __syncthreads();
        sort_falling(sh.list, kept);
        const unsigned long long f = tid < kept ? sh.list[tid] : 0;
        wt = tid < kept ? sh.sums[(uint32_t)f] : 0;
        const unsigned long long upto = block_scan(wt, sh.red, all) + wt;
        const double target = r.u * (double)all;
        if (wt && (double)upto > target && !((double)(upto - wt) > target)) {
            const int at = (int)~(uint32_t)(f >> 32);
            p.ids[row] = at;
            if (p.logp) p.logp[row] = (float)(sample_z(sc, logit(at)) - log((double)all / sc.unit));
        }
        return true;
    }

    // The cut: bins below lo are kept whole, those of lo .. hi logit by logit (keys above K, the first
    // `ties` at K, weights of at least min_p), the rest not
    int lo = NB, hi = NB - 1;
    uint32_t K = 0;
    unsigned ties = 0;
    constexpr int PER = CAP / ST;
    if (r.top_p < 1.f) {
        lo = hi = sh.at[0];
        unsigned long long above = sh.sum[0];
        if (lo < 0 || !gather(lo, hi)) return false;
        const double want = (double)r.top_p * (double)total;
        // K: the keys between the bin's edges cut into 1024 parts, then the part that reaches what
        // is wanted, until a part is one key (bf16: of 16 bits)
        constexpr int KS = sizeof(T) == 2 ? 16 : 0;
        uint32_t key[PER];
        unsigned long long wt[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = tid + k * ST;
            key[k] = i < n ? entry_key(sh.list[i]) : 0;
            wt[k] = i < n ? sample_weight(key_value(key[k]), mx, r.c, p.shift) : 0;
            key[k] >>= KS;
        }
        uint32_t khi = sample_key(bin_top(mx, lo)) >> KS, klo = max(sample_key(bin_bottom(mx, lo)) >> KS, 1u);
        while (true) {
            const int shift = klo == khi ? 0 : max(0, 22 - __builtin_clz(khi - klo));  // (khi - klo) >> shift < 1024
            sh.sums[tid] = 0;
            if (tid == 0) sh.at[1] = -1;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (wt[k] && key[k] >= klo && key[k] <= khi) atomicAdd(&sh.sums[(khi - key[k]) >> shift], wt[k]);
            __syncthreads();
            const unsigned long long a = sh.sums[tid];
            unsigned long long all;
            const unsigned long long before = above + block_scan(a, sh.red, all);
            if (a && ((double)before < want || before == 0) && (double)(before + a) >= want) sh.at[1] = tid, sh.sum[0] = before;
            __syncthreads();
            const int part = sh.at[1];
            if (part < 0) return false;
            above = sh.sum[0];
            khi -= (uint32_t)part << shift;
            klo = max(klo, khi - min(khi, (1u << shift) - 1));
            if (shift == 0) break;
            __syncthreads();
        }
        K = KS ? klo << KS | (klo >> 15 ? 0u : 0xffffu) : klo;  // (negative values' keys are complements)
        // of K's equals, as many as start below what is wanted; one at least where nothing lies above
        const unsigned long long each = sample_weight(key_value(K), mx, r.c, p.shift);
        const double q = each ? ceil((want - (double)above) / (double)each) : 0.0;
        ties = q < 1.0 ? 0u : q > (double)p.V ? (unsigned)p.V : (unsigned)q;
        while (ties && !((double)(above + (ties - 1) * each) < want)) --ties;
        while (each && ties < (unsigned)p.V && (double)(above + ties * each) < want) ++ties;
        if (ties == 0 && above == 0) ties = 1;
    }
    int mlo = NB;  // from this bin on weights are compared with min_p
    if (r.min_p > 0.0) {
        const double d = -(double)r.temp * log(r.min_p);
        mlo = max(0, sample_bin((float)(d * (1 - 0x1p-20))) - 1);
        const int mhi = min(sample_bin((float)(d * (1 + 0x1p-20))) + 1, NB - 1);
        const int nlo = min(lo, mlo), nhi = min(hi, mhi);
        if (nlo != lo || nhi != hi) {
            lo = nlo, hi = nhi;
            if (!gather(lo, hi)) return false;
        }
    }
    const auto heavy = [&](float v, int bin) { return !(r.min_p > 0.0 && bin >= mlo) || exp(sample_z(sc, v)) >= r.min_p; };
    // what each chunk keeps: its bins below the cut, the cut's keys above K, and its share of the ties
    __syncthreads();
    for (int c = w; c < p.C; c += ST / 64) {
        unsigned long long t = 0, h[NB / 64];
#pragma unroll
        for (int k = 0; k < NB / 64; ++k) h[k] = lane + 64 * k < lo ? hist[(long)c * NB + lane + 64 * k] : 0;
#pragma unroll
        for (int k = 0; k < NB / 64; ++k) t += h[k];
        t = wave_scan(t);
        if (lane == 63) sh.sums[c] = t, sh.tie[c] = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += ST) {
        const unsigned long long e = sh.list[i];
        const uint32_t key = entry_key(e);
        const float v = key_value(key);
        const int c = entry_index(e) / p.chunk;
        if (key < K || !heavy(v, sample_bin(mx - v))) continue;
        if (key == K) atomicAdd(&sh.tie[c], 1u);
        else atomicAdd(&sh.sums[c], sample_weight(v, mx, r.c, p.shift));
    }
    __syncthreads();
    unsigned long long mine = 0, tied;
    {
        const unsigned t = tid < p.C ? sh.tie[tid] : 0;
        const unsigned long long before = block_scan(t, sh.red, tied);
        if (tid < p.C) {
            mine = sh.sums[tid];
            if (t && before < ties) mine += (unsigned long long)min(t, ties - (unsigned)before) * sample_weight(key_value(K), mx, r.c, p.shift);
            sh.tie[tid] = (unsigned)before;
        }
    }
    const unsigned long long start = block_scan(mine, sh.red, total);
    const double target = r.u * (double)total;
    if (mine && !((double)start > target) && (double)(start + mine) > target) sh.at[3] = tid, sh.sum[1] = start;
    __syncthreads();
    // That chunk's logits, a stretch of neighbours a thread: what each keeps, the thread that holds
    // the target, and then its logits by the lanes of its wave.
    const int c0 = sh.at[3] * p.chunk, c1 = min(p.V, c0 + p.chunk);
    constexpr int Q = 16;  // a stretch; chunks of up to 16384 logits
    const int i0 = c0 + tid * Q;
    // a logit's weight if it is kept, or whether it is one of K's equals that count; most are
    // above or below the cut's bins for certain
    const float sure = lo == NB ? -INFINITY : bin_top(mx, lo), never = lo == NB ? -INFINITY : bin_bottom(mx, hi);
    auto weigh = [&](float v, bool &tie) {
        bool in = v > sure;
        tie = false;
        if (v <= sure && v >= never && v > -INFINITY) {
            const uint32_t key = sample_key(v);
            const int bin = sample_bin(mx - v);
            in = bin < lo || (bin <= hi && key >= K && heavy(v, bin));
            tie = in && bin >= lo && K && key == K;
        }
        return in && !tie ? sample_weight(v, mx, r.c, p.shift) : 0ull;
    };
    unsigned long long m = 0;
    unsigned t = 0;
    if (i0 < c1) {
        float v[Q];
        if (p.vec && i0 + Q <= c1) {
            constexpr int E = 16 / sizeof(T);
#pragma unroll
            for (int k = 0; k < Q / E; ++k) {
                const u32x4 u = *(const u32x4 *)(x + i0 + k * E);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if constexpr (sizeof(T) == 4) v[k * E + e] = __uint_as_float(u[e]);
                    else v[k * E + e] = __uint_as_float(e % 2 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
                    v[k * E + e] = fmaxf(v[k * E + e], -INFINITY);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < Q; ++k) v[k] = i0 + k < c1 ? logit(i0 + k) : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            bool tie;
            m += weigh(v[k], tie);
            t += tie;
        }
    }
    const unsigned long long each = K ? sample_weight(key_value(K), mx, r.c, p.shift) : 0;
    unsigned seen = sh.tie[sh.at[3]];  // K's equals before this stretch
    if (each) {
        unsigned long long all;
        seen += (unsigned)block_scan(t, sh.red, all);
        m += (seen < ties ? min(t, ties - seen) : 0) * each;
    }
    unsigned long long all;
    const unsigned long long run = sh.sum[1] + block_scan(m, sh.red, all);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(m && !((double)run > target) && (double)(run + m) > target);
    if (!hit) return true;
    {  // one wave is left: lane k has the stretch's logit k
        const int from = __builtin_ctzll(hit), at = __builtin_amdgcn_readlane(i0, from) + lane;
        const unsigned before = (unsigned)__builtin_amdgcn_readlane((int)seen, from);
        const unsigned long long base = lane_u64(run, from);
        const float v = lane < Q && at < c1 ? logit(at) : -INFINITY;
        bool tie;
        unsigned long long wt = weigh(v, tie);
        const unsigned long long eq = __builtin_amdgcn_ballot_w64(tie);
        if (tie && before + __popcll(eq & ((1ull << lane) - 1)) < ties) wt = each;
        const unsigned long long inc = row_scan(wt);
        const unsigned long long past = __builtin_amdgcn_ballot_w64(wt && (double)(base + inc) > target);
        if (past && lane == __builtin_ctzll(past)) {
            p.ids[row] = at;
            if (p.logp) p.logp[row] = (float)(sample_z(sc, v) - log((double)total / sc.unit));
        }
    }
    return true;
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_finish_kernel(const SampleArgs p)
{
    __shared__ FinishShared sh;
    if (!sample_finish<T>(p, blockIdx.x, sh)) {
        __syncthreads();
        sample_row_general<T>(p, blockIdx.x, sh.red);
    }
}

} // namespace jas

using namespace jas;

// Chunks of a row: of 4096 logits (a histogram of 12 KB each) up to 16384 (what the last step
// walks at once), as many as give some 1024 workgroups one
static void sample_chunks(int n, int V, int &C, int &chunk)
{
    C = std::max(std::min((1024 + n - 1) / n, (V + 4095) / 4096), (V + 16383) / 16384);
    chunk = ((V + C - 1) / C + 1023) / 1024 * 1024;
    C = (V + chunk - 1) / chunk;
}

extern "C" {

size_t jas_sample_workspace(int n, int V)
{
    if (n <= 0 || V <= 0 || V > 1 << 22) return 0;
    // chunks of all rows, at most (sample_chunks), and of every call of fewer or shorter ones
    const size_t rows = n, most = std::max(rows * ((V + 16383) / 16384), std::min(rows + 1023, rows * ((V + 4095) / 4096)));
    return most * (NB * sizeof(unsigned long long) + 2 * sizeof(uint32_t));
}

jas_status jas_sample(const void *x, int n, int V, int64_t ld, const float *temp, const int32_t *top_k, const float *top_p,
                      const float *min_p, const float *u, int32_t *ids, float *logp, int dtype, void *work, jas_stream_t stream)
{
    JAS_CHECK(x && u && ids, JAS_ERR_INVALID, "jas_sample: null logits, u or ids");
    JAS_CHECK(n >= 0 && V > 0 && V <= 1 << 22 && ld >= V, JAS_ERR_INVALID, "jas_sample: need n >= 0, V of 1 to 2^22 and ld >= V");
    JAS_CHECK(dtype == JAS_F32 || dtype == JAS_BF16, JAS_ERR_INVALID, "jas_sample: logits are JAS_F32 or JAS_BF16");
    JAS_CHECK((uintptr_t)x % (dtype == JAS_F32 ? 4 : 2) == 0, JAS_ERR_INVALID, "jas_sample: logits aligned to their elements");
    JAS_CHECK(((uintptr_t)temp | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)u | (uintptr_t)ids | (uintptr_t)logp) % 4 == 0,
              JAS_ERR_INVALID, "jas_sample: rows' values aligned to 4 bytes");
    if (!n) return JAS_OK;
    JAS_CHECK(n <= 65535, JAS_ERR_INVALID, "jas_sample: at most 65535 rows");
    JAS_CHECK(work && (uintptr_t)work % 16 == 0, JAS_ERR_INVALID, "jas_sample: need a workspace aligned to 16 bytes");
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    SampleArgs p{};
    p.x = x, p.n = n, p.V = V, p.shift = std::min(51, 62 - bits), p.ld = (long)ld;
    p.temp = temp, p.top_k = top_k, p.top_p = top_p, p.min_p = min_p, p.u = u, p.ids = ids, p.logp = logp;
    sample_chunks(n, V, p.C, p.chunk);
    p.vec = (uintptr_t)x % 16 == 0 && ld * (dtype == JAS_F32 ? 4 : 2) % 16 == 0;
    p.hist = (unsigned long long *)work;
    p.chunk_key = (uint32_t *)(p.hist + (size_t)n * p.C * NB);
    p.chunk_idx = (int32_t *)(p.chunk_key + (size_t)n * p.C);
    hipStream_t s = stream_or_default(stream);
    const dim3 grid(p.C, n);
    if (dtype == JAS_F32) {
        hipLaunchKernelGGL(sample_max_kernel<float>, grid, dim3(256), 0, s, p);
        hipLaunchKernelGGL(sample_hist_kernel<float>, grid, dim3(256), 0, s, p);
        hipLaunchKernelGGL(sample_finish_kernel<float>, dim3(n), dim3(ST), 0, s, p);
    } else {
        hipLaunchKernelGGL(sample_max_kernel<uint16_t>, grid, dim3(256), 0, s, p);
        hipLaunchKernelGGL(sample_hist_kernel<uint16_t>, grid, dim3(256), 0, s, p);
        hipLaunchKernelGGL(sample_finish_kernel<uint16_t>, dim3(n), dim3(ST), 0, s, p);
    }
    JAS_LAUNCH_CHECK();
    return JAS_OK;
}

} // extern "C"
