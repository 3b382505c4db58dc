// One token for each row of logits: temperature, top-k, top-p, min-p, and the draw from a given
// uniform number.
//
// Weights w = 2^shift exp((x - max) / T) are rounded to whole numbers (shift so that V of them fit
// 62 bits: 46 at 50257 logits), so sums are exact in any order and a threshold found by adding
// bins is the one found by adding values one by one.  The order by falling value, lowest index first
// among equals, is that of a whole-number key of the value; the kept set is always "keys above K,
// and the first `ties` at K", so no row is sorted: K is found digit by digit from histograms of
// counts (top-k) and of weights (top-p).
#include "jas_common.hpp"

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

constexpr int ST = 1024;  // threads of a row

// first of the ST threads' 64-bit sums in thread order: exclusive prefix and total
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long *red, unsigned long long &total)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned long long inc = v;
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long t = __shfl_up(inc, o, WAVE);
        if (lane >= o) inc += t;
    }
    __syncthreads();
    if (lane == 63) red[w] = inc;
    __syncthreads();
    unsigned long long before = 0, all = 0;
    for (int i = 0; i < ST / 64; ++i) {
        if (i < w) before += red[i];
        all += red[i];
    }
    total = all;
    return before + inc - v;
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_kernel(const SampleArgs p)
{
    __shared__ unsigned cnt[256];
    __shared__ unsigned long long mass[256], red[ST / 64];
    __shared__ unsigned s_key, s_ties;
    __shared__ unsigned long long s_mass;
    __shared__ float s_max[16];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
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

} // namespace jas

using namespace jas;

extern "C" {

size_t jas_sample_workspace(int n, int V) { return 0; }

jas_status jas_sample(const void *x, int n, int V, int64_t ld, const float *temp, const int32_t *top_k, const float *top_p,
                      const float *min_p, const float *u, int32_t *ids, float *logp, int dtype, void *work, jas_stream_t stream)
{
    JAS_CHECK(x && u && ids, JAS_ERR_INVALID, "jas_sample: null logits, u or ids");
    JAS_CHECK(n >= 0 && V > 0 && V <= 1 << 22 && ld >= V, JAS_ERR_INVALID, "jas_sample: need n >= 0, V of 1 to 2^22 and ld >= V");
    JAS_CHECK(dtype == JAS_F32 || dtype == JAS_BF16, JAS_ERR_INVALID, "jas_sample: logits are JAS_F32 or JAS_BF16");
    JAS_CHECK((uintptr_t)x % (dtype == JAS_F32 ? 4 : 2) == 0, JAS_ERR_INVALID, "jas_sample: logits aligned to their elements");
    if (!n) return JAS_OK;
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    SampleArgs p{x, n, V, std::min(52, 62 - bits), (long)ld, temp, top_p, min_p, u, top_k, ids, logp};
    hipStream_t s = stream_or_default(stream);
    if (dtype == JAS_F32) hipLaunchKernelGGL(sample_kernel<float>, dim3(n), dim3(ST), 0, s, p);
    else hipLaunchKernelGGL(sample_kernel<uint16_t>, dim3(n), dim3(ST), 0, s, p);
    JAS_LAUNCH_CHECK();
    return JAS_OK;
}

} // extern "C"
