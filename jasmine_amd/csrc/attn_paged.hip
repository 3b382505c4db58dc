// Attention of a ragged batch's rows over the paged cache: decode steps and chunks of prompts.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = 2^(scale log2(e) q . k_t - m), over the keys t that the
// row sees; one pass over the keys with the running maximum m and sum, in fp32.
#include "paged.hpp"

#include <cfloat>

namespace jas {

struct PagedAttnArgs {
    const void *q;
    void *o;
    PagedView kv;
    BatchView bt;
    int H, G, max_len, causal;  // G: query heads per key head
    FastDiv by_group;
    long q_st, q_sh, o_st, o_sh;
    float scale_log2;
};

template <int CK>
constexpr int cache_bytes = CK == CK_F32 ? 4 : CK == CK_BF16 ? 2 : 1;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Sequence b of the batch: its rows, and its length with them
struct PagedSeq {
    int row0, rows, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnArgs &p, int b)
{
    PagedSeq s;
    s.row0 = max(0, min(p.bt.cu[b], p.bt.n));
    s.rows = max(0, min(p.bt.cu[b + 1], p.bt.n) - s.row0);
    s.len = max(0, min(p.bt.lens[b], min(p.kv.cap, p.max_len)));
    return s;
}

// Where key t of sequence b lies: its page (-1: none) and slot
__device__ __forceinline__ int paged_page(const PagedAttnArgs &p, int b, int t, int &slot)
{
    const int q = (int)p.kv.by_page.div((uint32_t)t);
    slot = t - q * p.kv.page_size;
    const int page = p.kv.table[(long)b * p.kv.table_stride + q];
    return page >= 0 && page < p.kv.n_pages ? page : -1;
}

template <int CK>
__device__ __forceinline__ float cache_value(const void *pool, long at)
{
    if constexpr (CK == CK_F32) return ((const float *)pool)[at];
    else if constexpr (CK == CK_BF16) return bf16_to_f32(((const uint16_t *)pool)[at]);
    else if constexpr (CK == CK_I8) return (float)((const int8_t *)pool)[at];
    else return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)pool)[at], 0);
}

// One query row in fp32 arithmetic by one wave: keys [k_lo, k_hi) of sequence b, head hk; q: the
// row's D values in fp32 (LDS).  Every lane holds the maximum m (exponent units) and the sum l of
// the weights; out: elements lane + 64 e of the weighted mean of the values.  A mean of numbers
// near the end of fp32 is one itself though their sum is not: acc2 adds them times 2^-32.
template <int D, int CK>
__device__ __attribute__((noinline)) void paged_row(const PagedAttnArgs &p, int b, int hk, const float *q, int k_lo, int k_hi,
                                                    float &m, float &l, float (&out)[(D + 63) / 64])
{
    const int lane = threadIdx.x & 63;
    constexpr int E = (D + 63) / 64;
    float acc[E], acc2[E];
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc2[e] = 0.f;
    for (int k0 = k_lo; k0 < k_hi; k0 += 64) {
        const int t = k0 + lane;
        int slot = 0, page = -1;
        if (t < k_hi) page = paged_page(p, b, t, slot);
        const bool sees = page >= 0;
        const long at = (long)page * p.kv.page_stride + hk * p.kv.head_stride + slot * p.kv.tok_stride;
        const long sc = ((long)page * p.kv.n_kv + hk) * p.kv.page_size + slot;
        float s = -INFINITY, vs = 1.f;
        if (sees) {
            float d = 0.f;
            for (int e = 0; e < D; ++e) d = __builtin_fmaf(q[e], cache_value<CK>(p.kv.k, at + e), d);
            if (CK >= CK_I8) d *= p.kv.ks[sc], vs = p.kv.vs[sc];
            s = d * p.scale_log2;
        }
        const float mx = fmaxf(m, wave_max(s)), base = mx == -INFINITY ? 0.f : mx;
        const float corr = exp2_fast(m - base), pv = sees ? exp2_fast(s - base) : 0.f;
        l = l * corr + wave_sum(pv);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= corr, acc2[e] *= corr;
        const unsigned long long seen = __builtin_amdgcn_ballot_w64(sees);
        for (int k = 0; k < 64; ++k) {
            if (!(seen >> k & 1)) continue;
            const float pk = __shfl(pv, k, WAVE) * __shfl(vs, k, WAVE);
            const long vat = __shfl(at, k, WAVE);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane + 64 * e < D) {
                    const float v = cache_value<CK>(p.kv.v, vat + lane + 64 * e);
                    acc[e] = __builtin_fmaf(pk, v, acc[e]);
                    acc2[e] = __builtin_fmaf(pk, v * 0x1p-32f, acc2[e]);
                }
        }
        m = mx;
    }
    const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = fabsf(acc[e]) <= FLT_MAX ? acc[e] * inv : acc2[e] * inv * 0x1p32f;
}

// Four rows (token, query head) of the batch a workgroup, one a wave
template <int D, int CK, typename T>
__global__ void __launch_bounds__(256) paged_row_kernel(const PagedAttnArgs p)
{
    __shared__ float qs[4][D];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long id = (long)blockIdx.x * 4 + w;
    const int h = (int)(id % p.H);
    const long tok = id / p.H;
    if (tok >= p.bt.n) return;
    int lo = 0, hi = p.bt.B;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.bt.cu[mid] <= tok) lo = mid;
        else hi = mid - 1;
    }
    const int b = lo;
    if (b >= p.bt.B || p.bt.cu[b] > tok) return;
    const PagedSeq sq = paged_seq(p, b);
    const T *qr = (const T *)p.q + tok * p.q_st + h * p.q_sh;
    for (int e = lane; e < D; e += 64) {
        if constexpr (sizeof(T) == 4) qs[w][e] = qr[e];
        else qs[w][e] = bf16_to_f32(qr[e]);
    }
    __builtin_amdgcn_wave_barrier();
    const int pos = sq.len - sq.rows + (int)(tok - sq.row0);
    float m, l, acc[(D + 63) / 64];
    paged_row<D, CK>(p, b, h / p.G, qs[w], 0, p.causal ? min(sq.len, pos + 1) : sq.len, m, l, acc);
    T *o = (T *)p.o + tok * p.o_st + h * p.o_sh;
    for (int e = 0; e < (D + 63) / 64; ++e)
        if (lane + 64 * e < D) {
            if constexpr (sizeof(T) == 4) o[lane + 64 * e] = acc[e];
            else o[lane + 64 * e] = __builtin_bit_cast(uint16_t, (__bf16)acc[e]);
        }
}

template <int D, int CK, typename T>
static void paged_launch(const PagedAttnArgs &p, hipStream_t s)
{
    hipLaunchKernelGGL((paged_row_kernel<D, CK, T>), dim3(ceil_div((long)p.bt.n * p.H, 4)), dim3(256), 0, s, p);
}
template <int D>
static void paged_launch(const PagedAttnArgs &p, int cache, int dtype, hipStream_t s)
{
    if (dtype == JAS_F32) {
        if (cache == JAS_F32) paged_launch<D, CK_F32, float>(p, s);
        else if (cache == JAS_BF16) paged_launch<D, CK_BF16, float>(p, s);
        else if (cache == JAS_I8) paged_launch<D, CK_I8, float>(p, s);
        else paged_launch<D, CK_F8, float>(p, s);
    } else {
        if (cache == JAS_BF16) paged_launch<D, CK_BF16, uint16_t>(p, s);
        else if (cache == JAS_I8) paged_launch<D, CK_I8, uint16_t>(p, s);
        else paged_launch<D, CK_F8, uint16_t>(p, s);
    }
}

} // namespace jas

using namespace jas;

extern "C" {

size_t jas_attn_paged_workspace(int n, int B, int H, int n_kv, int dh, int max_q, int max_len) { return 0; }

jas_status jas_attn_paged(const void *q, void *o, const jas_paged_kv *kv, int n, int B, const int32_t *cu, const int32_t *lens,
                          int H, int max_q, int max_len, int64_t q_st, int64_t q_sh, int64_t o_st, int64_t o_sh, float scale,
                          int causal, int dtype, void *work, jas_stream_t stream)
{
    PagedAttnArgs p;
    jas_status rc = paged_view(kv, p.kv, "jas_attn_paged");
    if (rc != JAS_OK) return rc;
    rc = batch_view(n, B, cu, lens, p.bt, "jas_attn_paged");
    if (rc != JAS_OK) return rc;
    JAS_CHECK(q && o, JAS_ERR_INVALID, "jas_attn_paged: null q or o");
    JAS_CHECK(dtype == JAS_F32 || dtype == JAS_BF16, JAS_ERR_INVALID, "jas_attn_paged: rows are JAS_F32 or JAS_BF16");
    JAS_CHECK(dtype == JAS_F32 || kv->dtype != JAS_F32, JAS_ERR_INVALID, "jas_attn_paged: JAS_BF16 rows over a JAS_F32 cache");
    JAS_CHECK(H > 0 && H % kv->n_kv == 0, JAS_ERR_INVALID, "jas_attn_paged: H is a multiple of the cache's heads");
    JAS_CHECK(max_q >= 0 && max_len >= 0, JAS_ERR_INVALID, "jas_attn_paged: max_q and max_len are not negative");
    JAS_CHECK(((uintptr_t)q | (uintptr_t)o) % dtype_bytes(dtype) == 0, JAS_ERR_INVALID, "jas_attn_paged: rows aligned to their elements");
    JAS_CHECK((long)n * H <= 0x7fffffffl, JAS_ERR_RANGE, "jas_attn_paged: too many rows for one call");
    if (!n || !B) return JAS_OK;
    p.q = q, p.o = o, p.H = H, p.G = H / kv->n_kv, p.max_len = max_len, p.causal = causal != 0;
    p.by_group.set((uint32_t)p.G);
    p.q_st = q_st, p.q_sh = q_sh, p.o_st = o_st, p.o_sh = o_sh;
    p.scale_log2 = scale * 1.44269504088896340736f;
    hipStream_t s = stream_or_default(stream);
    if (kv->dh == 32) paged_launch<32>(p, kv->dtype, dtype, s);
    else if (kv->dh == 64) paged_launch<64>(p, kv->dtype, dtype, s);
    else paged_launch<128>(p, kv->dtype, dtype, s);
    JAS_LAUNCH_CHECK();
    return JAS_OK;
}

} // extern "C"
