// The paged key/value cache: rows written (and quantised to 8 bits on the way) and read back.
//
// A row is one token's dh values of one head.  The 8-bit types keep codes c and one fp32 scale
// s = max |x| / qmax; c = x / s rounded once, to nearest even, which the division's own rounding
// must not disturb: bf16 rows often put x / s within 2^-24 of a tie.  So the quotient is formed
// rounded to odd (cut towards zero, last bit set where anything was cut: quotient_to_odd), and the
// conversion's rounding is then the only one.
//
// Both kernels move each byte once: 16 bytes (8 values) a lane, dh / 8 lanes a row, the row's
// maximum met in registers.  Bound by memory; a decode step's few rows by the launch.  8 prompts of up to
// 2048 tokens, 8 heads of 128, fp32 to int8 and back: 268 MB in 62 us (4.3 TB/s; a copy of 1 GiB: 5.1); 61
// single tokens, bf16 to e4m3 and back: 9.5 us, the two launches.
#include "paged.hpp"

#include <cmath>

namespace jas {

jas_status paged_view(const jas_paged_kv *kv, PagedView &v, const char *who)
{
    JAS_CHECK(kv, JAS_ERR_INVALID, std::string(who) + ": null cache");
    JAS_CHECK(kv->d_k && kv->d_v && kv->d_table, JAS_ERR_INVALID, std::string(who) + ": null pool or table");
    JAS_CHECK(kv->dtype == JAS_F32 || kv->dtype == JAS_BF16 || dtype_eight(kv->dtype), JAS_ERR_INVALID,
              std::string(who) + ": the cache holds JAS_F32, JAS_BF16, JAS_I8 or JAS_F8E4M3");
    JAS_CHECK(!dtype_eight(kv->dtype) || (kv->d_k_scale && kv->d_v_scale), JAS_ERR_INVALID, std::string(who) + ": an 8-bit cache needs its scales");
    JAS_CHECK(kv->dh == 32 || kv->dh == 64 || kv->dh == 128, JAS_ERR_INVALID, std::string(who) + ": dh is 32, 64 or 128");
    JAS_CHECK(kv->n_pages > 0 && kv->page_size > 0 && kv->n_kv > 0 && kv->max_pages > 0 && kv->table_stride >= 0, JAS_ERR_INVALID,
              std::string(who) + ": n_pages, page_size, n_kv and max_pages are positive, table_stride is not negative");
    JAS_CHECK(kv->page_size <= 1 << 20, JAS_ERR_INVALID, std::string(who) + ": pages of at most 2^20 tokens");
    const long es = (long)dtype_bytes(kv->dtype);
    JAS_CHECK(kv->page_stride >= 0 && kv->head_stride >= 0 && kv->tok_stride >= kv->dh, JAS_ERR_INVALID,
              std::string(who) + ": strides are not negative, and tokens at least dh apart");
    JAS_CHECK(((uintptr_t)kv->d_k | (uintptr_t)kv->d_v) % 16 == 0 && kv->page_stride * es % 16 == 0 &&
                  kv->head_stride * es % 16 == 0 && kv->tok_stride * es % 16 == 0,
              JAS_ERR_INVALID, std::string(who) + ": rows of the cache start on 16 bytes");
    JAS_CHECK(((uintptr_t)kv->d_table | (uintptr_t)kv->d_k_scale | (uintptr_t)kv->d_v_scale) % 4 == 0, JAS_ERR_INVALID,
              std::string(who) + ": table and scales aligned to 4 bytes");
    v.k = kv->d_k, v.v = kv->d_v, v.ks = kv->d_k_scale, v.vs = kv->d_v_scale, v.table = kv->d_table;
    v.page_stride = kv->page_stride, v.head_stride = kv->head_stride, v.tok_stride = kv->tok_stride;
    v.table_stride = kv->table_stride, v.n_pages = kv->n_pages, v.page_size = kv->page_size, v.n_kv = kv->n_kv;
    const long cap = (long)kv->max_pages * kv->page_size;
    v.cap = (int)(cap < 0x7fff0000l ? cap : 0x7fff0000l);  // (a tile past the end stays below 2^31)
    v.by_page.set((uint32_t)kv->page_size);
    return JAS_OK;
}

jas_status batch_view(int n, int B, const int32_t *cu, const int32_t *lens, BatchView &v, const char *who)
{
    JAS_CHECK(n >= 0 && B >= 0, JAS_ERR_INVALID, std::string(who) + ": n and B are not negative");
    JAS_CHECK(B == 0 || (cu && lens), JAS_ERR_INVALID, std::string(who) + ": null cu or lens");
    JAS_CHECK(((uintptr_t)cu | (uintptr_t)lens) % 4 == 0, JAS_ERR_INVALID, std::string(who) + ": cu and lens aligned to 4 bytes");
    v = BatchView{cu, lens, B, n};
    return JAS_OK;
}

struct KvArgs {
    PagedView kv;
    BatchView bt;
    void *x[2];  // the batch's keys and values
    long st, sh;
    int vec;     // their rows start on 16 bytes
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight values at p as fp32
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const floatx4 a = __builtin_nontemporal_load((const floatx4 *)p), b = __builtin_nontemporal_load((const floatx4 *)(p + 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[e];
        }
    } else {
        if (vec) {
            const u32x4 t = __builtin_nontemporal_load((const u32x4 *)p);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[2 * e] = __uint_as_float(t[e] << 16), v[2 * e + 1] = __uint_as_float(t[e] & 0xffff0000u);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = bf16_to_f32(p[e]);
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, const float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            *(floatx4 *)p = floatx4{v[0], v[1], v[2], v[3]};
            *(floatx4 *)(p + 4) = floatx4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = v[e];
        }
    } else {
        u32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * e], (__bf16)v[2 * e + 1]});
        if (vec) *(u32x4 *)p = t;
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = (uint16_t)(t[e / 2] >> (16 * (e & 1)));
    }
}

// max over the L lanes of a row (L = 4, 8 or 16, aligned)
template <int L>
__device__ __forceinline__ float row_max(float v)
{
    v = fmaxf(v, dpp_f32<0xB1>(v));               // lane ^ 1
    v = fmaxf(v, dpp_f32<0x4E>(v));               // lane ^ 2
    if (L > 4) v = fmaxf(v, dpp_f32<0x141>(v));   // row_half_mirror
    if (L > 8) v = fmaxf(v, dpp_f32<0x140>(v));   // row_mirror
    return v;
}

// x / s rounded to odd, for s in [2^-60, 2^60] or so: t is within an ulp of the quotient (a
// reciprocal and one correction), the residual x - t s is exact, and its sign says on which
// side of t the quotient lies.
__device__ __forceinline__ float quotient_to_odd(float x, float s, float inv)
{
    const float t0 = x * inv;
    const float t = __builtin_fmaf(__builtin_fmaf(-t0, s, x), inv, t0);
    const float r = __builtin_fmaf(-t, s, x);
    uint32_t u = __float_as_uint(t);
    if ((__float_as_uint(r) ^ u) >> 31) u -= r != 0.f;  // |t| above the quotient: the value below
    return __uint_as_float(r != 0.f ? u | 1u : u);
}

// token tok of the batch: its sequence and position.  False: no row of the batch.
__device__ __forceinline__ bool find_token(const BatchView &bt, const int32_t *cu, int tok, int &b, int &pos)
{
    int lo = 0, hi = bt.B;  // the last b with cu[b] <= tok
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (mid < bt.B ? cu[mid] <= tok : cu[bt.B] <= tok) lo = mid;
        else hi = mid - 1;
    }
    b = lo;
    if (b >= bt.B || cu[b] > tok) return false;
    pos = max(0, bt.lens[b]) - (cu[b + 1] - tok);  // (both at least 0: a length of -2^31 does not wrap)
    return true;
}

constexpr int CU_LDS = 1024;  // batches up to this size are searched in LDS

// Eight values of the cache at element `at`, in fp32, and back
template <int CK>
__device__ __forceinline__ void cache_get(const void *pool, const float *scale, long at, long sc, float (&v)[8])
{
    if constexpr (CK == CK_F32) load8((const float *)pool + at, true, v);
    else if constexpr (CK == CK_BF16) load8((const uint16_t *)pool + at, true, v);
    else {
        const float s = scale[sc];
        const u32x2 c = *(const u32x2 *)((const uint8_t *)pool + at);
        if constexpr (CK == CK_I8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(c[e / 4] >> (8 * (e & 3))) * s;
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[e], false), d = __builtin_amdgcn_cvt_pk_f32_fp8(c[e], true);
                v[4 * e] = a[0] * s, v[4 * e + 1] = a[1] * s, v[4 * e + 2] = d[0] * s, v[4 * e + 3] = d[1] * s;
            }
        }
    }
}
// (every lane of a row comes here, whether the row is stored or not: they meet in its maximum)
template <int D, int CK>
__device__ __forceinline__ void cache_put(void *pool, float *scale, long at, long sc, bool there, int l, const float (&v)[8])
{
    if constexpr (CK == CK_F32) {
        if (there) store8((float *)pool + at, true, v);
    } else if constexpr (CK == CK_BF16) {
        if (there) store8((uint16_t *)pool + at, true, v);
    } else {
        // the row's largest magnitude; an infinity or NaN anywhere makes it one (fmaxf would drop a NaN)
        float mx = 0.f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mx = fmaxf(mx, fabsf(v[e]));
            bad |= !(fabsf(v[e]) <= 3.402823466e38f);
        }
        mx = row_max<D / 8>(bad ? INFINITY : mx);
        constexpr float QMAX = CK == CK_I8 ? 127.f : 448.f;
        float s = mx / QMAX;
        if (!(mx <= 3.402823466e38f)) s = __uint_as_float(0x7fc00000u);
        else if (s < 0x1p-126f) s = 0.f;
        // scaled into the middle of the range, where the residual of a quotient is exact
        const float up = s < 0x1p-40f ? 0x1p80f : s > 0x1p40f ? 0x1p-80f : 1.f;
        const float ss = s * up, inv = 1.0f / ss;
        u32x2 c = {0, 0};
        if (s > 0.f) {  // (a NaN scale too has codes of zero)
            float q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = quotient_to_odd(v[e] * up, ss, inv);
            if constexpr (CK == CK_I8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = (int)fminf(fmaxf(rintf(q[e]), -127.f), 127.f);
                    c[e / 4] |= ((uint32_t)k & 255u) << (8 * (e & 3));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e] = fminf(fmaxf(q[e], -448.f), 448.f);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int t = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * e], q[4 * e + 1], 0, false);
                    c[e] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * e + 2], q[4 * e + 3], t, true);
                }
            }
        }
        if (there) {
            *(u32x2 *)((uint8_t *)pool + at) = c;
            if (l == 0) scale[sc] = s;
        }
    }
}

// One thread: eight values of a row.  READ: cache to rows, of the keys and of the values, which lie
// alike, so that one look into the table serves both.  Else rows to cache, of one of them (blockIdx.y:
// the quantising is as long as the loads), read before the table is.
template <int D, int CK, typename T, bool READ>
__global__ void __launch_bounds__(256) kv_move_kernel(const KvArgs p)
{
    constexpr int L = D / 8;
    __shared__ int32_t cu_s[CU_LDS + 1];
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    const int l = (int)(id % L);
    const long row = id / L;
    const int h = (int)(row % p.kv.n_kv);
    const long tok = row / p.kv.n_kv;
    const long from = tok * p.st + h * p.sh + 8 * l;
    const int which = READ ? 0 : blockIdx.y;
    float k[8], v[8];
    // (whether the row is one of the batch is not known yet, but rows up to n are there to be read)
    if (!READ && tok < p.bt.n) load8((const T *)p.x[which] + from, p.vec, k);
    const int32_t *cu = p.bt.cu;
    if (p.bt.B <= CU_LDS) {
        for (int i = threadIdx.x; i <= p.bt.B; i += 256) cu_s[i] = cu[i];
        __syncthreads();
        cu = cu_s;
    }
    if (tok >= p.bt.n) return;
    int b, pos;
    if (!find_token(p.bt, cu, (int)tok, b, pos)) return;
    int page = -1, slot = 0;
    if (pos >= 0 && pos < p.kv.cap) {
        const int q = (int)p.kv.by_page.div((uint32_t)pos);
        slot = pos - q * p.kv.page_size;
        page = p.kv.table[(long)b * p.kv.table_stride + q];
    }
    const bool there = page >= 0 && page < p.kv.n_pages;
    const long at = (long)page * p.kv.page_stride + h * p.kv.head_stride + slot * p.kv.tok_stride + 8 * l;
    const long sc = ((long)page * p.kv.n_kv + h) * p.kv.page_size + slot;
    if constexpr (READ) {
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.f;
        if (there && p.x[0]) cache_get<CK>(p.kv.k, p.kv.ks, at, sc, k);
        if (there && p.x[1]) cache_get<CK>(p.kv.v, p.kv.vs, at, sc, v);
        if (p.x[0]) store8((T *)p.x[0] + from, p.vec, k);
        if (p.x[1]) store8((T *)p.x[1] + from, p.vec, v);
    } else {
        cache_put<D, CK>(which ? p.kv.v : p.kv.k, which ? p.kv.vs : p.kv.ks, at, sc, there, l, k);
    }
}

template <int D, int CK, bool READ>
static void kv_launch(const KvArgs &p, int dtype, hipStream_t s)
{
    const dim3 grid(ceil_div((long)p.bt.n * p.kv.n_kv * (D / 8), 256), READ ? 1 : 2), block(256);
    if (dtype == JAS_F32) hipLaunchKernelGGL((kv_move_kernel<D, CK, float, READ>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((kv_move_kernel<D, CK, uint16_t, READ>), grid, block, 0, s, p);
}
template <int D, bool READ>
static void kv_launch(const KvArgs &p, int cache, int dtype, hipStream_t s)
{
    if (cache == JAS_F32) kv_launch<D, CK_F32, READ>(p, dtype, s);
    else if (cache == JAS_BF16) kv_launch<D, CK_BF16, READ>(p, dtype, s);
    else if (cache == JAS_I8) kv_launch<D, CK_I8, READ>(p, dtype, s);
    else kv_launch<D, CK_F8, READ>(p, dtype, s);
}

template <bool READ>
static jas_status kv_move(const jas_paged_kv *kv, void *k, void *v, int n, int64_t st, int64_t sh, int B, const int32_t *cu,
                          const int32_t *lens, int dtype, jas_stream_t stream, const char *who)
{
    KvArgs p;
    jas_status rc = paged_view(kv, p.kv, who);
    if (rc != JAS_OK) return rc;
    rc = batch_view(n, B, cu, lens, p.bt, who);
    if (rc != JAS_OK) return rc;
    JAS_CHECK(dtype == JAS_F32 || dtype == JAS_BF16, JAS_ERR_INVALID, std::string(who) + ": rows are JAS_F32 or JAS_BF16");
    JAS_CHECK(READ || (k && v), JAS_ERR_INVALID, std::string(who) + ": null keys or values");
    const uintptr_t es = dtype_bytes(dtype);
    JAS_CHECK(((uintptr_t)k | (uintptr_t)v) % es == 0, JAS_ERR_INVALID, std::string(who) + ": rows aligned to their elements");
    if (!n || !B || (!k && !v)) return JAS_OK;
    // (a launch holds less than 2^32 threads)
    JAS_CHECK((double)n * kv->n_kv * (kv->dh / 8) * (READ ? 1 : 2) <= 4294966784.0, JAS_ERR_RANGE, std::string(who) + ": too many rows for one call");
    p.x[0] = k, p.x[1] = v, p.st = st, p.sh = sh;
    p.vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (st * (long)es) % 16 == 0 && (sh * (long)es) % 16 == 0;
    hipStream_t s = stream_or_default(stream);
    if (kv->dh == 32) kv_launch<32, READ>(p, kv->dtype, dtype, s);
    else if (kv->dh == 64) kv_launch<64, READ>(p, kv->dtype, dtype, s);
    else kv_launch<128, READ>(p, kv->dtype, dtype, s);
    JAS_LAUNCH_CHECK();
    return JAS_OK;
}

} // namespace jas

using namespace jas;

extern "C" {

jas_status jas_kv_append(const jas_paged_kv *kv, const void *k, const void *v, int n, int64_t st, int64_t sh, int B,
                         const int32_t *cu, const int32_t *lens, int dtype, jas_stream_t stream)
{
    return kv_move<false>(kv, (void *)k, (void *)v, n, st, sh, B, cu, lens, dtype, stream, "jas_kv_append");
}

jas_status jas_kv_read(const jas_paged_kv *kv, void *k, void *v, int n, int64_t st, int64_t sh, int B, const int32_t *cu,
                       const int32_t *lens, int dtype, jas_stream_t stream)
{
    return kv_move<true>(kv, k, v, n, st, sh, B, cu, lens, dtype, stream, "jas_kv_read");
}

} // extern "C"
