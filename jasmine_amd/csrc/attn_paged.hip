// Attention over the paged cache: checks, the choice of kernel and splits, and the launch.
#include "attn_paged.hpp"

#include <algorithm>

namespace jas {

static int paged_cus()
{
    static const int n = [] {
        int dev = 0, v = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) v = 256;
        return v;
    }();
    return n;
}

} // namespace jas

using namespace jas;

extern "C" {

size_t jas_attn_paged_workspace(int n, int B, int H, int n_kv, int dh, int max_q, int max_len)
{
    if (n <= 0 || B <= 0 || H <= 0 || n_kv <= 0 || H % n_kv != 0 || dh <= 0 || max_q < 0 || max_len < 0) return 0;
    return paged_workspace(n, B, H, n_kv, dh, max_q, max_len, paged_cus());
}

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
    JAS_CHECK(q != o, JAS_ERR_INVALID, "jas_attn_paged: o must not overlap q");
    JAS_CHECK(dtype == JAS_F32 || dtype == JAS_BF16, JAS_ERR_INVALID, "jas_attn_paged: rows are JAS_F32 or JAS_BF16");
    JAS_CHECK(dtype == JAS_F32 || kv->dtype != JAS_F32, JAS_ERR_INVALID, "jas_attn_paged: JAS_BF16 rows over a JAS_F32 cache");
    JAS_CHECK(H > 0 && H % kv->n_kv == 0, JAS_ERR_INVALID, "jas_attn_paged: H is a multiple of the cache's heads");
    JAS_CHECK(max_q >= 0 && max_len >= 0, JAS_ERR_INVALID, "jas_attn_paged: max_q and max_len are not negative");
    const long es = (long)dtype_bytes(dtype);
    JAS_CHECK(((uintptr_t)q | (uintptr_t)o) % es == 0, JAS_ERR_INVALID, "jas_attn_paged: rows aligned to their elements");
    JAS_CHECK((long)n * H <= 0x3fffffffl, JAS_ERR_RANGE, "jas_attn_paged: too many rows for one call");
    if (!n || !B) return JAS_OK;
    const PagedPlan plan = paged_plan(n, B, H, kv->n_kv, max_q, max_len, dtype, paged_cus());
    // (a launch holds less than 2^32 threads: 256 of a tile, and of four rows that are joined)
    JAS_CHECK((double)plan.tiles * kv->n_kv * std::max(plan.nsplit, plan.nsplit > 1 ? plan.rows / 4 : 1) <= 16777215.0, JAS_ERR_RANGE, "jas_attn_paged: too many tiles for one call");
    JAS_CHECK(plan.nsplit == 1 || work, JAS_ERR_INVALID, "jas_attn_paged: null workspace");
    JAS_CHECK(paged_need(plan, kv->n_kv, kv->dh) <= jas_attn_paged_workspace(n, B, H, kv->n_kv, kv->dh, max_q, max_len), JAS_ERR_RUNTIME,
              "jas_attn_paged: the plan exceeds its workspace");
    JAS_CHECK((uintptr_t)work % 16 == 0, JAS_ERR_INVALID, "jas_attn_paged: workspace aligned to 16 bytes");
    p.q = q, p.o = o, p.H = H, p.G = H / kv->n_kv, p.max_len = max_len, p.causal = causal != 0;
    p.by_group.set((uint32_t)p.G);
    p.q_st = q_st, p.q_sh = q_sh, p.o_st = o_st, p.o_sh = o_sh;
    p.q_vec = (uintptr_t)q % 16 == 0 && q_st * es % 16 == 0 && q_sh * es % 16 == 0;
    p.o_vec = (uintptr_t)o % 16 == 0 && o_st * es % 16 == 0 && o_sh * es % 16 == 0;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.tiles = (int)plan.tiles, p.nsplit = plan.nsplit, p.chunk = plan.chunk, p.sorted = plan.rows > 16 && plan.nsplit == 1 && B <= 256, p.cus = paged_cus(), p.part = (float *)work;
    hipStream_t s = stream_or_default(stream);
    if (kv->dh == 32) paged_launch_32(p, plan.rows, kv->dtype, dtype, s);
    else if (kv->dh == 64) paged_launch_64(p, plan.rows, kv->dtype, dtype, s);
    else paged_launch_128(p, plan.rows, kv->dtype, dtype, s);
    JAS_LAUNCH_CHECK();
    return JAS_OK;
}

} // extern "C"
