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

// Rounds of workgroups that tiles whose keys are split make, and the fewest keys of a split
static constexpr int paged_rounds(int rows) { return rows == 16 ? 8 : rows == 64 ? 4 : 2; }
static constexpr int paged_least(int rows) { return rows == 16 ? 128 : 256; }

// Tiles of 16 rows stream the keys once for each tile, without LDS: for sequences whose new rows
// (tokens times the query heads of a key head) fit one.  Otherwise tiles of 64 rows, or of 128, which
// read fragments from LDS for twice the products but come in half the number, less evenly loaded.
// (us, tiles of 128 and of 64; lengths spread up to what is named, heads of 128 but as said)
//   fp32 rows, 12 heads of 64: 16 x up to 200 tokens over 1024 keys 98, 55; 8 x 1024 92, 82; 2 x 333 over 2001
//     39.5, 38.7; 500 over 8000 93, 105: always 64
//   bf16 rows, 128 give a workgroup to every unit: 4 x 512 over 4096 125, 142; 24 x 256 over 2048, e4m3 92, 98
//   only 64 do, with some over: 2 x 512 over 4096 111, 88, int8 138, 112; 6 x 300 over 2048, 16 heads of 64 71, 48
//   neither does: 512 over 8192, int8 139, 208; 300 over 6000 45, 52
static PagedPlan paged_plan(int n, int B, int H, int n_kv, int max_q, int max_len, int dtype)
{
    PagedPlan r;
    max_len = std::min(max_len, 0x7fff0000);  // (no table's row holds more: PagedView)
    const long G = H / n_kv, most = std::min((long)max_q, (long)n) * G, cus = paged_cus();
    auto full = [&](int rows) { return std::max((long)B, (long)n * G / rows) * n_kv; };  // tiles, about
    r.rows = most <= 16 ? 16 : most <= 64 || dtype == JAS_F32 || (full(128) < cus && full(64) >= cus + cus / 8) ? 64 : 128;
    // sequence b owns tiles from floor(cu[b] G / rows) + b on
    r.tiles = (long)n * G / r.rows + B;
    // Splits of `chunk` keys: enough workgroups to fill the chip some times over, so that sequences of
    // different lengths even out; a split that a shorter sequence does not need ends at once.
    // Tiles of 16 rows: eight rounds of one workgroup a unit (32 sequences of 1024 to 4096 keys, 8
    // heads, bf16: 75.2, 71.0, 72.1, 78.9 us at 6, 8, 12, 16).  Larger tiles are bound by the matrix
    // cores and their partial results are large: split only where units would be left without one
    // (2 x 333 rows over 2001 keys, 12 heads of 64, fp32: 82, 38.7 us unsplit and split; 4 chunks of 512
    // over 4096, bf16: 125, 163), those of 64 into four rounds (that fp32: 42.4, 38.8, 38.7 at 2, 3, 4),
    // those of 128 into two (512 over 8192, int8: 172, 139, 169, 150 at 1.5, 2, 3, 4).  An odd number of
    // splits: see paged_block.
    if (r.rows > 16 && full(r.rows) >= cus) r.chunk = std::max(max_len, 1), r.nsplit = 1;
    else {
        const double share = (double)full(r.rows) * max_len / (paged_rounds(r.rows) * cus);
        r.chunk = (int)std::min(((long)std::max((double)paged_least(r.rows), std::min(share, (double)max_len)) + 127) / 128 * 128, 0x7fff0000L);
        r.nsplit = (int)std::max(1L, std::min(((long)max_len + r.chunk - 1) / r.chunk, 63L));
        if (r.nsplit > 1) r.nsplit |= 1;
    }
    return r;
}

// Bytes that hold the partial results of every call within the given numbers: fewer rows can need more
// than many, whose keys are not split.  With x = max(B, n G / rows) n_kv there are at most 2 x tiles of a
// head, of s = rounds cus / x + 1 splits, and one more to make them odd: 2 rounds cus + 4 x in all, where
// x is below rounds cus (s = 1 otherwise) and for tiles of 64 and 128 below cus (not split otherwise).
static size_t paged_bytes(int rows, int n, int B, int H, int n_kv, int D, int max_len)
{
    if (max_len <= paged_least(rows)) return 0;
    const double cus = paged_cus(), rounds = paged_rounds(rows), G = H / n_kv;
    const double x = std::min(std::max((double)B, n * G / rows) * n_kv, (rows == 16 ? rounds : 1.0) * cus);
    const double parts = std::min(2 * rounds * cus + 4 * x, (n * G / rows + B) * n_kv * std::min(63.0, (double)max_len / paged_least(rows) + 2));
    return (size_t)parts * rows * (D + 4) * sizeof(float);
}

} // namespace jas

using namespace jas;

extern "C" {

size_t jas_attn_paged_workspace(int n, int B, int H, int n_kv, int dh, int max_q, int max_len)
{
    if (n <= 0 || B <= 0 || H <= 0 || n_kv <= 0 || H % n_kv != 0 || dh <= 0 || max_q < 0 || max_len < 0) return 0;
    const double most = std::min((double)max_q, (double)n) * (H / n_kv);
    size_t bytes = paged_bytes(16, n, B, H, n_kv, dh, max_len);
    if (most > 16) bytes = std::max(bytes, paged_bytes(64, n, B, H, n_kv, dh, max_len));
    if (most > 64) bytes = std::max(bytes, paged_bytes(128, n, B, H, n_kv, dh, max_len));
    return bytes;
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
    const PagedPlan plan = paged_plan(n, B, H, kv->n_kv, max_q, max_len, dtype);
    // (a launch holds less than 2^32 threads: 256 of a tile, and of four rows that are joined)
    JAS_CHECK((double)plan.tiles * kv->n_kv * std::max(plan.nsplit, plan.nsplit > 1 ? plan.rows / 4 : 1) <= 16777215.0, JAS_ERR_RANGE, "jas_attn_paged: too many tiles for one call");
    JAS_CHECK(plan.nsplit == 1 || work, JAS_ERR_INVALID, "jas_attn_paged: null workspace");
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
