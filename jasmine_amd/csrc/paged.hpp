// The paged cache as kernels see it: pages, the table, and where a token of a ragged batch lies.
#pragma once
#include "jas_common.hpp"

namespace jas {

// t / d for 0 <= t < 2^31 by a product: q = (umulhi(m, t) + t) >> l with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1
struct FastDiv {
    uint32_t d, m, l;
    void set(uint32_t v)
    {
        d = v, l = 0;
        while ((1ull << l) < v) ++l;
        m = (uint32_t)((((1ull << l) - v) << 32) / v + 1);
    }
#ifdef __HIPCC__
    __device__ __forceinline__ uint32_t div(uint32_t t) const { return (__umulhi(m, t) + t) >> l; }
#endif
};

struct PagedView {
    void *k, *v;
    float *ks, *vs;
    const int32_t *table;
    long page_stride, head_stride, tok_stride;
    int table_stride, n_pages, page_size, n_kv, cap;  // cap: positions that a row of the table holds
    FastDiv by_page;
};

// A batch of rows: cu[B + 1], lens[B]
struct BatchView {
    const int32_t *cu, *lens;
    int B, n;
};

// What a cache holds, as kernels are instantiated for it
enum CacheKind : int { CK_F32 = 0, CK_BF16 = 1, CK_I8 = 2, CK_F8 = 3 };

jas_status paged_view(const jas_paged_kv *kv, PagedView &v, const char *who);
jas_status batch_view(int n, int B, const int32_t *cu, const int32_t *lens, BatchView &v, const char *who);
inline size_t dtype_bytes(int t) { return t == JAS_F32 ? 4 : t == JAS_BF16 ? 2 : 1; }
inline bool dtype_eight(int t) { return t == JAS_I8 || t == JAS_F8E4M3; }

} // namespace jas
