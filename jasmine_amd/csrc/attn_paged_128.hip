// Attention over the paged cache: the kernels of head dim 128.
#include "attn_paged.hpp"

namespace jas {
void paged_launch_128(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s) { paged_launch<128>(p, rows, cache, dtype, s); }
} // namespace jas
