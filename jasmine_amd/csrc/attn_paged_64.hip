// Attention over the paged cache: the kernels of head dim 64.
#include "attn_paged.hpp"

namespace jas {
void paged_launch_64(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s) { paged_launch<64>(p, rows, cache, dtype, s); }
} // namespace jas
