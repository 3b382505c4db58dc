// Attention over the paged cache: the kernels of head dim 32.
#include "attn_paged.hpp"

namespace jas {
void paged_launch_32(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s) { paged_launch<32>(p, rows, cache, dtype, s); }
} // namespace jas
