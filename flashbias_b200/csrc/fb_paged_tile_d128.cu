// Instantiations of the tile kernel of attention over pages at tile width 128.
#include "fb_paged_tile.cuh"

namespace fb {
int launch_paged_tile_d128(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) { return launch_paged_tile<128>(a, plan, st); }
}  // namespace fb
