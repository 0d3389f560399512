// Instantiations of the tile kernel of attention over pages at tile width 64.
#include "fb_paged_tile.cuh"

namespace fb {
int launch_paged_tile_d64(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) { return launch_paged_tile<64>(a, plan, st); }
}  // namespace fb
