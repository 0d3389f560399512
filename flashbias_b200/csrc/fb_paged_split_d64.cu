// Instantiations of the split kernel of attention over pages at tile width 64.
#include "fb_paged_split.cuh"

namespace fb {
int launch_paged_split_d64(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) { return launch_paged_split<64>(a, plan, st); }
}  // namespace fb
