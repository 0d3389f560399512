// Instantiations of the split kernel of attention over pages at tile width 128.
#include "fb_paged_split.cuh"

namespace fb {
int launch_paged_split_d128(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) { return launch_paged_split<128>(a, plan, st); }
}  // namespace fb
