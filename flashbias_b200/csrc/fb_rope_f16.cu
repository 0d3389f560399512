#include "fb_rope_vector.cuh"

namespace fb {
template void launch_rope_t<__half>(const RopeV&, int, unsigned, cudaStream_t);
}
