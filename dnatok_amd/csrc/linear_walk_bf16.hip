// Linear attention's walks over operands of bfloat16.
#include "linear_walk.hpp"

namespace dnatok {

template void launch_walk<__bf16>(const WalkArgs &w, hipStream_t s);
template void launch_pieces<__bf16>(const WalkArgs &w, hipStream_t s);

}  // namespace dnatok
