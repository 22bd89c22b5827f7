// Linear attention's walks over operands of 32 bits.
#include "linear_walk.hpp"

namespace dnatok {

template void launch_walk<float>(const WalkArgs &w, hipStream_t s);
template void launch_pieces<float>(const WalkArgs &w, hipStream_t s);

}  // namespace dnatok
