// Linear attention's walks over operands of float16.
#include "linear_walk.hpp"

namespace dnatok {

template void launch_walk<_Float16>(const WalkArgs &w, hipStream_t s);
template void launch_pieces<_Float16>(const WalkArgs &w, hipStream_t s);

}  // namespace dnatok
