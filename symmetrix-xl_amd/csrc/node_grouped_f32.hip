// Products by kind of row: the kernels of f32 values.
#include "node_grouped.hpp"

namespace smx {
namespace node {

template void launch_grouped<float, float>(const Grouped<float, float>&, Way, const Cut&, hipStream_t);


}  // namespace node
}  // namespace smx
