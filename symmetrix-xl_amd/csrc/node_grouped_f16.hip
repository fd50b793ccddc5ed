// Products by kind of row: the kernels of f16 values.
#include "node_grouped.hpp"

namespace smx {
namespace node {

template void launch_grouped<f16, float>(const Grouped<f16, float>&, Way, const Cut&, hipStream_t);
template void launch_grouped<f16, f16>(const Grouped<f16, f16>&, Way, const Cut&, hipStream_t);

}  // namespace node
}  // namespace smx
