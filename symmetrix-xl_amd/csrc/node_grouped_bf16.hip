// Products by kind of row: the kernels of bf16 values.
#include "node_grouped.hpp"

namespace smx {
namespace node {

template void launch_grouped<bf16, float>(const Grouped<bf16, float>&, Way, const Cut&, hipStream_t);
template void launch_grouped<bf16, bf16>(const Grouped<bf16, bf16>&, Way, const Cut&, hipStream_t);

}  // namespace node
}  // namespace smx
