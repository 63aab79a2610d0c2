// The layers on groups of rows (lm_grouped.hpp) in f16.
#include "lm_grouped_launch.hpp"

namespace edsl {
namespace lm {

template <>
hipError_t launch_grouped_rows<kF16>(const GroupedArgs& a, bool direct, hipStream_t stream) {
  return GroupedLaunch<f16>::rows(a, direct, stream);
}
template <>
hipError_t launch_grouped_skinny<kF16>(const GroupedArgs& a, hipStream_t stream) {
  return GroupedLaunch<f16>::skinny(a, stream);
}
template <>
hipError_t launch_grouped_weights<kF16>(const GroupedWeightArgs& a, bool direct, bool big, hipStream_t stream) {
  return GroupedLaunch<f16>::weights(a, direct, big, stream);
}

}  // namespace lm
}  // namespace edsl
