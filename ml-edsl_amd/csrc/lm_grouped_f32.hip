// The layers on groups of rows (lm_grouped.hpp) in f32.
#include "lm_grouped_launch.hpp"

namespace edsl {
namespace lm {

template <>
hipError_t launch_grouped_rows<kF32>(const GroupedArgs& a, bool direct, hipStream_t stream) {
  return GroupedLaunch<float>::rows(a, direct, stream);
}
template <>
hipError_t launch_grouped_skinny<kF32>(const GroupedArgs& a, hipStream_t stream) {
  return GroupedLaunch<float>::skinny(a, stream);
}
template <>
hipError_t launch_grouped_weights<kF32>(const GroupedWeightArgs& a, bool direct, bool big, hipStream_t stream) {
  return GroupedLaunch<float>::weights(a, direct, big, stream);
}

}  // namespace lm
}  // namespace edsl
