// The layers on groups of rows (lm_grouped.hpp) in f32.
#include "lm_grouped_launch.hpp"

namespace edsl {
namespace lm {

template <>
hipError_t launch_grouped_rows<kF32>(const GroupedArgs& a, int loads, hipStream_t stream) {
  return GroupedLaunch<float>::rows(a, loads, stream);
}
template <>
hipError_t launch_grouped_skinny<kF32>(const GroupedArgs& a, hipStream_t stream) {
  return GroupedLaunch<float>::skinny(a, stream);
}
template <>
hipError_t launch_grouped_weights<kF32>(const GroupedWeightArgs& a, int loads, bool big, hipStream_t stream) {
  return GroupedLaunch<float>::weights(a, loads, big, stream);
}

}  // namespace lm
}  // namespace edsl
