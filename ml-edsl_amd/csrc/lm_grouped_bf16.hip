// The layers on groups of rows (lm_grouped.hpp) in bf16.
#include "lm_grouped_launch.hpp"

namespace edsl {
namespace lm {

template <>
hipError_t launch_grouped_rows<kBf16>(const GroupedArgs& a, int loads, hipStream_t stream) {
  return GroupedLaunch<bf16>::rows(a, loads, stream);
}
template <>
hipError_t launch_grouped_skinny<kBf16>(const GroupedArgs& a, hipStream_t stream) {
  return GroupedLaunch<bf16>::skinny(a, stream);
}
template <>
hipError_t launch_grouped_weights<kBf16>(const GroupedWeightArgs& a, int loads, bool big, hipStream_t stream) {
  return GroupedLaunch<bf16>::weights(a, loads, big, stream);
}

}  // namespace lm
}  // namespace edsl
