// The 4-bit layer on up to 32 rows (q4_small.hpp), x in f32.
#include "q4_small.hpp"

namespace edsl {
namespace lm {
template hipError_t launch_q4_small<kF32>(const Q4Args& a, int nt, int waves, int spb, hipStream_t stream);
}  // namespace lm
}  // namespace edsl
