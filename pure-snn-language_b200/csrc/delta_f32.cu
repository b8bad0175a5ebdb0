// delta_f32.cu - the delta-rule scan's kernels for f32 tensors
#include "delta_launch.h"
namespace snnb_delta {
SNN_DELTA_LAUNCHES(float)
}  // namespace snnb_delta
