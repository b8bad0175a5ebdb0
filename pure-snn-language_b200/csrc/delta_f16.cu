// delta_f16.cu - the delta-rule scan's kernels for f16 tensors
#include "delta_launch.h"
namespace snnb_delta {
SNN_DELTA_LAUNCHES(__half)
}  // namespace snnb_delta
