// delta_bf16.cu - the delta-rule scan's kernels for bf16 tensors
#include "delta_launch.h"
namespace snnb_delta {
SNN_DELTA_LAUNCHES(__nv_bfloat16)
}  // namespace snnb_delta
