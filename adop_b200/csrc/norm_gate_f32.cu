// The kernels of norm_gate.cuh for images of this type.
#include "norm_gate.cuh"

namespace adop {

const void* norm_kernel_f32(int which, int vec, bool gated, int act) { return norm::norm_kernel<float>(which, vec, gated, act); }

}  // namespace adop
