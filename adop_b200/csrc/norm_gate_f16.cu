// The kernels of norm_gate.cuh for images of this type.
#include "norm_gate.cuh"

namespace adop {

const void* norm_kernel_f16(int which, int vec, bool gated, int act) { return norm::norm_kernel<__half>(which, vec, gated, act); }

}  // namespace adop
