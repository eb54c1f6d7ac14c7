// The convolution's kernels for float32 inputs.
#include "conv_kernels.h"

namespace ormi_hip {
int launch_conv_f32(const ConvParams& p, bool gradient, bool wide_dout) { return launch_conv<ORMI_DTYPE_F32>(p, gradient, wide_dout); }
}  // namespace ormi_hip
