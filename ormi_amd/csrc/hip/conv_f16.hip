// The convolution's kernels for float16 inputs.
#include "conv_kernels.h"

namespace ormi_hip {
int launch_conv_f16(const ConvParams& p, bool gradient, bool wide_dout) { return launch_conv<ORMI_DTYPE_F16>(p, gradient, wide_dout); }
}  // namespace ormi_hip
