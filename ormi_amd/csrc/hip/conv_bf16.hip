// The convolution's kernels for bfloat16 inputs.
#include "conv_kernels.h"

namespace ormi_hip {
int launch_conv_bf16(const ConvParams& p, bool gradient, bool wide_dout) { return launch_conv<ORMI_DTYPE_BF16>(p, gradient, wide_dout); }
}  // namespace ormi_hip
