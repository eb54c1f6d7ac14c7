// The recurrence's kernels for bfloat16 inputs.
#include "recurrence_kernels.h"

namespace ormi_hip {
int launch_recurrence_bf16(const RecParams& p, const RecCall& c) { return launch_recurrence<ORMI_DTYPE_BF16>(p, c); }
}  // namespace ormi_hip
