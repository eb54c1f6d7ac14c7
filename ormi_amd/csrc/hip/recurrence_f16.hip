// The recurrence's kernels for float16 inputs.
#include "recurrence_kernels.h"

namespace ormi_hip {
int launch_recurrence_f16(const RecParams& p, const RecCall& c) { return launch_recurrence<ORMI_DTYPE_F16>(p, c); }
}  // namespace ormi_hip
