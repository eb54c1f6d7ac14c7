// The recurrence's kernels for float32 inputs.
#include "recurrence_kernels.h"

namespace ormi_hip {
int launch_recurrence_f32(const RecParams& p, const RecCall& c) { return launch_recurrence<ORMI_DTYPE_F32>(p, c); }
}  // namespace ormi_hip
