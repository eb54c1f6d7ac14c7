// The attention kernels for one element type (see attention_kernels.h).
#include "attention_kernels.h"

namespace ormi_hip {

int launch_attention_fwd_f32(const AttnParams& p) {
    return p.dim <= 64    ? launch_attention_fwd_dp<TrF32, 64>(p)
           : p.dim <= 96  ? launch_attention_fwd_dp<TrF32, 96>(p)
           : p.dim <= 128 ? launch_attention_fwd_dp<TrF32, 128>(p)
                          : launch_attention_fwd_dp<TrF32, 256>(p);
}

int launch_attention_grad_f32(const AttnParams& p, float* delta, unsigned* bounds) {
    return p.dim <= 64    ? launch_attention_grad_dp<TrF32, 64>(p, delta, bounds)
           : p.dim <= 96  ? launch_attention_grad_dp<TrF32, 96>(p, delta, bounds)
           : p.dim <= 128 ? launch_attention_grad_dp<TrF32, 128>(p, delta, bounds)
                          : launch_attention_grad_dp<TrF32, 256>(p, delta, bounds);
}

}  // namespace ormi_hip
