// What the convolution's entry (conv.hip) and its kernels share.
#pragma once
#include <hip/hip_runtime.h>

#include "ormi_hip.h"

namespace ormi_hip {

constexpr int kConvLanes = 8;       // threads side by side over the channels
constexpr int kConvRuns = 32;       // runs of tokens of a tile
constexpr int kConvTokens = 8;      // of a run, forward
constexpr int kConvGradTokens = 8;  // of a run, backward

// Channels of a thread: a 16-byte access, half of one for 16-bit channels with
// more weights than registers hold beside their sums.
constexpr int conv_run(int dt, int width) { return dt == ORMI_DTYPE_F32 || width > 4 ? 4 : 8; }

struct ConvParams {
    const char *x, *initial, *dout;
    long long x_sb, x_sl, do_sb, do_sl;  // strides in elements; channels are neighbours
    int batch, length, channels, width, silu;
    int channel_blocks, tiles, parts;    // work-groups of a batch over the tiles: part k has tiles k, k + parts, ...
    const float *weight, *bias;
    const int *docs, *lengths;
    long long docs_sb;
    char *out, *last;
    // Gradient.
    const float* dlast;
    char *dx, *dinitial;
    float *dweight, *dbias;
    float* part_sums;  // (batch, parts, width + 1, channels), or null
};

int launch_conv_f32(const ConvParams& p, bool gradient, bool wide_dout);
int launch_conv_bf16(const ConvParams& p, bool gradient, bool wide_dout);
int launch_conv_f16(const ConvParams& p, bool gradient, bool wide_dout);

}  // namespace ormi_hip
