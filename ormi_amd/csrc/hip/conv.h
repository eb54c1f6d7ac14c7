// What the convolution's entry (conv.hip) and its kernels share.
#pragma once
#include <hip/hip_runtime.h>

#include "ormi_hip.h"

namespace ormi_hip {

constexpr int kConvLanes = 32;                 // threads side by side over the channels: 256 bytes of a 16-bit row
constexpr int kConvRun = 4;                    // channels of a thread
constexpr int kConvRuns = 256 / kConvLanes;    // runs of tokens of a tile
static_assert(kConvRuns >= ORMI_CONV_MAX_WIDTH - 1, "a run's threads for each row of the last state");
// Widths that kernels are built for: 3 and 4 without masks, and 4 and 8 with masks for
// all up to them, which other widths without masks use too. 8 x 2048 x 4096 bf16 with
// silu, forward / both passes: width 1 59 / 201 us, 2 63 / 190, 3 58 / 164, 4 58 / 164,
// 5 to 8 77-88 / 394-420 (the gradient's window, weights and sums of four channels fill
// 256 registers and more).
constexpr int conv_width(int width, bool masked) { return width == 3 && !masked ? 3 : width <= 4 ? 4 : 8; }
constexpr int run_tokens(int width) { return 32 / width * width; }  // of a thread's run: whole groups of that width

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
