// What the recurrence's entry (recurrence.hip) and its kernels share.
#pragma once
#include <hip/hip_runtime.h>

#include "ormi_hip.h"

namespace ormi_hip {

constexpr int kRecSegments = 32;                      // of a tile, one after the other in time
constexpr int kRecTokens = 4;                         // of a segment: a thread's
constexpr int kRecTile = kRecSegments * kRecTokens;   // tokens between the states kept for the gradient
static_assert(kRecTile == ORMI_RECURRENCE_TILE, "the header's tile");
constexpr int kRecLanes = 8;                          // threads side by side over the channels
constexpr int kRecMostSplits = 64;

struct RecParams {
    const char *gates, *x, *dout;
    long long g_sb, g_sl, x_sb, x_sl, do_sb, do_sl;  // strides in elements; channels are neighbours
    int batch, length, channels;
    int channel_blocks, splits, split_tiles, tiles;
    const float* initial;
    const int *docs, *lengths;
    long long docs_sb;
    char* out;
    float *last, *states;
    // Gradient.
    const float* dlast;
    char *dgates, *dx;
    float* dinitial;
    // Of each split, batch and channel: the product of its gates and what it leaves
    // of nothing, then (one per batch and split) whether its tokens forget.
    float2* part;
    int* part_cut;
};

// xt: the type of x and the result; gates and dout have it or are float32 (their flags).
struct RecCall {
    bool gates_f32, dout_f32, logits, gradient;
};
int launch_recurrence_f32(const RecParams& p, const RecCall& c);
int launch_recurrence_bf16(const RecParams& p, const RecCall& c);
int launch_recurrence_f16(const RecParams& p, const RecCall& c);

}  // namespace ormi_hip
