// What the recurrence's entry (recurrence.hip) and its kernels share.
#pragma once
#include <hip/hip_runtime.h>

#include "ormi_hip.h"

namespace ormi_hip {

constexpr int kRecLanes = 16;                         // threads side by side over the channels
constexpr int kRecRun = 4;                            // channels of a thread
constexpr int kRecChannels = kRecLanes * kRecRun;     // of a work-group
constexpr int kRecTokens = 8;                         // of a segment: a thread's
constexpr int kRecTile = 256 / kRecLanes * kRecTokens;  // tokens between the states kept for the gradient
constexpr int kRecGroup = 8;                          // chained tiles that share a state
constexpr int kRecWindow = 8;                         // groups that a tile looks at together
constexpr int kRecCounters = 16;                      // sets of chains
constexpr int kRecCounterStride = 64;                 // words between their counters
static_assert(kRecTile == ORMI_RECURRENCE_TILE, "the header's tile");

struct RecParams {
    const char *gates, *x, *dout;
    long long g_sb, g_sl, x_sb, x_sl, do_sb, do_sl;  // strides in elements; channels are neighbours
    int batch, length, channels;
    int channel_blocks, chains, tiles, chained;  // chains: channel blocks of all batches
    const float* initial;
    const int *docs, *lengths;
    long long docs_sb;
    char* out;
    float *last, *states;
    // Gradient.
    const float* dlast;
    char *dgates, *dx;
    float* dinitial;
    // Chained tiles, by tile or group, chain and channel: what is there of the tiles' and
    // the groups' spans and of the states before groups; and how many tiles of each set
    // of chains were given out.
    unsigned long long *chain_spans, *group_spans;
    unsigned* group_states;
    unsigned* tickets;
};

// Groups of a chain, the last one perhaps of fewer tiles; one more state than whole
// groups. 32-bit words of all spans and states, one after the other.
inline long long chain_groups(const RecParams& p) { return (p.tiles + kRecGroup - 1) / kRecGroup + 1; }
inline long long chain_words(const RecParams& p) { return (2ll * p.tiles + 3 * chain_groups(p)) * p.chains * kRecChannels; }

// xt: the type of x and the result; gates and dout have it or are float32 (their flags).
struct RecCall {
    bool gates_f32, dout_f32, logits, gradient;
};
int launch_recurrence_f32(const RecParams& p, const RecCall& c);
int launch_recurrence_bf16(const RecParams& p, const RecCall& c);
int launch_recurrence_f16(const RecParams& p, const RecCall& c);

}  // namespace ormi_hip
