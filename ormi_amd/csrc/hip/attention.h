// What the attention entry (attention.hip) and its kernels share.
#pragma once
#include <hip/hip_runtime.h>

namespace ormi_hip {

// What a score is beside a multiple of q.k: nothing, slopes, or a tanh and perhaps
// slopes. A cap multiplies what the tanh is off by: above kWideCap 16-bit scores
// take the tanh that is exact relative to itself, too (tanh_score).
constexpr int kPlain = 0, kBias = 1, kCap = 2, kCapWide = 3;
constexpr float kWideCap = 256.0f;

constexpr int kDocTile = 64;  // tokens per document range

// Keys per LDS tile of the forward kernel: two stages of keys and values. few:
// one wave per work-group, smaller tiles so that more of them fit a compute
// unit. 32-bit rows and 256 features take 32 keys so that the registers of the
// scores and the LDS of two stages fit.
constexpr int fwd_tile(int dp, int es, bool few) { return few || es == 4 || dp > 128 ? 32 : 64; }

struct AttnParams {
    const char *q, *k, *v;
    char* out;
    char* rest;  // 16-bit: what out's rounding left, rounded in turn, laid out like out
    float* lse;  // base-2 logarithm of a row's sum, (batch, kv head, row); +inf: the row sees no key
    long long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;  // strides in elements
    int batch, queries, keys, heads, kv_heads, group, dim;
    int rows;    // queries * group
    int chunks;  // 16-byte chunks of a row that exist
    int causal, form;
    float scale, scale2, cap2, scale_over_cap;  // scale2 = scale log2 e, cap2 = cap log2 e
    const float* slopes;
    const int *docs, *prefix, *lengths;
    long long docs_sb;
    const int2* ranges;
    int range_tiles;
    // Work split.
    int wide;  // 4 waves per work-group (128 rows), else one
    int row_blocks, splits;
    int split_tiles;  // tiles per split, or 0: an equal share of the row's tiles
    int spread;  // runs of blocks per head (Work)
    float* part;    // of out, or of dk and dv
    float* part_q;  // of dq
    float2* part_ml;
    // Gradient.
    const char* dout;
    long long do_sb, do_sl, do_sh;
    const float* delta;      // sum of out * dout of a row, laid out like lse
    const float* grad_scale; // float16: two squared norms per batch and key head (attention_delta_kernel)
    char *dq, *dk, *dv;
    int key_blocks, key_splits;
    unsigned group_m, group_s;  // division by group (ormi_fdiv)
};

int launch_attention_fwd_bf16(const AttnParams& p);
int launch_attention_fwd_f16(const AttnParams& p);
int launch_attention_fwd_f32(const AttnParams& p);
// bounds: two zeroed words per batch and key head where the score gradients are held scaled (float16), else null.
int launch_attention_grad_bf16(const AttnParams& p, float* delta, unsigned* bounds);
int launch_attention_grad_f16(const AttnParams& p, float* delta, unsigned* bounds);
int launch_attention_grad_f32(const AttnParams& p, float* delta, unsigned* bounds);

}  // namespace ormi_hip
