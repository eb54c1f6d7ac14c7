// C entry of the short causal convolution and its gradient: checks, work split and
// workspace. The kernels are in conv_kernels.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "conv.h"
#include "ormi_hip_internal.h"

namespace ormi_hip {
namespace {

constexpr long long kMostGroups = (1ll << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32
constexpr int kMostTokens = 1 << 30;                // token numbers of a last tile stay in 31 bits

constexpr int kMostStride = 1 << 20;                // elements between tokens: a tile's offsets stay in 32 bits

bool is_float(int dt) { return dt == ORMI_DTYPE_F32 || dt == ORMI_DTYPE_BF16 || dt == ORMI_DTYPE_F16; }

bool near(int length, int64_t stride) { return length <= 1 || (stride >= 0 && stride <= kMostStride); }

const char* check(const ormi_conv_desc* d) {
    if (!d) return "null descriptor";
    if (!is_float(d->dtype)) return "dtype must be float32, bfloat16 or float16";
    if (d->batch < 0 || d->length < 0 || d->channels < 0) return "negative extent";
    if (d->width < 1 || d->width > ORMI_CONV_MAX_WIDTH) return "width must be 1 to 8";
    if (d->length > kMostTokens) return "more than 2^30 tokens";
    if (d->channels > kMostStride) return "more than 2^20 channels";
    if (!near(d->length, d->x_strides[1])) return "tokens more than 2^20 elements apart";
    return nullptr;
}

// False: more work-groups than a launch holds.
bool plan(const ormi_conv_desc* d, bool gradient, ConvParams* p) {
    const int tokens = kConvRuns * run_tokens(conv_width(d->width, d->documents || d->lengths));
    p->batch = d->batch;
    p->length = d->length;
    p->channels = d->channels;
    p->width = d->width;
    p->silu = d->silu;
    p->channel_blocks = (int)((d->channels + kConvLanes * kConvRun - 1ll) / (kConvLanes * kConvRun));
    p->tiles = (d->length + tokens - 1) / tokens;
    p->parts = p->tiles;
    const long long rows = (long long)p->channel_blocks * d->batch;
    if (!gradient && p->tiles == 0) p->tiles = p->parts = 1;  // it leaves the initial inputs as the last state
    if (gradient) {
        // A work-group's sums of the weights' gradients are a row for the second
        // launch: no more of them than keep the card busy.
        p->parts = (int)std::min<long long>(p->tiles, (8ll * compute_units() + rows - 1) / std::max(1ll, rows));
    }
    return rows * p->parts <= kMostGroups;
}

size_t sums_bytes(const ConvParams& p) {
    return ((size_t)p.batch * p.parts * (p.width + 1) * p.channels * sizeof(float) + 255) / 256 * 256;
}

void fill(const ormi_conv_desc* d, ConvParams* p) {
    p->x = (const char*)d->x;
    p->x_sb = d->x_strides[0];
    p->x_sl = d->x_strides[1];
    p->initial = (const char*)d->initial;
    p->weight = d->weight;
    p->bias = d->bias;
    p->docs = d->documents;
    p->docs_sb = d->documents_batch_stride;
    p->lengths = d->lengths;
    p->out = (char*)d->out;
    p->last = (char*)d->last;
}

int launch(const ormi_conv_desc* d, const ConvParams& p, bool gradient, bool wide_dout, const char* name) {
    const int e = d->dtype == ORMI_DTYPE_F32    ? launch_conv_f32(p, gradient, wide_dout)
                  : d->dtype == ORMI_DTYPE_BF16 ? launch_conv_bf16(p, gradient, wide_dout)
                                                : launch_conv_f16(p, gradient, wide_dout);
    return e == 0 ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string(name) + ": " + hipGetErrorString((hipError_t)e));
}

}  // namespace
}  // namespace ormi_hip

using namespace ormi_hip;

extern "C" {

int ormi_hip_conv(const ormi_conv_desc* d) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_conv: ") + what); };
    if (const char* what = check(d)) return bad(what);
    if (d->batch == 0 || d->channels == 0) return ORMI_HIP_OK;
    if (!d->weight) return bad("null weight");
    if (d->length > 0 && (!d->x || !d->out)) return bad("null x or out");
    ConvParams p{};
    if (!plan(d, false, &p) || (long long)d->batch * d->channels > kMostGroups * 256) return bad("too large");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    fill(d, &p);
    return launch(d, p, false, false, "ormi_hip_conv");
}

int ormi_hip_conv_grad_workspace_size(const ormi_conv_grad_desc* g, size_t* bytes) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_conv_grad_workspace_size: ") + what); };
    if (!g || !bytes) return bad("null descriptor or bytes");
    if (const char* what = check(&g->forward)) return bad(what);
    *bytes = 0;
    if (!g->dweight && !g->dbias) return ORMI_HIP_OK;
    const int rc = ensure_init();
    if (rc != ORMI_HIP_OK) return rc;
    ConvParams p{};
    if (!plan(&g->forward, true, &p)) return bad("too large");
    *bytes = sums_bytes(p);
    return ORMI_HIP_OK;
}

int ormi_hip_conv_grad(const ormi_conv_grad_desc* g) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_conv_grad: ") + what); };
    if (!g) return bad("null descriptor");
    const ormi_conv_desc* d = &g->forward;
    if (const char* what = check(d)) return bad(what);
    if (g->dout && g->dout_dtype != d->dtype && g->dout_dtype != ORMI_DTYPE_F32) return bad("dout must have x's type or float32");
    if (g->dout && !near(d->length, g->dout_strides[1])) return bad("tokens more than 2^20 elements apart");
    if (d->channels == 0) return ORMI_HIP_OK;
    if (!d->weight) return bad("null weight");
    if (d->length > 0 && d->batch > 0 && !d->x) return bad("null x");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK) return rc;
    ConvParams p{};
    if (!plan(d, true, &p)) return bad("too large");
    const bool sums = g->dweight || g->dbias;
    if (sums && sums_bytes(p) > 0 && (!g->workspace || g->workspace_bytes < sums_bytes(p))) return bad("workspace too small");
    if ((rc = drain_queue()) != ORMI_HIP_OK) return rc;
    fill(d, &p);
    p.dout = (const char*)g->dout;
    p.do_sb = g->dout_strides[0];
    p.do_sl = g->dout_strides[1];
    p.dlast = g->dlast;
    p.dx = (char*)g->dx;
    p.dinitial = (char*)g->dinitial;
    p.dweight = g->dweight;
    p.dbias = g->dbias;
    p.part_sums = sums ? (float*)g->workspace : nullptr;
    return launch(d, p, true, g->dout && g->dout_dtype == ORMI_DTYPE_F32, "ormi_hip_conv_grad");
}

}  // extern "C"
