// C entry of the gated linear recurrence and its gradient: checks, work split and
// workspace. The kernels are in recurrence_kernels.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "ormi_hip.h"
#include "ormi_hip_internal.h"
#include "recurrence.h"

namespace ormi_hip {
namespace {

constexpr long long kMostGroups = (1ll << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32
constexpr int kMostTokens = 1 << 30;                // token numbers of a last tile stay in 31 bits

constexpr int kMostStride = 1 << 20;                // elements between tokens: a tile's offsets stay in 32 bits

bool is_float(int dt) { return dt == ORMI_DTYPE_F32 || dt == ORMI_DTYPE_BF16 || dt == ORMI_DTYPE_F16; }

bool near(int length, int64_t stride) { return length <= 1 || (stride >= 0 && stride <= kMostStride); }

const char* check(const ormi_recurrence_desc* d) {
    if (!d) return "null descriptor";
    if (!is_float(d->dtype)) return "dtype must be float32, bfloat16 or float16";
    if (d->gate_dtype != d->dtype && d->gate_dtype != ORMI_DTYPE_F32) return "gates must have x's type or float32";
    if (d->batch < 0 || d->length < 0 || d->channels < 0) return "negative extent";
    if (d->length > kMostTokens) return "more than 2^30 tokens";
    if (d->channels > kMostStride) return "more than 2^20 channels";
    if (!near(d->length, d->gate_strides[1]) || !near(d->length, d->x_strides[1])) return "tokens more than 2^20 elements apart";
    if ((long long)d->batch * ((d->channels + kRecChannels - 1ll) / kRecChannels) > kMostGroups) return "batch * channels too large";
    return nullptr;
}

bool nothing(const ormi_recurrence_desc* d) { return d->batch == 0 || d->channels == 0; }

// The tiles, and whether they are chained: with fewer than two work-groups to a
// compute unit the others do not keep the card's memory busy. Measured, chained and one
// after the other: 256 chains of 8 tiles (16 x 1000 x 1024 fp16) 31 and 40 us; chains of
// 16 tiles with their gradient (batches of 2048 x 4096 bf16), 320: 172 and 190, 384: 204
// and 201, 448: 234 and 210, 512: 263 and 233. Past 512 work-groups, as many as are on
// the card at once, the last ones have it to themselves: 640: 335 and 363, 832: 428 and
// 445, 1024: 537 and 496.
void plan(const ormi_recurrence_desc* d, RecParams* p) {
    p->batch = d->batch;
    p->length = d->length;
    p->channels = d->channels;
    p->tiles = (d->length + kRecTile - 1) / kRecTile;
    p->channel_blocks = (int)((d->channels + kRecChannels - 1ll) / kRecChannels);
    p->chains = p->channel_blocks * d->batch;
    p->chained = p->tiles > 1 && p->chains < 2 * compute_units();
}

// Spans, states, then the counters.
size_t workspace_bytes(const RecParams& p) {
    return p.chained ? (chain_words(p) * sizeof(unsigned) + 255) / 256 * 256 + kRecCounters * kRecCounterStride * sizeof(unsigned) : 0;
}

void fill(const ormi_recurrence_desc* d, RecParams* p) {
    p->gates = (const char*)d->gates;
    p->x = (const char*)d->x;
    p->g_sb = d->gate_strides[0];
    p->g_sl = d->gate_strides[1];
    p->x_sb = d->x_strides[0];
    p->x_sl = d->x_strides[1];
    p->initial = d->initial;
    p->docs = d->documents;
    p->docs_sb = d->documents_batch_stride;
    p->lengths = d->lengths;
    p->out = (char*)d->out;
    p->last = d->last;
    p->states = d->states;
    if (p->chained) {
        const long long row = (long long)p->chains * kRecChannels;
        p->chain_spans = (unsigned long long*)d->workspace;
        p->group_spans = p->chain_spans + p->tiles * row;
        p->group_states = (unsigned*)(p->group_spans + chain_groups(*p) * row);
        p->tickets = (unsigned*)((char*)d->workspace + workspace_bytes(*p)) - kRecCounters * kRecCounterStride;
    }
}

int launch(const ormi_recurrence_desc* d, const RecParams& p, const RecCall& c, const char* name) {
    const int e = d->dtype == ORMI_DTYPE_F32    ? launch_recurrence_f32(p, c)
                  : d->dtype == ORMI_DTYPE_BF16 ? launch_recurrence_bf16(p, c)
                                                : launch_recurrence_f16(p, c);
    return e == 0 ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string(name) + ": " + hipGetErrorString((hipError_t)e));
}

}  // namespace
}  // namespace ormi_hip

using namespace ormi_hip;

extern "C" {

int ormi_hip_recurrence_workspace_size(const ormi_recurrence_desc* d, size_t* bytes) {
    if (const char* what = check(d)) return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_recurrence_workspace_size: ") + what);
    if (!bytes) return fail(ORMI_HIP_ERR_INVALID, "ormi_hip_recurrence_workspace_size: null bytes");
    *bytes = 0;
    if (nothing(d)) return ORMI_HIP_OK;
    const int rc = ensure_init();
    if (rc != ORMI_HIP_OK) return rc;
    RecParams p{};
    plan(d, &p);
    *bytes = workspace_bytes(p);
    return ORMI_HIP_OK;
}

int ormi_hip_recurrence(const ormi_recurrence_desc* d) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_recurrence: ") + what); };
    if (const char* what = check(d)) return bad(what);
    if (nothing(d)) return ORMI_HIP_OK;
    if (d->length > 0 && (!d->gates || !d->x || !d->out)) return bad("null gates, x or out");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    RecParams p{};
    plan(d, &p);
    if (workspace_bytes(p) > 0 && (!d->workspace || d->workspace_bytes < workspace_bytes(p))) return bad("workspace too small");
    fill(d, &p);
    if (p.chained && (long long)p.chains * p.tiles > kMostGroups) return bad("batch * length * channels too large");
    return launch(d, p, RecCall{d->gate_dtype == ORMI_DTYPE_F32, false, d->logits != 0, false}, "ormi_hip_recurrence");
}

int ormi_hip_recurrence_grad(const ormi_recurrence_grad_desc* g) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_recurrence_grad: ") + what); };
    if (!g) return bad("null descriptor");
    const ormi_recurrence_desc* d = &g->forward;
    if (const char* what = check(d)) return bad(what);
    if (g->dout && g->dout_dtype != d->dtype && g->dout_dtype != ORMI_DTYPE_F32) return bad("dout must have x's type or float32");
    if (g->dout && !near(d->length, g->dout_strides[1])) return bad("tokens more than 2^20 elements apart");
    if (nothing(d)) return ORMI_HIP_OK;
    if (d->length > 0 && (!d->gates || !d->x || !d->states)) return bad("null gates, x or states");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    RecParams p{};
    plan(d, &p);
    if (workspace_bytes(p) > 0 && (!d->workspace || d->workspace_bytes < workspace_bytes(p))) return bad("workspace too small");
    fill(d, &p);
    p.dout = (const char*)g->dout;
    p.do_sb = g->dout_strides[0];
    p.do_sl = g->dout_strides[1];
    p.dlast = g->dlast;
    p.dgates = (char*)g->dgates;
    p.dx = (char*)g->dx;
    p.dinitial = g->dinitial;
    if (p.chained && (long long)p.chains * p.tiles > kMostGroups) return bad("batch * length * channels too large");
    return launch(d, p, RecCall{d->gate_dtype == ORMI_DTYPE_F32, g->dout && g->dout_dtype == ORMI_DTYPE_F32, d->logits != 0, true},
                  "ormi_hip_recurrence_grad");
}

}  // extern "C"
