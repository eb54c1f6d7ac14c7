// C entry of attention and its gradient: checks, operand packing, document
// ranges, work split and workspace. The kernels are in attention_kernels.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <string>

#include "attention.h"
#include "ormi_hip.h"
#include "ormi_hip_internal.h"

namespace ormi_hip {
namespace {

// A view with rows the kernels cannot read in 16-byte chunks, copied to
// (batch, token, head, padded features), the padding zero.
__global__ __launch_bounds__(256) void attention_pack_kernel(void* dst, const void* src, int es, int tokens, int heads, int dim,
                                                             int padded, long long sb, long long sl, long long sh, long long sd,
                                                             long long count) {
    for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < count; x += (long long)gridDim.x * 256) {
        const int d = (int)(x % padded);
        const long long y = x / padded;
        const int h = (int)(y % heads);
        const long long z = y / heads;
        const long long at = (z / tokens) * sb + (z % tokens) * sl + h * sh + d * sd;
        if (es == 4) ((float*)dst)[x] = d < dim ? ((const float*)src)[at] : 0.0f;
        else ((unsigned short*)dst)[x] = d < dim ? ((const unsigned short*)src)[at] : (unsigned short)0;
    }
}

// The lowest and highest document of each kDocTile tokens. A tile that also has
// tokens without one (negative) gets a range of two, so that no kernel takes it
// for a tile of a single document; one without any is empty.
__global__ __launch_bounds__(64) void attention_ranges_kernel(int2* ranges, const int* docs, long long sb, int keys, int tiles) {
    const int t = blockIdx.x % tiles, b = blockIdx.x / tiles, j = t * kDocTile + (int)threadIdx.x;
    const int doc = j < keys ? docs[b * sb + j] : -1;
    int lo = doc >= 0 ? doc : 0x7fffffff, hi = doc >= 0 ? doc : -1;
    const bool none = __any(doc < 0);
    for (int d = 1; d < 64; d <<= 1) {
        lo = min(lo, __shfl_xor(lo, d, 64));
        hi = max(hi, __shfl_xor(hi, d, 64));
    }
    if (none && lo == hi) {
        if (hi < 0x7fffffff) ++hi;
        else --lo;
    }
    if (threadIdx.x == 0) ranges[blockIdx.x] = make_int2(lo, hi);
}

__global__ __launch_bounds__(256) void attention_clear_kernel(unsigned* at, int n) {
    for (int i = (int)(blockIdx.x * 256 + threadIdx.x); i < n; i += (int)gridDim.x * 256) at[i] = 0;
}

// An operand as the kernels read it.
struct Operand {
    const void* ptr = nullptr;
    long long sb = 0, sl = 0, sh = 0, sd = 0;
    int tokens = 0, heads = 0;
    bool pack = false;
    size_t at = 0;  // of the packed copy in the workspace
};

struct Plan {
    AttnParams p{};
    Operand q, k, v, g;
    int es = 0, padded = 0;
    bool empty = false;
    size_t ranges = 0, part = 0, part_q = 0, part_ml = 0, delta = 0, bounds = 0, bytes = 0;
    bool hold = false;  // float16 gradients
};

size_t take(size_t& bytes, size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
}

Operand operand(const void* ptr, const int64_t (&s)[4], int batch, int tokens, int heads, int dim, int es, int group) {
    Operand o;
    o.ptr = ptr;
    o.tokens = tokens;
    o.heads = heads;
    o.sb = batch > 1 ? s[0] : 0;
    o.sl = tokens > 1 ? s[1] : 0;
    o.sh = heads > 1 ? s[2] : 0;
    o.sd = dim > 1 ? s[3] : 1;
    const long long tile = 66;  // tokens that one tile's 32-bit offsets span
    auto uneven = [&](long long v) { return v < 0 || v * es % 16 != 0; };
    o.pack = o.sd != 1 || (uintptr_t)ptr % 16 != 0 || dim * es % 16 != 0 || uneven(o.sb) || uneven(o.sl) || uneven(o.sh) ||
             (o.sl * tile + o.sh * group) * es >= (1ll << 31);
    return o;
}

int plan_attention(const ormi_attention_desc* d, const ormi_attention_grad_desc* g, const char* who, Plan* out) {
    auto bad = [&](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string(who) + ": " + what); };
    if (!d) return bad("null descriptor");
    if (d->dtype != ORMI_DTYPE_F32 && d->dtype != ORMI_DTYPE_BF16 && d->dtype != ORMI_DTYPE_F16)
        return bad("dtype must be float32, bfloat16 or float16");
    if (d->batch < 0 || d->queries < 0 || d->keys < 0 || d->heads < 1 || d->kv_heads < 1) return bad("negative extent or no heads");
    if (d->heads % d->kv_heads != 0) return bad("heads must be a multiple of kv_heads");
    if (d->dim < 1 || d->dim > ORMI_ATTENTION_MAX_DIM) return bad("head dim must be 1 to 256");
    if (!(d->cap >= 0.0f) || d->cap > 1e30f) return bad("cap must be zero or positive");
    if (!(d->scale >= -1e30f && d->scale <= 1e30f)) return bad("scale must be finite");
    if (d->prefix && !d->causal) return bad("a prefix needs causal");
    if (d->documents && d->documents_batch_stride < 0) return bad("negative document stride");
    Plan& pl = *out;
    AttnParams& p = pl.p;
    p.batch = d->batch;
    p.queries = d->queries;
    p.keys = d->keys;
    p.heads = d->heads;
    p.kv_heads = d->kv_heads;
    p.group = d->heads / d->kv_heads;
    p.dim = d->dim;
    if ((long long)d->queries * p.group >= (1ll << 30) || d->keys >= (1 << 30)) return bad("more than 2^30 rows or keys");
    if ((long long)d->batch * d->kv_heads >= (1 << 24)) return bad("more than 2^24 batches of key heads");
    p.rows = d->queries * p.group;
    pl.empty = d->batch == 0 || d->queries == 0;
    const bool none = pl.empty || d->keys == 0;
    if (!pl.empty && (!d->q || !d->out)) return bad("null q or out");
    if (!none && (!d->k || !d->v)) return bad("null k or v");
    if (g && !pl.empty && (!d->lse || !g->dout)) return bad("null lse or dout");
    p.causal = d->causal != 0;
    p.scale = d->scale;
    const double log2e = 1.4426950408889634;
    p.scale2 = (float)(d->scale * log2e);
    p.cap2 = (float)(d->cap * log2e);
    p.scale_over_cap = d->cap > 0.0f ? d->scale / d->cap : 0.0f;
    p.slopes = d->slopes;
    p.docs = d->documents;
    p.docs_sb = d->documents_batch_stride;
    p.prefix = d->prefix;
    p.lengths = d->lengths;
    p.out = (char*)d->out;
    p.lse = d->lse;
    p.rest = d->dtype == ORMI_DTYPE_F32 ? nullptr : (char*)d->rest;
    p.form = d->cap > kWideCap ? kCapWide : d->cap > 0.0f ? kCap : d->slopes ? kBias : kPlain;
    const int es = pl.es = d->dtype == ORMI_DTYPE_F32 ? 4 : 2, ve = 16 / es;
    pl.padded = (d->dim + ve - 1) / ve * ve;
    p.chunks = pl.padded / ve;
    // ceil(log2 group) and the multiplier of ormi_fdiv.
    while ((1ull << p.group_s) < (unsigned long long)p.group) ++p.group_s;
    p.group_m = (unsigned)(((1ull << 32) * ((1ull << p.group_s) - p.group)) / p.group + 1);

    pl.q = operand(d->q, d->q_strides, d->batch, d->queries, d->heads, d->dim, es, p.group);
    pl.k = operand(d->k, d->k_strides, d->batch, d->keys, d->kv_heads, d->dim, es, 1);
    pl.v = operand(d->v, d->v_strides, d->batch, d->keys, d->kv_heads, d->dim, es, 1);
    if (g) pl.g = operand(g->dout, g->dout_strides, d->batch, d->queries, d->heads, d->dim, es, p.group);
    for (Operand* o : {&pl.q, &pl.k, &pl.v, &pl.g}) {
        if (!o->pack) continue;
        o->at = take(pl.bytes, (size_t)d->batch * o->tokens * o->heads * pl.padded * es);
        o->sd = 1;
        o->sh = pl.padded;
        o->sl = (long long)o->heads * pl.padded;
        o->sb = o->sl * o->tokens;
        if ((o->sl * 66 + o->sh * p.group) * es >= (1ll << 31)) return bad("heads * dim too large");
    }
    p.range_tiles = (d->keys + kDocTile - 1) / kDocTile;
    if (d->documents) pl.ranges = take(pl.bytes, sizeof(int2) * (size_t)d->batch * std::max(p.range_tiles, 1));

    const int dp = d->dim <= 64 ? 64 : d->dim <= 96 ? 96 : d->dim <= 128 ? 128 : 256, cus = compute_units();
    const long long heads = (long long)d->batch * d->kv_heads;
    p.spread = heads % 8 == 0 ? 1 : heads % 4 == 0 ? 2 : heads % 2 == 0 ? 4 : 8;
    if (!g) {
        // Few rows (single tokens): one wave per work-group. Where the rows of
        // all heads leave compute units idle the keys are split over work-groups
        // and joined.
        p.wide = p.rows > 32;
        p.row_blocks = p.wide ? (p.rows + 127) / 128 : 1;
        const int bn = fwd_tile(dp, es, !p.wide);
        const long long items = heads * p.row_blocks, slots = (long long)cus * (p.wide ? (es == 4 ? 3 : 2) : 4);
        const int tiles = (d->keys + bn - 1) / bn;
        p.splits = 1;
        if (items > 0 && items * 2 <= slots) {
            // Single tokens over unequal lengths: splits of one size, twice as many as
            // fit, so that short sequences leave room instead of finishing early.
            const bool even = !p.wide && d->lengths;
            const long long want = std::min<long long>({(even ? 2 * slots : slots) / items, p.wide ? tiles / 2 : tiles, 64});
            p.splits = (int)std::max<long long>(1, want);
            if (even) p.split_tiles = (tiles + p.splits - 1) / p.splits;
        }
        if (p.splits > 1) {
            pl.part = take(pl.bytes, sizeof(float) * (size_t)p.splits * heads * p.rows * dp);
            pl.part_ml = take(pl.bytes, sizeof(float2) * (size_t)p.splits * heads * p.rows);
        }
        if (items * p.splits >= (1ll << 30)) return bad("too many work-groups");
    } else {
        p.row_blocks = (p.rows + 127) / 128;
        p.key_blocks = (d->keys + 127) / 128;
        // Rows are split so that causal work-groups of unequal length even out;
        // with documents most of a split would see nothing, so only to fill the card.
        const long long items = heads * p.key_blocks, slots = (long long)cus * (d->documents ? 1 : 4);
        const int tiles = (p.rows + 31) / 32;
        p.key_splits = items > 0 ? (int)std::max<long long>(1, std::min<long long>({slots / items, tiles / 8, 16})) : 1;
        if (p.key_splits > 1 && (g->dk || g->dv)) pl.part = take(pl.bytes, 2 * sizeof(float) * (size_t)p.key_splits * heads * d->keys * dp);
        const long long row_items = heads * p.row_blocks;
        const int key_tiles = (d->keys + 31) / 32;
        const long long row_slots = (long long)cus * (es == 4 ? 3 : 2);
        p.splits = row_items > 0 && row_items * 2 <= row_slots ? (int)std::max<long long>(1, std::min<long long>({row_slots / row_items, key_tiles / 4, 16})) : 1;
        if (p.splits > 1 && g->dq) pl.part_q = take(pl.bytes, sizeof(float) * (size_t)p.splits * heads * p.rows * dp);
        if (items * p.key_splits >= (1ll << 30) || heads * p.row_blocks >= (1ll << 30)) return bad("too many work-groups");
        pl.delta = take(pl.bytes, sizeof(float) * (size_t)heads * p.rows);
        pl.hold = d->dtype == ORMI_DTYPE_F16;
        if (pl.hold) pl.bounds = take(pl.bytes, 2 * sizeof(unsigned) * (size_t)heads);
        p.dq = (char*)g->dq;
        p.dk = (char*)g->dk;
        p.dv = (char*)g->dv;
    }
    return ORMI_HIP_OK;
}

int launched(const char* who, int e) {
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string(who) + ": " + hipGetErrorString((hipError_t)e));
}

// Packs the operands that have to be and fills in the kernels' pointers and strides.
void settle(Plan& pl, char* ws, const ormi_attention_desc* d, const ormi_attention_grad_desc* g) {
    AttnParams& p = pl.p;
    auto use = [&](const Operand& o, const int64_t (&s)[4], const char*& ptr, long long& sb, long long& sl, long long& sh) {
        ptr = (const char*)o.ptr;
        if (o.pack && o.tokens > 0) {
            const long long count = (long long)p.batch * o.tokens * o.heads * pl.padded;
            const unsigned grid = (unsigned)std::min<long long>((count + 255) / 256, (long long)compute_units() * 16);
            attention_pack_kernel<<<grid, 256>>>(ws + o.at, o.ptr, pl.es, o.tokens, o.heads, p.dim, pl.padded, s[0], s[1], s[2], s[3], count);
            ptr = ws + o.at;
        }
        sb = o.sb;
        sl = o.sl;
        sh = o.sh;
    };
    use(pl.q, d->q_strides, p.q, p.q_sb, p.q_sl, p.q_sh);
    use(pl.k, d->k_strides, p.k, p.k_sb, p.k_sl, p.k_sh);
    use(pl.v, d->v_strides, p.v, p.v_sb, p.v_sl, p.v_sh);
    if (g) use(pl.g, g->dout_strides, p.dout, p.do_sb, p.do_sl, p.do_sh);
    if (p.docs) {
        int2* r = (int2*)(ws + pl.ranges);
        attention_ranges_kernel<<<(unsigned)(p.batch * p.range_tiles), kDocTile>>>(r, p.docs, p.docs_sb, p.keys, p.range_tiles);
        p.ranges = r;
    }
    p.part = (float*)(ws + pl.part);
    p.part_q = (float*)(ws + pl.part_q);
    p.part_ml = (float2*)(ws + pl.part_ml);
}

int check_workspace(const char* who, const Plan& pl, const void* ws, size_t have) {
    if (pl.bytes == 0 || (ws && have >= pl.bytes)) return ORMI_HIP_OK;
    return fail(ORMI_HIP_ERR_INVALID, std::string(who) + ": needs " + std::to_string(pl.bytes) + " bytes of workspace");
}

// Zeros for an output whose every element has nothing to add up.
int zeros(void* out, size_t elements, int es) {
    const unsigned zero = 0;
    return out && elements ? ormi_hip_fill(out, &zero, (size_t)es, elements) : ORMI_HIP_OK;
}

}  // namespace
}  // namespace ormi_hip

using namespace ormi_hip;

extern "C" {

int ormi_hip_attention_workspace_size(const ormi_attention_desc* desc, size_t* bytes) {
    if (!bytes) return fail(ORMI_HIP_ERR_INVALID, "ormi_hip_attention_workspace_size: null output");
    Plan pl;
    const int rc = plan_attention(desc, nullptr, "ormi_hip_attention_workspace_size", &pl);
    if (rc == ORMI_HIP_OK) *bytes = pl.empty ? 0 : pl.bytes;
    return rc;
}

int ormi_hip_attention(const ormi_attention_desc* desc) {
    const char* who = "ormi_hip_attention";
    Plan pl;
    int rc = plan_attention(desc, nullptr, who, &pl);
    if (rc != ORMI_HIP_OK || pl.empty) return rc;
    if ((rc = check_workspace(who, pl, desc->workspace, desc->workspace_bytes)) != ORMI_HIP_OK) return rc;
    if ((rc = ensure_init()) != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    if (desc->keys == 0) {
        const float none = __builtin_huge_valf();
        const size_t rows = (size_t)desc->batch * desc->queries * desc->heads;
        if ((rc = zeros(desc->out, rows * desc->dim, pl.es)) != ORMI_HIP_OK) return rc;
        if ((rc = zeros(pl.p.rest, rows * desc->dim, pl.es)) != ORMI_HIP_OK) return rc;
        return desc->lse ? ormi_hip_fill(desc->lse, &none, 4, rows) : ORMI_HIP_OK;
    }
    settle(pl, (char*)desc->workspace, desc, nullptr);
    switch (desc->dtype) {
        case ORMI_DTYPE_F32: return launched(who, launch_attention_fwd_f32(pl.p));
        case ORMI_DTYPE_BF16: return launched(who, launch_attention_fwd_bf16(pl.p));
        default: return launched(who, launch_attention_fwd_f16(pl.p));
    }
}

int ormi_hip_attention_grad_workspace_size(const ormi_attention_grad_desc* desc, size_t* bytes) {
    const char* who = "ormi_hip_attention_grad_workspace_size";
    if (!bytes || !desc) return fail(ORMI_HIP_ERR_INVALID, std::string(who) + ": null argument");
    Plan pl;
    const int rc = plan_attention(&desc->forward, desc, who, &pl);
    if (rc == ORMI_HIP_OK) *bytes = pl.empty || desc->forward.keys == 0 ? 0 : pl.bytes;
    return rc;
}

int ormi_hip_attention_grad(const ormi_attention_grad_desc* desc) {
    const char* who = "ormi_hip_attention_grad";
    if (!desc) return fail(ORMI_HIP_ERR_INVALID, std::string(who) + ": null descriptor");
    const ormi_attention_desc* d = &desc->forward;
    Plan pl;
    int rc = plan_attention(d, desc, who, &pl);
    if (rc != ORMI_HIP_OK) return rc;
    if (!desc->dq && !desc->dk && !desc->dv) return ORMI_HIP_OK;
    if (pl.empty || d->keys == 0) {
        if ((rc = ensure_init()) != ORMI_HIP_OK) return rc;
        const size_t nq = (size_t)d->batch * d->queries * d->heads * d->dim, nk = (size_t)d->batch * d->keys * d->kv_heads * d->dim;
        if ((rc = zeros(desc->dq, nq, pl.es)) != ORMI_HIP_OK || (rc = zeros(desc->dk, nk, pl.es)) != ORMI_HIP_OK) return rc;
        return zeros(desc->dv, nk, pl.es);
    }
    if ((rc = check_workspace(who, pl, d->workspace, d->workspace_bytes)) != ORMI_HIP_OK) return rc;
    if ((rc = ensure_init()) != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    char* ws = (char*)d->workspace;
    settle(pl, ws, d, desc);
    float* delta = (float*)(ws + pl.delta);
    unsigned* bounds = pl.hold ? (unsigned*)(ws + pl.bounds) : nullptr;
    if (bounds) {
        const int n = 2 * d->batch * d->kv_heads;
        attention_clear_kernel<<<(unsigned)std::min((n + 255) / 256, 256), 256>>>(bounds, n);
    }
    pl.p.delta = delta;
    pl.p.grad_scale = (const float*)bounds;
    switch (d->dtype) {
        case ORMI_DTYPE_F32: return launched(who, launch_attention_grad_f32(pl.p, delta, bounds));
        case ORMI_DTYPE_BF16: return launched(who, launch_attention_grad_bf16(pl.p, delta, bounds));
        default: return launched(who, launch_attention_grad_f16(pl.p, delta, bounds));
    }
}

}  // extern "C"
