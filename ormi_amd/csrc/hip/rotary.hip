// Rotary positions: pairs of features turned by their token's angle.
//   a' = a cos - b sin,  b' = b cos + a sin
// Bound by memory: every element is read and written once for three flops. A
// thread turns the same V pairs of up to HEADS heads of one token, so a table
// row (8 bytes per pair, as much as a pair of fp32 features) is read once for
// them and their loads are in flight together.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "device/ormi_device.h"
#include "ormi_hip.h"
#include "ormi_hip_internal.h"

namespace ormi_hip {
namespace {

struct RotaryParams {
    const char* x;
    char* out;
    long long sb, sl, sh, sd;  // x, in elements
    const float *cos, *sin;
    const int* positions;
    long long pos_sb, pos_sl;
    int offset, rows;
    int length, heads, dim, part;
    float sign;
    unsigned units, turned, groups;  // V-pair units of a row (the turned ones first), head groups of a token
    unsigned first, total;           // tokens before this launch, threads of it
    unsigned units_m, units_s, groups_m, groups_s, length_m, length_s;
};

template <int DT> struct Elem { using type = unsigned short; };
template <> struct Elem<ORMI_DTYPE_F32> { using type = float; };

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::type v) {
    if constexpr (DT == ORMI_DTYPE_F32) return v;
    else return DT == ORMI_DTYPE_BF16 ? ormi_bf16_to_f32(v) : ormi_f16_to_f32(v);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::type from_f32(float v) {
    if constexpr (DT == ORMI_DTYPE_F32) return v;
    else return DT == ORMI_DTYPE_BF16 ? ormi_f32_to_bf16(v) : ormi_f32_to_f16(v);
}
// N elements in as few 16-byte (or smaller) accesses as they take.
template <int DT, int N>
struct alignas(N * sizeof(typename Elem<DT>::type) >= 16 ? 16 : N * sizeof(typename Elem<DT>::type)) Pack {
    typename Elem<DT>::type v[N];
};

constexpr int HEADS = 4;

template <int IN, int OUT, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
    using TI = typename Elem<IN>::type;
    using TO = typename Elem<OUT>::type;
    const unsigned id = blockIdx.x * 256 + threadIdx.x;
    if (id >= p.total) return;
    const unsigned rest = ormi_fdiv(id, p.units_m, p.units_s), u = id - rest * p.units;
    const unsigned tok0 = ormi_fdiv(rest, p.groups_m, p.groups_s), hg = rest - tok0 * p.groups;
    const unsigned tok = tok0 + p.first;
    const unsigned b = ormi_fdiv(tok, p.length_m, p.length_s), l = tok - b * (unsigned)p.length;
    const int h0 = (int)hg * HEADS, hn = min(HEADS, p.heads - h0);
    const TI* x = (const TI*)p.x + (b * p.sb + l * p.sl + (long long)h0 * p.sh);
    TO* out = (TO*)p.out + ((long long)tok * p.heads + h0) * p.dim;
    // The unit's 2 V elements: two runs of V, the second `apart` after the first.
    const bool turn = u < p.turned;
    int d, apart;
    if (turn) {
        d = INTERLEAVED ? (int)u * 2 * V : (int)u * V;
        apart = INTERLEAVED ? V : p.part / 2;
    } else {
        d = p.part + (int)(u - p.turned) * 2 * V;
        apart = V;
    }
    const bool second = turn || V > 1 || d + 1 < p.dim;  // one feature may be left over at V = 1
    float c[V], s[V];
    if (turn) {
        const long long at = p.positions ? p.positions[b * p.pos_sb + l * p.pos_sl] : (long long)p.offset + l;
        const bool inside = at >= 0 && at < p.rows;
        const long long row = (inside ? at : 0) * (p.part / 2) + (long long)u * V;
        const Pack<ORMI_DTYPE_F32, V> cv = *(const Pack<ORMI_DTYPE_F32, V>*)(p.cos + row);
        const Pack<ORMI_DTYPE_F32, V> sv = *(const Pack<ORMI_DTYPE_F32, V>*)(p.sin + row);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            c[e] = inside ? cv.v[e] : __builtin_nanf("");
            s[e] = inside ? sv.v[e] * p.sign : __builtin_nanf("");
        }
    }
    Pack<IN, V> r0[HEADS], r1[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (h >= hn) continue;
        const TI* at = x + h * p.sh;
        if (V > 1) {
            r0[h] = *(const Pack<IN, V>*)(at + d);
            r1[h] = *(const Pack<IN, V>*)(at + d + apart);
        } else {
            r0[h].v[0] = at[d * p.sd];
            if (second) r1[h].v[0] = at[(d + apart) * p.sd];
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (h >= hn) continue;
        Pack<OUT, V> o0, o1;
        if (!turn) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                o0.v[e] = from_f32<OUT>(to_f32<IN>(r0[h].v[e]));
                o1.v[e] = second ? from_f32<OUT>(to_f32<IN>(r1[h].v[e])) : TO(0);
            }
        } else if (INTERLEAVED && V > 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = 2 * e, j = 2 * e + 1;
                const float a = to_f32<IN>(i < V ? r0[h].v[i % V] : r1[h].v[i % V]);
                const float q = to_f32<IN>(j < V ? r0[h].v[j % V] : r1[h].v[j % V]);
                const TO na = from_f32<OUT>(a * c[e] - q * s[e]), nb = from_f32<OUT>(q * c[e] + a * s[e]);
                if (i < V) o0.v[i % V] = na;
                else o1.v[i % V] = na;
                if (j < V) o0.v[j % V] = nb;
                else o1.v[j % V] = nb;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float a = to_f32<IN>(r0[h].v[e]), q = to_f32<IN>(r1[h].v[e]);
                o0.v[e] = from_f32<OUT>(a * c[e] - q * s[e]);
                o1.v[e] = from_f32<OUT>(q * c[e] + a * s[e]);
            }
        }
        TO* at = out + (long long)h * p.dim;
        *(Pack<OUT, V>*)(at + d) = o0;
        if (second) *(Pack<OUT, V>*)(at + d + apart) = o1;
    }
}

template <int IN, int OUT, int V>
void launch_v(const RotaryParams& p, bool interleaved) {
    const unsigned grid = (p.total + 255) / 256;
    if (interleaved) rotary_kernel<IN, OUT, V, true><<<grid, 256>>>(p);
    else rotary_kernel<IN, OUT, V, false><<<grid, 256>>>(p);
}
template <int IN, int OUT>
void launch_types(const RotaryParams& p, int v, bool interleaved) {
    if (v == 8) launch_v<IN, OUT, 8>(p, interleaved);
    else if (v == 4) launch_v<IN, OUT, 4>(p, interleaved);
    else launch_v<IN, OUT, 1>(p, interleaved);
}
template <int IN>
void launch_in(const RotaryParams& p, int out, int v, bool interleaved) {
    switch (out) {
        case ORMI_DTYPE_F32: launch_types<IN, ORMI_DTYPE_F32>(p, v, interleaved); break;
        case ORMI_DTYPE_BF16: launch_types<IN, ORMI_DTYPE_BF16>(p, v, interleaved); break;
        default: launch_types<IN, ORMI_DTYPE_F16>(p, v, interleaved);
    }
}

void divider(unsigned d, unsigned* m, unsigned* s) {  // for ormi_fdiv
    *s = 0;
    while ((1ull << *s) < d) ++*s;
    *m = (unsigned)(((1ull << 32) * ((1ull << *s) - d)) / d + 1);
}

bool is_float(int dt) { return dt == ORMI_DTYPE_F32 || dt == ORMI_DTYPE_BF16 || dt == ORMI_DTYPE_F16; }

}  // namespace
}  // namespace ormi_hip

using namespace ormi_hip;

extern "C" int ormi_hip_rotary(const ormi_rotary_desc* d) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_rotary: ") + what); };
    if (!d) return bad("null descriptor");
    if (!is_float(d->dtype) || !is_float(d->out_dtype)) return bad("dtypes must be float32, bfloat16 or float16");
    if (d->batch < 0 || d->length < 0 || d->heads < 0 || d->dim < 0) return bad("negative extent");
    if (d->part < 0 || d->part > d->dim || d->part % 2 != 0) return bad("part must be even and at most dim");
    if (d->table_rows < 0) return bad("negative table rows");
    if (d->batch == 0 || d->length == 0 || d->heads == 0 || d->dim == 0) return ORMI_HIP_OK;
    if (!d->x || !d->out) return bad("null x or out");
    if (d->part > 0 && (!d->cos || !d->sin || d->table_rows == 0)) return bad("no tables");
    const long long tokens = (long long)d->batch * d->length;
    if (tokens >= (1ll << 31)) return bad("2^31 tokens or more");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;

    RotaryParams p{};
    p.x = (const char*)d->x;
    p.out = (char*)d->out;
    p.sb = d->x_strides[0];
    p.sl = d->x_strides[1];
    p.sh = d->x_strides[2];
    p.sd = d->x_strides[3];
    p.cos = d->cos;
    p.sin = d->sin;
    p.positions = d->positions;
    p.pos_sb = d->positions_strides[0];
    p.pos_sl = d->positions_strides[1];
    p.offset = d->offset;
    p.rows = d->table_rows;
    p.length = d->length;
    p.heads = d->heads;
    p.dim = d->dim;
    p.part = d->part;
    p.sign = d->inverse ? -1.0f : 1.0f;
    // Pairs per thread: the most whose runs are whole and aligned on both sides.
    const int es_in = d->dtype == ORMI_DTYPE_F32 ? 4 : 2, es_out = d->out_dtype == ORMI_DTYPE_F32 ? 4 : 2;
    auto fits = [&](int v) {
        const long long in = std::min(16, v * es_in), out = std::min(16, v * es_out);
        auto whole = [&](long long stride, int extent) { return extent <= 1 || stride * es_in % in == 0; };
        return (d->dim == 1 || p.sd == 1) && d->part / 2 % v == 0 && (d->dim - d->part) % (2 * v) == 0 &&
               (uintptr_t)d->x % in == 0 && (uintptr_t)d->out % out == 0 && (long long)d->dim * es_out % out == 0 &&
               (uintptr_t)d->cos % 16 == 0 && (uintptr_t)d->sin % 16 == 0 && whole(p.sb, d->batch) && whole(p.sl, d->length) &&
               whole(p.sh, d->heads);
    };
    const int v = fits(8) ? 8 : fits(4) ? 4 : 1;
    p.turned = (unsigned)(d->part / 2 / v);
    p.units = p.turned + (unsigned)((d->dim - d->part + 2 * v - 1) / (2 * v));
    p.groups = (unsigned)((d->heads + HEADS - 1) / HEADS);
    divider(p.units, &p.units_m, &p.units_s);
    divider(p.groups, &p.groups_m, &p.groups_s);
    divider((unsigned)p.length, &p.length_m, &p.length_s);
    // Threads are counted in 31 bits: a longer tensor goes in several launches.
    const long long per_token = (long long)p.units * p.groups, most = std::max<long long>(1, ((1ll << 31) - 512) / per_token);
    for (long long at = 0; at < tokens; at += most) {
        p.first = (unsigned)at;
        p.total = (unsigned)(std::min(most, tokens - at) * per_token);
        switch (d->dtype) {
            case ORMI_DTYPE_F32: launch_in<ORMI_DTYPE_F32>(p, d->out_dtype, v, d->interleaved != 0); break;
            case ORMI_DTYPE_BF16: launch_in<ORMI_DTYPE_BF16>(p, d->out_dtype, v, d->interleaved != 0); break;
            default: launch_in<ORMI_DTYPE_F16>(p, d->out_dtype, v, d->interleaved != 0);
        }
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string("ormi_hip_rotary: ") + hipGetErrorString(e));
}
