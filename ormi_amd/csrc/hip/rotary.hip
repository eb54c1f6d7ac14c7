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
constexpr long long kMostThreads = (1ll << 31) - 512;  // of a launch: they are counted in 31 bits

// Every element is read once and written once, so where each access covers whole
// 128-byte lines (runs of that many bytes) it goes past the caches, which stay
// with the tables: 4 x 4096 x 16 x 128 float32 to bfloat16 45 -> 33 us, 6.0 TB/s.
// Shorter runs share lines between accesses and would fetch them again (float16
// runs of 48 bytes: 15.8 -> 31 us).
template <bool PAST, class P>
__device__ __forceinline__ P stream_in(const void* at) {
    if constexpr (PAST && sizeof(P) % 16 == 0) {
        P r;
#pragma unroll
        for (unsigned i = 0; i < sizeof(P) / 16; ++i) {
            const ormi_f4 w = __builtin_nontemporal_load((const ormi_f4*)at + i);
            __builtin_memcpy((char*)&r + 16 * i, &w, 16);
        }
        return r;
    } else {
        return *(const P*)at;
    }
}
template <bool PAST, class P>
__device__ __forceinline__ void stream_out(void* at, const P& v) {
    if constexpr (PAST && sizeof(P) % 16 == 0) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(P) / 16; ++i) {
            ormi_f4 w;
            __builtin_memcpy(&w, (const char*)&v + 16 * i, 16);
            __builtin_nontemporal_store(w, (ormi_f4*)at + i);
        }
    } else if constexpr (PAST && sizeof(P) == 8) {
        unsigned long long w;
        __builtin_memcpy(&w, &v, 8);
        __builtin_nontemporal_store(w, (unsigned long long*)at);
    } else {
        *(P*)at = v;
    }
}

template <int IN, int OUT, int V, bool INTERLEAVED, bool PAST>
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
    // The unit's 2 V elements: a run of V in each half of the turned features (or
    // of the others), so that the lanes of one access are neighbours, with
    // interleaved pairs too.
    constexpr bool SINGLE = INTERLEAVED && V == 1;  // a pair of neighbours
    const bool turn = u < p.turned;
    int d, apart;
    if (turn) {
        d = SINGLE ? (int)u * 2 : (int)u * V;
        apart = SINGLE ? 1 : p.part / 2;
    } else {
        d = p.part + (int)(u - p.turned) * (V > 1 ? V : 2);
        apart = V > 1 ? (p.dim - p.part) / 2 : 1;
    }
    const bool second = turn || V > 1 || d + 1 < p.dim;  // one feature may be left over at V = 1
    // Cosine and sine of the pairs: V of the two runs' elements, or with
    // interleaved pairs V / 2 of each run.
    float c[V], s[V];
    if (turn) {
        const long long at = p.positions ? p.positions[b * p.pos_sb + l * p.pos_sl] : (long long)p.offset + l;
        const bool inside = at >= 0 && at < p.rows;
        const long long row = (inside ? at : 0) * (p.part / 2);
        constexpr int H = INTERLEAVED && V > 1 ? V / 2 : V;
#pragma unroll
        for (int k = 0; k < V / H; ++k) {
            const long long from = row + (long long)u * H + k * (p.part / 4);
            const Pack<ORMI_DTYPE_F32, H> cv = *(const Pack<ORMI_DTYPE_F32, H>*)(p.cos + from);
            const Pack<ORMI_DTYPE_F32, H> sv = *(const Pack<ORMI_DTYPE_F32, H>*)(p.sin + from);
#pragma unroll
            for (int e = 0; e < H; ++e) {
                c[k * H + e] = inside ? cv.v[e] : __builtin_nanf("");
                s[k * H + e] = inside ? sv.v[e] * p.sign : __builtin_nanf("");
            }
        }
    }
    Pack<IN, V> r0[HEADS], r1[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (h >= hn) continue;
        const TI* at = x + h * p.sh;
        if (V > 1) {
            r0[h] = stream_in<PAST, Pack<IN, V>>(at + d);
            r1[h] = stream_in<PAST, Pack<IN, V>>(at + d + apart);
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
                const Pack<IN, V>& r = e < V / 2 ? r0[h] : r1[h];
                Pack<OUT, V>& o = e < V / 2 ? o0 : o1;
                const int i = 2 * e % V;
                const float a = to_f32<IN>(r.v[i]), q = to_f32<IN>(r.v[i + 1]);
                o.v[i] = from_f32<OUT>(a * c[e] - q * s[e]);
                o.v[i + 1] = from_f32<OUT>(q * c[e] + a * s[e]);
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
        stream_out<PAST>(at + d, o0);
        if (second) stream_out<PAST>(at + d + apart, o1);
    }
}

template <int IN, int OUT, int V, bool PAST>
void launch_v(const RotaryParams& p, bool interleaved) {
    const unsigned grid = (p.total + 255) / 256;
    if (interleaved) rotary_kernel<IN, OUT, V, true, PAST><<<grid, 256>>>(p);
    else rotary_kernel<IN, OUT, V, false, PAST><<<grid, 256>>>(p);
}
template <int IN, int OUT>
void launch_types(const RotaryParams& p, int v, bool interleaved, bool past) {
    if constexpr (IN != ORMI_DTYPE_F32 && OUT != ORMI_DTYPE_F32)
        if (v == 8) return past ? launch_v<IN, OUT, 8, true>(p, interleaved) : launch_v<IN, OUT, 8, false>(p, interleaved);
    if (v == 4) past ? launch_v<IN, OUT, 4, true>(p, interleaved) : launch_v<IN, OUT, 4, false>(p, interleaved);
    else launch_v<IN, OUT, 1, false>(p, interleaved);
}
template <int IN>
void launch_in(const RotaryParams& p, int out, int v, bool interleaved, bool past) {
    switch (out) {
        case ORMI_DTYPE_F32: launch_types<IN, ORMI_DTYPE_F32>(p, v, interleaved, past); break;
        case ORMI_DTYPE_BF16: launch_types<IN, ORMI_DTYPE_BF16>(p, v, interleaved, past); break;
        default: launch_types<IN, ORMI_DTYPE_F16>(p, v, interleaved, past);
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
    // Threads of one token, at most a launch's (below): a pair of features of four heads each.
    if (((long long)d->dim + 1) / 2 * (((long long)d->heads + HEADS - 1) / HEADS) > kMostThreads) return bad("heads * dim too large");
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
    const bool wide = es_in == 4 || es_out == 4;  // 4 fp32 elements are a whole access
    const int v = !wide && fits(8) ? 8 : fits(4) ? 4 : 1;
    const int run = d->part / 2, rest = (d->dim - d->part) / 2;
    const bool past = run * std::min(es_in, es_out) % 128 == 0 && rest * std::min(es_in, es_out) % 128 == 0;
    p.turned = (unsigned)(d->part / 2 / v);
    p.units = p.turned + (unsigned)((d->dim - d->part + 2 * v - 1) / (2 * v));
    p.groups = (unsigned)((d->heads + HEADS - 1) / HEADS);
    divider(p.units, &p.units_m, &p.units_s);
    divider(p.groups, &p.groups_m, &p.groups_s);
    divider((unsigned)p.length, &p.length_m, &p.length_s);
    // A longer tensor goes in several launches.
    const long long per_token = (long long)p.units * p.groups, most = kMostThreads / per_token;
    for (long long at = 0; at < tokens; at += most) {
        p.first = (unsigned)at;
        p.total = (unsigned)(std::min(most, tokens - at) * per_token);
        switch (d->dtype) {
            case ORMI_DTYPE_F32: launch_in<ORMI_DTYPE_F32>(p, d->out_dtype, v, d->interleaved != 0, past); break;
            case ORMI_DTYPE_BF16: launch_in<ORMI_DTYPE_BF16>(p, d->out_dtype, v, d->interleaved != 0, past); break;
            default: launch_in<ORMI_DTYPE_F16>(p, d->out_dtype, v, d->interleaved != 0, past);
        }
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string("ormi_hip_rotary: ") + hipGetErrorString(e));
}
