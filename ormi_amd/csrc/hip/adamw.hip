// One AdamW step over a list of tensors, moments in 32 or in 8 bits.
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g g
//   p -= lr ((m / c1) / (sqrt(v / c2) + eps) + decay p)
// Bound by memory (28 bytes per fp32 parameter, 16 with 8-bit moments), so the
// work is one pass; the tensors of a list share launches, since a network's
// biases and norms are far smaller than a launch. Their pointers travel in the
// kernel's arguments: nothing is uploaded, and a work-group finds its tensor by
// its first work-group number.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "device/ormi_device.h"
#include "ormi_hip.h"
#include "ormi_hip_internal.h"

namespace ormi_hip {
namespace {

constexpr int kMost = 32;      // tensors per launch: their entries and the scalars fit 4 KB of arguments
constexpr int kPerGroup = 2048;  // elements per work-group: two groups of four per thread
constexpr unsigned long long kMostGroups = (1ull << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32

struct AdamEntry {
    const void *p, *g, *m, *v;
    void *out, *m_out, *v_out;
    const float *m_scale, *v_scale;
    float *m_scale_out, *v_scale_out;
    long long count;
    unsigned first;  // its first work-group
    unsigned char p_dtype, g_dtype, vec, unused;
};
struct AdamParams {
    float lr, b1, ob1, b2, ob2, eps, decay, c1, c2, r1, r2;
    int n;
    AdamEntry t[kMost];
};
static_assert(sizeof(AdamParams) <= 4096, "kernel arguments");

struct f32x4 { float v[4]; };

// Elements [i, i + 4) as fp32; n of them exist.
__device__ __forceinline__ f32x4 load4(const void* base, int dt, long long i, int n, bool vec) {
    f32x4 r = {{0.0f, 0.0f, 0.0f, 0.0f}};
    if (vec && n == 4) {
        if (dt == ORMI_DTYPE_F32) {
            const ormi_f4 q = __builtin_nontemporal_load((const ormi_f4*)((const float*)base + i));
#pragma unroll
            for (int e = 0; e < 4; ++e) r.v[e] = q[e];
        } else {
            const ormi_u16x4 q = __builtin_nontemporal_load((const ormi_u16x4*)((const unsigned short*)base + i));
#pragma unroll
            for (int e = 0; e < 4; ++e) r.v[e] = dt == ORMI_DTYPE_BF16 ? ormi_bf16_to_f32(q[e]) : ormi_f16_to_f32(q[e]);
        }
        return r;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) {
            if (dt == ORMI_DTYPE_F32) r.v[e] = ((const float*)base)[i + e];
            else {
                const unsigned short h = ((const unsigned short*)base)[i + e];
                r.v[e] = dt == ORMI_DTYPE_BF16 ? ormi_bf16_to_f32(h) : ormi_f16_to_f32(h);
            }
        }
    return r;
}
__device__ __forceinline__ void store4(void* base, int dt, long long i, int n, bool vec, const f32x4& x) {
    if (vec && n == 4) {
        if (dt == ORMI_DTYPE_F32) {
            const ormi_f4 q = {x.v[0], x.v[1], x.v[2], x.v[3]};
            __builtin_nontemporal_store(q, (ormi_f4*)((float*)base + i));
        } else {
            ormi_u16x4 q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = dt == ORMI_DTYPE_BF16 ? ormi_f32_to_bf16(x.v[e]) : ormi_f32_to_f16(x.v[e]);
            __builtin_nontemporal_store(q, (ormi_u16x4*)((unsigned short*)base + i));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) {
            if (dt == ORMI_DTYPE_F32) ((float*)base)[i + e] = x.v[e];
            else ((unsigned short*)base)[i + e] = dt == ORMI_DTYPE_BF16 ? ormi_f32_to_bf16(x.v[e]) : ormi_f32_to_f16(x.v[e]);
        }
}

__device__ __forceinline__ int find_tensor(const AdamParams& a) {
    int t = 0;
    for (int step = kMost / 2; step > 0; step >>= 1)
        if (t + step < a.n && a.t[t + step].first <= blockIdx.x) t += step;
    return t;
}

// x / c, rounded correctly, for a c whose correctly rounded reciprocal r is at
// hand (Markstein: a quotient within a unit, corrected by its exact remainder).
// Where the remainder could underflow, or r is 0 (the host found c to be one the
// theorem leaves out), by the division itself.
__device__ __forceinline__ float divide(float x, float c, float r) {
    const float a = __builtin_fabsf(x);
    if (r == 0.0f || !(a <= 0x1p100f) || (a < 0x1p-100f && a != 0.0f)) return x / c;
    const float q = x * r;
    return __builtin_fmaf(__builtin_fmaf(-q, c, x), r, q);
}
// Compiled without contraction: each operation rounds on its own.
__device__ __forceinline__ void update(const AdamParams& a, float g, float& p, float& m, float& v) {
    m = m * a.b1 + g * a.ob1;
    v = v * a.b2 + (g * g) * a.ob2;
    const float rate = divide(m, a.c1, a.r1) / (__builtin_sqrtf(divide(v, a.c2, a.r2)) + a.eps);
    p = p - a.lr * (rate + a.decay * p);
}

// SCALED: every gradient times *factor.
template <bool SCALED>
__global__ __launch_bounds__(256) void adamw_kernel(AdamParams a, const float* factor) {
    const float scale = SCALED ? *factor : 1.0f;
    const AdamEntry& t = a.t[find_tensor(a)];
    const long long base = (long long)(blockIdx.x - t.first) * kPerGroup;
    f32x4 p[2], g[2], m[2], v[2];
    long long i[2];
    int n[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        i[k] = base + k * 1024 + threadIdx.x * 4;
        n[k] = (int)max(0ll, min(4ll, t.count - i[k]));
        p[k] = load4(t.p, t.p_dtype, i[k], n[k], t.vec);
        g[k] = load4(t.g, t.g_dtype, i[k], n[k], t.vec);
        m[k] = load4(t.m, ORMI_DTYPE_F32, i[k], n[k], t.vec);
        v[k] = load4(t.v, ORMI_DTYPE_F32, i[k], n[k], t.vec);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) update(a, SCALED ? g[k].v[e] * scale : g[k].v[e], p[k].v[e], m[k].v[e], v[k].v[e]);
        store4(t.out, t.p_dtype, i[k], n[k], t.vec, p[k]);
        store4(t.m_out, ORMI_DTYPE_F32, i[k], n[k], t.vec, m[k]);
        store4(t.v_out, ORMI_DTYPE_F32, i[k], n[k], t.vec, v[k]);
    }
}

// Codes. The first moment's spacing is finest near zero (its sign apart, the
// square of the code); the second's fourth power lets the root that the step
// divides by span four decades, and no second moment above zero becomes zero.
__device__ __forceinline__ float decode_m(int c, float scale) {
    const float w = (float)(c < 0 ? -c : c) * (float)(1.0 / 127.0), x = w * w * scale;
    return c < 0 ? -x : x;
}
__device__ __forceinline__ float decode_v(int c, float scale) {
    float w = (float)c * (float)(1.0 / 255.0);
    w = w * w;
    return w * w * scale;
}
// Codes of exactly rint(127 sqrt(|x| / scale)) and rint(255 sqrt(sqrt(x / scale))),
// each operation rounded: which integer that is shows from the hardware's
// approximations (a few units in 2^24 of at most 255, so within 2^-12) unless
// they lie that close to half way; only then is it computed in full. The full
// divisions and roots of every element took longer than the memory (25 M
// parameters: 124 us).
__device__ __forceinline__ int code_m(float x, float scale, float inv) {
    const float a = __builtin_fabsf(x);
    float w = __builtin_amdgcn_sqrtf(a * inv) * 127.0f, c = __builtin_rintf(w);
    if (!(__builtin_fabsf(w - c) < 0.5f - 0x1p-12f)) c = __builtin_rintf(__builtin_sqrtf(scale == 0.0f ? 0.0f : a / scale) * 127.0f);
    const int k = (int)fminf(c, 127.0f);
    return x < 0.0f ? -k : k;
}
__device__ __forceinline__ int code_v(float x, float scale, float inv) {
    const float a = __builtin_fabsf(x);
    float w = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(a * inv)) * 255.0f, c = __builtin_rintf(w);
    if (!(__builtin_fabsf(w - c) < 0.5f - 0x1p-12f))
        c = __builtin_rintf(__builtin_sqrtf(__builtin_sqrtf(scale == 0.0f ? 0.0f : a / scale)) * 255.0f);
    const int k = (int)fminf(c, 255.0f);
    return x > 0.0f && k < 1 ? 1 : k;
}
// The approximate reciprocal of a block's scale; NaN (which takes the full way)
// where it or its products could leave the normal range.
__device__ __forceinline__ float scale_inverse(float scale) {
    return scale > 0x1p-90f && scale < 0x1p90f ? __builtin_amdgcn_rcpf(scale) : __builtin_nanf("");
}

// A wave per block of 256 elements, four per lane (their codes one word).
template <bool SCALED>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamParams a, const float* factor) {
    const float scale = SCALED ? *factor : 1.0f;
    const AdamEntry& t = a.t[find_tensor(a)];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long blocks = (t.count + ORMI_ADAMW_BLOCK - 1) / ORMI_ADAMW_BLOCK;
    long long blk[2], i[2];
    int n[2];
    f32x4 p[2], g[2];
    unsigned mc[2], vc[2];
    float ms[2], vs[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        blk[k] = (long long)(blockIdx.x - t.first) * (kPerGroup / ORMI_ADAMW_BLOCK) + k * 4 + wave;
        const long long bc = min(blk[k], blocks - 1);
        i[k] = blk[k] * ORMI_ADAMW_BLOCK + lane * 4;
        n[k] = (int)max(0ll, min(4ll, t.count - i[k]));
        p[k] = load4(t.p, t.p_dtype, i[k], n[k], t.vec);
        g[k] = load4(t.g, t.g_dtype, i[k], n[k], t.vec);
        mc[k] = ((const unsigned*)t.m)[bc * 64 + lane];
        vc[k] = ((const unsigned*)t.v)[bc * 64 + lane];
        ms[k] = t.m_scale[bc];
        vs[k] = t.v_scale[bc];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (blk[k] >= blocks) continue;  // the whole wave
        f32x4 m, v;
        float mt = 0.0f, vt = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m.v[e] = decode_m((int)(signed char)(mc[k] >> (8 * e)), ms[k]);
            v.v[e] = decode_v((int)(unsigned char)(vc[k] >> (8 * e)), vs[k]);
            update(a, SCALED ? g[k].v[e] * scale : g[k].v[e], p[k].v[e], m.v[e], v.v[e]);
            if (e >= n[k]) m.v[e] = v.v[e] = 0.0f;  // padding past the tensor's end
            mt = ormi_maximum(mt, __builtin_fabsf(m.v[e]));
            vt = ormi_maximum(vt, __builtin_fabsf(v.v[e]));
        }
        mt = ormi_lanes_max<64>(mt);
        vt = ormi_lanes_max<64>(vt);
        const float mi = scale_inverse(mt), vi = scale_inverse(vt);
        unsigned mo = 0, vo = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mo |= (unsigned)(code_m(m.v[e], mt, mi) & 255) << (8 * e);
            vo |= (unsigned)(code_v(v.v[e], vt, vi) & 255) << (8 * e);
        }
        store4(t.out, t.p_dtype, i[k], n[k], t.vec, p[k]);
        ((unsigned*)t.m_out)[blk[k] * 64 + lane] = mo;
        ((unsigned*)t.v_out)[blk[k] * 64 + lane] = vo;
        if (lane == 0) {
            t.m_scale_out[blk[k]] = mt;
            t.v_scale_out[blk[k]] = vt;
        }
    }
}

__global__ __launch_bounds__(256) void adamw_values_kernel(float* m, float* v, const unsigned* mc, const float* ms, const unsigned* vc,
                                                           const float* vs, long long count) {
    const long long word = (long long)blockIdx.x * 256 + threadIdx.x, i = word * 4;
    if (i >= count) return;
    const unsigned cm = mc[word], cv = vc[word];
    const float sm = ms[word >> 6], sv = vs[word >> 6];
    const int n = (int)min(4ll, count - i);
    f32x4 a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a.v[e] = decode_m((int)(signed char)(cm >> (8 * e)), sm);
        b.v[e] = decode_v((int)(unsigned char)(cv >> (8 * e)), sv);
    }
    const bool vec = (((uintptr_t)m | (uintptr_t)v) & 15) == 0;
    store4(m, ORMI_DTYPE_F32, i, n, vec, a);
    store4(v, ORMI_DTYPE_F32, i, n, vec, b);
}

bool is_float(int dt) { return dt == ORMI_DTYPE_F32 || dt == ORMI_DTYPE_BF16 || dt == ORMI_DTYPE_F16; }
int size_of(int dt) { return dt == ORMI_DTYPE_F32 ? 4 : 2; }

}  // namespace
}  // namespace ormi_hip

using namespace ormi_hip;

static int adamw_step(const ormi_adamw_desc* d, const float* factor) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_adamw: ") + what); };
    if (!d) return bad("null descriptor");
    if (d->num_tensors < 0 || (d->num_tensors > 0 && !d->tensors)) return bad("bad tensor list");
    if (d->state_bits != 32 && d->state_bits != 8) return bad("state_bits must be 32 or 8");
    if (d->step < 1) return bad("step counts from 1");
    if (!(d->beta1 >= 0.0 && d->beta1 < 1.0) || !(d->beta2 >= 0.0 && d->beta2 < 1.0)) return bad("betas must be in [0, 1)");
    if (!(d->eps >= 0.0)) return bad("eps must not be negative");
    const bool small = d->state_bits == 8;
    for (int k = 0; k < d->num_tensors; ++k) {
        const ormi_adamw_tensor& t = d->tensors[k];
        if (t.count < 0 || t.count > (long long)kMostGroups * kPerGroup) return bad("element count out of range");
        if (!is_float(t.p_dtype) || !is_float(t.g_dtype)) return bad("p and g must be float32, bfloat16 or float16");
        if (t.count == 0) continue;
        if (!t.p || !t.g || !t.out || !t.m || !t.v || !t.m_out || !t.v_out) return bad("null tensor");
        if (small && (!t.m_scale || !t.v_scale || !t.m_scale_out || !t.v_scale_out)) return bad("null scales");
    }
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;

    AdamParams a{};
    a.lr = (float)d->lr;
    a.b1 = (float)d->beta1;
    a.ob1 = (float)(1.0 - d->beta1);
    a.b2 = (float)d->beta2;
    a.ob2 = (float)(1.0 - d->beta2);
    a.eps = (float)d->eps;
    a.decay = (float)d->weight_decay;
    a.c1 = (float)(1.0 - std::pow(d->beta1, (double)d->step));
    a.c2 = (float)(1.0 - std::pow(d->beta2, (double)d->step));
    auto reciprocal = [](float c) {  // 0: not one that divide() may use
        int e;
        const float m = std::frexp(c, &e);
        return !(c > 0x1p-60f && c <= 1.0f) || m == 1.0f - 0x1p-24f ? 0.0f : (float)(1.0 / (double)c);
    };
    a.r1 = reciprocal(a.c1);
    a.r2 = reciprocal(a.c2);
    unsigned long long groups = 0;
    auto flush = [&] {
        if (a.n == 0) return;
        if (small) factor ? adamw8_kernel<true><<<(unsigned)groups, 256>>>(a, factor) : adamw8_kernel<false><<<(unsigned)groups, 256>>>(a, factor);
        else factor ? adamw_kernel<true><<<(unsigned)groups, 256>>>(a, factor) : adamw_kernel<false><<<(unsigned)groups, 256>>>(a, factor);
        a.n = 0;
        groups = 0;
    };
    for (int k = 0; k < d->num_tensors; ++k) {
        const ormi_adamw_tensor& t = d->tensors[k];
        if (t.count == 0) continue;
        const unsigned long long need = (unsigned long long)(t.count + kPerGroup - 1) / kPerGroup;
        if (a.n == kMost || groups + need > kMostGroups) flush();
        AdamEntry& e = a.t[a.n++];
        e.p = t.p;
        e.g = t.g;
        e.m = t.m;
        e.v = t.v;
        e.out = t.out;
        e.m_out = t.m_out;
        e.v_out = t.v_out;
        e.m_scale = t.m_scale;
        e.v_scale = t.v_scale;
        e.m_scale_out = t.m_scale_out;
        e.v_scale_out = t.v_scale_out;
        e.count = t.count;
        e.first = (unsigned)groups;
        e.p_dtype = (unsigned char)t.p_dtype;
        e.g_dtype = (unsigned char)t.g_dtype;
        const uintptr_t ps = 4 * size_of(t.p_dtype), gs = 4 * size_of(t.g_dtype);
        e.vec = (uintptr_t)t.p % ps == 0 && (uintptr_t)t.out % ps == 0 && (uintptr_t)t.g % gs == 0 &&
                (small || (((uintptr_t)t.m | (uintptr_t)t.v | (uintptr_t)t.m_out | (uintptr_t)t.v_out) & 15) == 0);
        groups += need;
    }
    flush();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string("ormi_hip_adamw: ") + hipGetErrorString(e));
}

extern "C" {

int ormi_hip_adamw(const ormi_adamw_desc* d) { return adamw_step(d, nullptr); }

int ormi_hip_adamw_scaled(const ormi_adamw_desc* d, const float* factor) {
    if (!factor) return fail(ORMI_HIP_ERR_INVALID, "ormi_hip_adamw_scaled: null factor");
    return adamw_step(d, factor);
}

int ormi_hip_adamw_values(float* m, float* v, const void* m_codes, const float* m_scale, const void* v_codes, const float* v_scale,
                          int64_t count) {
    if (count < 0 || count >= (1ll << 40)) return fail(ORMI_HIP_ERR_INVALID, "ormi_hip_adamw_values: element count out of range");
    if (count == 0) return ORMI_HIP_OK;
    if (!m || !v || !m_codes || !m_scale || !v_codes || !v_scale) return fail(ORMI_HIP_ERR_INVALID, "ormi_hip_adamw_values: null pointer");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    for (int64_t at = 0, most = (int64_t)(kMostGroups / 4 * 4) * 1024; at < count; at += most) {  // whole blocks of codes
        const int64_t n = std::min(most, count - at);
        adamw_values_kernel<<<(unsigned)((n + 1023) / 1024), 256>>>(m + at, v + at, (const unsigned*)m_codes + at / 4, m_scale + at / ORMI_ADAMW_BLOCK,
                                                                    (const unsigned*)v_codes + at / 4, v_scale + at / ORMI_ADAMW_BLOCK, n);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string("ormi_hip_adamw_values: ") + hipGetErrorString(e));
}

}  // extern "C"
