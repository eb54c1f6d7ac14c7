// Kernels of the short causal convolution per channel
//   z_t = bias + sum_j w_j x_{t - W + 1 + j},  y = z or z sigmoid(z)
// and its gradient, with dz = dy, or dy (s + z s (1 - s)), s = sigmoid(z):
//   dx_t = sum_j w_j dz_{t + W - 1 - j},  dw_j = sum_t dz_t x_{t - W + 1 + j},  db = sum_t dz_t.
// Bound by memory: 2 W flops an element forward, 4 W more backward. A thread has four
// channels and goes through a run of tokens, W at a time: the inputs that they read
// and the gradients still being summed stay in registers, the next W rows are on
// their way. A work-group is 8 such runs by 128 channels. (All of a run's rows in
// registers at once took 256 of them, one wave to a SIMD: 229 us for the gradient of
// 8 x 2048 x 4096 bf16; now 105, 3.8 TB/s, and 64 forward, 4.2. 128 bytes of a row to a
// work-group in place of 256: 5% more there, 14% in float32.)
// dw and db are summed by a thread over its tokens, then over a work-group, which
// goes through several tiles; each leaves one partial row, and a second launch adds
// those up in their order.
#pragma once
#include "conv.h"
#include "row_access.h"

namespace ormi_hip {
namespace {

// 1 / (1 + e^-z). For 16-bit results without what rounding -z log2 e leaves, at most
// 2 |z| 2^-24 of e^-z.
template <bool PRECISE>
__device__ __forceinline__ float conv_sigmoid(float z) {
    if (PRECISE) return ormi_sigmoid(z);
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269502f));
}
// s + z s (1 - s): for large z the difference loses its own accuracy, not the sum.
template <bool PRECISE>
__device__ __forceinline__ float silu_grad(float z) {
    const float s = conv_sigmoid<PRECISE>(z);
    return __builtin_fmaf(z * s, 1.0f - s, s);
}

struct ConvPlace {
    int b, c, n, part, end, run;
};
__device__ __forceinline__ ConvPlace conv_place(const ConvParams& p) {
    ConvPlace w;
    const int cb = (int)(blockIdx.x % p.channel_blocks), rest = (int)(blockIdx.x / p.channel_blocks);
    w.part = rest % p.parts;
    w.b = rest / p.parts;
    w.run = threadIdx.x / kConvLanes;
    w.c = (cb * kConvLanes + (int)(threadIdx.x % kConvLanes)) * kConvRun;
    w.n = max(0, min(kConvRun, p.channels - w.c));
    w.end = p.length;
    if (p.lengths) w.end = max(0, min(p.length, p.lengths[w.b]));
    return w;
}

// Kernels without masks are for widths 3 and 4; MASKED ones of W also take smaller widths, whose
// first W - width taps no token reads.
template <int W, bool MASKED>
__device__ __forceinline__ int width_of(const ConvParams& p) {
    return MASKED ? p.width : W;
}
template <int W, bool MASKED>
__device__ __forceinline__ void load_weights(const ConvParams& p, const ConvPlace& w, float (&weight)[W][kConvRun], float (&bias)[kConvRun]) {
    const int width = width_of<W, MASKED>(p), pad = W - width;
#pragma unroll
    for (int e = 0; e < kConvRun; ++e) {
#pragma unroll
        for (int j = 0; j < W; ++j) weight[j][e] = e < w.n && j >= pad ? p.weight[(long long)(w.c + e) * width + j - pad] : 0.0f;
        bias[e] = p.bias && e < w.n ? p.bias[w.c + e] : 0.0f;
    }
}

// The rows of one batch of x or dout. `initial` (or null): the `back` rows before them.
struct Source {
    const char* rows;
    long long step;  // bytes between tokens
    const char* initial;
    long long initial_step;
    int back, end;
};
// A thread's N rows from token `first` on, of which [0, end) and the initial ones are
// there; others are 0. tile0: the work-group's first token, so that the 64-bit part of
// the addresses is the same for all its threads. Inside a sequence no row needs a
// branch; at its ends one that is not there is read where token 0 is.
template <int DT, int N>
__device__ __forceinline__ void load_run(Run<DT, kConvRun> (&rows)[N], const Source& x, int tile0, int ahead, int first, const ConvPlace& w) {
    constexpr int size = sizeof(typename ElemOf<DT>::type), V = kConvRun;
    const unsigned c = (unsigned)w.c * size;
    if (__all(first >= 0 && first + N <= x.end && w.n == V)) {
        const char* tile = x.rows + (long long)(tile0 + ahead) * x.step;
        const unsigned off = (unsigned)(first - ahead - tile0) * (unsigned)x.step + c;
#pragma unroll
        for (int i = 0; i < N; ++i) rows[i].load(tile + i * x.step + off);
        return;
    }
    if (w.n == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) rows[i].fill(0.0f);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = first + i;
        const bool here = t >= 0 && t < x.end, before = t < 0 && t >= -x.back && x.initial;
        rows[i].load((here ? x.rows + t * x.step : before ? x.initial + (t + x.back) * x.initial_step : x.rows) + c, w.n);
        if (!here && !before) rows[i].fill(0.0f);
    }
}

// Of the tokens from t0 - W to t0 + R + W - 1 of a thread's run (bit i: token
// t0 - W + i): which count, and which go on with the document of the one before.
// Initial inputs are the first token's document's. A run's threads look at a token or
// two each.
struct Flow {
    unsigned long long on, on_with;
};
template <int W, bool MASKED>
__device__ __forceinline__ Flow flow_of(const int* docs, int length, int t0, int end) {
    static_assert(run_tokens(W) + 2 * W <= 64, "bits");
    Flow f = {~0ull, ~0ull};
    if (!MASKED) return f;
    const int first = t0 - W, lane = threadIdx.x % kConvLanes, at = (int)(threadIdx.x & 63) - lane;
    f = {0, 0};
#pragma unroll
    for (int k = 0; k < 64; k += kConvLanes) {
        const int t = first + k + lane, here = max(0, min(t, length - 1)), before = max(0, min(t - 1, length - 1));
        const int d = docs ? docs[here] : 0, last = docs ? docs[before] : 0;
        const unsigned long long on = __ballot(t >= 0 && t < end && d >= 0) >> at, with = __ballot(d == last) >> at;
        f.on |= (on & 0xffffffffull) << k;
        f.on_with |= (with & 0xffffffffull) << k;
    }
    return f;
}
// The window of the group from token t0 + g on: the W - 1 tokens before it, then its own.
template <int W, bool MASKED>
struct GroupFlow {
    unsigned on = 0, on_with = 0;
    __device__ __forceinline__ GroupFlow(const Flow& f, int g) {
        if (MASKED) on = (unsigned)(f.on >> (g + 1)), on_with = (unsigned)(f.on_with >> (g + 1));
    }
    __device__ __forceinline__ bool counts(int i) const { return !MASKED || (on >> (i + W - 1) & 1); }
    // Whether token i reads the input q tokens before it.
    __device__ __forceinline__ bool reads(int i, int q, int width) const {
        if (!MASKED) return true;
        const unsigned span = (1u << q) - 1;
        return counts(i) && q < width && (on_with >> (i + W - q) & span) == span;
    }
};

// The fp32 inputs that a group of W tokens reads: W - 1 before it, then its own.
template <int W>
struct Window {
    float x[2 * W - 1][kConvRun];
    template <int DT>
    __device__ __forceinline__ void start(const Run<DT, kConvRun> (&r)[W]) {  // rows -W .. -1: the last W - 1 are taken
#pragma unroll
        for (int i = 1; i < W; ++i)
#pragma unroll
            for (int e = 0; e < kConvRun; ++e) x[W - 1 + i][e] = r[i].get(e);
    }
    template <int DT>
    __device__ __forceinline__ void next(const Run<DT, kConvRun> (&r)[W]) {
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
#pragma unroll
            for (int e = 0; e < kConvRun; ++e) x[i][e] = x[W + i][e];
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int e = 0; e < kConvRun; ++e) x[W - 1 + i][e] = r[i].get(e);
    }
};

// z of token i of the group.
template <int W, bool MASKED>
__device__ __forceinline__ float preact(const float (&weight)[W][kConvRun], const float (&bias)[kConvRun], const Window<W>& in, int i, const GroupFlow<W, MASKED>& f,
                                        int width, int e) {
    float z = bias[e];
#pragma unroll
    for (int j = 0; j < W; ++j) z = __builtin_fmaf(weight[j][e], f.reads(i, W - 1 - j, width) ? in.x[i + j][e] : 0.0f, z);
    return z;
}

// The first token that a token after `end` of the last one's document reads no further
// back than: token numbers from 1 - width (the initial inputs') on.
__device__ __forceinline__ int last_run(const int* docs, int end, int width) {
    const int first = end - (width - 1);
    if (end == 0 || !docs) return first;
    if (docs[end - 1] < 0) return end;
    int from = end - 1;
    while (from > first && !(from > 0 && docs[from - 1] != docs[from])) --from;
    return from;
}
// Row j of the inputs that a next token reads, a thread's channels of it.
template <int DT>
__device__ __forceinline__ void put_last(const ConvParams& p, const ConvPlace& w, const Source& x, const int* docs, int width, int j) {
    constexpr int size = sizeof(typename ElemOf<DT>::type);
    const int t = w.end - (width - 1) + j;
    const bool here = t >= 0, before = !here && x.initial, kept = (here || before) && t >= last_run(docs, w.end, width);
    Run<DT, kConvRun> r;
    if (kept) r.load((here ? x.rows + t * x.step : x.initial + (t + x.back) * x.initial_step) + (long long)w.c * size, w.n);
    else r.fill(0.0f);
    r.store(p.last + (((long long)w.b * (width - 1) + j) * p.channels + w.c) * size, w.n);
}

template <int DT, int W, bool MASKED>
__global__ __launch_bounds__(256) void conv_kernel(ConvParams p) {
    constexpr int V = kConvRun, R = run_tokens(W);
    constexpr bool PRECISE = DT == ORMI_DTYPE_F32;
    constexpr int size = sizeof(typename ElemOf<DT>::type);
    const ConvPlace w = conv_place(p);
    const int width = width_of<W, MASKED>(p);
    const int tile0 = w.part * kConvRuns * R, t0 = tile0 + w.run * R;
    const int* docs = p.docs ? p.docs + w.b * p.docs_sb : nullptr;
    const Source x{p.x + w.b * p.x_sb * size, p.x_sl * size, p.initial ? p.initial + (long long)w.b * (width - 1) * p.channels * size : nullptr,
                   (long long)p.channels * size, width - 1, w.end};
    if (p.length == 0) {  // no row is there
        if (p.last && w.run < width - 1 && w.n > 0) put_last<DT>(p, w, x, nullptr, width, w.run);
        return;
    }
    float weight[W][V], bias[V];
    Run<DT, V> before[W], rows[W];
    load_run<DT, W>(before, x, tile0, -W, t0 - W, w);
    load_run<DT, W>(rows, x, tile0, 0, t0, w);
    load_weights<W, MASKED>(p, w, weight, bias);
    Window<W> in;
    in.start(before);
    const Flow flow = flow_of<W, MASKED>(docs, p.length, t0, w.end);
    char* tile = p.out + ((long long)w.b * p.length + tile0) * p.channels * size;
    const unsigned off = ((unsigned)(w.run * R) * (unsigned)p.channels + (unsigned)w.c) * size;
    if (p.last && w.part == p.parts - 1 && w.run < width - 1 && w.n > 0) put_last<DT>(p, w, x, docs, width, w.run);
#pragma unroll 1
    for (int g = 0; g < R; g += W) {
        if (!__any(t0 + g < p.length)) break;
        in.next(rows);
        if (g + W < R) load_run<DT, W>(rows, x, tile0, g + W, t0 + g + W, w);
        const GroupFlow<W, MASKED> f(flow, g);
        const bool whole = __all(t0 + g + W <= p.length && w.n == V);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            Run<DT, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float z = preact<W, MASKED>(weight, bias, in, i, f, width, e);
                if (p.silu) z *= conv_sigmoid<PRECISE>(z);
                o.set(e, f.counts(i) ? z : 0.0f);
            }
            char* to = tile + (long long)(g + i) * p.channels * size;
            if (whole) o.store_past(to + off);
            else if (t0 + g + i < p.length) o.store(to + off, w.n);
        }
    }
}

// The gradient of the initial inputs, a thread per channel: the tokens of the first
// width - 1 that read each, and the last state's where it still holds it.
template <int DT, int GT>
__global__ __launch_bounds__(256) void conv_initial_grad_kernel(ConvParams p) {
    using T = typename ElemOf<DT>::type;
    using TG = typename ElemOf<GT>::type;
    const int width = p.width;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long long)p.batch * p.channels) return;
    const int b = (int)(id / p.channels), c = (int)(id % p.channels);
    const int end = p.lengths ? max(0, min(p.length, p.lengths[b])) : p.length;
    const int* docs = p.docs ? p.docs + b * p.docs_sb : nullptr;
    const T* x = (const T*)p.x + b * p.x_sb + c;
    const T* initial = p.initial ? (const T*)p.initial + (long long)b * (width - 1) * p.channels + c : nullptr;
    const float* weight = p.weight + (long long)c * width;
    // Tokens that go on with what was before the first.
    int tokens = 0;
    while (tokens < min(end, width - 1) && !(docs && (docs[tokens] < 0 || docs[tokens] != docs[0]))) ++tokens;
    const int from = last_run(docs, end, width);
    for (int k = 0; k < width - 1; ++k) {  // input k - (width - 1)
        float g = 0.0f;
        for (int t = 0; t < min(tokens, k + 1); ++t) {
            float dz = p.dout ? elem_to_f32<GT>(((const TG*)p.dout)[b * p.do_sb + t * p.do_sl + c]) : 0.0f;
            if (p.silu) {
                float z = p.bias ? p.bias[c] : 0.0f;
                for (int j = 0; j < width; ++j) {
                    const int at = t - (width - 1) + j;
                    const float v = at >= 0 ? elem_to_f32<DT>(x[at * p.x_sl]) : initial ? elem_to_f32<DT>(initial[(long long)(at + width - 1) * p.channels]) : 0.0f;
                    z = __builtin_fmaf(weight[j], v, z);
                }
                dz *= silu_grad<true>(z);
            }
            g = __builtin_fmaf(weight[k - t], dz, g);
        }
        const int at = k - (width - 1), j = at - (end - (width - 1));
        if (p.dlast && j >= 0 && at >= from) g += p.dlast[((long long)b * (width - 1) + j) * p.channels + c];
        ((T*)p.dinitial)[((long long)b * (width - 1) + k) * p.channels + c] = elem_from_f32<DT>(g);
    }
}

template <int DT, int GT, int W, bool MASKED>
__global__ __launch_bounds__(256) void conv_grad_kernel(ConvParams p) {
    constexpr int V = kConvRun, R = run_tokens(W);
    constexpr bool PRECISE = DT == ORMI_DTYPE_F32;
    constexpr int size = sizeof(typename ElemOf<DT>::type), gsize = sizeof(typename ElemOf<GT>::type);
    __shared__ float lds[4][kConvLanes][(W + 1) * V];
    const ConvPlace w = conv_place(p);
    const int width = width_of<W, MASKED>(p);
    const int* docs = p.docs ? p.docs + w.b * p.docs_sb : nullptr;
    const Source x{p.x + w.b * p.x_sb * size, p.x_sl * size, p.initial ? p.initial + (long long)w.b * (width - 1) * p.channels * size : nullptr,
                   (long long)p.channels * size, width - 1, w.end};
    const Source dout{p.dout + w.b * p.do_sb * gsize, p.do_sl * gsize, nullptr, 0, 0, w.end};
    float weight[W][V], bias[V], dw[W][V], db[V];
    load_weights<W, MASKED>(p, w, weight, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][e] = 0.0f;
        db[e] = 0.0f;
    }
    // The inputs that the last state holds have its gradient too.
    const float* dlast = p.dlast ? p.dlast + (long long)w.b * (width - 1) * p.channels + w.c : nullptr;
    const int last_from = p.dlast ? last_run(docs, w.end, width) : 0;
    for (int tile = w.part; tile < p.tiles; tile += p.parts) {
        const int tile0 = tile * kConvRuns * R, t0 = tile0 + w.run * R;
        Run<DT, V> before[W], rows[W];
        Run<GT, V> rd[W];
        auto fetch = [&](int g) {
            load_run<DT, W>(rows, x, tile0, g, t0 + g, w);
            if (p.dout) load_run<GT, W>(rd, dout, tile0, g, t0 + g, w);
        };
        if (!p.dout) {
#pragma unroll
            for (int i = 0; i < W; ++i) rd[i].fill(0.0f);
        }
        load_run<DT, W>(before, x, tile0, -W, t0 - W, w);
        fetch(0);
        Window<W> in;
        in.start(before);
        const Flow flow = flow_of<W, MASKED>(docs, p.length, t0, w.end);
        float d[W][V];  // of inputs whose gradients are still being summed: that of token t0 + k in d[k % W]
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) d[i][e] = 0.0f;
        char* dx_tile = p.dx + ((long long)w.b * p.length + tile0) * p.channels * size;
        const unsigned off = ((unsigned)(w.run * R) * (unsigned)p.channels + (unsigned)w.c) * size;
        // One group more than the run's: its tokens read the last inputs.
#pragma unroll 1
        for (int g = 0; g <= R; g += W) {
            if (!__any(t0 + g < p.length + W - 1)) break;
            in.next(rows);
            float dy[W][V];
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) dy[i][e] = rd[i].get(e);
            if (g < R) fetch(g + W);
            const GroupFlow<W, MASKED> f(flow, g);
            const bool whole = __all(t0 + g + 1 <= p.length && w.n == V);  // inputs up to t0 + g are written
#pragma unroll
            for (int i = 0; i < W; ++i) {
#pragma unroll
                for (int e = 0; e < V; ++e) d[i][e] = 0.0f;
                // Past the last token stand the inputs before it with a gradient of zero, and zero
                // times infinity is not zero. (101 us without the question; asked of a whole group,
                // with its body twice: 190 registers for 150.)
                if (MASKED || t0 + g + i < p.length) {
                    float dz[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        dz[e] = f.counts(i) ? dy[i][e] : 0.0f;
                        if (p.silu) dz[e] *= silu_grad<PRECISE>(preact<W, MASKED>(weight, bias, in, i, f, width, e));
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const int q = W - 1 - j, slot = (i - q + W) % W;
                        const bool skip = !f.reads(i, q, width);
#pragma unroll
                        for (int e = 0; e < V; ++e) d[slot][e] = __builtin_fmaf(weight[j][e], skip ? 0.0f : dz[e], d[slot][e]);
                    }
                    if (g < R) {
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            const bool skip = !f.reads(i, W - 1 - j, width);
#pragma unroll
                            for (int e = 0; e < V; ++e) dw[j][e] = __builtin_fmaf(skip ? 0.0f : dz[e], skip ? 0.0f : in.x[i + j][e], dw[j][e]);
                        }
#pragma unroll
                        for (int e = 0; e < V; ++e) db[e] += dz[e];
                    }
                }
                const int done = g + i - (W - 1), slot = (i + 1) % W;  // the input that no later token reads
                if (done >= 0 && done < R && p.dx) {
                    const int t = t0 + done, j = t - (w.end - (width - 1));
                    if (dlast && j >= 0 && t < w.end && t >= last_from) {
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (e < w.n) d[slot][e] += dlast[(long long)j * p.channels + e];
                    }
                    Run<DT, V> o;
#pragma unroll
                    for (int e = 0; e < V; ++e) o.set(e, d[slot][e]);
                    char* to = dx_tile + (long long)done * p.channels * size;
                    if (whole) o.store_past(to + off);
                    else if (t < p.length) o.store(to + off, w.n);
                }
            }
        }
    }
    if (!p.part_sums) return;
    // Over the runs of a wave, then the four waves.
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j <= W; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float v = j < W ? dw[j < W ? j : 0][e] : db[e];
#pragma unroll
            for (int step = kConvLanes; step < 32; step *= 2) v += __shfl_xor(v, step, 64);
            v += __shfl_xor(v, 32, 64);
            if (lane < kConvLanes) lds[wave][lane][j * V + e] = v;
        }
    __syncthreads();
    float* sums = p.part_sums + ((long long)w.b * p.parts + w.part) * (width + 1) * p.channels;
    const int pad = W - width;
    for (int k = threadIdx.x; k < kConvLanes * (W + 1) * V; k += 256) {
        const int e = k % V, l = k / V % kConvLanes, j = k / (V * kConvLanes);
        const int c = ((int)(blockIdx.x % p.channel_blocks) * kConvLanes + l) * V + e;
        if (c >= p.channels || j < pad) continue;
        const int at = j * V + e;
        sums[(long long)(j - pad) * p.channels + c] = (lds[0][l][at] + lds[1][l][at]) + (lds[2][l][at] + lds[3][l][at]);
    }
}

// The partial rows added up, 16 at a time side by side; 64 sums to a work-group of
// four waves that share the rows.
__global__ __launch_bounds__(256) void conv_sums_kernel(ConvParams p) {
    __shared__ float lds[4][64];
    const long long width = (p.width + 1ll) * p.channels, at = (long long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int rows = p.batch * p.parts, wave = threadIdx.x >> 6;
    float s = 0.0f;
    if (at < width) {
        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        int r = wave;
        for (; r + 12 < rows; r += 16)
#pragma unroll
            for (int u = 0; u < 4; ++u) a[u] += p.part_sums[(long long)(r + 4 * u) * width + at];
        for (int u = 0; r < rows; r += 4, ++u) a[u & 3] += p.part_sums[(long long)r * width + at];
        s = (a[0] + a[1]) + (a[2] + a[3]);
    }
    lds[wave][threadIdx.x & 63] = s;
    __syncthreads();
    if (wave != 0 || at >= width) return;
    const int l = threadIdx.x;
    s = (lds[0][l] + lds[1][l]) + (lds[2][l] + lds[3][l]);
    const int j = (int)(at / p.channels), c = (int)(at % p.channels);
    if (j == p.width) {
        if (p.dbias) p.dbias[c] = s;
    } else if (p.dweight) {
        p.dweight[(long long)c * p.width + j] = s;
    }
}

template <int DT, int GT, int W, bool MASKED>
void launch_grad(const ConvParams& p) {
    const unsigned grid = (unsigned)((long long)p.channel_blocks * p.parts * p.batch);
    if (grid > 0) conv_grad_kernel<DT, GT, W, MASKED><<<grid, 256>>>(p);
    const long long threads = (long long)p.batch * p.channels;
    if (p.dinitial && p.width > 1 && threads > 0) conv_initial_grad_kernel<DT, GT><<<(unsigned)((threads + 255) / 256), 256>>>(p);
    if (p.dweight || p.dbias) conv_sums_kernel<<<(unsigned)(((p.width + 1ll) * p.channels + 63) / 64), 256>>>(p);
}
template <int DT, int W, bool MASKED>
void launch_masked(const ConvParams& p, bool gradient, bool wide_dout) {
    if (gradient) return wide_dout ? launch_grad<DT, ORMI_DTYPE_F32, W, MASKED>(p) : launch_grad<DT, DT, W, MASKED>(p);
    conv_kernel<DT, W, MASKED><<<(unsigned)((long long)p.channel_blocks * p.parts * p.batch), 256>>>(p);
}
template <int DT>
int launch_conv(const ConvParams& p, bool gradient, bool wide_dout) {
    const bool masked = p.docs || p.lengths || p.width < 3 || p.width > 4;
    switch (conv_width(p.width, masked)) {
        case 3: launch_masked<DT, 3, false>(p, gradient, wide_dout); break;
        case 4: masked ? launch_masked<DT, 4, true>(p, gradient, wide_dout) : launch_masked<DT, 4, false>(p, gradient, wide_dout); break;
        default: launch_masked<DT, 8, true>(p, gradient, wide_dout);
    }
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace ormi_hip
