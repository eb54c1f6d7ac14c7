// Kernels of the short causal convolution per channel
//   z_t = bias + sum_j w_j x_{t - W + 1 + j},  y = z or z sigmoid(z)
// and its gradient, with dz = dy, or dy (s + z s (1 - s)), s = sigmoid(z):
//   dx_t = sum_j w_j dz_{t + W - 1 - j},  dw_j = sum_t dz_t x_{t - W + 1 + j},  db = sum_t dz_t.
// Bound by memory: 2 W flops an element forward, 4 W more backward. A thread has the
// channels of a 16-byte access and a run of tokens; the rows before (and, backward,
// after) its run come out of the caches, where its neighbours' reads left them. A
// work-group is 32 such runs by 128 bytes of a row.
// dw and db are summed by a thread over its tokens, then over a work-group, which
// goes through several tiles; each leaves one partial row, and a second launch adds
// those up in their order.
#pragma once
#include "conv.h"
#include "row_access.h"

namespace ormi_hip {
namespace {

// The inputs of one batch: x, and `initial` before it.
template <int DT>
struct Inputs {
    using T = typename ElemOf<DT>::type;
    const T *x, *initial;  // at the thread's channels
    long long stride, initial_stride;
};

// The first token of token t's run of one document within width - 1 tokens before
// it (initial inputs have negative numbers): no farther than that matters.
__device__ __forceinline__ int run_start(const int* docs, int t, int width) {
    int from = t;
    const int first = t - (width - 1);
    if (!docs) return first;
    const int own = docs[t];
    while (from > first) {
        if (from > 0 && docs[from - 1] != own) break;
        --from;
    }
    return from;
}

__device__ __forceinline__ float silu(float z) { return z * ormi_sigmoid(z); }
// s + z s (1 - s): for large z the difference loses its own accuracy, not the sum.
__device__ __forceinline__ float silu_grad(float z) {
    const float s = ormi_sigmoid(z);
    return __builtin_fmaf(z * s, 1.0f - s, s);
}

struct ConvPlace {
    int b, c, n, part, end;
};
template <int V>
__device__ __forceinline__ ConvPlace conv_place(const ConvParams& p) {
    ConvPlace w;
    const int cb = blockIdx.x % p.channel_blocks, rest = blockIdx.x / p.channel_blocks;
    w.part = rest % p.parts;
    w.b = rest / p.parts;
    w.c = (cb * kConvLanes + (threadIdx.x & 7)) * V;
    w.n = max(0, min(V, p.channels - w.c));
    w.end = p.length;
    if (p.lengths) w.end = max(0, min(p.length, p.lengths[w.b]));
    return w;
}

// Input t (t < 0: an initial one), 0 where there is none.
template <int DT, int V>
__device__ __forceinline__ void load_input(Run<DT, V>& r, const Inputs<DT>& in, int t, int end, int back, int n) {
    if (t >= 0 && t < end) r.load(in.x + t * in.stride, n);
    else if (t < 0 && t >= -back && in.initial) r.load(in.initial + (t + back) * in.initial_stride, n);
    else r.fill(0.0f);
}

// Kernels exist for widths 3 and 4; MASKED ones of W also take smaller widths, whose
// first W - width taps no token reads.
template <int W, bool MASKED>
__device__ __forceinline__ int width_of(const ConvParams& p) {
    return MASKED ? p.width : W;
}

template <int W, int V, bool MASKED>
__device__ __forceinline__ void load_weights(const ConvParams& p, const ConvPlace& w, float (&weight)[W][V], float (&bias)[V]) {
    const int width = width_of<W, MASKED>(p), pad = W - width;
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int j = 0; j < W; ++j) weight[j][e] = e < w.n && j >= pad ? p.weight[(long long)(w.c + e) * width + j - pad] : 0.0f;
        bias[e] = p.bias && e < w.n ? p.bias[w.c + e] : 0.0f;
    }
}

// What a token of number t is: whether it counts, and the first input that it reads.
struct Reach {
    bool on;
    int from;
};
template <int W, bool MASKED>
__device__ __forceinline__ Reach reach_of(const int* docs, int t, int end, int width) {
    Reach r;
    r.on = t < end;
    r.from = t - (width - 1);
    if (MASKED && r.on && docs) {
        r.on = docs[t] >= 0;
        r.from = run_start(docs, t, width);
    }
    if (MASKED && !r.on) r.from = t + 1;
    return r;
}
template <int DT, int W, int V, int N, bool MASKED>
__device__ __forceinline__ void load_inputs(Run<DT, V> (&rows)[N], const Inputs<DT>& in, const int* docs, int t0, const ConvPlace& w, int width) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // Rows that no token here reads are not read either: those past the end, and
        // those of tokens without a document.
        const int t = t0 + i - (W - 1);
        const bool dead = t0 >= w.end || (MASKED && docs && t >= 0 && t < w.end && docs[t] < 0);
        load_input<DT, V>(rows[i], in, dead ? w.end : t, w.end, width - 1, w.n);
    }
}
// z of token t of a thread whose row `at` is its first input.
template <int W, bool MASKED, int DT, int V, int N>
__device__ __forceinline__ float preact(const float (&weight)[W][V], const float (&bias)[V], const Run<DT, V> (&rows)[N], int at, int t, const Reach& r, int e) {
    float z = bias[e];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const float v = rows[at + j].get(e);
        z = __builtin_fmaf(weight[j][e], MASKED && t - (W - 1) + j < r.from ? 0.0f : v, z);
    }
    return z;
}

template <int DT, int W, int S, bool MASKED>
__global__ __launch_bounds__(256) void conv_kernel(ConvParams p) {
    constexpr int V = conv_run(DT, W);
    using T = typename ElemOf<DT>::type;
    const ConvPlace w = conv_place<V>(p);
    const int width = width_of<W, MASKED>(p);
    if (w.n == 0) return;
    const int t0 = (w.part * kConvRuns + (int)(threadIdx.x >> 3)) * S;
    const int* docs = p.docs ? p.docs + w.b * p.docs_sb : nullptr;
    const Inputs<DT> in{(const T*)p.x + w.b * p.x_sb + w.c, p.initial ? (const T*)p.initial + (long long)w.b * (width - 1) * p.channels + w.c : nullptr,
                        p.x_sl, p.channels};
    float weight[W][V], bias[V];
    load_weights<W, V, MASKED>(p, w, weight, bias);
    Run<DT, V> rows[S + W - 1];
    load_inputs<DT, W, V, S + W - 1, MASKED>(rows, in, docs, t0, w, width);
    T* out = (T*)p.out + (long long)w.b * p.length * p.channels + w.c;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int t = t0 + i;
        if (t >= p.length) break;
        const Reach r = reach_of<W, MASKED>(docs, t, w.end, width);
        Run<DT, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float z = preact<W, MASKED, DT, V, S + W - 1>(weight, bias, rows, i, t, r, e);
            if (p.silu) z = silu(z);
            o.set(e, MASKED && !r.on ? 0.0f : z);
        }
        o.store(out + (long long)t * p.channels, w.n);
    }
}

// The inputs that a next token reads. A thread per channel.
template <int DT>
__global__ __launch_bounds__(256) void conv_last_kernel(ConvParams p) {
    using T = typename ElemOf<DT>::type;
    const int width = p.width;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long long)p.batch * p.channels) return;
    const int b = (int)(id / p.channels), c = (int)(id % p.channels);
    const int end = p.lengths ? max(0, min(p.length, p.lengths[b])) : p.length;
    const int* docs = p.docs ? p.docs + b * p.docs_sb : nullptr;
    const int from = end == 0 ? 1 - width : docs && docs[end - 1] < 0 ? end : run_start(docs, end - 1, width);
    T* last = (T*)p.last + (long long)b * (width - 1) * p.channels + c;
    for (int j = 0; j < width - 1; ++j) {
        const int t = end - (width - 1) + j;
        T v = T(0);
        if (t >= from) {
            if (t >= 0) v = ((const T*)p.x)[b * p.x_sb + t * p.x_sl + c];
            else if (p.initial) v = ((const T*)p.initial)[((long long)b * (width - 1) + t + width - 1) * p.channels + c];
        }
        last[(long long)j * p.channels] = v;
    }
}

template <int DT, int GT, int W, int S, bool MASKED>
__global__ __launch_bounds__(256) void conv_grad_kernel(ConvParams p) {
    constexpr int V = conv_run(DT, W), M = S + W - 1, N = M + W - 1;  // M: tokens that read the thread's inputs
    using T = typename ElemOf<DT>::type;
    using TG = typename ElemOf<GT>::type;
    __shared__ float lds[4][kConvLanes][(W + 1) * V];
    const ConvPlace w = conv_place<V>(p);
    const int width = width_of<W, MASKED>(p);
    const int run = threadIdx.x >> 3;
    const int* docs = p.docs ? p.docs + w.b * p.docs_sb : nullptr;
    const Inputs<DT> in{(const T*)p.x + w.b * p.x_sb + w.c, p.initial ? (const T*)p.initial + (long long)w.b * (width - 1) * p.channels + w.c : nullptr,
                        p.x_sl, p.channels};
    const TG* dout = p.dout ? (const TG*)p.dout + w.b * p.do_sb + w.c : nullptr;
    T* dx = p.dx ? (T*)p.dx + (long long)w.b * p.length * p.channels + w.c : nullptr;
    float weight[W][V], bias[V], dw[W][V], db[V];
    load_weights<W, V, MASKED>(p, w, weight, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][e] = 0.0f;
        db[e] = 0.0f;
    }
    // The inputs that the last state holds have its gradient too.
    const float* dlast = p.dlast ? p.dlast + (long long)w.b * (width - 1) * p.channels + w.c : nullptr;
    const int last_from = w.end == 0 ? 1 - width : docs && docs[w.end - 1] < 0 ? w.end : run_start(docs, w.end - 1, width);
    auto add_last = [&](int t, float (&g)[V]) {
        const int j = t - (w.end - (width - 1));
        if (!dlast || j < 0 || t >= w.end || t < last_from) return;
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < w.n) g[e] += dlast[(long long)j * p.channels + e];
    };
    for (int tile = w.part; tile < p.tiles; tile += p.parts) {
        const int t0 = (tile * kConvRuns + run) * S;
        Run<DT, V> rows[N];
        Run<GT, V> rd[M];
        load_inputs<DT, W, V, N, MASKED>(rows, in, docs, t0, w, width);
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int t = t0 + i;
            const bool on = dout && t < w.end && !(MASKED && docs && docs[t] < 0);
            if (on) rd[i].load(dout + t * p.do_sl, w.n);
            else rd[i].fill(0.0f);
        }
        float d[W][V];  // the gradients of the last W inputs that are still being summed: input t0 + k in d[k % W]
        float dz[V];
        auto dz_of = [&](int i, const Reach& r) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                dz[e] = rd[i].get(e);
                if (p.silu) dz[e] *= silu_grad(preact<W, MASKED, DT, V, N>(weight, bias, rows, i, t0 + i, r, e));
            }
        };
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int t = t0 + i;
            const Reach r = reach_of<W, MASKED>(docs, t, w.end, width);
            dz_of(i, r);
            if (i < S) {
#pragma unroll
                for (int e = 0; e < V; ++e) d[i % W][e] = 0.0f, db[e] += MASKED && !r.on ? 0.0f : dz[e];
            }
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const bool skip = MASKED && t - (W - 1) + j < r.from;
                const int to = i - (W - 1) + j;  // the input among the thread's
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float g = skip ? 0.0f : dz[e];
                    if (to >= 0 && to < S) d[to % W][e] = __builtin_fmaf(weight[j][e], g, d[to % W][e]);
                    if (i < S) dw[j][e] = __builtin_fmaf(g, skip ? 0.0f : rows[i + j].get(e), dw[j][e]);
                }
            }
            const int done = i - (W - 1), td = t - (W - 1);
            if (done >= 0 && dx && td < p.length) {
                Run<DT, V> o;
                add_last(td, d[done % W]);
#pragma unroll
                for (int e = 0; e < V; ++e) o.set(e, d[done % W][e]);
                o.store(dx + (long long)td * p.channels, w.n);
            }
        }
        if (p.dinitial && t0 == 0) {  // the inputs before the first token's
            for (int k = 0; k < width - 1; ++k) {
                float g[V];
#pragma unroll
                for (int e = 0; e < V; ++e) g[e] = 0.0f;
#pragma unroll
                for (int i = 0; i < W - 1; ++i) {  // the tokens that read it: i <= k
                    if (i > k || i >= M) continue;
                    const Reach r = reach_of<W, MASKED>(docs, i, w.end, width);
                    dz_of(i, r);
                    if (!(k - (width - 1) < r.from))
#pragma unroll
                        for (int e = 0; e < V; ++e) g[e] = __builtin_fmaf(e < w.n ? p.weight[(long long)(w.c + e) * width + k - i] : 0.0f, dz[e], g[e]);
                }
                add_last(k - (width - 1), g);
                Run<DT, V> o;
#pragma unroll
                for (int e = 0; e < V; ++e) o.set(e, g[e]);
                o.store((T*)p.dinitial + ((long long)w.b * (width - 1) + k) * p.channels + w.c, w.n);
            }
        }
    }
    if (!p.part_sums) return;
    // Over the eight runs of a wave, then the four waves.
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j <= W; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float v = j < W ? dw[j < W ? j : 0][e] : db[e];
            v += __shfl_xor(v, 8, 64);
            v += __shfl_xor(v, 16, 64);
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

template <int DT, int W, bool MASKED>
void launch_masked(const ConvParams& p, bool gradient, bool wide_dout) {
    const unsigned grid = (unsigned)((long long)p.channel_blocks * p.parts * p.batch);
    if (!gradient) {
        if (p.tiles > 0) conv_kernel<DT, W, kConvTokens, MASKED><<<grid, 256>>>(p);
        if (p.width > 1 && p.last) conv_last_kernel<DT><<<(unsigned)(((long long)p.batch * p.channels + 255) / 256), 256>>>(p);
        return;
    }
    if (grid > 0) {
        if (wide_dout) conv_grad_kernel<DT, ORMI_DTYPE_F32, W, kConvGradTokens, MASKED><<<grid, 256>>>(p);
        else conv_grad_kernel<DT, DT, W, kConvGradTokens, MASKED><<<grid, 256>>>(p);
    }
    if (p.dweight || p.dbias) conv_sums_kernel<<<(unsigned)(((p.width + 1ll) * p.channels + 63) / 64), 256>>>(p);
}
template <int DT>
int launch_conv(const ConvParams& p, bool gradient, bool wide_dout) {
    const bool masked = p.docs || p.lengths;
    if (p.width == 4 && !masked) launch_masked<DT, 4, false>(p, gradient, wide_dout);
    else if (p.width == 3 && !masked) launch_masked<DT, 3, false>(p, gradient, wide_dout);
    else if (p.width <= 4) launch_masked<DT, 4, true>(p, gradient, wide_dout);
    else launch_masked<DT, 8, true>(p, gradient, wide_dout);
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace ormi_hip
