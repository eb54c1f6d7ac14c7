// Kernels of the gated linear recurrence, per channel
//   h_t = a_t h_{t-1} + b_t
// with the gates as values (b = x) or logits (a = sigmoid(g), b = (1 - a) x), and
// its gradient: l_t = dh_t + a_{t+1} l_{t+1} is the whole gradient of h_t, and
//   values: dx = l, dg = l h_{t-1};   logits: dx = l (1 - a), dg = l (h_{t-1} - x) a (1 - a).
// Bound by memory: a handful of flops per element besides the sigmoid.
//
// A span of tokens takes the state before it to A h + B, A the product of its
// gates and B what it makes of nothing, and spans join by (A1 A2, A2 B1 + B2). A
// tile is 32 segments of 4 tokens by 8 threads' channels (128 bytes of a row, a
// cache line). A thread takes its own segment's span, segments join by lane
// exchanges in a wave and through LDS across the four waves, and each thread then
// walks its tokens again from the state before them. One work-group goes through
// the tiles of its channels with the state in registers; where batch and channels
// give too few of them, the length is split: a first launch takes each split's
// span, the second starts from the joined ones.
//
// Where a token forgets (a document's first one, or one of none) the state before
// it must not matter at all, NaN included, so spans carry a flag: a product that
// is zero would let infinities through as NaN.
// All states and products are fp32; results are rounded once.
#pragma once
#include "recurrence.h"
#include "row_access.h"

namespace ormi_hip {
namespace {

constexpr float kPassLogit = 200.0f;  // its sigmoid is 1 and what it takes 0, in every type

// a = sigmoid(g) and 1 - a = e^-g a, each accurate relative to itself. e^-g is
// 2^hi (1 + r), hi = fl(-g log2 e) and r what that leaves. Logits below -87, whose
// sigmoid leaves the normal range, count as -87.
__device__ __forceinline__ void gate_of(float g, float& a, float& take) {
    g = __builtin_elementwise_minimum(__builtin_elementwise_maximum(g, -87.0f), kPassLogit);
    const float hi = g * -1.44269502f;
    float r = __builtin_fmaf(-hi, 0.693147182f, -g);
    r = __builtin_fmaf(-hi, -1.90465432e-09f, r);
    float e = __builtin_amdgcn_exp2f(hi);
    e = __builtin_fmaf(e, r, e);
    a = __builtin_amdgcn_rcpf(1.0f + e);
    take = e * a;
}

// Which of a segment's tokens count, and which forget what came before them (bits).
struct Rules {
    unsigned on, cut;
};
template <bool MASKED>
__device__ __forceinline__ Rules token_rules(const RecParams& p, int b, int end, int t0) {
    Rules r = {0, 0};
#pragma unroll
    for (int i = 0; i < kRecTokens; ++i) {
        const int t = t0 + i;
        if (t >= end) continue;
        bool on = true, cut = false;
        if constexpr (MASKED)
            if (p.docs) {
                const int* d = p.docs + b * p.docs_sb + t;
                on = d[0] >= 0;
                cut = !on || (t > 0 && d[-1] != d[0]);
            }
        r.on |= (unsigned)on << i;
        r.cut |= (unsigned)cut << i;
    }
    return r;
}

// Rows t0 + i of a tensor, as `other` where the token does not count.
template <int DT, int V>
__device__ __forceinline__ void load_rows(Run<DT, V> (&r)[kRecTokens], const typename ElemOf<DT>::type* at, long long stride, unsigned on, int n, float other) {
#pragma unroll
    for (int i = 0; i < kRecTokens; ++i) {
        if (on >> i & 1) r[i].load(at + i * stride, n);
        else r[i].fill(other);
    }
}

// Spans of V channels.
template <int V>
struct Span {
    float a[V], b[V];
    bool cut;
};

// The state that span s makes of h.
template <bool MASKED>
__device__ __forceinline__ float after(float a, float b, bool cut, float h) {
    const float r = __builtin_fmaf(a, h, b);
    return MASKED && cut ? b : r;
}

// s joined with the spans of the lanes before it (those `up` lanes lower) or, with
// DOWN, after it: inclusive over the eight segments of a wave, then exclusive.
template <int V, bool MASKED, bool DOWN>
__device__ __forceinline__ void scan_wave(Span<V>& s, Span<V>& whole) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int step = kRecLanes; step < 64; step *= 2) {
        const bool has = DOWN ? lane + step < 64 : lane >= step;
        const int from = DOWN ? lane + step : lane - step;
        const bool ocut = MASKED ? __shfl((int)s.cut, from & 63, 64) != 0 : false;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float oa = __shfl(s.a[e], from & 63, 64), ob = __shfl(s.b[e], from & 63, 64);
            if (has) {
                s.b[e] = after<MASKED>(s.a[e], s.b[e], s.cut, ob);
                s.a[e] *= oa;
            }
        }
        if (MASKED && has) s.cut = s.cut || ocut;
    }
    // The wave's whole span stands in its last (first) segment.
    const int full = (DOWN ? 0 : 56) + (lane & 7), from = DOWN ? lane + kRecLanes : lane - kRecLanes;
    const bool has = DOWN ? lane < 56 : lane >= kRecLanes;
    const bool wcut = MASKED ? __shfl((int)s.cut, full, 64) != 0 : false, ecut = MASKED ? __shfl((int)s.cut, from & 63, 64) != 0 : false;
    whole.cut = wcut;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        whole.a[e] = __shfl(s.a[e], full, 64);
        whole.b[e] = __shfl(s.b[e], full, 64);
        const float oa = __shfl(s.a[e], from & 63, 64), ob = __shfl(s.b[e], from & 63, 64);
        s.a[e] = has ? oa : 1.0f;
        s.b[e] = has ? ob : 0.0f;
    }
    s.cut = MASKED && has && ecut;
}

// A tile's waves' whole spans, twice: the next tile's are written while some wave
// may still read these.
template <int V>
struct WaveSpans {
    float2 s[2][4][kRecLanes][V];
    int cut[2][4];
};
template <int V>
__device__ __forceinline__ void put_wave(WaveSpans<V>& l, int at, const Span<V>& whole) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < kRecLanes) {
#pragma unroll
        for (int e = 0; e < V; ++e) l.s[at][wave][lane][e] = make_float2(whole.a[e], whole.b[e]);
        if (lane == 0) l.cut[at][wave] = whole.cut;
    }
}
// The state before this wave's first segment (after its last with DOWN) in h, and
// the one past the tile in `carry`, which holds the one before it.
template <int V, bool MASKED, bool DOWN>
__device__ __forceinline__ void cross_waves(const WaveSpans<V>& l, int at, float (&carry)[V], float (&h)[V]) {
    const int lane = threadIdx.x & 7, wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int w = DOWN ? 3 - k : k;
        const bool cut = MASKED && l.cut[at][w] != 0;
        if (w == wave) {
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = carry[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 s = l.s[at][w][lane][e];
            carry[e] = after<MASKED>(s.x, s.y, cut, carry[e]);
        }
    }
}

// What a work-group has: its channels, batch and tiles.
struct Place {
    int b, c, n, split, first, tiles, end;
};
template <int V>
__device__ __forceinline__ Place place_of(const RecParams& p) {
    Place w;
    const int blocks = p.channel_blocks, id = blockIdx.x;
    const int cb = id % blocks, rest = id / blocks;
    w.split = rest % p.splits;
    w.b = rest / p.splits;
    w.c = (cb * kRecLanes + (threadIdx.x & 7)) * V;
    w.n = max(0, min(V, p.channels - w.c));
    w.first = w.split * p.split_tiles;
    w.tiles = max(0, min(p.split_tiles, p.tiles - w.first));
    w.end = p.length;
    if (p.lengths) w.end = max(0, min(p.length, p.lengths[w.b]));
    return w;
}
// The carry that a split starts from: `start` and the splits before it (after it).
template <int V, bool MASKED, bool DOWN>
__device__ __forceinline__ void join_splits(const RecParams& p, const Place& w, const float* start, float (&carry)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) carry[e] = start && e < w.n ? start[(long long)w.b * p.channels + w.c + e] : 0.0f;
    const int others = DOWN ? p.splits - 1 - w.split : w.split;
    for (int k = 0; k < others; ++k) {
        const long long row = (long long)w.b * p.splits + (DOWN ? p.splits - 1 - k : k);
        const bool cut = MASKED && p.part_cut[row] != 0;
        const float2* at = p.part + row * p.channels + w.c;
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < w.n) carry[e] = after<MASKED>(at[e].x, at[e].y, cut, carry[e]);
    }
}
template <int V>
__device__ __forceinline__ void put_split(const RecParams& p, const Place& w, const Span<V>& s) {
    if (threadIdx.x >= kRecLanes) return;
    const long long row = (long long)w.b * p.splits + w.split;
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < w.n) p.part[row * p.channels + w.c + e] = make_float2(s.a[e], s.b[e]);
    if (w.c == 0) p.part_cut[row] = s.cut;
}

// Forward; SPANS: only the splits' spans.
template <int GT, int XT, bool LOGIT, bool MASKED, bool SPANS>
__global__ __launch_bounds__(256) void recurrence_kernel(RecParams p) {
    constexpr int V = XT == ORMI_DTYPE_F32 ? 4 : 8, S = kRecTokens;
    using TG = typename ElemOf<GT>::type;
    using TX = typename ElemOf<XT>::type;
    __shared__ WaveSpans<V> lds;
    const Place w = place_of<V>(p);
    if (SPANS && w.split == p.splits - 1) return;  // nothing starts from it
    const int seg = threadIdx.x >> 3;
    const TG* gates = (const TG*)p.gates + w.b * p.g_sb + w.c;
    const TX* x = (const TX*)p.x + w.b * p.x_sb + w.c;
    TX* out = (TX*)p.out + (long long)w.b * p.length * p.channels + w.c;
    float carry[V];
    Span<V> total;
    total.cut = false;
#pragma unroll
    for (int e = 0; e < V; ++e) total.a[e] = 1.0f, total.b[e] = 0.0f;
    if (!SPANS) join_splits<V, MASKED, false>(p, w, p.initial, carry);
    for (int k = 0; k < w.tiles; ++k) {
        const int tile = w.first + k, t0 = tile * kRecTile + seg * S;
        const Rules rule = token_rules<MASKED>(p, w.b, w.end, t0);
        Run<GT, V> rg[S];
        Run<XT, V> rx[S];
        load_rows<GT, V>(rg, gates + t0 * p.g_sl, p.g_sl, rule.on, w.n, LOGIT ? kPassLogit : 1.0f);
        load_rows<XT, V>(rx, x + t0 * p.x_sl, p.x_sl, rule.on, w.n, 0.0f);
        float a[S][V], b[S][V];
        Span<V> s;
        s.cut = MASKED && rule.cut != 0;
#pragma unroll
        for (int e = 0; e < V; ++e) s.a[e] = 1.0f, s.b[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (rule.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (LOGIT) {
                    float take;
                    gate_of(rg[i].get(e), a[i][e], take);
                    b[i][e] = take * rx[i].get(e);
                } else {
                    a[i][e] = rg[i].get(e);
                    b[i][e] = rx[i].get(e);
                }
                s.b[e] = after<MASKED>(a[i][e], b[i][e], cut, s.b[e]);
                s.a[e] *= a[i][e];
            }
        }
        Span<V> whole;
        scan_wave<V, MASKED, false>(s, whole);
        put_wave<V>(lds, k & 1, whole);
        __syncthreads();
        float h[V];
        if (SPANS) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bool cut = MASKED && lds.cut[k & 1][q] != 0;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float2 o = lds.s[k & 1][q][threadIdx.x & 7][e];
                    total.b[e] = after<MASKED>(o.x, o.y, cut, total.b[e]);
                    total.a[e] *= o.x;
                }
                total.cut = total.cut || cut;
            }
            continue;
        }
        if (p.states && seg == 0) {
            float* at = p.states + ((long long)w.b * p.tiles + tile) * p.channels + w.c;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < w.n) at[e] = carry[e];
        }
        cross_waves<V, MASKED, false>(lds, k & 1, carry, h);
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = after<MASKED>(s.a[e], s.b[e], s.cut, h[e]);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (rule.cut >> i & 1), on = rule.on >> i & 1;
            Run<XT, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = after<MASKED>(a[i][e], b[i][e], cut, h[e]);
                o.set(e, MASKED && !on ? 0.0f : h[e]);
            }
            if (t0 + i < p.length) o.store(out + (long long)(t0 + i) * p.channels, w.n);
        }
    }
    if (SPANS) put_split<V>(p, w, total);
    else if (p.last && w.split == p.splits - 1 && threadIdx.x < kRecLanes) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < w.n) p.last[(long long)w.b * p.channels + w.c + e] = carry[e];
    }
}

// Gradient, tiles from the last to the first. m is the gradient of the state before
// a token but for that state's own output: m_t = a_t (dh_t + m_{t+1}), a recurrence
// of the same gates the other way. The states before a tile's tokens are made again
// from the one that the forward pass kept, in full precision.
template <int GT, int XT, int DT, bool LOGIT, bool MASKED, bool SPANS>
__global__ __launch_bounds__(256) void recurrence_grad_kernel(RecParams p) {
    constexpr int V = XT == ORMI_DTYPE_F32 ? 4 : 8, S = kRecTokens;
    using TG = typename ElemOf<GT>::type;
    using TX = typename ElemOf<XT>::type;
    using TD = typename ElemOf<DT>::type;
    __shared__ WaveSpans<V> back, forth;
    const Place w = place_of<V>(p);
    if (SPANS && w.split == 0) return;
    const int seg = threadIdx.x >> 3;
    const TG* gates = (const TG*)p.gates + w.b * p.g_sb + w.c;
    const TX* x = (const TX*)p.x + w.b * p.x_sb + w.c;
    const TD* dout = (const TD*)p.dout + w.b * p.do_sb + w.c;
    const long long base = (long long)w.b * p.length * p.channels + w.c;
    float carry[V];
    Span<V> total;
    total.cut = false;
#pragma unroll
    for (int e = 0; e < V; ++e) total.a[e] = 1.0f, total.b[e] = 0.0f;
    if (!SPANS) join_splits<V, MASKED, true>(p, w, p.dlast, carry);
    for (int k = w.tiles - 1; k >= 0; --k) {
        const int tile = w.first + k, t0 = tile * kRecTile + seg * S;
        const Rules rule = token_rules<MASKED>(p, w.b, w.end, t0);
        Run<GT, V> rg[S];
        Run<XT, V> rx[S];
        Run<DT, V> rd[S];
        load_rows<GT, V>(rg, gates + t0 * p.g_sl, p.g_sl, rule.on, w.n, LOGIT ? kPassLogit : 1.0f);
        load_rows<DT, V>(rd, dout + t0 * p.do_sl, p.do_sl, p.dout ? rule.on : 0u, w.n, 0.0f);
        if (!SPANS) load_rows<XT, V>(rx, x + t0 * p.x_sl, p.x_sl, rule.on, w.n, 0.0f);
        float a[S][V], take[S][V], before[V];
        if (!SPANS) {
            const float* at = p.states + ((long long)w.b * p.tiles + tile) * p.channels + w.c;
#pragma unroll
            for (int e = 0; e < V; ++e) before[e] = e < w.n ? at[e] : 0.0f;
        }
        Span<V> f, r;
        f.cut = r.cut = MASKED && rule.cut != 0;
#pragma unroll
        for (int e = 0; e < V; ++e) f.a[e] = 1.0f, f.b[e] = r.b[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (rule.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (LOGIT) gate_of(rg[i].get(e), a[i][e], take[i][e]);
                else a[i][e] = rg[i].get(e);
                f.a[e] *= a[i][e];
                if (!SPANS) {
                    const float v = rx[i].get(e);
                    f.b[e] = after<MASKED>(a[i][e], LOGIT ? take[i][e] * v : v, cut, f.b[e]);
                }
            }
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const bool cut = MASKED && (rule.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) r.b[e] = MASKED && cut ? 0.0f : a[i][e] * (rd[i].get(e) + r.b[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) r.a[e] = f.a[e];
        Span<V> whole;
        scan_wave<V, MASKED, true>(r, whole);
        put_wave<V>(back, k & 1, whole);
        if (!SPANS) {
            scan_wave<V, MASKED, false>(f, whole);
            put_wave<V>(forth, k & 1, whole);
        }
        __syncthreads();
        if (SPANS) {
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                const bool cut = MASKED && back.cut[k & 1][q] != 0;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float2 o = back.s[k & 1][q][threadIdx.x & 7][e];
                    total.b[e] = after<MASKED>(o.x, o.y, cut, total.b[e]);
                    total.a[e] *= o.x;
                }
                total.cut = total.cut || cut;
            }
            continue;
        }
        float m[V], h[V], prev[S][V];
        cross_waves<V, MASKED, true>(back, k & 1, carry, m);
        cross_waves<V, MASKED, false>(forth, k & 1, before, h);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            m[e] = after<MASKED>(r.a[e], r.b[e], r.cut, m[e]);
            h[e] = after<MASKED>(f.a[e], f.b[e], f.cut, h[e]);
        }
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (rule.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                prev[i][e] = MASKED && cut ? 0.0f : h[e];
                const float v = rx[i].get(e);
                h[e] = __builtin_fmaf(a[i][e], prev[i][e], LOGIT ? take[i][e] * v : v);
            }
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const bool cut = MASKED && (rule.cut >> i & 1), on = rule.on >> i & 1;
            Run<GT, V> og;
            Run<XT, V> ox;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float l = rd[i].get(e) + m[e];
                float dx = l, dg = l * prev[i][e];
                if (LOGIT) {
                    dx = l * take[i][e];
                    dg = dx * a[i][e] * (prev[i][e] - rx[i].get(e));
                }
                m[e] = MASKED && cut ? 0.0f : a[i][e] * l;
                og.set(e, MASKED && !on ? 0.0f : dg);
                ox.set(e, MASKED && !on ? 0.0f : dx);
            }
            if (t0 + i < p.length) {
                const long long at = base + (long long)(t0 + i) * p.channels;
                if (p.dgates) og.store((TG*)p.dgates + at, w.n);
                if (p.dx) ox.store((TX*)p.dx + at, w.n);
            }
        }
    }
    if (SPANS) put_split<V>(p, w, total);
    else if (p.dinitial && w.split == 0 && threadIdx.x < kRecLanes) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < w.n) p.dinitial[(long long)w.b * p.channels + w.c + e] = carry[e];
    }
}

template <int GT, int XT, int DT, bool LOGIT, bool MASKED>
void launch_masked(const RecParams& p, bool gradient) {
    const unsigned grid = (unsigned)(p.channel_blocks * p.splits * p.batch);
    if (gradient) {
        if (p.splits > 1) recurrence_grad_kernel<GT, XT, DT, LOGIT, MASKED, true><<<grid, 256>>>(p);
        recurrence_grad_kernel<GT, XT, DT, LOGIT, MASKED, false><<<grid, 256>>>(p);
    } else if constexpr (DT == XT) {
        if (p.splits > 1) recurrence_kernel<GT, XT, LOGIT, MASKED, true><<<grid, 256>>>(p);
        recurrence_kernel<GT, XT, LOGIT, MASKED, false><<<grid, 256>>>(p);
    }
}
template <int GT, int XT, int DT>
void launch_types(const RecParams& p, const RecCall& c) {
    const bool masked = p.docs || p.lengths;
    if (c.logits) masked ? launch_masked<GT, XT, DT, true, true>(p, c.gradient) : launch_masked<GT, XT, DT, true, false>(p, c.gradient);
    else masked ? launch_masked<GT, XT, DT, false, true>(p, c.gradient) : launch_masked<GT, XT, DT, false, false>(p, c.gradient);
}
template <int XT>
int launch_recurrence(const RecParams& p, const RecCall& c) {
    constexpr int F = ORMI_DTYPE_F32;
    const bool wide_dout = c.gradient && c.dout_f32;
    if constexpr (XT == F) {
        launch_types<F, F, F>(p, c);
    } else {
        if (c.gates_f32) wide_dout ? launch_types<F, XT, F>(p, c) : launch_types<F, XT, XT>(p, c);
        else wide_dout ? launch_types<XT, XT, F>(p, c) : launch_types<XT, XT, XT>(p, c);
    }
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace ormi_hip
