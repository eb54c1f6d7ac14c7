// Kernels of the gated linear recurrence, per channel
//   h_t = a_t h_{t-1} + b_t
// with the gates as values (b = x) or logits (a = sigmoid(g), b = (1 - a) x), and
// its gradient: l_t = dh_t + a_{t+1} l_{t+1} is the whole gradient of h_t, and
//   values: dx = l, dg = l h_{t-1};   logits: dx = l (1 - a), dg = l (h_{t-1} - x) a (1 - a).
// Bound by memory: a handful of flops per element besides the sigmoid. 8 x 2048 x 4096
// bf16: 90 us forward, 146 backward, 4.5 TB/s (a copy: 5.3).
//
// A span of tokens takes the state before it to A h + B, A the product of its
// gates and B what it makes of nothing, and spans join by (A1 A2, A2 B1 + B2). A
// tile is 16 segments of 8 tokens by 16 threads of 4 channels. A thread takes its
// own segment's span, segments join by lane exchanges in a wave and through LDS
// across the four waves, and each thread then walks its tokens again from the
// state before them.
//
// Where batch and channels give enough work-groups, one goes through all tiles of
// its channels, the state in registers, the next tile's loads in flight. Otherwise
// (CHAINED) a work-group has one tile, and the state before it comes from what the
// tiles before publish (chained_state). Inputs are read once either way.
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
// 2^hi (1 + r), hi = fl(-g log2 e) and r what that leaves, which is at most 2 |g|
// 2^-24: it is left out for 16-bit logits, themselves rounded to |g| 2^-12 or worse.
// Logits below -87, whose sigmoid leaves the normal range, count as -87.
template <bool PRECISE>
__device__ __forceinline__ void gate_of(float g, float& a, float& take) {
    float e;
    if (PRECISE) {
        g = __builtin_elementwise_minimum(__builtin_elementwise_maximum(g, -87.0f), kPassLogit);
        const float hi = g * -1.44269502f;
        float r = __builtin_fmaf(-hi, 0.693147182f, -g);
        r = __builtin_fmaf(-hi, -1.90465432e-09f, r);
        e = __builtin_amdgcn_exp2f(hi);
        e = __builtin_fmaf(e, r, e);
    } else {
        e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -1.44269502f, 125.5f));
    }
    a = __builtin_amdgcn_rcpf(1.0f + e);
    take = e * a;
}

// What a thread has: its channels, batch and tokens that exist.
struct Place {
    int b, c, n, end;
};
__device__ __forceinline__ Place place_of(const RecParams& p, int chain) {
    Place w;
    const int cb = chain % p.channel_blocks;
    w.b = chain / p.channel_blocks;
    w.c = cb * kRecChannels + (int)(threadIdx.x % kRecLanes) * kRecRun;
    w.n = max(0, min(kRecRun, p.channels - w.c));
    w.end = p.length;
    if (p.lengths) w.end = max(0, min(p.length, p.lengths[w.b]));
    return w;
}

// Which of a segment's tokens count, and which forget what came before them (bits).
struct Rules {
    unsigned on, cut;
};
template <bool MASKED>
__device__ __forceinline__ Rules token_rules(const RecParams& p, int b, int end, int t0) {
    constexpr unsigned all = (1u << kRecTokens) - 1;
    const int left = end - t0;
    Rules r = {left >= kRecTokens ? all : left > 0 ? (1u << left) - 1 : 0u, 0};
    if constexpr (MASKED)
        if (p.docs) {  // a thread of the segment looks at a token
            const int* docs = p.docs + b * p.docs_sb;
            const int lane = threadIdx.x % kRecLanes, at = (int)(threadIdx.x & 63) - lane, t = t0 + lane;
            const int d = docs[min(t, p.length - 1)], last = docs[max(0, min(t - 1, p.length - 1))];  // token 0 goes on with itself
            const unsigned none = (unsigned)(__ballot(d < 0) >> at), other = (unsigned)(__ballot(d != last) >> at);
            r.cut = (none | other) & r.on;
            r.on &= ~none;
        }
    return r;
}

// A thread's rows of a tensor: the tile's first token, the same for all threads,
// so that the 64-bit part of an address stays in scalar registers, the thread's
// offset from it (the entry keeps tiles within 2^31 bytes), and the tokens' stride.
struct Rows {
    const char* tile;
    unsigned off;
    long long step;
    __device__ __forceinline__ const char* at(int i) const { return tile + i * step + off; }
};
template <int DT>
__device__ __forceinline__ Rows rows_of(const char* base, long long sb, long long sl, const Place& w, int tile) {
    constexpr int size = sizeof(typename ElemOf<DT>::type);
    Rows r;
    r.tile = base + (w.b * sb + (long long)tile * kRecTile * sl) * size;
    r.off = ((unsigned)(threadIdx.x / kRecLanes * kRecTokens) * (unsigned)sl + (unsigned)w.c) * size;
    r.step = sl * size;
    return r;
}

// A thread's tokens of a tensor, as `other` where the token does not count. whole:
// all of the wave's tokens count and all channels exist, which takes no branch per row.
template <int DT, int V>
__device__ __forceinline__ void load_rows(Run<DT, V> (&r)[kRecTokens], const Rows& at, bool whole, unsigned on, int n, float other) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < kRecTokens; ++i) r[i].load(at.at(i));
        return;
    }
#pragma unroll
    for (int i = 0; i < kRecTokens; ++i) {
        if (on >> i & 1) r[i].load(at.at(i), n);
        else r[i].fill(other);
    }
}
template <int DT, int V>
__device__ __forceinline__ void store_row(const Run<DT, V>& r, const Rows& to, int i, bool whole, bool exists, int n) {
    if (whole) r.store_past((void*)to.at(i));
    else if (exists) r.store((void*)to.at(i), n);
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

// s joined with the spans of the lanes before it (of higher lanes with DOWN):
// inclusive over a wave's segments, then exclusive; `whole` is the wave's.
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
    whole = s;  // in the last (first) segment's lanes
    const int from = DOWN ? lane + kRecLanes : lane - kRecLanes;
    const bool has = DOWN ? lane < 64 - kRecLanes : lane >= kRecLanes;
    const bool ecut = MASKED ? __shfl((int)s.cut, from & 63, 64) != 0 : false;
#pragma unroll
    for (int e = 0; e < V; ++e) {
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
template <int V, bool DOWN>
__device__ __forceinline__ void put_wave(WaveSpans<V>& l, int at, const Span<V>& whole) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = DOWN ? lane : lane - (64 - kRecLanes);
    if (k >= 0 && k < kRecLanes) {
#pragma unroll
        for (int e = 0; e < V; ++e) l.s[at][wave][k][e] = make_float2(whole.a[e], whole.b[e]);
        if (k == 0) l.cut[at][wave] = whole.cut;
    }
}
// The state before this wave's first segment (after its last with DOWN) in h, and
// the one past the tile in `carry`, which holds the one before it.
template <int V, bool MASKED, bool DOWN>
__device__ __forceinline__ void cross_waves(const WaveSpans<V>& l, int at, float (&carry)[V], float (&h)[V]) {
    const int lane = threadIdx.x % kRecLanes, wave = threadIdx.x >> 6;
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

// ------------------------------------------------------------ chained tiles --
// The state before a tile is found from what other tiles publish, per channel: each
// tile its span, and the last tile of every kRecGroup the span of the group and, once
// it knows it, the state past it. A tile applies the spans of the groups from the
// nearest state that is there on, one after the other, then those of its own group's
// tiles before it. A group's state came about in the same way, so which one is there
// in time makes no difference to any bit. Nothing waits for a state: spans depend on
// their own tiles alone, groups' on their tiles'.
// A span is one word (its gates' product above the rest), so that no order between
// words matters. All bits set: not there yet. Published NaN have other bits, and a span
// that forgets has them in the product's place.
constexpr unsigned kNone = 0xffffffffu;
constexpr unsigned long long kNoSpan = ~0ull;
// Looks at a span that is not there yet, seconds' worth: the tiles that a tile waits
// for were begun before it and wait for none after them, so this ends a wait only
// where a work-group was lost; the states are NaN then.
constexpr int kMostLooks = 1 << 21;

__device__ __forceinline__ unsigned published(float v) { return v == v ? __float_as_uint(v) : 0x7fc00000u; }
__device__ __forceinline__ unsigned long long as_word(float a, float b, bool cut) {
    return (unsigned long long)(cut ? kNone : published(a)) << 32 | published(b);
}
__device__ __forceinline__ float apply(unsigned long long span, float h) {
    const unsigned a = (unsigned)(span >> 32);
    const float b = __uint_as_float((unsigned)span);
    return a == kNone ? b : __builtin_fmaf(__uint_as_float(a), h, b);
}
template <class T>
__device__ __forceinline__ T look(const T* at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ void publish(T* at, T v) {
    __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Of one channel: the state before tile `pos` of a chain (counted in the order that
// the tiles go), whose span is (a, b, cut).
__device__ __forceinline__ float chained_state(const RecParams& p, int chain, int pos, int channel, float start, float a, float b, bool cut) {
    constexpr int G = kRecGroup;
    const long long stride = (long long)p.chains * kRecChannels, column = (long long)chain * kRecChannels + channel;
    const int group = pos / G, before = pos % G;
    unsigned long long* const spans = p.chain_spans + (long long)group * G * stride + column;  // of the group's tiles
    const unsigned long long* const groups = p.group_spans + column;
    unsigned* const states = p.group_states + column;
    const unsigned long long own = as_word(a, b, cut);
    publish(spans + before * stride, own);
    // The group's tiles before this one.
    unsigned long long tile[G - 1];
    unsigned got;
    int looks = 0;
    while (true) {
        got = look(states + group * stride);
#pragma unroll
        for (int k = 0; k < G - 1; ++k) tile[k] = k < before ? look(spans + k * stride) : 0;
        bool there = true;
#pragma unroll
        for (int k = 0; k < G - 1; ++k) there = there && tile[k] != kNoSpan;
        if (there) break;
        if (++looks > kMostLooks) return __builtin_nanf("");
        __builtin_amdgcn_s_sleep(1);
    }
    float ga = 1.0f, gb = 0.0f;
    bool gcut = false;
    if (before == G - 1) {
#pragma unroll
        for (int k = 0; k < G; ++k) {
            const unsigned long long s = k < G - 1 ? tile[k < G - 1 ? k : 0] : own;
            gb = apply(s, gb);
            gcut = gcut || (unsigned)(s >> 32) == kNone;
            ga *= __uint_as_float((unsigned)(s >> 32));
        }
        publish(p.group_spans + group * stride + column, as_word(ga, gb, gcut));
    }
    float h = start;
    if (group > 0 && got != kNone) {
        h = __uint_as_float(got);
    } else if (group > 0) {
        int from = 0;  // h is the state before group `from`
        for (int back = 1; back < group && from == 0; back += kRecWindow) {
            unsigned state[kRecWindow];
#pragma unroll
            for (int k = 0; k < kRecWindow; ++k) state[k] = look(states + max(group - back - k, 1) * stride);
#pragma unroll
            for (int k = 0; k < kRecWindow; ++k)
                if (from == 0 && group - back - k > 0 && state[k] != kNone) {
                    from = group - back - k;
                    h = __uint_as_float(state[k]);
                }
        }
        while (from < group) {
            unsigned long long span[kRecWindow];
#pragma unroll
            for (int k = 0; k < kRecWindow; ++k) span[k] = look(groups + min(from + k, group - 1) * stride);
            bool there = true;
#pragma unroll
            for (int k = 0; k < kRecWindow; ++k) {
                there = there && span[k] != kNoSpan;
                if (!there || from == group) continue;
                h = apply(span[k], h);
                ++from;
            }
            if (!there) {
                if (++looks > kMostLooks) return __builtin_nanf("");
                __builtin_amdgcn_s_sleep(1);
            }
        }
    }
    if (before == G - 1) publish(states + (group + 1) * stride, published(gcut ? gb : __builtin_fmaf(ga, h, gb)));
#pragma unroll
    for (int k = 0; k < G - 1; ++k)
        if (k < before) h = apply(tile[k], h);
    return h;
}
// A tile's whole span of one channel, from its waves'.
template <int V, bool MASKED, bool DOWN>
__device__ __forceinline__ void tile_span(const WaveSpans<V>& l, int at, int channel, float& a, float& b, bool& cut) {
    a = 1.0f;
    b = 0.0f;
    cut = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int w = DOWN ? 3 - k : k;
        const float2 s = l.s[at][w][channel / V][channel % V];
        const bool c = MASKED && l.cut[at][w] != 0;
        b = after<MASKED>(s.x, s.y, c, b);
        a *= s.x;
        cut = cut || c;
    }
}

// What a work-group goes through: all tiles of a chain, or one tile that it is given.
// Tiles are given out when their work-groups begin, a chain's in their order, so that
// a tile waits only for tiles that run or are done. Chains are in kRecCounters sets,
// each with a counter of its own: additions to one word of memory take about 12 ns
// each (7504 tiles of one counter: 21 us more). A work-group whose set is through takes
// from the next; there are as many work-groups as tiles.
template <bool CHAINED, bool DOWN>
struct Walk {
    int chain, tile;
    bool on;
    __device__ __forceinline__ void first(const RecParams& p, int* lds) {
        if (!CHAINED) {
            chain = (int)blockIdx.x;
            tile = DOWN ? p.tiles - 1 : 0;
            on = p.tiles > 0;
            return;
        }
        if (threadIdx.x == 0) {
            int pos = -1, of = 0;
            for (int k = 0; k < kRecCounters && pos < 0; ++k) {
                const int set = (int)((blockIdx.x + k) % kRecCounters), n = (p.chains - set + kRecCounters - 1) / kRecCounters;
                if (set >= p.chains) continue;
                const unsigned item = __hip_atomic_fetch_add(p.tickets + set * kRecCounterStride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (item >= (unsigned)n * (unsigned)p.tiles) continue;
                pos = (int)(item / (unsigned)n);
                of = set + (int)(item % (unsigned)n) * kRecCounters;
            }
            lds[0] = pos;
            lds[1] = of;
        }
        __syncthreads();
        const int pos = __builtin_amdgcn_readfirstlane(lds[0]);
        chain = __builtin_amdgcn_readfirstlane(lds[1]);
        tile = DOWN ? p.tiles - 1 - pos : pos;
        on = pos >= 0;
    }
    __device__ __forceinline__ void next(const RecParams& p) {
        tile += DOWN ? -1 : 1;
        on = !CHAINED && (DOWN ? tile >= 0 : tile < p.tiles);
    }
};

__global__ __launch_bounds__(256) void recurrence_clear_kernel(unsigned* at, long long count, unsigned* tickets) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (blockIdx.x == 0 && threadIdx.x < kRecCounters) tickets[threadIdx.x * kRecCounterStride] = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (i + k < count) at[i + k] = kNone;
}

template <int V>
__device__ __forceinline__ void start_from(const float* start, const RecParams& p, const Place& w, float (&carry)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) carry[e] = start && e < w.n ? start[(long long)w.b * p.channels + w.c + e] : 0.0f;
}
template <int V>
__device__ __forceinline__ void put_state(float* to, const Place& w, const float (&h)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < w.n) to[e] = h[e];
}

template <int GT, int XT, bool LOGIT, bool MASKED, bool CHAINED>
__global__ __launch_bounds__(256) void recurrence_kernel(RecParams p) {
    constexpr int V = kRecRun, S = kRecTokens;
    __shared__ WaveSpans<V> lds;
    __shared__ float chain_carry[CHAINED ? kRecChannels : 1];
    __shared__ int given[2];
    const long long out_sb = (long long)p.length * p.channels;
    const int seg = threadIdx.x / kRecLanes;
    Walk<CHAINED, false> walk;
    walk.first(p, given);
    const Place w = place_of(p, walk.chain);
    float carry[V];
    start_from<V>(p.initial, p, w, carry);
    Run<GT, V> rg[S];
    Run<XT, V> rx[S];
    Rules rule;
    bool whole = false;
    auto fetch = [&](int tile) {
        rule = token_rules<MASKED>(p, w.b, w.end, tile * kRecTile + seg * S);
        whole = __all(rule.on == (1u << S) - 1 && w.n == V);
        load_rows<GT, V>(rg, rows_of<GT>(p.gates, p.g_sb, p.g_sl, w, tile), whole, rule.on, w.n, LOGIT ? kPassLogit : 1.0f);
        load_rows<XT, V>(rx, rows_of<XT>(p.x, p.x_sb, p.x_sl, w, tile), whole, rule.on, w.n, 0.0f);
    };
    if (walk.on) fetch(walk.tile);
    for (int k = 0; walk.on; ++k) {
        const int tile = walk.tile, chain = walk.chain, t0 = tile * kRecTile + seg * S;
        const Rules now = rule;
        const bool all = whole;
        float a[S][V], b[S][V];
        Span<V> s;
        s.cut = MASKED && now.cut != 0;
#pragma unroll
        for (int e = 0; e < V; ++e) s.a[e] = 1.0f, s.b[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (now.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (LOGIT) {
                    float take;
                    gate_of<GT == ORMI_DTYPE_F32>(rg[i].get(e), a[i][e], take);
                    b[i][e] = take * rx[i].get(e);
                } else {
                    a[i][e] = rg[i].get(e);
                    b[i][e] = rx[i].get(e);
                }
                s.b[e] = after<MASKED>(a[i][e], b[i][e], cut, s.b[e]);
                s.a[e] *= a[i][e];
            }
        }
        walk.next(p);
        if (!CHAINED && walk.on) fetch(walk.tile);
        Span<V> sum;
        scan_wave<V, MASKED, false>(s, sum);
        put_wave<V, false>(lds, k & 1, sum);
        __syncthreads();
        if (CHAINED) {
            if (threadIdx.x < kRecChannels) {
                const int c = w.c - (int)(threadIdx.x % kRecLanes) * V + (int)threadIdx.x;  // this lane's one channel
                float sa, sb, h = 0.0f;
                bool cut;
                tile_span<V, MASKED, false>(lds, k & 1, threadIdx.x, sa, sb, cut);
                if (c < p.channels)
                    h = chained_state(p, chain, tile, threadIdx.x, p.initial ? p.initial[(long long)w.b * p.channels + c] : 0.0f, sa, sb, cut);
                chain_carry[threadIdx.x] = h;
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e) carry[e] = chain_carry[threadIdx.x % kRecLanes * V + e];
        }
        if (p.states && seg == 0) put_state<V>(p.states + ((long long)w.b * p.tiles + tile) * p.channels + w.c, w, carry);
        const Rows to = rows_of<XT>(p.out, out_sb, p.channels, w, tile);
        float h[V];
        cross_waves<V, MASKED, false>(lds, k & 1, carry, h);
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = after<MASKED>(s.a[e], s.b[e], s.cut, h[e]);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (now.cut >> i & 1), on = now.on >> i & 1;
            Run<XT, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = after<MASKED>(a[i][e], b[i][e], cut, h[e]);
                o.set(e, MASKED && !on ? 0.0f : h[e]);
            }
            store_row<XT, V>(o, to, i, all, t0 + i < p.length, w.n);
        }
    }
    if (p.last && seg == 0 && (!CHAINED || walk.tile == p.tiles)) put_state<V>(p.last + (long long)w.b * p.channels + w.c, w, carry);
}

// Gradient, tiles from the last to the first. m is the gradient of the state before
// a token but for that state's own output: m_t = a_t (dh_t + m_{t+1}), a recurrence
// of the same gates the other way. The states before a tile's tokens are made again
// from the one that the forward pass kept, in full precision.
// AHEAD: the next tile's loads go out before this one is finished, where x and the
// gradient have 16 bits. With 16-bit gates the registers hold both tiles; with float32
// logits 10 to 14 of them spill (8 x 2048 x 4096 bf16, both passes: 324 us, 342 over
// documents; 303 and 300 with loads when a tile is reached).
template <int GT, int XT, int DT, bool LOGIT, bool MASKED, bool CHAINED>
__global__ __launch_bounds__(256, 2) void recurrence_grad_kernel(RecParams p) {
    constexpr int V = kRecRun, S = kRecTokens;
    constexpr bool AHEAD = !CHAINED && sizeof(typename ElemOf<XT>::type) == 2 && sizeof(typename ElemOf<DT>::type) == 2;
    __shared__ WaveSpans<V> back, forth;
    __shared__ float chain_carry[CHAINED ? kRecChannels : 1];
    __shared__ int given[2];
    const long long out_sb = (long long)p.length * p.channels;
    const int seg = threadIdx.x / kRecLanes;
    Walk<CHAINED, true> walk;
    walk.first(p, given);
    const Place w = place_of(p, walk.chain);
    float carry[V];
    start_from<V>(p.dlast, p, w, carry);
    Run<GT, V> rg[S];
    Run<XT, V> rx[S];
    Run<DT, V> rd[S];
    float kept[V];
    Rules rule;
    bool whole = false;
    auto fetch = [&](int tile) {
        rule = token_rules<MASKED>(p, w.b, w.end, tile * kRecTile + seg * S);
        whole = __all(rule.on == (1u << S) - 1 && w.n == V);
        load_rows<GT, V>(rg, rows_of<GT>(p.gates, p.g_sb, p.g_sl, w, tile), whole, rule.on, w.n, LOGIT ? kPassLogit : 1.0f);
        load_rows<XT, V>(rx, rows_of<XT>(p.x, p.x_sb, p.x_sl, w, tile), whole, rule.on, w.n, 0.0f);
        load_rows<DT, V>(rd, rows_of<DT>(p.dout, p.do_sb, p.do_sl, w, tile), whole && p.dout, p.dout ? rule.on : 0u, w.n, 0.0f);
        const float* at = p.states + ((long long)w.b * p.tiles + tile) * p.channels + w.c;
#pragma unroll
        for (int e = 0; e < V; ++e) kept[e] = e < w.n ? at[e] : 0.0f;
    };
    if (AHEAD && walk.on) fetch(walk.tile);
    for (int k = 0; walk.on; ++k) {
        if (!AHEAD) fetch(walk.tile);
        const int tile = walk.tile, chain = walk.chain, t0 = tile * kRecTile + seg * S;
        const Rules now = rule;
        const bool all = whole;
        float a[S][V], take[S][V], before[V];
        Run<XT, V> nx[S];
        Run<DT, V> nd[S];
#pragma unroll
        for (int e = 0; e < V; ++e) before[e] = kept[e];
        Span<V> f, r;
        f.cut = r.cut = MASKED && now.cut != 0;
#pragma unroll
        for (int e = 0; e < V; ++e) f.a[e] = 1.0f, f.b[e] = r.b[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (now.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (LOGIT) gate_of<GT == ORMI_DTYPE_F32>(rg[i].get(e), a[i][e], take[i][e]);
                else a[i][e] = rg[i].get(e);
                f.a[e] *= a[i][e];
                const float v = rx[i].get(e);
                f.b[e] = after<MASKED>(a[i][e], LOGIT ? take[i][e] * v : v, cut, f.b[e]);
            }
            nx[i] = rx[i];
            nd[i] = rd[i];
            nx[i].stay_packed();
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const bool cut = MASKED && (now.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) r.b[e] = MASKED && cut ? 0.0f : a[i][e] * (nd[i].get(e) + r.b[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) r.a[e] = f.a[e];
#pragma unroll
        for (int i = 0; i < S; ++i) nd[i].stay_packed();
        walk.next(p);
        if (AHEAD && walk.on) fetch(walk.tile);
        Span<V> sum;
        scan_wave<V, MASKED, true>(r, sum);
        put_wave<V, true>(back, k & 1, sum);
        scan_wave<V, MASKED, false>(f, sum);
        put_wave<V, false>(forth, k & 1, sum);
        __syncthreads();
        if (CHAINED) {
            if (threadIdx.x < kRecChannels) {
                const int c = w.c - (int)(threadIdx.x % kRecLanes) * V + (int)threadIdx.x;  // this lane's one channel
                float sa, sb, h = 0.0f;
                bool cut;
                tile_span<V, MASKED, true>(back, k & 1, threadIdx.x, sa, sb, cut);
                if (c < p.channels)
                    h = chained_state(p, chain, p.tiles - 1 - tile, threadIdx.x, p.dlast ? p.dlast[(long long)w.b * p.channels + c] : 0.0f, sa, sb, cut);
                chain_carry[threadIdx.x] = h;
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e) carry[e] = chain_carry[threadIdx.x % kRecLanes * V + e];
        }
        const Rows to_gates = rows_of<GT>(p.dgates, out_sb, p.channels, w, tile), to_x = rows_of<XT>(p.dx, out_sb, p.channels, w, tile);
        float m[V], h[V], q[S][V];  // q: what a token's gate gets of its l
        cross_waves<V, MASKED, true>(back, k & 1, carry, m);
        cross_waves<V, MASKED, false>(forth, k & 1, before, h);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            m[e] = after<MASKED>(r.a[e], r.b[e], r.cut, m[e]);
            h[e] = after<MASKED>(f.a[e], f.b[e], f.cut, h[e]);
        }
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool cut = MASKED && (now.cut >> i & 1);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float prev = MASKED && cut ? 0.0f : h[e], v = nx[i].get(e);
                q[i][e] = LOGIT ? a[i][e] * take[i][e] * (prev - v) : prev;
                // As the forward pass joins them. Of a restart's gate nothing is left where it is a value;
                // a logit's is finite, or its b is NaN too.
                h[e] = after<MASKED && !LOGIT>(a[i][e], LOGIT ? take[i][e] * v : v, cut, prev);
            }
        }
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const bool cut = MASKED && (now.cut >> i & 1), on = now.on >> i & 1;
            Run<GT, V> og;
            Run<XT, V> ox;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float l = nd[i].get(e) + m[e], dg = l * q[i][e], dx = LOGIT ? l * take[i][e] : l;
                m[e] = MASKED && cut ? 0.0f : a[i][e] * l;
                og.set(e, MASKED && !on ? 0.0f : dg);
                ox.set(e, MASKED && !on ? 0.0f : dx);
            }
            if (p.dgates) store_row<GT, V>(og, to_gates, i, all, t0 + i < p.length, w.n);
            if (p.dx) store_row<XT, V>(ox, to_x, i, all, t0 + i < p.length, w.n);
        }
    }
    if (p.dinitial && seg == 0 && (!CHAINED || walk.tile < 0)) put_state<V>(p.dinitial + (long long)w.b * p.channels + w.c, w, carry);
}

template <int GT, int XT, int DT, bool LOGIT, bool MASKED>
void launch_masked(const RecParams& p, bool gradient) {
    const unsigned tiles = (unsigned)p.chains * (unsigned)p.tiles;
    if (p.chained) {
        const long long words = chain_words(p);
        recurrence_clear_kernel<<<(unsigned)((words + 1023) / 1024), 256>>>((unsigned*)p.chain_spans, words, p.tickets);
    }
    const unsigned groups = p.chained ? tiles : (unsigned)p.chains;
    if (gradient) {
        if (p.chained) recurrence_grad_kernel<GT, XT, DT, LOGIT, MASKED, true><<<groups, 256>>>(p);
        else recurrence_grad_kernel<GT, XT, DT, LOGIT, MASKED, false><<<groups, 256>>>(p);
    } else if constexpr (DT == XT) {
        if (p.chained) recurrence_kernel<GT, XT, LOGIT, MASKED, true><<<groups, 256>>>(p);
        else recurrence_kernel<GT, XT, LOGIT, MASKED, false><<<groups, 256>>>(p);
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
