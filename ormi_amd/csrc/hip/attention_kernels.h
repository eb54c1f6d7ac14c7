// Attention kernels (attention_bf16.hip, attention_f16.hip and attention_f32.hip
// each instantiate them for one element type; attention.hip holds the C entry).
//
// For query row i and key j of one head
//   t_ij = scale q_i.k_j;  t = cap tanh(t / cap);  t -= slope |pos_i - j|
//   p_ij = 2^(t log2 e - lse_i) over the visible keys, o_i = sum_j p_ij v_j
// with a running maximum and sum, so that no score leaves the registers.
//
// Rows. The query heads that share a key/value head are folded into the rows:
// row r is query r / group of head kv * group + r % group, so shared keys and
// values are read once for all of them and their gradients add up in order in
// one work-group's registers, without atomics.
//
// Masks. Row i sees key j when j < lim_i and (with documents) both belong to the
// same one: causal, prefix and length rules all bound j from above, and one
// integer per row, lim = min(length, max(pos + 1, prefix)), holds them.
//
// Tiles. The product of a tile of keys (rows of the first MFMA operand, from
// LDS) and a wave's 32 query rows (second operand, in registers) puts one query
// in each lane's column: a row's maximum and sum are reductions over the lane's
// own registers and one exchange of the wave's halves. The accumulator's
// register order (keys 8 b + 4 half + 0..3) is taken as the order of the second
// product's depth, so p goes from the first product's accumulators into the
// second product's operand without leaving its lane; the values follow that
// order through transposing LDS reads (16-bit) or plain ones (32-bit).
// Keys and values come straight from memory into two LDS stages, one 16-byte
// chunk per lane, their chunks exchanged by row (swz) so that neither the row
// reads nor the transposing reads meet in a bank.
#pragma once
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>

#include "attention.h"
#include "device/ormi_device.h"
#include "gemm_mfma.h"

namespace ormi_hip {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) float lds_float;
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;
typedef __attribute__((address_space(3))) i32x4_t lds_i32x4;

constexpr float kInf = __builtin_huge_valf();

// ---------------------------------------------------------------- helpers --
__device__ __forceinline__ unsigned pack2(TrBF16, float a, float b) {
    const f32x2_t f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, bf16x2_t));
}
__device__ __forceinline__ unsigned pack2(TrF16, float a, float b) {
    const f32x2_t f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, f16x2_t));
}
template <class Tr> struct IsF16 { static constexpr bool value = false; };
template <> struct IsF16<TrF16> { static constexpr bool value = true; };
template <class Tr>
__device__ __forceinline__ float unpack(unsigned low16) {
    return IsF16<Tr>::value ? ormi_f16_to_f32((unsigned short)low16) : ormi_bf16_to_f32((unsigned short)low16);
}
// NaN when any is: a row with a NaN score is NaN whatever its maximum.
__device__ __forceinline__ float max3(float a, float b, float c) { return ormi_maximum(ormi_maximum(a, b), c); }
// Both halves of the wave hold the result for lane % 32.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return ormi_maximum(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = min(v, __shfl_xor(v, d, 64));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = max(v, __shfl_xor(v, d, 64));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ const char* uniform_ptr(const char* p) {
    const unsigned long long t = (unsigned long long)(uintptr_t)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)t);
    const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)(t >> 32));
    return (const char*)(((unsigned long long)hi << 32) | lo);
}
// tanh for scores. 1 - 2 / (1 + e^2y) is off by up to 2.4e-7, whatever y: times a cap
// of at most kWideCap that moves a weight by an eighth of float16's half step. Wider
// caps and 32-bit scores take the form whose error shrinks with y (8192 tokens in 24
// documents, 8 heads of 128, float16, forward and gradient: 417 us instead of 372).
template <class Tr, bool WIDE>
__device__ __forceinline__ float tanh_score(float y) {
    if constexpr (WIDE || Tr::ESIZE == 4) return ormi_tanh(y);
    const float e = __builtin_amdgcn_exp2f(y * 2.88539004f);
    return __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + e), -2.0f, 1.0f);
}

// The wait states between a matrix instruction and a vector instruction that
// reads its result, spelled out: 12 after a 32x32x16 product (its 8 passes and
// four more), 18 after a 32x32x2 one (16 and two), which is what the compiler
// puts there itself in straight-line code. Across the branches that masks bring,
// it (ROCm 7.2) has left too few of them, and rows came out wrong now and then.
// tests/test_mfma_wait_states.py checks the counts and the assembly.
template <class Tr>
__device__ __forceinline__ void settle(f32x16_t& a) {
    if constexpr (Tr::ESIZE == 4) asm("s_nop 15\n\ts_nop 1" : "+v"(a));
    else asm("s_nop 11" : "+v"(a));
}

// 16-bit probabilities are held 2^kShift above their value (of at most 1, or
// 2^8 before a row's maximum is brought up to date), so that those of long rows
// stay in float16's normal range; the sums they go into undo it.
template <class Tr> struct Shift { static constexpr float fwd = 0.0f, bwd = 0.0f; };
template <> struct Shift<TrF16> { static constexpr float fwd = 7.0f, bwd = 12.0f; };

// ------------------------------------------------------------------ tiles --
// A tile of rows of DP features in LDS, 16-byte chunks exchanged by row.
template <class Tr, int DP>
struct Tile {
    static constexpr int ES = Tr::ESIZE, VE = Tr::VE, ROWB = DP * ES, CPR = ROWB / 16;
    static constexpr int NF = DP / (2 * VE);  // operand fragments along the features
    static constexpr int DT = DP / 32;        // accumulator tiles along the features

    // A direct load fills 1 KB, RPS rows; such segments lie SEGB apart, and within
    // a row chunk c stands at c ^ swz(row). Between them sixteen rows in a row meet
    // in no bank (row reads), and neither do four rows' 64-byte pieces (transposing
    // reads), while most steps along a row stay constant offsets of few addresses
    // (an exchange over all 16 chunks took 16 address registers instead of 8, which
    // the gradient kernels do not have).
    // Rows of 96 features (12 or 24 chunks) do not divide a segment and lie without
    // gaps: their stride itself takes rows to different banks.
    static constexpr bool EVEN = 64 % CPR == 0;
    static constexpr int RPS = EVEN ? 64 / CPR : 1, SEGB = 1024 + (EVEN ? CPR == 32 ? 128 : 16 : 0);
    __device__ __forceinline__ static int swz(int row) {
        return CPR == 8    ? (((row >> 1) & 1) << 2) | (((row >> 2) & 1) << 1)
               : CPR == 12 ? (row >> 2) & 3
               : CPR == 16 ? (row & 3) << 2
               : CPR == 24 ? (row >> 1) & 7
               : CPR == 32 ? ((row & 1) << 2) | ((row >> 2) & 3)
                           : 0;
    }
    __device__ __forceinline__ static constexpr int at(int row) { return EVEN ? row / RPS * SEGB + row % RPS * ROWB : row * ROWB; }
    static constexpr int bytes(int rows) { return EVEN ? rows / RPS * SEGB : rows * ROWB; }
    // Rows [row0, row0 + 32), fragment f: lane l holds the chunk 2 f + l / 32 of row l % 32.
    __device__ __forceinline__ static u32x4_t frag(const lds_char* t, int row0, int f) {
        const int lane = threadIdx.x & 63, row = lane & 31;
        // The bits of f that the exchange leaves alone are a constant step.
        constexpr int kept = CPR == 8 ? 0 : CPR == 12 ? ~1 : CPR == 16 ? 1 : CPR == 64 ? ~0 : ~3;
        const int fx = f & ~kept, step = (f & kept) * 32;
        const int lane_at = at(row) + (((2 * fx + (lane >> 5)) ^ swz(row)) << 4);
        return *(const __attribute__((address_space(3))) u32x4_t*)(t + at(row0) + step + lane_at);
    }
    // 16-bit: features [32 dt, 32 dt + 32) as rows, the depth the tile rows
    // row0 + 16 step + {4 half + 0..3, 8 + 4 half + 0..3}, accumulator order.
    __device__ __forceinline__ static u32x4_t turned(const lds_char* t, int row0, int step, int dt) {
        const int lane = threadIdx.x & 63, i = lane & 15;
        const int col = dt * 32 + ((lane >> 4) & 1) * 16 + 4 * (i & 3);
        u32x4_t out;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 8 * h + 4 * (lane >> 5) + (i >> 2);  // row % 16
            const lds_char* p = t + at(row0 + 16 * step + 8 * h) + at(k - 8 * h) + (((col >> 3) ^ swz(k)) << 4) + ((col & 4) << 1);
            const s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)p);
            const uint2 w = __builtin_bit_cast(uint2, v);
            out[2 * h] = w.x;
            out[2 * h + 1] = w.y;
        }
        return out;
    }
    // 32-bit: feature 32 dt + l % 32 of the tile row that accumulator register r of the lane's half stands for.
    __device__ __forceinline__ static float turned1(const lds_char* t, int row0, int r, int dt) {
        const int lane = threadIdx.x & 63, row = 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        const int d = dt * 32 + (lane & 31);
        return *(const lds_float*)(t + at(row0) + at(row) + (((d >> 2) ^ swz(row)) << 4) + (d & 3) * 4);
    }
    // acc[dt] += (the tile's rows row0.. turned) x (accumulator `a` as 16- or 32-bit
    // operand); SUM: sum += its columns' sums, by a product with ones. The matrix
    // instruction takes 16-bit operands, so weights and score gradients are rounded here;
    // a second product with what that leaves (leave_rest) would cost as much again, and is
    // made where it counts: one tile of a row or key, and all of them where memory bounds.
    template <bool SUM = false>
    __device__ __forceinline__ static void second(const lds_char* t, int row0, const f32x16_t& a, f32x16_t (&acc)[DT], f32x16_t* sum = nullptr) {
        if constexpr (ES == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4_t b;
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = pack2(Tr{}, a[8 * s + 2 * e], a[8 * s + 2 * e + 1]);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) Tr::mma(turned(t, row0, s, dt), b, acc[dt]);
                if constexpr (SUM) {
                    constexpr unsigned one = IsF16<Tr>::value ? 0x3C003C00u : 0x3F803F80u;
                    Tr::mma(u32x4_t{one, one, one, one}, b, *sum);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(turned1(t, row0, r, dt), a[r], acc[dt], 0, 0, 0);
        }
    }
    // What second() rounded off its 16-bit operand.
    __device__ __forceinline__ static void leave_rest(f32x16_t& a) {
        if constexpr (ES == 2) {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const unsigned w = pack2(Tr{}, a[e], a[e + 1]);
                a[e] -= unpack<Tr>(w);
                a[e + 1] -= unpack<Tr>(w >> 16);
            }
        }
    }
    // Zeros for the chunks that rows of fewer features do not fill, in `rows` rows of
    // tiles that lie one after the other, by all `threads` of the work-group; before
    // any load into them.
    __device__ __forceinline__ static void clear_padding(lds_char* t, int rows, int chunks, int threads) {
        if (chunks == CPR) return;
        const int pad = CPR - chunks;
        for (int x = threadIdx.x; x < rows * pad; x += threads) {
            const int row = x / pad, c = chunks + x % pad;
            *(__attribute__((address_space(3))) u32x4_t*)(t + at(row) + ((c ^ swz(row)) << 4)) = u32x4_t{0, 0, 0, 0};
        }
        __syncthreads();
    }
    // A row's fragments from memory: lane l holds row `row`'s chunks 2 f + l / 32 (zero past the row's end).
    __device__ __forceinline__ static void row_frags(const char* row, int chunks, u32x4_t (&out)[NF]) {
        const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int c = 2 * f + half;
            out[f] = c < chunks ? *(const u32x4_t*)(row + c * 16) : u32x4_t{0, 0, 0, 0};
        }
    }
};

// Direct loads of a tile's 16-byte chunks into LDS: 1 KB per instruction, whose
// lanes' chunks land one after the other; the exchange of chunks is made on the
// source side. Inline assembly, as in the GEMMs: the compiler would make every
// LDS read of the current stage wait for the next stage's loads. The kernels
// wait themselves before the barrier that publishes a stage.
// Chunks past the row's end are not loaded but cleared once (clear_padding): zero has
// to meet zero there, not an infinity that stands elsewhere in the row. Each load runs
// with the lanes whose chunks exist; a branch for whole rows instead parted the loop's
// instructions (dk and dv of 2 x 1025 tokens, 6 heads of 80, float32: 111 us, so 106).
template <class Tr, int DP, int ROWS, int NW>
struct Loader {
    using T = Tile<Tr, DP>;
    static constexpr int SEGS = ROWS * T::CPR / 64, PER = (SEGS + NW - 1) / NW;
    static_assert(ROWS * T::CPR % 64 == 0 && T::CPR <= 64, "whole segments");

    __device__ __forceinline__ static int seg_lane(int s) {  // this lane's chunk of the tile in segment s
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        return min((wave * PER + s) * 64 + lane, ROWS * T::CPR - 1);
    }
    __device__ __forceinline__ static int seg_row(int s) { return seg_lane(s) / T::CPR; }
    __device__ __forceinline__ static int seg_at(int s, int row) {  // chunk within the row
        return (T::EVEN ? (int)(threadIdx.x & 63) % T::CPR : seg_lane(s) % T::CPR) ^ T::swz(row);
    }
    __device__ __forceinline__ static unsigned seg_chunk(int s, int row, int chunks) {  // bytes within the row
        const int c = seg_at(s, row);
        return c < chunks ? (unsigned)c * 16u : 0u;
    }
    // The lanes whose chunks exist, of each of the segments after which the lanes'
    // chunks come again (pairs of them are alike with 32 chunks a row).
    static constexpr int ALIKE = T::CPR == 32 ? 2 : 1, KINDS = T::CPR == 32 ? 4 : T::CPR == 12 ? 3 : T::CPR == 24 ? 6 : 1;
    struct Live {
        unsigned long long m[KINDS < PER ? KINDS : PER];
        __device__ __forceinline__ explicit Live(int chunks) {
#pragma unroll
            for (int k = 0; k < KINDS && k * ALIKE < PER; ++k) m[k] = __ballot(seg_at(k * ALIKE, seg_row(k * ALIKE)) < chunks);
        }
        __device__ __forceinline__ unsigned long long of(int s) const { return m[s / ALIKE % KINDS]; }
    };
    // All of the wave's segments from base + off[s], up to four per asm block. The
    // assembler's text is not checked for hazards, so the waits are written out:
    // five cycles before a memory instruction reads a scalar register that a
    // vector instruction (a lane read that restores a spilled one, say) may have
    // written, one between a write of m0 and a load to LDS. All lanes of the wave are
    // active here, and are again after it.
    __device__ __forceinline__ static void load(lds_char* dst, const char* base, const unsigned (&off)[PER], const Live& live) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const unsigned d = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(dst + wave * PER * T::SEGB));
        constexpr int N = SEGS % NW != 0 || !T::EVEN ? 1 : PER % 4 == 0 ? 4 : PER % 2 == 0 ? 2 : 1;
#pragma unroll
        for (int s = 0; s < PER; s += N) {
            if (SEGS % NW != 0 && wave * PER + s >= SEGS) break;  // the last wave's share is shorter
            if constexpr (N == 4)
                asm volatile(
                    "s_nop 3\n\ts_mov_b64 exec, %7\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\t"
                    "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %5\n\t"
                    "s_mov_b64 exec, %8\n\ts_add_u32 m0, m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5\n\t"
                    "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %5\n\ts_mov_b64 exec, -1" ::"s"(d + s * T::SEGB),
                    "v"(off[s]), "v"(off[s + 1]), "v"(off[s + 2]), "v"(off[s + 3]), "s"(base), "i"(T::SEGB), "s"(live.of(s)), "s"(live.of(s + 2))
                    : "memory", "m0", "scc");
            else if constexpr (N == 2)
                asm volatile(
                    "s_nop 3\n\ts_mov_b64 exec, %5\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
                    "s_add_u32 m0, m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, -1" ::"s"(d + s * T::SEGB),
                    "v"(off[s]), "v"(off[s + 1]), "s"(base), "i"(T::SEGB), "s"(live.of(s))
                    : "memory", "m0", "scc");
            else
                asm volatile("s_nop 3\n\ts_mov_b64 exec, %3\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1" ::"s"(
                                 d + s * T::SEGB),
                             "v"(off[s]), "s"(base), "s"(live.of(s))
                             : "memory", "m0");
        }
    }
    // Rows base + row * row_bytes, rows past `last` re-reading it.
    __device__ __forceinline__ static void rows(lds_char* dst, const char* base, unsigned row_bytes, int last, int chunks, const Live& live) {
        unsigned off[PER];
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            const int row = seg_row(s);
            off[s] = (unsigned)min(row, last) * row_bytes + seg_chunk(s, row, chunks);
        }
        load(dst, uniform_ptr(base), off, live);
    }
};

// One 4-byte value per lane into 256 bytes of LDS, from an address of its own.
__device__ __forceinline__ void load_words(const void* dst, const void* from) {
    const unsigned d = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_char*)dst);
    asm volatile("s_nop 3\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(d), "v"(from) : "memory", "m0");
}

// Waits for this wave's direct loads and LDS reads, then for the other waves.
__device__ __forceinline__ void publish() {
    wait_vmcnt_lds<0>();
    lds_barrier();
}

// Work item of a work-group: a block of rows (or keys) of one key head, and its
// split. Consecutive work-groups go to different XCDs, each with an L2 of its
// own, so the heads (or, where their number is not a multiple of 8, each head's
// blocks dealt out to `spread` runs) are the fastest index: a run always meets
// the same XCD. Blocks are the slowest and go from long to short under a causal
// mask, over all heads at once: run by run, the last head's longest block
// started when the others were nearly done (float32, 32 heads of 32 blocks: 69%
// of the compute units' time in use).
struct Work {
    int bh, block, split;
    __device__ __forceinline__ Work(const AttnParams& p, int splits) {
        const int runs = p.batch * p.kv_heads * p.spread, id = (int)blockIdx.x;
        const int run = id % runs, q = id / runs;
        split = q % splits;
        block = q / splits * p.spread + run % p.spread;
        bh = run / p.spread;
    }
    static unsigned grid(const AttnParams& p, int blocks, int splits) {
        return (unsigned)(p.batch * p.kv_heads * p.spread * splits * ((blocks + p.spread - 1) / p.spread));
    }
};

// ------------------------------------------------------------------ masks --
// Per batch: keys that exist, position of query 0, prefix.
struct Span {
    int end, off, prefix;
    __device__ __forceinline__ Span(const AttnParams& p, int b) {
        end = p.lengths ? min(max(p.lengths[b], 0), p.keys) : p.keys;
        off = end - p.queries;
        prefix = p.prefix ? min(max(p.prefix[b], 0), end) : 0;
    }
    __device__ __forceinline__ int limit(const AttnParams& p, int pos) const {
        return p.causal ? min(end, max(max(pos + 1, prefix), 0)) : end;
    }
};
__device__ __forceinline__ int doc_at(const AttnParams& p, int b, int pos) {
    return pos >= 0 && pos < p.keys ? p.docs[b * p.docs_sb + pos] : -1;
}
// Documents of a set of tokens as a range; a token without one makes the range
// wider than a single document, so that the set never counts as uniform.
__device__ __forceinline__ int2 widen(int lo, int hi, bool none) {
    if (lo > hi || !none || lo != hi) return make_int2(lo, hi);
    return hi < 0x7fffffff ? make_int2(lo, hi + 1) : make_int2(lo - 1, hi);
}

// Walks the tiles of BN keys that share a document with a work-group's rows: 64
// ranges at a time become two masks, of those that share one with the group and
// of those whose keys and the wave's rows all have one and the same (no mask).
template <int BN>
struct DocTiles {
    static constexpr int RT = kDocTile / BN;  // tiles per range
    const int2* ranges;
    int count, base = -1;
    int2 group, wave;
    unsigned long long meet = 0, one = 0;
    // The next tile from t on, or end.
    __device__ __forceinline__ int next(int t, int end) {
        while (t < end) {
            const int rt = t / RT;
            if (base < 0 || rt >= base + 64) {
                base = rt;
                const int at = rt + (int)(threadIdx.x & 63);
                const int2 r = at < count ? ranges[at] : make_int2(0x7fffffff, -1);
                meet = __ballot(r.x <= group.y && group.x <= r.y);
                one = __ballot(r.x == r.y && wave.x == wave.y && r.x == wave.x);
            }
            const unsigned long long left = meet >> (rt - base);
            if (left & 1) return t;
            t = left ? (rt + __builtin_ctzll(left)) * RT : (base + 64) * RT;
        }
        return end;
    }
    // Whether tile t, the last that next gave, needs no document mask.
    __device__ __forceinline__ bool same(int t) const { return one >> (t / RT - base) & 1; }
};

// A score in powers of two, plus base; its derivative with respect to scale q.k
// in slope (kCap, kCapWide).
template <class Tr, int FORM>
__device__ __forceinline__ float score2(const AttnParams& p, float s, float slope2, float away, float base, float& slope) {
    if constexpr (FORM != kPlain) base = __builtin_fmaf(-slope2, __builtin_fabsf(away), base);
    if constexpr (FORM >= kCap) {
        const float u = tanh_score<Tr, FORM == kCapWide>(s * p.scale_over_cap);
        slope = __builtin_fmaf(-u, u, 1.0f);
        return __builtin_fmaf(u, p.cap2, base);
    }
    return __builtin_fmaf(s, p.scale2, base);
}

// 2^x for the gradients' weights. The hardware's is zero below 2^-126; a key far down
// a slope has no other weights, and its float32 gradient, in the normal range once they
// are times dout and q, would miss them (a tenth of a dk of 1.2e-36). The square of a
// root reaches 2^-149 (2 x 1025 tokens, 6 heads of 80: dq 76.7 us instead of 76.2, the
// library's own 2^x 82). 16-bit weights below 2^-126 count as zero.
template <class Tr>
__device__ __forceinline__ float weight2(float x) {
    if constexpr (Tr::ESIZE == 2) return __builtin_amdgcn_exp2f(x);
    const float root = __builtin_amdgcn_exp2f(0.5f * x);
    return root * root;
}

// ---------------------------------------------------------------- outputs --
// Accumulators acc[dt][r], feature 32 dt + 8 (r / 4) + 4 half + r % 4 of the
// lane's row, times f, rounded once to the output's type; what that left goes to
// `rest` (or null), rounded in turn.
template <class Tr, int DT>
__device__ __forceinline__ void store_row(char* row, int dim, const f32x16_t (&acc)[DT], float f, char* rest = nullptr) {
    const int half = (threadIdx.x & 63) >> 5;
    const bool vec = dim % 4 == 0;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = dt * 32 + 8 * q + 4 * half;
            if (d >= dim) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[dt][4 * q + e] * f;
            if constexpr (Tr::ESIZE == 4) {
                float* o = (float*)row + d;
                if (vec) *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < dim) o[e] = v[e];
            } else {
                uint2 w = make_uint2(pack2(Tr{}, v[0], v[1]), pack2(Tr{}, v[2], v[3]));
                auto put = [&](char* to) {
                    unsigned short* o = (unsigned short*)to + d;
                    if (vec) *(uint2*)o = w;
                    else {
                        o[0] = (unsigned short)w.x;
                        if (d + 1 < dim) o[1] = (unsigned short)(w.x >> 16);
                        if (d + 2 < dim) o[2] = (unsigned short)w.y;
                        if (d + 3 < dim) o[3] = (unsigned short)(w.y >> 16);
                    }
                };
                put(row);
                if (rest) {
                    w = make_uint2(pack2(Tr{}, v[0] - unpack<Tr>(w.x), v[1] - unpack<Tr>(w.x >> 16)),
                                   pack2(Tr{}, v[2] - unpack<Tr>(w.y), v[3] - unpack<Tr>(w.y >> 16)));
                    put(rest);
                }
            }
        }
}
// The same as fp32 partial values, DT * 32 a row.
template <int DT>
__device__ __forceinline__ void store_part(float* row, const f32x16_t (&acc)[DT]) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *(float4*)(row + dt * 32 + 8 * q + 4 * half) =
                make_float4(acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]);
}

// ----------------------------------------------------------------- repair --
// A masked position has the weight zero, and zero times an infinity or a NaN that
// stands there is a NaN in the matrix products. Rows (and keys) that end up not
// finite though their own sums are finite are therefore added up again, in plain
// order and over what they see alone; nothing else pays for it but one look at
// the accumulators. One row at a time, the wave's lanes along the features, about
// 1 us for each key: an infinite value in the tile that all rows of 2 x 4096 causal
// tokens, 16 heads of 128, begin with takes 128 ms instead of 0.2, one in a row of
// dout 116 ms instead of 0.7.
template <class Tr>
__device__ __forceinline__ float load1(const char* row, int d) {
    if constexpr (Tr::ESIZE == 4) return ((const float*)row)[d];
    else return unpack<Tr>(((const unsigned short*)row)[d]);
}

template <class Tr>
__device__ __forceinline__ float row_dot(const char* a, const char* b, int dim) {
    float v = 0.0f;
    for (int d = threadIdx.x & 63; d < dim; d += 64) v = __builtin_fmaf(load1<Tr>(a, d), load1<Tr>(b, d), v);
    return ormi_wave_sum(v);
}
// sum += w times a row's features lane, lane + 64, ...
template <class Tr>
__device__ __forceinline__ void add_row(const char* row, int dim, float w, float (&sum)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = e * 64 + (int)(threadIdx.x & 63);
        if (d < dim) sum[e] = __builtin_fmaf(w, load1<Tr>(row, d), sum[e]);
    }
}
template <class Tr>
__device__ __forceinline__ void put_row(char* row, int dim, const float (&sum)[4], float f, char* rest) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = e * 64 + (int)(threadIdx.x & 63);
        if (d >= dim) continue;
        const float v = sum[e] * f;
        if constexpr (Tr::ESIZE == 4) ((float*)row)[d] = v;
        else {
            const unsigned w = pack2(Tr{}, v, v);
            ((unsigned short*)row)[d] = (unsigned short)w;
            if (rest) {
                const float left = v - unpack<Tr>(w);
                ((unsigned short*)rest)[d] = (unsigned short)pack2(Tr{}, left, left);
            }
        }
    }
}
// Whether any of the lane's row's accumulators, in either half, is not finite.
template <int DT>
__device__ __forceinline__ bool not_finite(const f32x16_t (&acc)[DT]) {
    float z = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) z = __builtin_fmaf(acc[dt][e], 0.0f, z);
    return !(halves_sum(z) == 0.0f);
}
template <int DT>
__device__ __forceinline__ void clear_if(bool yes, f32x16_t (&acc)[DT]) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = yes ? 0.0f : acc[dt][e];
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }

// The launch's arguments read once more, and what follows from them: a repair takes
// nothing but its row or key from the loop before it, which would have to keep it in
// registers (it did: dk and dv of 4096 x 16 heads of 128 took 407 us instead of 370).
__device__ __forceinline__ const AttnParams& arguments_again() {
    auto at = (const __attribute__((address_space(4))) AttnParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const AttnParams*)at;
}
struct Repair {
    const AttnParams& p;
    const Work work;
    const int b, kvh;
    const Span span;
    __device__ __forceinline__ Repair(const AttnParams& p, int splits)
        : p(p), work(p, splits), b(work.bh / p.kv_heads), kvh(work.bh % p.kv_heads), span(p, b) {}
    __device__ __forceinline__ long long row_at(int rr) const { return (long long)work.bh * p.rows + rr; }
    __device__ __forceinline__ long long part_at(int rr) const {
        return ((long long)work.split * p.batch * p.kv_heads + work.bh) * p.rows + rr;
    }
};
// A row of a repair, and where its values begin.
template <class Tr, int FORM>
struct RepairRow {
    int i, head, pos;
    float slope2;
    __device__ __forceinline__ RepairRow(const Repair& w, int rr) {
        i = rr / w.p.group, head = w.kvh * w.p.group + rr - i * w.p.group, pos = i + w.span.off;
        slope2 = FORM != kPlain && w.p.slopes ? w.p.slopes[head] * 1.44269504f : 0.0f;
    }
    __device__ __forceinline__ bool sees(const Repair& w, int j) const {
        if (j >= w.span.limit(w.p, pos)) return false;
        const int doc = w.p.docs ? doc_at(w.p, w.b, pos) : 0;
        return doc >= 0 && (!w.p.docs || doc_at(w.p, w.b, j) == doc);
    }
    __device__ __forceinline__ const char* q(const Repair& w) const {
        return w.p.q + (w.b * w.p.q_sb + (long long)i * w.p.q_sl + head * w.p.q_sh) * Tr::ESIZE;
    }
    __device__ __forceinline__ const char* dout(const Repair& w) const {
        return w.p.dout + (w.b * w.p.do_sb + (long long)i * w.p.do_sl + head * w.p.do_sh) * Tr::ESIZE;
    }
    // Where the row begins in out, in its rest and in dq.
    __device__ __forceinline__ long long at(const Repair& w) const {
        return (((long long)w.b * w.p.queries + i) * w.p.heads + head) * w.p.dim * Tr::ESIZE;
    }
    __device__ __forceinline__ float weight(const Repair& w, const char* k, int j, float base, float& slope) const {
        return weight2<Tr>(score2<Tr, FORM>(w.p, row_dot<Tr>(q(w), k, w.p.dim), slope2, (float)(pos - j), base, slope));
    }
};
template <class Tr>
__device__ __forceinline__ const char* key_row(const Repair& w, int j) {
    return w.p.k + (w.b * w.p.k_sb + (long long)j * w.p.k_sl + w.kvh * w.p.k_sh) * Tr::ESIZE;
}
template <class Tr>
__device__ __forceinline__ const char* value_row(const Repair& w, int j) {
    return w.p.v + (w.b * w.p.v_sb + (long long)j * w.p.v_sl + w.kvh * w.p.v_sh) * Tr::ESIZE;
}
// Whether a row holds a value that is not finite.
template <class Tr>
__device__ __forceinline__ bool row_bad(const char* row, int dim) {
    bool bad = false;
    for (int d = threadIdx.x & 63; d < dim; d += 64) bad = bad | !(__builtin_fabsf(load1<Tr>(row, d)) < kInf);
    return __any(bad);
}
// Whether one of the keys in [j0, j1) that a row of the wave (rows from r0 on) does not
// see is such; with documents any of them. In the keys [w0, w1) also one that is seen:
// what rounding left of a weight has either sign, and an infinity times that is not the
// infinity it has to be. Without any the sums are right as they are: an infinity that
// all rows see elsewhere costs this look, not a repair.
template <class Tr, class F>
__device__ __forceinline__ bool repair_needed(const Repair& w, int r0, int j0, int j1, int w0, int w1, F&& row_of) {
    const int lim = min(w.p.docs ? 0 : w.span.limit(w.p, r0 / w.p.group + w.span.off), max(w.span.end - 1, 0));
    for (int j = j0; j < min(j1, w.span.end); ++j)  // keys past the end read the last one
        if ((j >= lim || (Tr::ESIZE == 2 && j >= w0 && j < w1)) && row_bad<Tr>(row_of(j), w.p.dim)) return true;
    return false;
}
// Nothing brings a sum back from NaN.
__device__ __forceinline__ bool all_nan(const float (&sum)[4], int dim) {
    bool yes = true;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e * 64 + (int)(threadIdx.x & 63) < dim) yes = yes & (sum[e] != sum[e]);
    return __all(yes);
}
// A row of a split's partial sums.
template <int DP>
__device__ __forceinline__ void put_part(float* row, const float (&sum)[4], float f) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (const int d = e * 64 + (int)(threadIdx.x & 63); d < DP) row[d] = sum[e] * f;
}

// ---------------------------------------------------------------- forward --
// NW waves of 32 rows; BN keys per tile. Many rows: four waves share the tiles in LDS,
// bound by the matrix pipes with the exponentials beside them (causal, bf16, 2 x 4096
// tokens x 16 heads of 128 on 4 key heads: 161 us, 854 TF; 12 heads of 64 over 8191
// keys with slopes: 254 us, 814 TF, the exponentials nearly as long as the products).
// Up to 32 rows: one wave, keys split over the chip, bound by reading them (16 single
// tokens over up to 8192 keys x 8 heads of 128: 62 us, 5.4 TB/s of those that exist).
// Up to 96 features three groups of waves share a CU, whatever that spills (with two, as
// the compiler alone would have it, those 12 heads of 64 take 1.4 times as long).
template <class Tr, int DP, int NW, int BN, int FORM>
__global__ __launch_bounds__(64 * NW, DP * Tr::ESIZE > 512 || DP > 128 ? 1 : NW == 4 && DP * Tr::ESIZE <= 192 ? 3 : 2) void attention_fwd_kernel(AttnParams p) {
    using T = Tile<Tr, DP>;
    constexpr int MT = BN / 32, TILEB = T::bytes(BN);
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILEB];
    __shared__ int shared_i[3 * NW];
    __shared__ __attribute__((aligned(16))) int key_doc[2][64];  // of a stage's keys
    lds_char* lds = (lds_char*)smem;

    const Work work(p, p.splits);
    if (work.block >= p.row_blocks) return;
    const int split = work.split, bh = work.bh, rb = p.row_blocks - 1 - work.block;
    const int b = bh / p.kv_heads, kvh = bh % p.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

    // This lane's row.
    const Span span(p, b);
    const int r = (rb * NW + wave) * 32 + (lane & 31);
    const int rc = min(r, p.rows - 1), i = rc / p.group, head = kvh * p.group + rc % p.group;
    const int pos = i + span.off;
    int lim = span.limit(p, pos), doc = 0;
    if (p.docs) {
        doc = doc_at(p, b, pos);
        if (doc < 0) lim = 0;
    }
    const float slope2 = FORM != kPlain && p.slopes ? p.slopes[head] * 1.44269504f : 0.0f;
    u32x4_t qf[T::NF];
    T::row_frags(p.q + (b * p.q_sb + (long long)i * p.q_sl + head * p.q_sh) * T::ES, p.chunks, qf);

    // What the wave and the work-group see.
    const int lim_min = wave_min_i(lim), lim_max = wave_max_i(lim);
    int2 docs_wave = make_int2(0, 0), docs_group = make_int2(0, 0);
    int lim_group = lim_max;
    if (NW > 1 || p.docs) {
        if (p.docs) {
            const int lo = wave_min_i(lim > 0 ? doc : 0x7fffffff), hi = wave_max_i(lim > 0 ? doc : -1);
            docs_wave = widen(lo, hi, __any(lim <= 0));
            docs_group = docs_wave;
        }
        if (NW > 1) {
            if (lane == 0) {
                shared_i[wave] = lim_max;
                shared_i[NW + wave] = docs_wave.x;
                shared_i[2 * NW + wave] = docs_wave.y;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                lim_group = max(lim_group, shared_i[w]);
                docs_group.x = min(docs_group.x, shared_i[NW + w]);
                docs_group.y = max(docs_group.y, shared_i[2 * NW + w]);
            }
            lim_group = __builtin_amdgcn_readfirstlane(lim_group);
        }
    }
    const int tiles = (lim_group + BN - 1) / BN;
    const int per = p.split_tiles ? p.split_tiles : (tiles + p.splits - 1) / p.splits;
    const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);

    DocTiles<BN> walk{p.docs ? p.ranges + (long long)b * p.range_tiles : nullptr, p.range_tiles, -1, docs_group, docs_wave};
    // With slopes the tiles nearest to the rows come first: the maximum then seldom
    // moves, and tiles too far off for any weight cost their scores alone.
    const int near = FORM != kPlain && p.slopes && !p.docs ? min(max((rb * NW * 32 / p.group + span.off) / BN, t0), max(t1 - 1, t0)) : t0;
    auto after = [&](int t) {
        if (p.docs) return walk.next(t + 1, t1);
        if (t >= near) return t + 1 < t1 ? t + 1 : near > t0 ? near - 1 : t1;
        return t > t0 ? t - 1 : t1;
    };
    const char* kb = p.k + (b * p.k_sb + kvh * p.k_sh) * T::ES;
    const char* vb = p.v + (b * p.v_sb + kvh * p.v_sh) * T::ES;
    using L = Loader<Tr, DP, BN, NW>;
    const typename L::Live live(p.chunks);
    auto issue = [&](int t, int stage) {
        const int last = span.end - 1 - t * BN;
        L::rows(lds + stage * 2 * TILEB, kb + (long long)t * BN * p.k_sl * T::ES, (unsigned)(p.k_sl * T::ES), last, p.chunks, live);
        L::rows(lds + stage * 2 * TILEB + TILEB, vb + (long long)t * BN * p.v_sl * T::ES, (unsigned)(p.v_sl * T::ES), last, p.chunks, live);
        if (p.docs && wave == 0) load_words(key_doc[stage], p.docs + b * p.docs_sb + min(t * BN + lane, p.keys - 1));
    };

    f32x16_t acc[T::DT];
#pragma unroll
    for (int dt = 0; dt < T::DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.0f;
    // m: the row's maximum, in powers of two; it may lag by up to 2^8 (the sums then
    // grow by as much). base: what turns a score into the exponent of what is held.
    float m = -kInf, l = 0.0f, base = Shift<Tr>::fwd;
    // At 64 features the exponentials bound the kernel and the matrix pipes have
    // time to add up their sums.
    constexpr bool SUM = T::ES == 2 && DP == 64;
    f32x16_t sum;
    if constexpr (SUM)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[e] = 0.0f;

    T::clear_padding(lds, 4 * BN, p.chunks, 64 * NW);
    int t = p.docs ? walk.next(t0, t1) : near, stage = 0;
    // The weights are rounded to 16 bits for their product with the values. In the tile
    // that a row begins with, what that leaves is multiplied too: it holds all keys of a
    // row that sees few, where single weights count (and the gradient's delta, a sum over
    // the row, would carry their rounding into every score's: dq 1.5 times as far off as
    // rounding the result alone, now 1.05), and with slopes the heaviest. With many keys
    // the roundings average out, and the matrix pipes bound the kernel. Rows by the
    // wave (NW 1) wait for memory: there it is every tile, in the same time.
    const int whole = t;
    bool same = !p.docs || (t < t1 && walk.same(t));
    if (t < t1) issue(t, 0);
    while (t < t1) {
        publish();
        const int tn = after(t);
        const bool same_next = !p.docs || (tn < t1 && walk.same(tn));
        if (tn < t1) issue(tn, stage ^ 1);
        const int j0 = t * BN;
        if (j0 < lim_max) {
            const lds_char* kt = lds + stage * 2 * TILEB;
            const lds_char* vt = kt + TILEB;
            const float away = (float)(pos - j0 - 4 * half);  // of the lane's first key
            f32x16_t s[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[mt][e] = 0.0f;
#pragma unroll
                for (int f = 0; f < T::NF; ++f) Tr::mma(T::frag(kt, mt * 32, f), qf[f], s[mt]);
                settle<Tr>(s[mt]);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float slope;
                    s[mt][e] = score2<Tr, FORM>(p, s[mt][e], slope2, away - (float)(mt * 32 + 8 * (e >> 2) + (e & 3)), base, slope);
                }
            }
            if (j0 + BN > lim_min || !same) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int j = j0 + mt * 32 + 8 * (e >> 2) + 4 * half + (e & 3);
                        s[mt][e] = j < lim ? s[mt][e] : -kInf;
                    }
                if (!same) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const i32x4_t kd = *(const lds_i32x4*)&key_doc[stage][mt * 32 + 8 * q + 4 * half];
                            s[mt][4 * q] = kd.x == doc ? s[mt][4 * q] : -kInf;
                            s[mt][4 * q + 1] = kd.y == doc ? s[mt][4 * q + 1] : -kInf;
                            s[mt][4 * q + 2] = kd.z == doc ? s[mt][4 * q + 2] : -kInf;
                            s[mt][4 * q + 3] = kd.w == doc ? s[mt][4 * q + 3] : -kInf;
                        }
                }
            }
            float top = -kInf;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 16; e += 2) top = max3(top, s[mt][e], s[mt][e + 1]);
            top = halves_max(top);
            if (__any(m == -kInf ? top > -kInf : top > 8.0f + Shift<Tr>::fwd)) {
                const float mn = fmaxf(m, top - base);
                const float a = mn == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                const float to = mn == -kInf ? base : Shift<Tr>::fwd - mn, by = to - base;
                if constexpr (SUM) sum[0] *= a;
                else l *= a;
#pragma unroll
                for (int dt = 0; dt < T::DT; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[dt][e] *= a;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[mt][e] += by;
                top += by;
                m = mn;
                base = to;
            }
            // Under a steep slope exponents below float32's least make every weight of
            // a tile far off zero.
            if (FORM != kBias || __any(!(top < -152.0f))) {
                float part[2] = {0.0f, 0.0f};
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        s[mt][e] = __builtin_amdgcn_exp2f(s[mt][e]);
                        if constexpr (!SUM) part[e & 1] += s[mt][e];
                    }
                if constexpr (!SUM) l += part[0] + part[1];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) T::template second<SUM>(vt, mt * 32, s[mt], acc, &sum);
                if (T::ES == 2 && (NW == 1 || t == whole)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        T::leave_rest(s[mt]);
                        T::template second<SUM>(vt, mt * 32, s[mt], acc, &sum);
                    }
                }
            }
        }
        t = tn;
        same = same_next;
        stage ^= 1;
    }

#pragma unroll
    for (int dt = 0; dt < T::DT; ++dt) settle<Tr>(acc[dt]);
    if constexpr (SUM) {
        settle<Tr>(sum);
        l = sum[0];
    } else {
        l = halves_sum(l);
    }
    clear_if(l == 0.0f, acc);
    const bool bad = not_finite(acc);  // by all lanes: it adds up the wave's halves
    unsigned todo = (unsigned)__ballot(half == 0 && r < p.rows && l < kInf && bad);
    if (__builtin_expect(todo != 0, 0)) {
        const Repair w(arguments_again(), arguments_again().splits);
        if (!repair_needed<Tr>(w, __builtin_amdgcn_readfirstlane(r), t0 * BN, t1 * BN, NW == 1 ? 0 : whole * BN, NW == 1 ? t1 * BN : whole * BN + BN,
                               [&](int j) { return value_row<Tr>(w, j); }))
            todo = 0;
    }
    const bool repaired = todo >> (lane & 31) & 1;
    if (__builtin_expect(todo != 0, 0)) {
        const Repair w(arguments_again(), arguments_again().splits);
        for (; todo; todo &= todo - 1) {
            const int from = __builtin_ctz(todo), rr = __builtin_amdgcn_readlane(r, from);
            const RepairRow<Tr, FORM> row(w, rr);
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, slope = 1.0f;
            for (int j = t0 * BN; j < t1 * BN && !all_nan(o, w.p.dim); ++j)
                if (row.sees(w, j)) add_row<Tr>(value_row<Tr>(w, j), w.p.dim, row.weight(w, key_row<Tr>(w, j), j, lane_of(base, from), slope), o);
            if (w.p.splits > 1) put_part<DP>(w.p.part + w.part_at(rr) * DP, o, 1.0f);
            else put_row<Tr>(w.p.out + row.at(w), w.p.dim, o, 1.0f / lane_of(l, from), w.p.rest ? w.p.rest + row.at(w) : nullptr);
        }
    }
    if (r >= p.rows) return;
    if (p.splits > 1) {
        const long long at = ((long long)split * p.batch * p.kv_heads + bh) * p.rows + r;
        if (!(l == 0.0f) && !repaired) store_part(p.part + at * DP, acc);
        if (half == 0) p.part_ml[at] = make_float2(m == -kInf ? -kInf : m - Shift<Tr>::fwd, l);
        return;
    }
    const long long to = (((long long)b * p.queries + i) * p.heads + head) * p.dim * T::ES;
    if (!repaired)
        store_row<Tr, T::DT>(p.out + to, p.dim, acc, l == 0.0f ? 0.0f : 1.0f / l, p.rest ? p.rest + to : nullptr);
    if (p.lse && half == 0) p.lse[(long long)bh * p.rows + r] = l == 0.0f ? kInf : m - Shift<Tr>::fwd + __builtin_log2f(l);
}

// Joins the splits of a row: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s,
// in split order. One wave per row: lane s holds split s's maximum and sum (at
// most 64 splits), then the lanes go along the features; a split that saw no key
// has stored no values. Bound by the wait for three loads in turn (5.9-7 us for one
// to 512 rows).
template <class Tr, int DP>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnParams p) {
    const long long total = (long long)p.batch * p.kv_heads * p.rows;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= total) return;
    constexpr int NE = (DP + 63) / 64;
    const float2 ml = lane < p.splits ? p.part_ml[lane * total + row] : make_float2(-kInf, 0.0f);
    const bool some = !(ml.y == 0.0f);
    const float top = ormi_lanes_max<64>(some ? ml.x : -kInf);
    const float weight = some ? __builtin_amdgcn_exp2f(ml.x - top) : 0.0f;
    const float l = ormi_lanes_sum<64>(some ? weight * ml.y : 0.0f);
    const unsigned long long live = __ballot(some);
    float o[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        if (!(live >> s & 1)) continue;
        const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), s));
#pragma unroll
        for (int e = 0; e < NE; ++e) o[e] += a * p.part[(s * total + row) * DP + min(e * 64 + lane, DP - 1)];
    }
    const int bh = (int)(row / p.rows), r = (int)(row % p.rows), b = bh / p.kv_heads;
    const int i = r / p.group, head = (bh % p.kv_heads) * p.group + r % p.group;
    const long long at = (((long long)b * p.queries + i) * p.heads + head) * p.dim;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const int d = e * 64 + lane;
        if (d < p.dim) {
            const float v = o[e] * inv;
            if constexpr (Tr::ESIZE == 4) ((float*)p.out)[at + d] = v;
            else {
                const unsigned w = pack2(Tr{}, v, v);
                ((unsigned short*)p.out)[at + d] = (unsigned short)w;
                if (p.rest) {
                    const float left = v - unpack<Tr>(w);
                    ((unsigned short*)p.rest)[at + d] = (unsigned short)pack2(Tr{}, left, left);
                }
            }
        }
    }
    if (p.lse && lane == 0) p.lse[row] = l == 0.0f ? kInf : top + __builtin_log2f(l);
}

template <class Tr, int DP, int FORM>
void launch_attention_fwd_form(const AttnParams& p) {
    const unsigned grid = Work::grid(p, p.row_blocks, p.splits);
    if (p.wide) attention_fwd_kernel<Tr, DP, 4, fwd_tile(DP, Tr::ESIZE, false), FORM><<<grid, 256>>>(p);
    else attention_fwd_kernel<Tr, DP, 1, fwd_tile(DP, Tr::ESIZE, true), FORM><<<grid, 64>>>(p);
}

template <class Tr, int DP>
int launch_attention_fwd_dp(const AttnParams& p) {
    if (p.form == kPlain) launch_attention_fwd_form<Tr, DP, kPlain>(p);
    else if (p.form == kBias) launch_attention_fwd_form<Tr, DP, kBias>(p);
    else if (Tr::ESIZE == 4 || p.form == kCap) launch_attention_fwd_form<Tr, DP, kCap>(p);
    else if constexpr (Tr::ESIZE == 2) launch_attention_fwd_form<Tr, DP, kCapWide>(p);
    if (p.splits > 1) {
        const long long rows = (long long)p.batch * p.kv_heads * p.rows;
        attention_join_kernel<Tr, DP><<<(unsigned)((rows + 3) / 4), 256>>>(p);
    }
    return (int)hipGetLastError();
}

// --------------------------------------------------------------- gradient --
// delta = sum of out * dout of a row; 16 lanes per row. out comes with what its
// rounding left: an error of delta is common to a row's score gradients, and in
// short rows it would be as large as their own rounding. float16 also collects
// the largest squared norms of a dout row and of a value row: |score gradient|
// <= p (|dp| + |delta|) <= 2 |dout| |v|, and held times the power of two that
// takes that bound to 2^15 the score gradients keep to float16's normal range
// whatever the scale of the loss, each batch's key head by its own two norms (a
// sequence or a head of a far larger loss takes nothing from the others). A
// maximum does not depend on its order. What
// stands at masked positions has no part in it: rows that see nothing (their
// score gradients are zero whatever dout holds) and values past the length or
// without a document; nor have rows that are not finite, whose own score
// gradients are not finite at any scale.
template <class Tr>
__device__ __forceinline__ void load_chunk(const char* at, float (&v)[Tr::VE]) {
    const u32x4_t w = *(const u32x4_t*)at;
#pragma unroll
    for (int e = 0; e < Tr::VE; ++e) {
        if constexpr (Tr::ESIZE == 4) v[e] = __uint_as_float(w[e]);
        else v[e] = unpack<Tr>(e & 1 ? w[e >> 1] >> 16 : w[e >> 1]);
    }
}
template <class Tr>
__global__ __launch_bounds__(256) void attention_delta_kernel(AttnParams p, float* delta, unsigned* bounds, unsigned row_groups) {
    const int sub = threadIdx.x & 15;
    const bool rows = blockIdx.x < row_groups;
    const int group = (int)(rows ? blockIdx.x : blockIdx.x - row_groups), groups = (int)(rows ? row_groups : gridDim.x - row_groups);
    // Without bounds the rows in out's order; with them each key head's own, some
    // (or one) of the work-groups' runs of rows for each, heads the fastest.
    const int all_heads = p.batch * p.kv_heads, heads = bounds ? min(all_heads, groups) : 1, slices = groups / heads;
    const long long n = bounds ? (rows ? p.rows : p.keys) : (long long)p.batch * p.queries * p.heads;
    for (int bh = group % heads; bh < (bounds ? all_heads : 1); bh += heads) {
        float most_norm = 0.0f;
        for (long long at = (long long)(group / heads) * 16 + (threadIdx.x >> 4); at - (threadIdx.x >> 4) < n; at += (long long)slices * 16) {
            const bool live = at < n;
            const long long row = live ? at : n - 1;
            float dot = 0.0f, norm = 0.0f;
            if (rows) {
                int b, i, head;
                if (bounds) {
                    b = bh / p.kv_heads;
                    i = (int)row / p.group;
                    head = bh % p.kv_heads * p.group + (int)row % p.group;
                } else {
                    head = (int)(row % p.heads);
                    const long long bi = row / p.heads;
                    b = (int)(bi / p.queries);
                    i = (int)(bi % p.queries);
                }
                const long long from = (((long long)b * p.queries + i) * p.heads + head) * p.dim * Tr::ESIZE;
                const char* o = p.out + from;
                const char* rest = p.rest ? p.rest + from : nullptr;
                const char* g = p.dout + (b * p.do_sb + (long long)i * p.do_sl + head * p.do_sh) * Tr::ESIZE;
                if (p.dim % Tr::VE == 0) {
                    for (int c = sub; c < p.dim / Tr::VE; c += 16) {
                        float x[Tr::VE], y[Tr::VE];
                        load_chunk<Tr>(o + c * 16, x);
                        load_chunk<Tr>(g + c * 16, y);
                        if (rest) {
                            float z[Tr::VE];
                            load_chunk<Tr>(rest + c * 16, z);
#pragma unroll
                            for (int e = 0; e < Tr::VE; ++e) x[e] += z[e];
                        }
#pragma unroll
                        for (int e = 0; e < Tr::VE; ++e) {
                            dot = __builtin_fmaf(x[e], y[e], dot);
                            norm = __builtin_fmaf(y[e], y[e], norm);
                        }
                    }
                } else {
                    for (int d = sub; d < p.dim; d += 16) {
                        const float y = load1<Tr>(g, d);
                        dot = __builtin_fmaf(load1<Tr>(o, d) + (rest ? load1<Tr>(rest, d) : 0.0f), y, dot);
                        norm = __builtin_fmaf(y, y, norm);
                    }
                }
                dot = ormi_lanes_sum<16>(dot);
                const long long to = ((long long)b * p.kv_heads + head / p.group) * p.rows + (long long)i * p.group + head % p.group;
                if (live && sub == 0) delta[to] = dot;
                if (bounds && p.lse[to] == kInf) norm = 0.0f;
            } else {
                const int b = bh / p.kv_heads, j = (int)row;
                if (j < Span(p, b).end && !(p.docs && p.docs[b * p.docs_sb + j] < 0)) {
                    const char* v = p.v + (b * p.v_sb + (long long)j * p.v_sl + bh % p.kv_heads * p.v_sh) * Tr::ESIZE;
                    for (int c = sub; c < p.chunks; c += 16) {
                        float y[Tr::VE];
                        load_chunk<Tr>(v + c * 16, y);
#pragma unroll
                        for (int e = 0; e < Tr::VE; ++e) norm = __builtin_fmaf(y[e], y[e], norm);
                    }
                }
            }
            if (bounds) {
                norm = ormi_lanes_sum<16>(norm);
                if (norm < kInf) most_norm = fmaxf(most_norm, norm);
            }
        }
        if (!bounds) return;
        float norm = most_norm;
        norm = fmaxf(norm, __shfl_xor(norm, 16, 64));
        norm = fmaxf(norm, __shfl_xor(norm, 32, 64));
        __shared__ float most[4];
        __syncthreads();  // the last head's have been read
        if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = norm;
        __syncthreads();
        if (threadIdx.x == 0)
            atomicMax(bounds + 2 * bh + (rows ? 0 : 1), __float_as_uint(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]))));
    }
}
// The power of two that the score gradients of a batch's key head are held times.
template <class Tr>
__device__ __forceinline__ float grad_hold(const AttnParams& p, int bh) {
    if (Shift<Tr>::bwd == 0.0f) return 1.0f;
    const float bound = 2.0f * __builtin_sqrtf(p.grad_scale[2 * bh] * p.grad_scale[2 * bh + 1]);
    if (!(bound > 0.0f && bound < 1e30f)) return 1.0f;
    return __builtin_amdgcn_ldexpf(1.0f, min(100, max(-100, 15 - __builtin_amdgcn_frexp_expf(bound))));
}

// dq. Rows, tiles and masks as in the forward kernel, with both products of a
// tile's keys and values against the row's q and dout; the score gradients then
// meet the keys again, turned. Bound by the matrix pipes (2 x 4096 tokens x 16 heads
// of 128, causal: 207 us, 996 TF; 8192 tokens without a mask: 1158 TF).
template <class Tr, int DP, int BN, int FORM>
__global__ __launch_bounds__(256, DP * Tr::ESIZE > 384 ? 1 : 2) void attention_dq_kernel(AttnParams p) {
    using T = Tile<Tr, DP>;
    constexpr int NW = 4, MT = BN / 32, TILEB = T::bytes(BN);
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILEB];
    __shared__ int shared_i[3 * NW];
    __shared__ __attribute__((aligned(16))) int key_doc[2][64];  // of a stage's keys
    lds_char* lds = (lds_char*)smem;

    const Work work(p, p.splits);
    if (work.block >= p.row_blocks) return;
    const int split = work.split, bh = work.bh, rb = p.row_blocks - 1 - work.block;
    const int b = bh / p.kv_heads, kvh = bh % p.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

    const Span span(p, b);
    const int r = (rb * NW + wave) * 32 + (lane & 31);
    const int rc = min(r, p.rows - 1), i = rc / p.group, head = kvh * p.group + rc % p.group;
    const int pos = i + span.off;
    int lim = r < p.rows ? span.limit(p, pos) : 0, doc = 0;
    if (p.docs) {
        doc = doc_at(p, b, pos);
        if (doc < 0) lim = 0;
    }
    const float slope2 = FORM != kPlain && p.slopes ? p.slopes[head] * 1.44269504f : 0.0f;
    const float lse = p.lse[(long long)bh * p.rows + rc], delta = p.delta[(long long)bh * p.rows + rc];
    const float hold = grad_hold<Tr>(p, bh);
    u32x4_t qf[T::NF], gf[T::NF];
    T::row_frags(p.q + (b * p.q_sb + (long long)i * p.q_sl + head * p.q_sh) * T::ES, p.chunks, qf);
    T::row_frags(p.dout + (b * p.do_sb + (long long)i * p.do_sl + head * p.do_sh) * T::ES, p.chunks, gf);

    const int lim_min = wave_min_i(lim), lim_max = wave_max_i(lim);
    int2 docs_wave = make_int2(0, 0), docs_group;
    if (p.docs) docs_wave = widen(wave_min_i(lim > 0 ? doc : 0x7fffffff), wave_max_i(lim > 0 ? doc : -1), __any(lim <= 0));
    docs_group = docs_wave;
    int lim_group = lim_max;
    if (lane == 0) {
        shared_i[wave] = lim_max;
        shared_i[NW + wave] = docs_wave.x;
        shared_i[2 * NW + wave] = docs_wave.y;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        lim_group = max(lim_group, shared_i[w]);
        docs_group.x = min(docs_group.x, shared_i[NW + w]);
        docs_group.y = max(docs_group.y, shared_i[2 * NW + w]);
    }
    lim_group = __builtin_amdgcn_readfirstlane(lim_group);
    const int tiles = (lim_group + BN - 1) / BN;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);

    DocTiles<BN> walk{p.docs ? p.ranges + (long long)b * p.range_tiles : nullptr, p.range_tiles, -1, docs_group, docs_wave};
    auto next = [&](int t) { return p.docs ? walk.next(t, t1) : t; };
    const char* kb = p.k + (b * p.k_sb + kvh * p.k_sh) * T::ES;
    const char* vb = p.v + (b * p.v_sb + kvh * p.v_sh) * T::ES;
    using L = Loader<Tr, DP, BN, NW>;
    const typename L::Live live(p.chunks);
    auto issue = [&](int t, int stage) {
        const int last = span.end - 1 - t * BN;
        L::rows(lds + stage * 2 * TILEB, kb + (long long)t * BN * p.k_sl * T::ES, (unsigned)(p.k_sl * T::ES), last, p.chunks, live);
        L::rows(lds + stage * 2 * TILEB + TILEB, vb + (long long)t * BN * p.v_sl * T::ES, (unsigned)(p.v_sl * T::ES), last, p.chunks, live);
        if (p.docs && wave == 0) load_words(key_doc[stage], p.docs + b * p.docs_sb + min(t * BN + lane, p.keys - 1));
    };

    f32x16_t acc[T::DT];
#pragma unroll
    for (int dt = 0; dt < T::DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.0f;

    T::clear_padding(lds, 4 * BN, p.chunks, 64 * NW);
    int t = next(t0), stage = 0;
    // As in the forward pass, one tile's score gradients go in with what rounding left of them.
    const int whole = FORM != kPlain && p.slopes && !p.docs ? min(max((rb * NW * 32 / p.group + span.off) / BN, t0), max(t1 - 1, t0)) : t;
    bool same = !p.docs || (t < t1 && walk.same(t));
    if (t < t1) issue(t, 0);
    while (t < t1) {
        publish();
        const int tn = next(t + 1);
        const bool same_next = !p.docs || (tn < t1 && walk.same(tn));
        if (tn < t1) issue(tn, stage ^ 1);
        const int j0 = t * BN;
        if (j0 < lim_max) {
            const lds_char* kt = lds + stage * 2 * TILEB;
            const lds_char* vt = kt + TILEB;
            const bool masked = j0 + BN > lim_min || !same;
            const float away = (float)(pos - j0 - 4 * half);  // of the lane's first key
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                f32x16_t s, g;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = g[e] = 0.0f;
#pragma unroll
                for (int f = 0; f < T::NF; ++f) {
                    Tr::mma(T::frag(kt, mt * 32, f), qf[f], s);
                    Tr::mma(T::frag(vt, mt * 32, f), gf[f], g);
                }
                settle<Tr>(s);
                settle<Tr>(g);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float slope = 1.0f;
                    const float pr = weight2<Tr>(
                        score2<Tr, FORM>(p, s[e], slope2, away - (float)(mt * 32 + 8 * (e >> 2) + (e & 3)), -lse, slope));
                    float ds = pr * (g[e] - delta);
                    if (FORM >= kCap) ds *= slope;
                    if (Shift<Tr>::bwd != 0.0f) ds *= hold;
                    s[e] = ds;
                }
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int j = j0 + mt * 32 + 8 * (e >> 2) + 4 * half + (e & 3);
                        s[e] = j < lim ? s[e] : 0.0f;
                    }
                    if (!same) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const i32x4_t kd = *(const lds_i32x4*)&key_doc[stage][mt * 32 + 8 * q + 4 * half];
                            s[4 * q] = kd.x == doc ? s[4 * q] : 0.0f;
                            s[4 * q + 1] = kd.y == doc ? s[4 * q + 1] : 0.0f;
                            s[4 * q + 2] = kd.z == doc ? s[4 * q + 2] : 0.0f;
                            s[4 * q + 3] = kd.w == doc ? s[4 * q + 3] : 0.0f;
                        }
                    }
                }
                T::second(kt, mt * 32, s, acc);
                if (T::ES == 2 && t == whole) {
                    T::leave_rest(s);
                    T::second(kt, mt * 32, s, acc);
                }
            }
        }
        t = tn;
        same = same_next;
        stage ^= 1;
    }
#pragma unroll
    for (int dt = 0; dt < T::DT; ++dt) settle<Tr>(acc[dt]);
    clear_if(lse == kInf, acc);
    const bool bad = not_finite(acc);
    unsigned todo = (unsigned)__ballot(half == 0 && r < p.rows && __builtin_fabsf(lse) < kInf && __builtin_fabsf(delta) < kInf && bad);
    if (__builtin_expect(todo != 0, 0)) {
        const Repair w(arguments_again(), arguments_again().splits);
        if (!repair_needed<Tr>(w, __builtin_amdgcn_readfirstlane(r), t0 * BN, t1 * BN, whole * BN, whole * BN + BN,
                               [&](int j) { return key_row<Tr>(w, j); }))
            todo = 0;
    }
    const bool repaired = todo >> (lane & 31) & 1;
    if (__builtin_expect(todo != 0, 0)) {
        const Repair w(arguments_again(), arguments_again().splits);
        for (; todo; todo &= todo - 1) {
            const int rr = __builtin_amdgcn_readlane(r, __builtin_ctz(todo));
            const RepairRow<Tr, FORM> row(w, rr);
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, slope = 1.0f;
            for (int j = t0 * BN; j < t1 * BN && !all_nan(o, w.p.dim); ++j) {
                if (!row.sees(w, j)) continue;
                const float e = row.weight(w, key_row<Tr>(w, j), j, -w.p.lse[w.row_at(rr)], slope);
                const float ds = e * (row_dot<Tr>(row.dout(w), value_row<Tr>(w, j), w.p.dim) - w.p.delta[w.row_at(rr)]) * slope;
                add_row<Tr>(key_row<Tr>(w, j), w.p.dim, ds, o);
            }
            if (w.p.splits > 1) put_part<DP>(w.p.part_q + w.part_at(rr) * DP, o, grad_hold<Tr>(w.p, w.work.bh));
            else put_row<Tr>(w.p.dq + row.at(w), w.p.dim, o, w.p.scale, nullptr);
        }
    }
    if (r >= p.rows || repaired) return;
    if (p.splits > 1) {
        store_part(p.part_q + (((long long)split * p.batch * p.kv_heads + bh) * p.rows + r) * DP, acc);
        return;
    }
    store_row<Tr, T::DT>(p.dq + (((long long)b * p.queries + i) * p.heads + head) * p.dim * T::ES, p.dim, acc, p.scale / hold);
}

// The tiles of BM rows that a split goes over for the keys from k0 on: of those that
// can see them, its share.
template <int BM>
__device__ __forceinline__ int2 row_tiles(const AttnParams& p, const Span& span, int k0, int split) {
    const int tiles = (p.rows + BM - 1) / BM;
    int lo = 0, hi = tiles;
    if (k0 >= span.end) hi = 0;
    else if (p.causal && span.prefix <= k0) lo = min(tiles, (int)((long long)max(0, k0 - span.off) * p.group / BM));
    const int per = (max(hi - lo, 0) + p.key_splits - 1) / p.key_splits, t0 = min(lo + split * per, hi);
    return make_int2(t0, min(t0 + per, hi));
}

// Values in LDS instead of registers: where 32 keys' k, v and both gradients
// (16-bit rows of 128 features: 192 registers) leave too few for two waves a SIMD.
constexpr bool values_in_lds(int dp, int es) { return dp * es >= 256 && dp * es <= 512; }

// dk and dv. A wave owns 32 keys, one per lane's column: their k and v stay in
// registers as second operands, and tiles of BM rows of q and dout pass through
// LDS. Here the accumulators of the first products hold rows in their registers
// and a key per lane, so what belongs to a row (its sum, delta, limit, position)
// comes from LDS, four rows at a time. DV, DK: which gradients this launch makes
// (rows of 256 features leave the registers for one at a time; both at once
// spilled 208 of them and took 1911 us where two launches take 807, 4096 x 16 heads).
// Bound by the matrix pipes and, with both operands of three products in LDS, by its
// reads: 2 x 4096 tokens x 16 heads of 128, causal, 305 us, 901 TF (8192 tokens without a
// mask: 1035 TF). 8192 tokens in 24 documents with capped scores, 8 heads: 186 us; its 512
// work-groups all run at once and end when those of the longest documents do.
template <class Tr, int DP, int FORM, bool DK, bool DV>
__global__ __launch_bounds__(256, DP * Tr::ESIZE > 256 ? 1 : 2) void attention_dkv_kernel(AttnParams p) {
    using T = Tile<Tr, DP>;
    constexpr int NW = 4, BM = 32, TILEB = T::bytes(BM);
    constexpr bool VL = DK && values_in_lds(DP, T::ES);
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILEB + (VL ? NW * TILEB : 0)];
    // Of a stage's rows: sums and deltas, slopes and documents, positions, limits.
    __shared__ __attribute__((aligned(16))) float row_sums[2][2 * BM], row_pos[2][BM];
    __shared__ __attribute__((aligned(16))) int row_rule[2][2 * BM], row_lim[2][BM];
    lds_char* lds = (lds_char*)smem;

    const Work work(p, p.key_splits);
    if (work.block >= p.key_blocks) return;
    const int split = work.split, bh = work.bh, kblock = work.block;
    const int b = bh / p.kv_heads, kvh = bh % p.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

    const Span span(p, b);
    const int k0 = kblock * NW * 32, kw = k0 + wave * 32;  // first key of the group, of the wave
    const int key = kw + (lane & 31), keyc = min(key, max(span.end - 1, 0));
    const int doc = p.docs && key < span.end ? doc_at(p, b, key) : -1;
    const int first_doc = p.docs ? __builtin_amdgcn_readfirstlane(doc) : 0;
    const bool one_doc = p.docs && __all(doc == first_doc) && first_doc >= 0;
    const float keyf = (float)(key - k0);  // with row_pos: positions from k0 on, so that near ones are exact past 2^24
    const bool sloped = FORM != kPlain && p.slopes;
    const int key_live = p.docs && doc < 0 ? 0x7fffffff : key;  // a key without a document is seen by no row
    const float hold = grad_hold<Tr>(p, bh), shift = Shift<Tr>::bwd;
    const float hold_p = Shift<Tr>::bwd != 0.0f ? hold * __builtin_amdgcn_exp2f(-shift) : 1.0f;
    u32x4_t kf[T::NF], vf[VL ? 1 : T::NF];
    T::row_frags(p.k + (b * p.k_sb + (long long)keyc * p.k_sl + kvh * p.k_sh) * T::ES, p.chunks, kf);
    const lds_char* vt = lds + 4 * TILEB + wave * TILEB;
    if constexpr (DK && !VL) T::row_frags(p.v + (b * p.v_sb + (long long)keyc * p.v_sl + kvh * p.v_sh) * T::ES, p.chunks, vf);

    // Tiles of rows that can see the group's keys.
    const int2 part = row_tiles<BM>(p, span, k0, split);
    const int t0 = part.x, t1 = part.y;

    // With documents, tiles whose positions share none with the group's keys are passed over.
    const int2* ranges = p.docs ? p.ranges + (long long)b * p.range_tiles : nullptr;
    int2 mine = make_int2(0x7fffffff, -1);
    if (p.docs)
        for (int c = k0 / kDocTile; c < min(p.range_tiles, (k0 + NW * 32 + kDocTile - 1) / kDocTile); ++c) {
            const int2 q = ranges[c];
            mine.x = min(mine.x, q.x);
            mine.y = max(mine.y, q.y);
        }
    unsigned long long meet = 0;
    int meet_base = -1;
    auto next = [&](int t) {
        if (!p.docs) return t;
        while (t < t1) {
            if (meet_base < 0 || t >= meet_base + 64) {
                meet_base = t;
                const int at = t + lane;
                bool yes = false;
                if (at < t1) {
                    const int a = max(at * BM / p.group + span.off, 0);
                    const int z = min((min(at * BM + BM, p.rows) - 1) / p.group + span.off, p.keys - 1);
                    for (int c = a / kDocTile; z >= 0 && c <= z / kDocTile; ++c)
                        yes = yes || (ranges[c].x <= mine.y && mine.x <= ranges[c].y);
                }
                meet = __ballot(yes);
            }
            const unsigned long long left = meet >> (t - meet_base);
            if (left & 1) return t;
            t = left ? t + __builtin_ctzll(left) : meet_base + 64;
        }
        return t1;
    };
    const char* qb = p.q + (b * p.q_sb + (long long)kvh * p.group * p.q_sh) * T::ES;
    const char* gb = p.dout + (b * p.do_sb + (long long)kvh * p.group * p.do_sh) * T::ES;
    using L = Loader<Tr, DP, BM, NW>;
    const typename L::Live live(p.chunks);
    auto issue = [&](int t, int stage) {
        const int r0 = t * BM, i0 = r0 / p.group;
        const char* qt = uniform_ptr(qb + (long long)i0 * p.q_sl * T::ES);
        const char* gt = uniform_ptr(gb + (long long)i0 * p.do_sl * T::ES);
        unsigned qo[L::PER], go[L::PER];
#pragma unroll
        for (int s = 0; s < L::PER; ++s) {
            const int row = L::seg_row(s), rr = min(r0 + row, p.rows - 1);
            const int i = (int)ormi_fdiv((unsigned)rr, p.group_m, p.group_s), g = rr - i * p.group;
            const unsigned c = L::seg_chunk(s, row, p.chunks);
            qo[s] = ((unsigned)(i - i0) * (unsigned)p.q_sl + (unsigned)g * (unsigned)p.q_sh) * T::ES + c;
            go[s] = ((unsigned)(i - i0) * (unsigned)p.do_sl + (unsigned)g * (unsigned)p.do_sh) * T::ES + c;
        }
        L::load(lds + stage * 2 * TILEB, qt, qo, live);
        L::load(lds + stage * 2 * TILEB + TILEB, gt, go, live);
        // What belongs to the rows, one per lane of the first wave's halves; a row
        // past the last has the limit 0, as has one without a document of its own.
        if (wave == 0) {
            const int rr = min(r0 + (lane & 31), p.rows - 1);
            const int i = (int)ormi_fdiv((unsigned)rr, p.group_m, p.group_s), pos = i + span.off;
            load_words(row_sums[stage], (half == 0 ? p.lse : p.delta) + (long long)bh * p.rows + rr);
            if (p.docs || sloped)
                load_words(row_rule[stage], half == 0 && sloped ? (const int*)p.slopes + kvh * p.group + rr - i * p.group
                                            : p.docs ? p.docs + b * p.docs_sb + min(max(pos, 0), p.keys - 1)
                                                     : (const int*)p.slopes);
            if (half == 0) {
                row_lim[stage][lane] = r0 + lane >= p.rows || (p.docs && pos < 0) ? 0 : span.limit(p, pos);
                if (FORM != kPlain) row_pos[stage][lane] = (float)(pos - k0);
            }
        }
    };
    f32x16_t acc_k[T::DT], acc_v[T::DT];
#pragma unroll
    for (int dt = 0; dt < T::DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc_k[dt][e] = acc_v[dt][e] = 0.0f;

    T::clear_padding(lds, (VL ? 4 + NW : 4) * BM, p.chunks, 64 * NW);
    int t = next(t0), stage = 0;
    // One tile's weights and score gradients go in with what rounding left of them: the
    // only tile of keys that few rows see.
    const int whole = sloped && !p.docs ? min(max((int)((long long)max(0, k0 - span.off) * p.group / BM), t0), max(t1 - 1, t0)) : t;
    if (t < t1) {
        issue(t, 0);
        if constexpr (VL) {
            lds_char* vg = lds + 4 * TILEB;
            const char* vb = p.v + (b * p.v_sb + kvh * p.v_sh + (long long)k0 * p.v_sl) * T::ES;
            using V = Loader<Tr, DP, NW * 32, NW>;
            V::rows(vg, vb, (unsigned)(p.v_sl * T::ES), span.end - 1 - k0, p.chunks, typename V::Live(p.chunks));
        }
    }
    while (t < t1) {
        publish();
        const int tn = next(t + 1);
        if (tn < t1) issue(tn, stage ^ 1);
        const int lim_lane = row_lim[stage][lane & 31];
        if (__any(lim_lane > kw)) {
            const lds_char* qt = lds + stage * 2 * TILEB;
            const lds_char* gt = qt + TILEB;
            bool same = true;
            if (p.docs) same = one_doc && __all(row_rule[stage][BM + (lane & 31)] == first_doc);
            const bool masked = !__all(lim_lane >= kw + 32) || !same;
            f32x16_t s, g;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = g[e] = 0.0f;
#pragma unroll
            for (int f = 0; f < T::NF; ++f) {
                Tr::mma(T::frag(qt, 0, f), kf[f], s);
                if constexpr (VL) Tr::mma(T::frag(gt, 0, f), T::frag(vt, 0, f), g);
                else if (DK) Tr::mma(T::frag(gt, 0, f), vf[f], g);
            }
            settle<Tr>(s);
            if (DK) settle<Tr>(g);
            // s becomes p, g the score gradient.
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const int row = 8 * q4 + 4 * half;
                const f32x4_t ls = *(const lds_f32x4*)&row_sums[stage][row];
                f32x4_t de, sl, ps;
                if (DK) de = *(const lds_f32x4*)&row_sums[stage][BM + row];
                if (FORM != kPlain) {
                    sl = *(const lds_f32x4*)&row_rule[stage][row];
                    ps = *(const lds_f32x4*)&row_pos[stage][row];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = 4 * q4 + e;
                    float slope = 1.0f;
                    s[x] = weight2<Tr>(
                        score2<Tr, FORM>(p, s[x], sloped ? sl[e] * 1.44269504f : 0.0f, ps[e] - keyf, shift - ls[e], slope));
                    if (!DK) continue;
                    g[x] = s[x] * (g[x] - de[e]);
                    if (FORM >= kCap) g[x] *= slope;
                    if (Shift<Tr>::bwd != 0.0f) g[x] *= hold_p;
                }
            }
            if (masked) {
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const int row = 8 * q4 + 4 * half;
                    const i32x4_t li = *(const lds_i32x4*)&row_lim[stage][row];
                    i32x4_t dc = {0, 0, 0, 0};
                    if (!same) dc = *(const lds_i32x4*)&row_rule[stage][BM + row];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int x = 4 * q4 + e;
                        const bool seen = key_live < li[e] && (same || dc[e] == doc);
                        s[x] = seen ? s[x] : 0.0f;
                        if (DK) g[x] = seen ? g[x] : 0.0f;
                    }
                }
            }
            if (DV) T::second(gt, 0, s, acc_v);
            if (DK) T::second(qt, 0, g, acc_k);
            if (T::ES == 2 && t == whole) {
                if (DV) {
                    T::leave_rest(s);
                    T::second(gt, 0, s, acc_v);
                }
                if (DK) {
                    T::leave_rest(g);
                    T::second(qt, 0, g, acc_k);
                }
            }
        }
        t = tn;
        stage ^= 1;
    }
#pragma unroll
    for (int dt = 0; dt < T::DT; ++dt) {
        if (DK) settle<Tr>(acc_k[dt]);
        if (DV) settle<Tr>(acc_v[dt]);
    }
    bool bad = false;
    if (DK) bad = not_finite(acc_k);
    if (DV) bad = bad | not_finite(acc_v);
    unsigned todo = (unsigned)__ballot(half == 0 && key < p.keys && bad);
    if (__builtin_expect(todo != 0, 0)) {  // is a row not finite that does not see all of the wave's keys, or is in the tile `whole`?
        const Repair w(arguments_again(), arguments_again().key_splits);
        const int first = w.work.block * NW * 32, past = first + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32 + 32;
        const int2 tiles = row_tiles<BM>(w.p, w.span, first, w.work.split);
        bool hidden = false;
        for (int rr = tiles.x * BM; rr < min(tiles.y * BM, w.p.rows) && !hidden; ++rr) {
            const RepairRow<Tr, FORM> row(w, rr);  // rows past the last read it again
            if (w.p.docs || rr == w.p.rows - 1 || w.span.limit(w.p, row.pos) < past || (T::ES == 2 && rr / BM == whole))
                hidden = row_bad<Tr>(row.q(w), w.p.dim) || row_bad<Tr>(row.dout(w), w.p.dim);
        }
        if (!hidden) todo = 0;
    }
    const bool repaired = todo >> (lane & 31) & 1;
    if (__builtin_expect(todo != 0, 0)) {
        for (; todo; todo &= todo - 1) {
            const AttnParams& a = arguments_again();
            const Work at(a, a.key_splits);
            const int at_k0 = at.block * NW * 32, j = at_k0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32 + __builtin_ctz(todo);
            const int2 tiles = row_tiles<BM>(a, Span(a, at.bh / a.kv_heads), at_k0, at.split);
            float ok[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ov[4] = {0.0f, 0.0f, 0.0f, 0.0f}, slope = 1.0f;
            for (int rr = tiles.x * BM; rr < min(tiles.y * BM, arguments_again().rows); ++rr) {
                if ((!DK || all_nan(ok, arguments_again().dim)) && (!DV || all_nan(ov, arguments_again().dim))) break;
                const Repair w(arguments_again(), arguments_again().key_splits);
                const RepairRow<Tr, FORM> row(w, rr);
                if (!row.sees(w, j)) continue;
                const float e = row.weight(w, key_row<Tr>(w, j), j, -w.p.lse[w.row_at(rr)], slope);
                if (DV) add_row<Tr>(row.dout(w), w.p.dim, e, ov);
                if (DK)
                    add_row<Tr>(row.q(w), w.p.dim,
                                e * (row_dot<Tr>(row.dout(w), value_row<Tr>(w, j), w.p.dim) - w.p.delta[w.row_at(rr)]) * slope, ok);
            }
            const Repair w(arguments_again(), arguments_again().key_splits);
            const long long n = (long long)w.p.batch * w.p.kv_heads * w.p.keys, row = (long long)w.work.bh * w.p.keys + j;
            const long long to = (((long long)w.b * w.p.keys + j) * w.p.kv_heads + w.kvh) * w.p.dim * T::ES;
            if (w.p.key_splits > 1) {
                if (DK) put_part<DP>(w.p.part + (w.work.split * n + row) * DP, ok, grad_hold<Tr>(w.p, w.work.bh));
                if (DV) put_part<DP>(w.p.part + ((w.p.key_splits + w.work.split) * n + row) * DP, ov, __builtin_amdgcn_exp2f(Shift<Tr>::bwd));
            } else {
                if (DK && w.p.dk) put_row<Tr>(w.p.dk + to, w.p.dim, ok, w.p.scale, nullptr);
                if (DV && w.p.dv) put_row<Tr>(w.p.dv + to, w.p.dim, ov, 1.0f, nullptr);
            }
        }
    }
    if (key >= p.keys || repaired) return;
    if (p.key_splits > 1) {
        const long long n = (long long)p.batch * p.kv_heads * p.keys, at = (long long)bh * p.keys + key;
        if (DK) store_part(p.part + (split * n + at) * DP, acc_k);
        if (DV) store_part(p.part + ((p.key_splits + split) * n + at) * DP, acc_v);
        return;
    }
    const long long at = (((long long)b * p.keys + key) * p.kv_heads + kvh) * p.dim * T::ES;
    if (DK && p.dk) store_row<Tr, T::DT>(p.dk + at, p.dim, acc_k, p.scale / hold);
    if (DV && p.dv) store_row<Tr, T::DT>(p.dv + at, p.dim, acc_v, __builtin_amdgcn_exp2f(-shift));
}

// Adds the splits' partial gradients in split order, one wave per row: first dq's
// rows, then each key's dk and dv. Bound by memory (four splits of
// 8 x 4096 keys of 128 features: 134 MB read and 17 written in 25 us).
template <class Tr, int DP>
__global__ __launch_bounds__(256) void attention_grad_join_kernel(AttnParams p) {
    const long long nq = p.dq && p.splits > 1 ? (long long)p.batch * p.kv_heads * p.rows : 0;
    const long long nk = (p.dk || p.dv) && p.key_splits > 1 ? (long long)p.batch * p.kv_heads * p.keys : 0;
    long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    auto add = [&](const float* part, int splits, long long n, char* out, long long at, float f) {
#pragma unroll
        for (int e = 0; e < (DP + 63) / 64; ++e) {
            const int d = e * 64 + lane;
            if (d >= p.dim) continue;
            float v = 0.0f;
#pragma unroll 4
            for (int s = 0; s < splits; ++s) v += part[(s * n + row) * DP + d];
            v *= f;
            if constexpr (Tr::ESIZE == 4) ((float*)out)[at + d] = v;
            else ((unsigned short*)out)[at + d] = (unsigned short)pack2(Tr{}, v, v);
        }
    };
    if (row < nq) {
        const int bh = (int)(row / p.rows), r = (int)(row % p.rows), b = bh / p.kv_heads;
        const int i = r / p.group, head = (bh % p.kv_heads) * p.group + r % p.group;
        add(p.part_q, p.splits, nq, p.dq, (((long long)b * p.queries + i) * p.heads + head) * p.dim, p.scale / grad_hold<Tr>(p, bh));
        return;
    }
    row -= nq;
    if (row >= nk) return;
    const int bh = (int)(row / p.keys), j = (int)(row % p.keys), b = bh / p.kv_heads, kvh = bh % p.kv_heads;
    const long long at = (((long long)b * p.keys + j) * p.kv_heads + kvh) * p.dim;
    if (p.dk) add(p.part, p.key_splits, nk, p.dk, at, p.scale / grad_hold<Tr>(p, bh));
    if (p.dv) add(p.part + p.key_splits * nk * DP, p.key_splits, nk, p.dv, at, __builtin_amdgcn_exp2f(-Shift<Tr>::bwd));
}

template <class Tr, int DP, int FORM>
void launch_attention_grad_form(const AttnParams& p) {
    if (p.dq) attention_dq_kernel<Tr, DP, fwd_tile(DP, Tr::ESIZE, false), FORM><<<Work::grid(p, p.row_blocks, p.splits), 256>>>(p);
    if (p.dk || p.dv) {
        const unsigned grid = Work::grid(p, p.key_blocks, p.key_splits);
        if constexpr (DP > 128) {
            if (p.dk) attention_dkv_kernel<Tr, DP, FORM, true, false><<<grid, 256>>>(p);
            if (p.dv) attention_dkv_kernel<Tr, DP, FORM, false, true><<<grid, 256>>>(p);
        } else {
            attention_dkv_kernel<Tr, DP, FORM, true, true><<<grid, 256>>>(p);
        }
    }
}

// Work-groups over the rows of dout, and over those of v, where both also give their
// largest norms: the words of all heads lie in a few lines, in which the maxima of all
// work-groups meet (8192 tokens, 8 heads of 128: 1024 work-groups 33 us, 4096 98 us).
constexpr int kDeltaGroups = 1024;

template <class Tr, int DP>
int launch_attention_grad_dp(const AttnParams& p, float* delta, unsigned* bounds) {
    const long long rows = (long long)p.batch * p.queries * p.heads, values = (long long)p.batch * p.keys * p.kv_heads;
    unsigned row_groups = (unsigned)std::min<long long>((rows + 15) / 16, 1 << 22), value_groups = 0;  // a launch holds fewer than 2^24 of 256 threads
    if (bounds) {
        const int heads = std::min(p.batch * p.kv_heads, 1 << 16), slices = std::max(1, kDeltaGroups / heads);
        row_groups = (unsigned)(heads * std::min((p.rows + 15) / 16, slices));
        value_groups = (unsigned)(heads * std::min((p.keys + 15) / 16, slices));
    }
    attention_delta_kernel<Tr><<<row_groups + value_groups, 256>>>(p, delta, bounds, row_groups);
    if (p.form == kPlain) launch_attention_grad_form<Tr, DP, kPlain>(p);
    else if (p.form == kBias) launch_attention_grad_form<Tr, DP, kBias>(p);
    else if (Tr::ESIZE == 4 || p.form == kCap) launch_attention_grad_form<Tr, DP, kCap>(p);
    else if constexpr (Tr::ESIZE == 2) launch_attention_grad_form<Tr, DP, kCapWide>(p);
    const long long join = (p.dq && p.splits > 1 ? rows : 0) + ((p.dk || p.dv) && p.key_splits > 1 ? values : 0);
    if (join > 0) attention_grad_join_kernel<Tr, DP><<<(unsigned)((join + 3) / 4), 256>>>(p);
    return (int)hipGetLastError();
}

}  // namespace ormi_hip
