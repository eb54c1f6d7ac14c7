// The norm over a list of tensors, and their values times a factor.
//   norm = sqrt(sum of all squares), factor = min(1, max_norm / norm)
// Bound by memory: one read for the norm, a read and a write for the product.
// Squares are added in 64 bits: those of float32 are exact there, neither
// overflow nor vanish, and cost less than the memory (a conversion and a
// multiply-add an element). Pointers travel in the kernels' arguments as
// AdamW's do. A work-group leaves one partial sum, and a last launch of one
// work-group adds those up: the order is fixed by the sizes. 25 M float32 parameters:
// 20 us (5.0 TB/s), 4 and 31 (the second read comes partly out of the Infinity Cache).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "ormi_hip.h"
#include "ormi_hip_internal.h"
#include "row_access.h"

namespace ormi_hip {
namespace {

constexpr int kMostNorm = 160, kMostScale = 120;  // tensors per launch: their entries fit 4 KB of arguments
constexpr int kPerGroup = 8192;                   // elements per work-group
constexpr long long kMostGroups = (1ll << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32

struct NormEntry {
    const void* data;
    long long count;
    unsigned first;  // its first work-group
    int dtype;
};
struct NormParams {
    double* part;  // of this launch's first work-group
    int n;
    NormEntry t[kMostNorm];
};
struct ScaleEntry {
    const void* data;
    void* out;
    long long count;
    unsigned first;
    int dtype;
};
struct ScaleParams {
    const float* factor;
    int n;
    ScaleEntry t[kMostScale];
};
static_assert(sizeof(NormParams) <= 4096 && sizeof(ScaleParams) <= 4096, "kernel arguments");

template <class P>
__device__ __forceinline__ int find_tensor(const P& a) {
    int t = 0;
    for (int step = 128; step > 0; step >>= 1)
        if (t + step < a.n && a.t[t + step].first <= blockIdx.x) t += step;
    return t;
}

template <int DT>
__device__ __forceinline__ double squares(const void* data, long long base, long long count) {
    constexpr int V = DT == ORMI_DTYPE_F32 ? 4 : 8, K = kPerGroup / 256 / V;
    using T = typename ElemOf<DT>::type;
    Run<DT, V> r[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = base + (k * 256 + (int)threadIdx.x) * V;
        r[k].load((const T*)data + i, (int)max(0ll, min((long long)V, count - i)));
    }
    double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double x = r[k].get(e);
            s[e % 4] = __builtin_fma(x, x, s[e % 4]);
        }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// v of all threads of a work-group of N waves, in thread 0.
template <int N>
__device__ __forceinline__ double group_sum(double v) {
    __shared__ double lds[N];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    if (threadIdx.x == 0)
        for (int i = 0; i < N; ++i) s += lds[i];
    return s;
}

__global__ __launch_bounds__(256) void norm_kernel(NormParams a) {
    const NormEntry& t = a.t[find_tensor(a)];
    const long long base = (long long)(blockIdx.x - t.first) * kPerGroup;
    const double s = t.dtype == ORMI_DTYPE_F32    ? squares<ORMI_DTYPE_F32>(t.data, base, t.count)
                     : t.dtype == ORMI_DTYPE_BF16 ? squares<ORMI_DTYPE_BF16>(t.data, base, t.count)
                                                  : squares<ORMI_DTYPE_F16>(t.data, base, t.count);
    const double total = group_sum<4>(s);
    if (threadIdx.x == 0) a.part[blockIdx.x] = total;
}

__global__ __launch_bounds__(1024) void norm_join_kernel(const double* part, long long count, double max_norm, float* norm, float* factor) {
    double s = 0.0;
    for (long long i = threadIdx.x; i < count; i += 1024) s += part[i];
    s = group_sum<16>(s);
    if (threadIdx.x != 0) return;
    const double n = sqrt(s);
    if (norm) *norm = (float)n;
    if (factor) *factor = (float)(n <= max_norm ? 1.0 : max_norm / n);
}

template <int DT>
__device__ __forceinline__ void scale(const ScaleEntry& t, long long base, float factor) {
    constexpr int V = DT == ORMI_DTYPE_F32 ? 4 : 8, K = kPerGroup / 256 / V;
    using T = typename ElemOf<DT>::type;
    Run<DT, V> r[K];
    int n[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = base + (k * 256 + (int)threadIdx.x) * V;
        n[k] = (int)max(0ll, min((long long)V, t.count - i));
        r[k].load((const T*)t.data + i, n[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) r[k].set(e, r[k].get(e) * factor);
        r[k].store((T*)t.out + base + (k * 256 + (int)threadIdx.x) * V, n[k]);
    }
}
__global__ __launch_bounds__(256) void scale_kernel(ScaleParams a) {
    const ScaleEntry& t = a.t[find_tensor(a)];
    const long long base = (long long)(blockIdx.x - t.first) * kPerGroup;
    const float factor = *a.factor;
    if (t.dtype == ORMI_DTYPE_F32) scale<ORMI_DTYPE_F32>(t, base, factor);
    else if (t.dtype == ORMI_DTYPE_BF16) scale<ORMI_DTYPE_BF16>(t, base, factor);
    else scale<ORMI_DTYPE_F16>(t, base, factor);
}

const char* check(const ormi_tensor_ref* tensors, int n, bool out) {
    if (n < 0 || (n > 0 && !tensors)) return "bad tensor list";
    for (int k = 0; k < n; ++k) {
        const ormi_tensor_ref& t = tensors[k];
        if (t.dtype != ORMI_DTYPE_F32 && t.dtype != ORMI_DTYPE_BF16 && t.dtype != ORMI_DTYPE_F16) return "tensors must be float32, bfloat16 or float16";
        if (t.count < 0 || t.count > kMostGroups * kPerGroup) return "element count out of range";
        if (t.count > 0 && (!t.data || (out && !t.out))) return "null tensor";
    }
    return nullptr;
}
long long groups_of(const ormi_tensor_ref& t) { return (t.count + kPerGroup - 1) / kPerGroup; }
size_t part_bytes(const ormi_tensor_ref* tensors, int n) {
    long long groups = 0;
    for (int k = 0; k < n; ++k) groups += groups_of(tensors[k]);
    return (size_t)(groups * (long long)sizeof(double) + 255) / 256 * 256;
}

// Calls launch(params, work-groups) for as many tensors at a time as its arguments
// and a launch hold.
template <int MOST, class P, class Entry, class Launch>
void in_launches(const ormi_tensor_ref* tensors, int n, P& a, Entry entry, Launch launch) {
    long long groups = 0;
    a.n = 0;
    auto flush = [&] {
        if (a.n > 0) launch(groups);
        a.n = 0;
        groups = 0;
    };
    for (int k = 0; k < n; ++k) {
        if (tensors[k].count == 0) continue;
        const long long need = groups_of(tensors[k]);
        if (a.n == MOST || groups + need > kMostGroups) flush();
        auto& e = a.t[a.n++];
        e.data = tensors[k].data;
        e.count = tensors[k].count;
        e.dtype = tensors[k].dtype;
        e.first = (unsigned)groups;
        entry(e, tensors[k]);
        groups += need;
    }
    flush();
}

}  // namespace
}  // namespace ormi_hip

using namespace ormi_hip;

extern "C" {

int ormi_hip_norm_workspace_size(const ormi_tensor_ref* tensors, int num_tensors, size_t* bytes) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_norm_workspace_size: ") + what); };
    if (const char* what = check(tensors, num_tensors, false)) return bad(what);
    if (!bytes) return bad("null bytes");
    *bytes = part_bytes(tensors, num_tensors);
    return ORMI_HIP_OK;
}

int ormi_hip_norm(const ormi_tensor_ref* tensors, int num_tensors, double max_norm, float* norm, float* factor, void* workspace,
                  size_t workspace_bytes) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_norm: ") + what); };
    if (const char* what = check(tensors, num_tensors, false)) return bad(what);
    if (factor && !(max_norm >= 0.0)) return bad("max_norm must not be negative");
    const size_t need = part_bytes(tensors, num_tensors);
    if (need > 0 && (!workspace || workspace_bytes < need)) return bad("workspace too small");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    NormParams a{};
    double* const part = (double*)workspace;
    long long done = 0;
    in_launches<kMostNorm>(tensors, num_tensors, a, [](NormEntry&, const ormi_tensor_ref&) {}, [&](long long groups) {
        a.part = part + done;
        norm_kernel<<<(unsigned)groups, 256>>>(a);
        done += groups;
    });
    norm_join_kernel<<<1, 1024>>>(part, done, max_norm, norm, factor);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string("ormi_hip_norm: ") + hipGetErrorString(e));
}

int ormi_hip_scale(const ormi_tensor_ref* tensors, int num_tensors, const float* factor) {
    auto bad = [](const char* what) { return fail(ORMI_HIP_ERR_INVALID, std::string("ormi_hip_scale: ") + what); };
    if (const char* what = check(tensors, num_tensors, true)) return bad(what);
    if (!factor) return bad("null factor");
    int rc = ensure_init();
    if (rc != ORMI_HIP_OK || (rc = drain_queue()) != ORMI_HIP_OK) return rc;
    ScaleParams a{};
    a.factor = factor;
    in_launches<kMostScale>(tensors, num_tensors, a, [](ScaleEntry& e, const ormi_tensor_ref& t) { e.out = t.out; },
                            [&](long long groups) { scale_kernel<<<(unsigned)groups, 256>>>(a); });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ORMI_HIP_OK : fail(ORMI_HIP_ERR_RUNTIME, std::string("ormi_hip_scale: ") + hipGetErrorString(e));
}

}  // extern "C"
