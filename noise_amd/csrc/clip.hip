// Global norm of many gradients, and the gradients scaled in place to a bound on it:
//   norm = sqrt(sum of squares),  factor = min(1, max_norm / (norm + 1e-6)),  g <- factor g.
// Memory bound: everything is read once for the norm, then read and written once where the factor is below 1. Two launches per
// table of 192 tensors: the first leaves one partial sum per workgroup, and every workgroup of the second adds those up itself, in
// the same order, so that nothing waits for a launch in between and results do not depend on timing. Squares are summed in fp64:
// no finite fp32 or bf16 value's square overflows or vanishes there; the factor, which may then be too small for fp32, is 24 bits and
// a power of two.
// A workgroup takes a contiguous range of the bytes, forwards for the norm and backwards for the scaling, which starts with what
// was read last and is still in the caches. 37.75 M fp32 values in 60 tensors: 29 us for the norm (5.2 TB/s) and 53 for the scaling
// (5.7 TB/s read and written); 1e9 values in 300 tensors, fp32 and bf16: 736 us (5.1) and 1630 (4.6).
#include "common.hpp"
#include "mfma.hpp"

#include <stdlib.h>

namespace noise {
namespace {

constexpr int kTensors = 192;        // of a launch's table, which travels as a kernel argument (3.9 KB)
constexpr int kThreads = 256, kUnroll = 4;
constexpr int64_t kUnit = 16 * kThreads * kUnroll;   // bytes that a workgroup takes at a time
constexpr int kGroups = 2048;        // workgroups of all launches together, at most one more per launch

struct ClipArgs {
    void *ptr[kTensors];
    int64_t numel[kTensors];         // bf16 tensors: -numel
    uint32_t unit[kTensors];         // a tensor's first unit
    int count;
    uint32_t units, groups, first;   // of this launch; first: where its partial sums go
};
struct ClipBound {
    double *partials;
    float *norm;
    float max_norm;
    uint32_t total;                  // partial sums
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <class E>
__device__ __forceinline__ float element(const u32x4 &v, int e) {
    if constexpr (sizeof(E) == 4) return __uint_as_float(v[e]);
    return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
}

// Elements before the first 16 B address, whole 16 B pieces, elements after them
template <class E>
struct Span {
    E *head, *tail;
    u32x4 *body;
    int heads, tails;
    int64_t pieces;
    __device__ Span(void *p, int64_t n) {
        constexpr int N = 16 / sizeof(E);
        head = static_cast<E *>(p);
        heads = (int)((0 - (uintptr_t)p) % 16 / sizeof(E));
        if (heads > n) heads = (int)n;
        pieces = (n - heads) / N;
        body = reinterpret_cast<u32x4 *>(head + heads);
        tail = head + heads + pieces * N;
        tails = (int)(n - heads - pieces * N);
    }
};

template <class E>
__device__ __forceinline__ void add_unit(void *p, int64_t n, int64_t unit, double (&s)[kUnroll]) {
    constexpr int N = 16 / sizeof(E);
    const Span<E> sp(p, n);
    const int64_t at = unit * (kThreads * kUnroll) + threadIdx.x;
    u32x4 v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) v[i] = at + i * kThreads < sp.pieces ? sp.body[at + i * kThreads] : u32x4{0, 0, 0, 0};
    double x = 0.;
    if (unit == 0) {
        if ((int)threadIdx.x < sp.heads) x = (double)(float)sp.head[threadIdx.x];
        else if ((int)threadIdx.x - N >= 0 && (int)threadIdx.x - N < sp.tails) x = (double)(float)sp.tail[threadIdx.x - N];
    }
    s[0] += x * x;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double d = (double)element<E>(v[i], e);
            s[i] += d * d;
        }
}

// factor = part 2^power with part of 24 bits in 1/2 .. 1: no factor is too small for fp32, and its products are rounded as any
struct Factor {
    float part;
    int power;
    __device__ __forceinline__ float times(float v) const { return ldexpf(v * part, power); }
};

template <class E>
__device__ __forceinline__ void scale_unit(void *p, int64_t n, int64_t unit, const Factor &factor) {
    constexpr int N = 16 / sizeof(E);
    const Span<E> sp(p, n);
    const int64_t at = unit * (kThreads * kUnroll) + threadIdx.x;
    u32x4 v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
        if (at + i * kThreads < sp.pieces) v[i] = sp.body[at + i * kThreads];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
        if (at + i * kThreads < sp.pieces) {
            E o[N];
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = (E)factor.times(element<E>(v[i], e));
            __builtin_memcpy(&v[i], o, 16);
            sp.body[at + i * kThreads] = v[i];
        }
    if (unit == 0) {
        E *x = (int)threadIdx.x < sp.heads ? sp.head + threadIdx.x
               : (int)threadIdx.x - N >= 0 && (int)threadIdx.x - N < sp.tails ? sp.tail + (threadIdx.x - N)
                                                                              : nullptr;
        if (x) *x = (E)factor.times((float)*x);
    }
}

// Sum over the workgroup, which every thread gets
__device__ __forceinline__ double group_sum(double s) {
    __shared__ double slots[kThreads / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) s += slots[w];
    return s;
}

// The last tensor that begins at or before a unit (tensors without elements have no units and are not in the table)
__device__ __forceinline__ int tensor_of(const ClipArgs &a, uint32_t unit) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.unit[mid] <= unit) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ __launch_bounds__(kThreads) void clip_norm_kernel(ClipArgs a, double *partials) {
    const uint32_t begin = (uint32_t)((uint64_t)a.units * blockIdx.x / a.groups);
    const uint32_t end = (uint32_t)((uint64_t)a.units * (blockIdx.x + 1) / a.groups);
    double s[kUnroll] = {};
    int t = begin < end ? tensor_of(a, begin) : 0;
    for (uint32_t u = begin; u < end; ++u) {
        while (t + 1 < a.count && a.unit[t + 1] <= u) ++t;
        const int64_t n = a.numel[t];
        if (n < 0) add_unit<__bf16>(a.ptr[t], -n, u - a.unit[t], s);
        else add_unit<float>(a.ptr[t], n, u - a.unit[t], s);
    }
    double all = 0.;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) all += s[i];
    all = group_sum(all);
    if (threadIdx.x == 0) partials[a.first + blockIdx.x] = all;
}

__device__ __forceinline__ double total_norm(const ClipBound &b) {
    double s = 0.;
    for (uint32_t i = threadIdx.x; i < b.total; i += kThreads) s += b.partials[i];
    return sqrt(group_sum(s));
}

__global__ __launch_bounds__(kThreads) void clip_scale_kernel(ClipArgs a, ClipBound b) {
    const double norm = total_norm(b);
    if (a.first + blockIdx.x == 0 && threadIdx.x == 0) *b.norm = (float)norm;
    const double quotient = (double)b.max_norm / (norm + 1e-6);
    if (quotient >= 1.) return;   // (a NaN goes on, into every gradient)
    Factor factor;
    factor.part = (float)frexp(quotient, &factor.power);
    const uint32_t begin = (uint32_t)((uint64_t)a.units * blockIdx.x / a.groups);
    const uint32_t end = (uint32_t)((uint64_t)a.units * (blockIdx.x + 1) / a.groups);
    if (begin == end) return;
    int t = tensor_of(a, end - 1);
    for (uint32_t u = end; u-- > begin;) {
        while (a.unit[t] > u) --t;
        const int64_t n = a.numel[t];
        if (n < 0) scale_unit<__bf16>(a.ptr[t], -n, u - a.unit[t], factor);
        else scale_unit<float>(a.ptr[t], n, u - a.unit[t], factor);
    }
}

// The norm alone
__global__ __launch_bounds__(kThreads) void clip_total_kernel(ClipBound b) {
    const double norm = total_norm(b);
    if (threadIdx.x == 0) *b.norm = (float)norm;
}

int by_address(const void *p, const void *q) {
    const uintptr_t a = (uintptr_t)(*static_cast<const noise_gradient_t *const *>(p))->ptr,
                    b = (uintptr_t)(*static_cast<const noise_gradient_t *const *>(q))->ptr;
    return a < b ? -1 : a > b;
}

int64_t bytes_of(const noise_gradient_t &g) { return g.numel * (g.type == NOISE_BF16 ? 2 : 4); }
// units of a tensor: at least one, whose workgroup also takes what stands before and after the whole 16 B pieces
int64_t units_of(const noise_gradient_t &g) { return g.numel == 0 ? 0 : (bytes_of(g) + kUnit - 1) / kUnit; }

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int64_t noise_clip_workspace_bytes(int64_t count) {
    clear_error();
    NOISE_CHECK_ARG(count > 0 && count <= (1 << 24), "noise_clip_workspace_bytes: 1 .. 2^24 gradients required, got %lld", (long long)count);
    return 8 * (int64_t)(kGroups + count / kTensors + 1);
}

extern "C" int noise_clip_gradients(const noise_gradient_t *gradients, int64_t count, float max_norm, float *norm,
                                    void *workspace, int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_clip_gradients";
    NOISE_CHECK_ARG(gradients && count > 0 && count <= (1 << 24), "%s: bad table of gradients", fn);
    NOISE_CHECK_ARG(max_norm >= 0.f, "%s: max_norm must not be negative", fn);
    NOISE_CHECK_ARG(norm && aligned(norm, 4), "%s: norm NULL or not 4 B aligned", fn);
    NOISE_CHECK_ARG(workspace && aligned(workspace, 8) && workspace_bytes >= noise_clip_workspace_bytes(count),
                    "%s: workspace of %lld bytes (8 B aligned) required", fn, (long long)noise_clip_workspace_bytes(count));
    int64_t units = 0, tensors = 0;
    bool sorted = true;
    uintptr_t end = 0;
    for (int64_t i = 0; i < count; ++i) {
        const noise_gradient_t &g = gradients[i];
        NOISE_CHECK_ARG(g.type == NOISE_BF16 || g.type == NOISE_FP32, "%s: gradient %lld: unknown type %lld", fn, (long long)i,
                        (long long)g.type);
        NOISE_CHECK_ARG(g.numel >= 0 && g.numel <= (1ll << 40), "%s: gradient %lld: bad number of elements", fn, (long long)i);
        if (g.numel == 0) continue;
        NOISE_CHECK_ARG(g.ptr && aligned(g.ptr, g.type == NOISE_BF16 ? 2 : 4), "%s: gradient %lld: NULL or not aligned to its type",
                        fn, (long long)i);
        if ((uintptr_t)g.ptr < end) sorted = false;
        end = (uintptr_t)g.ptr + bytes_of(g);
        units += units_of(g);
        ++tensors;
    }
    NOISE_CHECK_ARG(units < (1ll << 32), "%s: too many elements", fn);
    if (!sorted) {
        // gradients that share memory would be counted and scaled twice, by workgroups that race
        const noise_gradient_t **order = static_cast<const noise_gradient_t **>(malloc(tensors * sizeof(*order)));
        NOISE_CHECK_ARG(order, "%s: out of host memory", fn);
        int64_t n = 0;
        for (int64_t i = 0; i < count; ++i)
            if (gradients[i].numel) order[n++] = gradients + i;
        qsort(order, n, sizeof(*order), by_address);
        bool overlap = false;
        for (int64_t i = 1; i < n; ++i)
            overlap |= (uintptr_t)order[i]->ptr < (uintptr_t)order[i - 1]->ptr + bytes_of(*order[i - 1]);
        free(order);
        NOISE_CHECK_ARG(!overlap, "%s: gradients share memory", fn);
    }
    ClipBound b;
    b.partials = static_cast<double *>(workspace);
    b.norm = norm;
    b.max_norm = max_norm;
    // workgroups: in proportion to a launch's share of the work, kGroups together (or one per unit)
    const int64_t groups = units < kGroups ? units : kGroups;
    for (int pass = 0; pass < 2; ++pass) {
        ClipArgs a;
        a.count = 0, a.units = 0, a.first = 0;
        for (int64_t i = 0; i < count; ++i) {
            const int64_t n = units_of(gradients[i]);
            if (n) {
                a.ptr[a.count] = gradients[i].ptr;
                a.numel[a.count] = gradients[i].type == NOISE_BF16 ? -gradients[i].numel : gradients[i].numel;
                a.unit[a.count++] = a.units;
                a.units += (uint32_t)n;
            }
            if (a.count && (a.count == kTensors || i + 1 == count)) {
                const int64_t share = (int64_t)((__int128)groups * a.units / units);
                a.groups = (uint32_t)(share ? share : 1);
                if (pass == 0)
                    hipLaunchKernelGGL(clip_norm_kernel, dim3(a.groups), dim3(kThreads), 0, (hipStream_t)stream, a, b.partials);
                else
                    hipLaunchKernelGGL(clip_scale_kernel, dim3(a.groups), dim3(kThreads), 0, (hipStream_t)stream, a, b);
                a.first += a.groups;
                a.count = 0, a.units = 0;
            }
        }
        b.total = a.first;
        if (pass == 0 && (b.total == 0 || max_norm > 3.4028234663852886e38f)) {
            hipLaunchKernelGGL(clip_total_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, b);
            break;
        }
    }
    return launch_status(fn);
}
