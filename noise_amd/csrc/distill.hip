// Distillation from a teacher's top logits, forward and backward: per row of logits x, with z = cap(x) / tau and the teacher's
// softmax p over its entries in use,
//   loss = tau^2 sum_k p_k (log p_k - z[i_k] + log sum exp z),
//   dx_v = weight tau (softmax(z)_v - sum_{k: i_k = v} p_k) cap'(x_v),  cap'(x) = 1 - tanh(x / softcap)^2.
// Memory bound: the row is read once and the gradient written once. One workgroup per row.
#include "common.hpp"
#include "mfma.hpp"

namespace noise {
namespace {

constexpr int kThreads = 256;

struct DistillArgs {
    const void *x, *teacher, *index;
    const float *weight;
    float *loss;
    void *grad;
    int64_t vocab, stride, entries, width, grad_stride, first;
    int type, teacher_type, index_wide;
    float tau, cap;
};

__device__ __forceinline__ float load_any(const void *p, int type, int64_t i) {
    return type == NOISE_BF16 ? (float)static_cast<const __bf16 *>(p)[i] : static_cast<const float *>(p)[i];
}

// over the workgroup; every thread gets the result
template <class Op>
__device__ __forceinline__ float group_reduce(float v, Op op, float *shared) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = shared[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) r = op(r, shared[w]);
    return r;
}

__global__ __launch_bounds__(kThreads) void distill_kernel(DistillArgs a) {
    __shared__ float shared[kThreads / 64];
    const int64_t row = a.first + blockIdx.x;
    const int64_t xb = row * a.stride, tb = row * a.entries;
    const float inv_tau = 1.0f / a.tau;
    auto max2 = [](float p, float q) { return fmaxf(p, q); };
    auto add2 = [](float p, float q) { return p + q; };
    auto index_at = [&](int64_t k) {
        const int64_t i = a.index_wide ? static_cast<const int64_t *>(a.index)[tb + k]
                                       : (int64_t)static_cast<const int32_t *>(a.index)[tb + k];
        return i >= 0 && i < a.vocab ? i : -1;
    };
    auto capped = [&](int64_t i) {
        const float x = load_any(a.x, a.type, xb + i);
        return a.cap > 0.f ? a.cap * tanhf(x / a.cap) : x;
    };
    // the teacher
    float tm = -__builtin_inff();
    for (int64_t k = threadIdx.x; k < a.entries; k += kThreads)
        if (index_at(k) >= 0) tm = fmaxf(tm, load_any(a.teacher, a.teacher_type, tb + k) * inv_tau);
    tm = group_reduce(tm, max2, shared);
    const bool some = tm > -__builtin_inff() || tm != tm;
    float ts = 0.f;
    if (some)
        for (int64_t k = threadIdx.x; k < a.entries; k += kThreads)
            if (index_at(k) >= 0) ts += expf(load_any(a.teacher, a.teacher_type, tb + k) * inv_tau - tm);
    ts = group_reduce(ts, add2, shared);
    // the student
    float m = -__builtin_inff();
    for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) m = fmaxf(m, capped(j) * inv_tau);
    m = group_reduce(m, max2, shared);
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) s += expf(capped(j) * inv_tau - m);
    s = group_reduce(s, add2, shared);
    const float log_s = logf(s), log_ts = logf(ts);
    float loss = 0.f;
    if (some)
        for (int64_t k = threadIdx.x; k < a.entries; k += kThreads) {
            const int64_t i = index_at(k);
            if (i < 0) continue;
            const float t = load_any(a.teacher, a.teacher_type, tb + k) * inv_tau - tm, p = expf(t) / ts;
            if (p != 0.f) loss += p * (t - log_ts - (capped(i) * inv_tau - m - log_s));
        }
    loss = group_reduce(loss, add2, shared);
    if (threadIdx.x == 0) a.loss[row] = a.tau * a.tau * loss;
    if (!a.grad) return;
    const float scale = a.tau * (a.weight ? a.weight[row] : 1.f);
    for (int64_t j = threadIdx.x; j < a.width; j += kThreads) {
        float g = 0.f;
        if (j < a.vocab && some) {
            const float z = capped(j);
            g = expf(z * inv_tau - m) / s;
            for (int64_t k = 0; k < a.entries; ++k)
                if (index_at(k) == j) g -= expf(load_any(a.teacher, a.teacher_type, tb + k) * inv_tau - tm) / ts;
            g *= scale;
            if (a.cap > 0.f) g *= 1.f - (z / a.cap) * (z / a.cap);
        }
        if (a.type == NOISE_BF16)
            static_cast<__bf16 *>(a.grad)[row * a.grad_stride + j] = (__bf16)g;
        else
            static_cast<float *>(a.grad)[row * a.grad_stride + j] = g;
    }
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int noise_distill(const void *x, int type, int64_t rows, int64_t vocab, int64_t stride, const void *teacher,
                             int teacher_type, const void *index, int index_wide, int64_t entries, const float *weight,
                             float temperature, float softcap, float *loss, void *grad, int64_t width,
                             int64_t grad_stride, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_distill";
    NOISE_CHECK_ARG(type == NOISE_BF16 || type == NOISE_FP32, "%s: unknown type %d", fn, type);
    NOISE_CHECK_ARG(teacher_type == NOISE_BF16 || teacher_type == NOISE_FP32, "%s: unknown teacher type %d", fn, teacher_type);
    NOISE_CHECK_ARG(rows >= 0 && vocab > 0 && vocab <= (1 << 30) && entries > 0 && entries <= (1 << 20),
                    "%s: rows >= 0, vocab 1 .. 2^30 and entries 1 .. 2^20 required", fn);
    NOISE_CHECK_ARG(temperature > 0.f && temperature < __builtin_inff(), "%s: temperature must be positive", fn);
    NOISE_CHECK_ARG(softcap >= 0.f && softcap < __builtin_inff(), "%s: softcap must be positive, or 0 for none", fn);
    if (rows == 0) return NOISE_OK;
    NOISE_CHECK_ARG(x && teacher && index && loss, "%s: NULL pointer", fn);
    const size_t size = type == NOISE_BF16 ? 2 : 4;
    NOISE_CHECK_ARG(aligned(x, size) && aligned(teacher, teacher_type == NOISE_BF16 ? 2 : 4) &&
                        aligned(index, index_wide ? 8 : 4) && aligned(loss, 4) && aligned(weight, 4),
                    "%s: a pointer is not aligned to its type", fn);
    NOISE_CHECK_ARG(!grad || (aligned(grad, size) && width >= vocab && width <= (1 << 30) && grad_stride >= width),
                    "%s: grad needs vocab <= width <= grad_stride", fn);
    DistillArgs a;
    a.x = x; a.teacher = teacher; a.index = index; a.weight = weight; a.loss = loss; a.grad = grad;
    a.vocab = vocab; a.stride = stride; a.entries = entries; a.width = width; a.grad_stride = grad_stride;
    a.type = type; a.teacher_type = teacher_type; a.index_wide = index_wide; a.tau = temperature; a.cap = softcap;
    constexpr int64_t kLaunchGroups = 1 << 22;  // a launch has fewer than 2^32 threads
    for (a.first = 0; a.first < rows; a.first += kLaunchGroups) {
        const int64_t n = rows - a.first < kLaunchGroups ? rows - a.first : kLaunchGroups;
        hipLaunchKernelGGL(distill_kernel, dim3((unsigned)n), dim3(kThreads), 0, (hipStream_t)stream, a);
    }
    return launch_status(fn);
}
