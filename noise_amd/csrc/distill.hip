// Distillation from a teacher's top logits, forward and backward: per row of logits x, with z = cap(x) / tau and the teacher's
// softmax p over its entries in use,
//   loss = tau^2 sum_k p_k (log p_k - z[i_k] + log sum exp z),
//   dx_v = weight tau (softmax(z)_v - sum_{k: i_k = v} p_k) cap'(x_v),  cap'(x) = 1 - tanh(x / softcap)^2.
// Memory bound: a workgroup takes a row, reads it once into registers (16 B of consecutive elements per thread and step), and
// takes the maximum, the sum, the loss and the gradient from there. Rows past 393 KB do not fit; they are read twice.
// The teacher's entries go through LDS. Their terms reach the gradient last: an entry's thread writes the whole gradient of
// its index over what the row's pass left there (summing the entries that share the index, so that they write the same: it
// compares its index with all others, work that grows with their square).
//
// 16384 fp32 rows of 4096 soft-capped logits, 64 entries, loss and gradient: 122 us (545 MB, 4.5 TB/s, where a large copy runs at
// 4.9); 4096 bf16 rows of 65536: 251 us (1.08 GB, 4.3 TB/s; 512 threads with twice the chunks 258; streaming stores 242, but
// 136 us for the former). The loss alone of 100 bf16 rows of 4000: 4.9 us. With more entries (another run) the former
// 135 us at 64, 153 at 128, 221 at 256, 572 at 512 and 2027 at 1024, where the comparisons are all there is (the
// loss alone 74, 72, 81, 91, 127); the latter, soft-capped, 412, 429, 475, 610 and 900.
#include "common.hpp"
#include "mfma.hpp"

namespace noise {
namespace {

constexpr int kMaxEntries = 1024;

struct DistillArgs {
    const void *x, *teacher, *index;
    const float *weight;
    float *loss;
    void *grad;
    int64_t stride, grad_stride, first;
    int vocab, width, entries;
    int teacher_type, index_wide;
    float tau, cap;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 B of consecutive elements at any address of their type
template <class E>
struct Chunk {
    static constexpr int N = 16 / sizeof(E);
    u32x4 v;
    __device__ __forceinline__ void load(const E *p) { __builtin_memcpy(&v, p, 16); }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(E) == 4) return __uint_as_float(v[i]);
        return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
    }
};
template <class E>
__device__ __forceinline__ void store_chunk(E *p, const float (&g)[16 / sizeof(E)]) {
    E out[16 / sizeof(E)];
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(E)); ++i) out[i] = (E)g[i];
    __builtin_memcpy(p, out, 16);
}

// tanh: its odd series up to y^11 below 0.35 (the next term is 1.2e-8 of the value there), 1 - 2 / (e^2y + 1) above (8 roundings
// of the quotient, which is below 2/3). Compared with the device library's, half the instructions.
__device__ __forceinline__ float tanh_of(float y) {
    const float a = fabsf(y), s = a * a;
    float p = __builtin_fmaf(s, -1382.f / 155925.f, 62.f / 2835.f);
    p = __builtin_fmaf(s, p, -17.f / 315.f);
    p = __builtin_fmaf(s, p, 2.f / 15.f);
    p = __builtin_fmaf(s, p, -1.f / 3.f);
    const float near = __builtin_fmaf(a * s, p, a);
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(exp2_fast(a * 2.885390081777927f) + 1.f);
    return copysignf(a < 0.35f ? near : far, y);
}

// The larger of two, or NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

// Both values over the workgroup, every thread gets the results. Each call has its own `slots` (2 per wave): one barrier.
template <int NT, class F, class G>
__device__ __forceinline__ void reduce2(float &a, float &b, F f, G g, float *slots) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a = f(a, __shfl_xor(a, o, 64));
        b = g(b, __shfl_xor(b, o, 64));
    }
    constexpr int NW = NT / 64;
    if ((threadIdx.x & 63) == 0) {
        slots[threadIdx.x >> 6] = a;
        slots[NW + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = slots[0], b = slots[NW];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
        a = f(a, slots[w]);
        b = g(b, slots[NW + w]);
    }
}

// NT threads, C chunks each (0: rows of any length, read twice)
template <class E, int NT, int C, bool CAP>
__global__ __launch_bounds__(NT, NT == 1024 && C == 8 ? 8 : 4) void distill_kernel(DistillArgs a) {
    constexpr int N = Chunk<E>::N;
    __shared__ int s_index[kMaxEntries];
    __shared__ float s_t[kMaxEntries], s_x[kMaxEntries], slots[3][2 * NT / 64];
    const int64_t row = a.first + blockIdx.x;
    const int tid = threadIdx.x, chunks = a.vocab / N, tail = a.vocab - chunks * N;
    const E *x = static_cast<const E *>(a.x) + row * a.stride;
    const float c = 1.4426950408889634f / a.tau, inv_tau = 1.f / a.tau, inv_cap = CAP ? 1.f / a.cap : 0.f;
    auto capped = [&](float v) { return CAP ? a.cap * tanh_of(v * inv_cap) : v; };
    // the row, and its last elements past the chunks, one per thread
    Chunk<E> ch[C > 0 ? C : 1];
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (tid + i * NT < chunks) ch[i].load(x + (int64_t)(tid + i * NT) * N);
    }
    float rest = tid < tail ? (float)x[chunks * N + tid] : -__builtin_inff();
    // the teacher: the entries in use
    float tm = -__builtin_inff();
    const int64_t tb = row * a.entries;
    for (int k = tid; k < a.entries; k += NT) {
        const int64_t i = a.index_wide ? static_cast<const int64_t *>(a.index)[tb + k]
                                       : (int64_t)static_cast<const int32_t *>(a.index)[tb + k];
        const float t = a.teacher_type == NOISE_BF16 ? (float)static_cast<const __bf16 *>(a.teacher)[tb + k]
                                                     : static_cast<const float *>(a.teacher)[tb + k];
        const bool used = i >= 0 && i < a.vocab && !(t == -__builtin_inff());
        s_index[k] = used ? (int)i : -1;
        s_t[k] = t;
        s_x[k] = used ? (float)x[i] : 0.f;
        if (used) tm = max_nan(tm, t);
    }
    // the row's maximum (of the uncapped values: the cap keeps their order), with fp32 rows capped in place
    float m = rest, s = 0.f;
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (tid + i * NT < chunks) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    m = fmaxf(m, ch[i].get(e));
                    if constexpr (CAP && sizeof(E) == 4) ch[i].v[e] = __float_as_uint(capped(ch[i].get(e)));
                }
            }
    } else {
        for (int i = tid; i < chunks; i += NT) {
            Chunk<E> t;
            t.load(x + (int64_t)i * N);
            float top = t.get(0);
#pragma unroll
            for (int e = 1; e < N; ++e) top = fmaxf(top, t.get(e));
            // Under the cap -inf is a value like others, -softcap, and so is a maximum of it. Without one, a thread that has met
            // nothing but -inf and NaN holds 0 or, for good, NaN in s.
            const bool counts = CAP || m > -__builtin_inff();
            if (top > m) {
                if (counts) s *= exp2_fast((capped(m) - capped(top)) * c);
                m = top;
            }
            const float at = capped(m);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float v = t.get(e);
                s += CAP || m > -__builtin_inff() ? exp2_fast((capped(v) - at) * c) : v != v ? v : 0.f;
            }
        }
    }
    const float m_own = m;
    auto max2 = [](float p, float q) { return fmaxf(p, q); };
    auto add2 = [](float p, float q) { return p + q; };
    reduce2<NT>(m, tm, max2, max_nan, slots[0]);
    const float top = capped(m);
    rest = tid < tail ? (capped(rest) - top) * c : -__builtin_inff();
    auto value = [&](const Chunk<E> &t, int e) {   // the exponent (log2) of an element
        return ((CAP && (sizeof(E) == 2 || C == 0) ? capped(t.get(e)) : t.get(e)) - top) * c;
    };
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (tid + i * NT < chunks) {
#pragma unroll
                for (int e = 0; e < N; ++e) s += exp2_fast(value(ch[i], e));
            }
    } else if (s != 0.f) {
        s *= exp2_fast((capped(m_own) - top) * c);
    }
    if (C > 0 || tid < tail) s += exp2_fast(rest);
    const bool some = !(tm == -__builtin_inff());
    float ts = 0.f;
    if (some)
        for (int k = tid; k < a.entries; k += NT)
            if (s_index[k] >= 0) ts += exp2_fast((s_t[k] - tm) * c);
    reduce2<NT>(s, ts, add2, add2, slots[1]);
    const float inv_s = 1.f / s, log_s = logf(s), log_ts = logf(ts), inv_ts = 1.f / ts;
    float loss = 0.f, none = 0.f;
    if (some)
        for (int k = tid; k < a.entries; k += NT)
            if (s_index[k] >= 0) {
                const float p = exp2_fast((s_t[k] - tm) * c) * inv_ts;
                if (p != 0.f) loss += p * ((s_t[k] - tm) * inv_tau - log_ts - ((capped(s_x[k]) - top) * inv_tau - log_s));
                s_t[k] = p;   // (read by the other threads after the barrier below)
            }
    reduce2<NT>(loss, none, add2, add2, slots[2]);
    if (tid == 0) a.loss[row] = a.tau * a.tau * loss;
    if (!a.grad) return;

    E *grad = static_cast<E *>(a.grad) + row * a.grad_stride;
    const float scale = some ? a.tau * (a.weight ? a.weight[row] : 1.f) : 0.f;
    // of the softmax's part q at a capped value z: (scale q) cap'
    auto slope = [&](float z) { return CAP ? 1.f - (z * inv_cap) * (z * inv_cap) : 1.f; };
    const float qs = some ? scale * inv_s : 0.f;
    auto chunk_grad = [&](const Chunk<E> &t, int i) {
        float g[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float z = CAP && (sizeof(E) == 2 || C == 0) ? capped(t.get(e)) : t.get(e);
            g[e] = some ? qs * exp2_fast((z - top) * c) * slope(z) : 0.f;
        }
        store_chunk<E>(grad + (int64_t)i * N, g);
    };
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (tid + i * NT < chunks) chunk_grad(ch[i], tid + i * NT);
    } else {
        for (int i = tid; i < chunks; i += NT) {
            Chunk<E> t;
            t.load(x + (int64_t)i * N);
            chunk_grad(t, i);
        }
    }
    if (tid < tail) {
        const float z = capped((float)x[chunks * N + tid]);
        grad[chunks * N + tid] = (E)(some ? qs * exp2_fast(rest) * slope(z) : 0.f);
    }
    for (int j = a.vocab + tid; j < a.width; j += NT) grad[j] = (E)0.f;
    if (!some) return;
    __syncthreads();   // the row's stores before the entries'
    for (int k = tid; k < a.entries; k += NT) {
        const int i = s_index[k];
        if (i < 0) continue;
        float p = 0.f;
        for (int o = 0; o < a.entries; ++o) p += s_index[o] == i ? s_t[o] : 0.f;
        const float z = capped(s_x[k]);
        grad[i] = (E)(scale * (exp2_fast((z - top) * c) * inv_s - p) * slope(z));
    }
}

template <class E, bool CAP>
void (*pick(int64_t vocab, int *threads))(DistillArgs) {
    const int64_t chunks = vocab / Chunk<E>::N;
    *threads = chunks <= 1024 ? 256 : chunks <= 4096 ? 512 : 1024;
    return chunks <= 256     ? distill_kernel<E, 256, 1, CAP>
           : chunks <= 1024  ? distill_kernel<E, 256, 4, CAP>
           : chunks <= 4096  ? distill_kernel<E, 512, 8, CAP>
           : chunks <= 8192  ? distill_kernel<E, 1024, 8, CAP>
           : chunks <= 24576 ? distill_kernel<E, 1024, 24, CAP>
                             : distill_kernel<E, 1024, 0, CAP>;
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
    NOISE_CHECK_ARG(rows >= 0 && vocab > 0 && vocab <= (1 << 30) && entries > 0 && entries <= kMaxEntries,
                    "%s: rows >= 0, vocab 1 .. 2^30 and entries 1 .. %d required", fn, kMaxEntries);
    NOISE_CHECK_ARG(temperature >= 1e-6f && temperature <= 1e6f, "%s: temperature must be 1e-6 .. 1e6", fn);
    NOISE_CHECK_ARG(softcap == 0.f || (softcap >= 1e-6f && softcap <= 1e6f), "%s: softcap must be 1e-6 .. 1e6, or 0 for none", fn);
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
    a.vocab = (int)vocab; a.stride = stride; a.entries = (int)entries; a.width = (int)width; a.grad_stride = grad_stride;
    a.teacher_type = teacher_type; a.index_wide = index_wide; a.tau = temperature; a.cap = softcap;
    int threads;
    auto kernel = type == NOISE_BF16 ? (softcap > 0.f ? pick<__bf16, true>(vocab, &threads) : pick<__bf16, false>(vocab, &threads))
                                     : (softcap > 0.f ? pick<float, true>(vocab, &threads) : pick<float, false>(vocab, &threads));
    constexpr int64_t kLaunchGroups = 1 << 21;  // a launch has fewer than 2^32 threads
    for (a.first = 0; a.first < rows; a.first += kLaunchGroups) {
        const int64_t n = rows - a.first < kLaunchGroups ? rows - a.first : kLaunchGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads), 0, (hipStream_t)stream, a);
    }
    return launch_status(fn);
}
