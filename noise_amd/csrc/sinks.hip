// Attention with a sliding window and first tokens that stay visible: query i sees the keys j <= i with i - j <= W or j < n.
// The keys that a query sees are at most two runs, 0 .. n' - 1 and first .. last (first = max(0, i - W), n' = min(n, first)).
//
// One wave per query (forward, dq, decode) or per key (dk, dv); a lane takes a key (or query) of every 64 for the products
// over the head dimension, then dims lane, lane + 64 for the sums over keys.
#include "common.hpp"
#include "mfma.hpp"

namespace noise {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kFar = 1ll << 62;  // sums of a position and a window stay in 64 bits
constexpr int kGroup = 4;  // waves per workgroup

struct Rows {
    __bf16 *ptr;
    int64_t s_b, s_t, s_h;
};

struct SinkArgs {
    Rows q, k, v, o, d_o, dq, dk, dv;
    float *lse, *delta;
    const void *lengths, *start;   // [batch] int32 (int64 where wide)
    int64_t units, first;          // waves' units of work in all, this launch's first workgroup
    int64_t window, sinks;
    int wide, tokens, slots, heads, kv_heads;
    float scale;
};

__device__ __forceinline__ int64_t at_wide(const void *p, int wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
}

// keys of the sequence
__device__ __forceinline__ int seq_len(const SinkArgs &a, int64_t b) {
    if (!a.lengths) return a.slots;
    const int64_t n = at_wide(a.lengths, a.wide, b);
    return n < 0 ? 0 : n > a.slots ? a.slots : (int)n;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <int D>
__device__ __forceinline__ float dot(const float *q, const __bf16 *k) {
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < D; d += 8) {
        const bf16x8 x = load_bf16x8(k + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += q[d + e] * (float)x[e];
    }
    return s;
}

// the query's position and the keys that it sees: u < n -> key u < sunk ? u : u - sunk + lo
struct Seen {
    int sunk, lo, n;
};
__device__ __forceinline__ Seen seen_by(const SinkArgs &a, int64_t pos, int len) {
    Seen s{0, 0, 0};
    if (pos < 0 || len == 0) return s;
    const int64_t lo = pos > a.window ? pos - a.window : 0;
    const int64_t hi = pos < len ? pos + 1 : len;  // end
    s.lo = (int)(lo < len ? lo : len);
    s.sunk = (int)(a.sinks < s.lo ? a.sinks : s.lo);
    s.n = s.sunk + (hi > s.lo ? (int)hi - s.lo : 0);
    return s;
}

template <int D>
__global__ __launch_bounds__(64 * kGroup) void sink_fwd_kernel(SinkArgs a) {
    __shared__ float sq[kGroup][D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t unit = (a.first + blockIdx.x) * kGroup + wave;
    if (unit >= a.units) return;
    const int t = (int)(unit % a.tokens), h = (int)(unit / a.tokens % a.heads);
    const int64_t b = unit / a.tokens / a.heads;
    const int len = seq_len(a, b), hk = h / (a.heads / a.kv_heads);
    const int64_t pos = a.start ? at_wide(a.start, a.wide, b) + t : t < len ? t : -1;
    const __bf16 *q = a.q.ptr + b * a.q.s_b + t * a.q.s_t + h * a.q.s_h;
    for (int d = lane; d < D; d += 64) sq[wave][d] = (float)q[d] * a.scale * kLog2e;
    wave_lds_sync();
    const Seen seen = seen_by(a, pos, len);
    float m = -__builtin_inff(), l = 0.f, o[D / 64] = {};
    for (int u0 = 0; u0 < seen.n; u0 += 64) {
        const int u = u0 + lane, n = seen.n - u0 < 64 ? seen.n - u0 : 64;
        const int key = u < seen.sunk ? u : u - seen.sunk + seen.lo;
        float s = -__builtin_inff();
        if (u < seen.n) s = dot<D>(sq[wave], a.k.ptr + b * a.k.s_b + key * a.k.s_t + hk * a.k.s_h);
        const float mn = fmaxf(m, wave_max(s)), alpha = mn == -__builtin_inff() ? 1.f : exp2f(m - mn);
        const float p = u < seen.n && mn > -__builtin_inff() ? exp2f(s - mn) : 0.f;
        m = mn;
        l = l * alpha + wave_sum(p);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) o[i] *= alpha;
        for (int e = 0; e < n; ++e) {
            const float pe = __shfl(p, e, 64);
            const int64_t ke = u0 + e < seen.sunk ? u0 + e : u0 + e - seen.sunk + seen.lo;
            const __bf16 *v = a.v.ptr + b * a.v.s_b + ke * a.v.s_t + hk * a.v.s_h;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) o[i] += pe * (float)v[lane + 64 * i];
        }
    }
    __bf16 *out = a.o.ptr + b * a.o.s_b + t * a.o.s_t + h * a.o.s_h;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) out[lane + 64 * i] = (__bf16)(seen.n ? o[i] / l : 0.f);
    if (a.lse && lane == 0 && seen.n) a.lse[(b * a.heads + h) * a.tokens + t] = m + log2f(l);
}

// dq, and delta = sum_d dO o for the next kernel
template <int D>
__global__ __launch_bounds__(64 * kGroup) void sink_dq_kernel(SinkArgs a) {
    __shared__ float sq[kGroup][D], sd[kGroup][D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t unit = (a.first + blockIdx.x) * kGroup + wave;
    if (unit >= a.units) return;
    const int t = (int)(unit % a.tokens), h = (int)(unit / a.tokens % a.heads);
    const int64_t b = unit / a.tokens / a.heads;
    const int len = seq_len(a, b), hk = h / (a.heads / a.kv_heads);
    const Seen seen = seen_by(a, t < len ? t : -1, len);
    const __bf16 *q = a.q.ptr + b * a.q.s_b + t * a.q.s_t + h * a.q.s_h;
    const __bf16 *o = a.o.ptr + b * a.o.s_b + t * a.o.s_t + h * a.o.s_h;
    const __bf16 *d_o = a.d_o.ptr + b * a.d_o.s_b + t * a.d_o.s_t + h * a.d_o.s_h;
    float delta = 0.f, dq[D / 64] = {};
    for (int d = lane; d < D; d += 64) {
        sq[wave][d] = (float)q[d] * a.scale * kLog2e;
        sd[wave][d] = (float)d_o[d];
        delta += (float)o[d] * (float)d_o[d];
    }
    delta = wave_sum(delta);
    wave_lds_sync();
    const int64_t li = (b * a.heads + h) * a.tokens + t;
    const float lse = seen.n ? a.lse[li] : 0.f;
    if (lane == 0) a.delta[li] = delta;
    for (int u0 = 0; u0 < seen.n; u0 += 64) {
        const int u = u0 + lane, n = seen.n - u0 < 64 ? seen.n - u0 : 64;
        const int64_t key = u < seen.sunk ? u : u - seen.sunk + seen.lo;
        float ds = 0.f;
        if (u < seen.n)
            ds = exp2f(dot<D>(sq[wave], a.k.ptr + b * a.k.s_b + key * a.k.s_t + hk * a.k.s_h) - lse) *
                 (dot<D>(sd[wave], a.v.ptr + b * a.v.s_b + key * a.v.s_t + hk * a.v.s_h) - delta);
        for (int e = 0; e < n; ++e) {
            const float de = __shfl(ds, e, 64);
            const int64_t ke = u0 + e < seen.sunk ? u0 + e : u0 + e - seen.sunk + seen.lo;
            const __bf16 *k = a.k.ptr + b * a.k.s_b + ke * a.k.s_t + hk * a.k.s_h;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) dq[i] += de * (float)k[lane + 64 * i];
        }
    }
    __bf16 *out = a.dq.ptr + b * a.dq.s_b + t * a.dq.s_t + h * a.dq.s_h;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) out[lane + 64 * i] = (__bf16)(dq[i] * a.scale);
}

template <int D>
__global__ __launch_bounds__(64 * kGroup) void sink_dkv_kernel(SinkArgs a) {
    __shared__ float sk[kGroup][D], sv[kGroup][D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t unit = (a.first + blockIdx.x) * kGroup + wave;
    if (unit >= a.units) return;
    const int j = (int)(unit % a.tokens), hk = (int)(unit / a.tokens % a.kv_heads);
    const int64_t b = unit / a.tokens / a.kv_heads;
    const int len = seq_len(a, b), G = a.heads / a.kv_heads;
    const __bf16 *k = a.k.ptr + b * a.k.s_b + j * a.k.s_t + hk * a.k.s_h;
    const __bf16 *v = a.v.ptr + b * a.v.s_b + j * a.v.s_t + hk * a.v.s_h;
    for (int d = lane; d < D; d += 64) {
        sk[wave][d] = (float)k[d] * a.scale * kLog2e;
        sv[wave][d] = (float)v[d];
    }
    wave_lds_sync();
    float dk[D / 64] = {}, dv[D / 64] = {};
    const int64_t last = j < a.sinks ? len : (int64_t)j + a.window + 1;
    const int end = j < len ? (int)(last < len ? last : len) : j;
    for (int g = 0; g < G; ++g) {
        const int h = hk * G + g;
        const int64_t li = (b * a.heads + h) * a.tokens;
        for (int i0 = j; i0 < end; i0 += 64) {
            const int i = i0 + lane, n = end - i0 < 64 ? end - i0 : 64;
            float p = 0.f, ds = 0.f;
            if (i < end) {
                p = exp2f(dot<D>(sk[wave], a.q.ptr + b * a.q.s_b + i * a.q.s_t + h * a.q.s_h) - a.lse[li + i]);
                ds = p * (dot<D>(sv[wave], a.d_o.ptr + b * a.d_o.s_b + i * a.d_o.s_t + h * a.d_o.s_h) - a.delta[li + i]);
            }
            for (int e = 0; e < n; ++e) {
                const float pe = __shfl(p, e, 64), de = __shfl(ds, e, 64);
                const __bf16 *q = a.q.ptr + b * a.q.s_b + (int64_t)(i0 + e) * a.q.s_t + h * a.q.s_h;
                const __bf16 *d_o = a.d_o.ptr + b * a.d_o.s_b + (int64_t)(i0 + e) * a.d_o.s_t + h * a.d_o.s_h;
#pragma unroll
                for (int x = 0; x < D / 64; ++x) {
                    dv[x] += pe * (float)d_o[lane + 64 * x];
                    dk[x] += de * (float)q[lane + 64 * x];
                }
            }
        }
    }
    __bf16 *ok = a.dk.ptr + b * a.dk.s_b + j * a.dk.s_t + hk * a.dk.s_h;
    __bf16 *ov = a.dv.ptr + b * a.dv.s_b + j * a.dv.s_t + hk * a.dv.s_h;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
        ok[lane + 64 * x] = (__bf16)(dk[x] * a.scale);
        ov[lane + 64 * x] = (__bf16)dv[x];
    }
}

int check_heads(const char *fn, const char *name, const noise_heads_t *h, Rows *out) {
    NOISE_CHECK_ARG(h && h->ptr && aligned(h->ptr, 16), "%s: %s NULL or not 16 B aligned", fn, name);
    NOISE_CHECK_ARG(h->s_b % 8 == 0 && h->s_t % 8 == 0 && h->s_h % 8 == 0, "%s: %s strides must be multiples of 8", fn, name);
    *out = Rows{static_cast<__bf16 *>(h->ptr), h->s_b, h->s_t, h->s_h};
    return NOISE_OK;
}

int check_sizes(const char *fn, int64_t batch, int64_t tokens, int64_t slots, int64_t heads, int64_t kv_heads,
                int64_t head_dim, int64_t window, int64_t sinks) {
    NOISE_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128, got %lld", fn, (long long)head_dim);
    NOISE_CHECK_ARG(batch >= 0 && tokens >= 0 && tokens <= (1 << 30) && slots >= 0 && slots <= (1 << 30),
                    "%s: bad batch/tokens/capacity", fn);
    NOISE_CHECK_ARG(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= (1 << 16),
                    "%s: %lld query heads for %lld key heads", fn, (long long)heads, (long long)kv_heads);
    NOISE_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window and sinks must not be negative", fn);
    NOISE_CHECK_ARG(tokens == 0 || batch * heads <= INT64_MAX / 64 / tokens, "%s: too many rows", fn);
    return NOISE_OK;
}

void fill_args(SinkArgs *a, const void *lengths, const void *start, int wide, int64_t tokens, int64_t slots,
               int64_t heads, int64_t kv_heads, int64_t window, int64_t sinks, float scale) {
    a->lengths = lengths; a->start = start; a->wide = wide;
    a->tokens = (int)tokens; a->slots = (int)slots; a->heads = (int)heads; a->kv_heads = (int)kv_heads;
    a->window = window < kFar ? window : kFar;
    a->sinks = sinks < kFar ? sinks : kFar;
    a->scale = scale;
    a->lse = a->delta = nullptr;
}

constexpr int64_t kLaunchGroups = 1 << 22;  // a launch has fewer than 2^32 threads

int launch_units(void (*kernel)(SinkArgs), SinkArgs &a, int64_t units, hipStream_t stream, const char *fn) {
    a.units = units;
    const int64_t groups = (units + kGroup - 1) / kGroup;
    for (a.first = 0; a.first < groups; a.first += kLaunchGroups) {
        const int64_t n = groups - a.first < kLaunchGroups ? groups - a.first : kLaunchGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(64 * kGroup), 0, stream, a);
    }
    return launch_status(fn);
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int64_t noise_sink_decode_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                     int64_t capacity, int64_t head_dim, int64_t window,
                                                     int64_t sinks) {
    clear_error();
    const int st = check_sizes("noise_sink_decode_workspace_bytes", batch, tokens, capacity, heads, kv_heads, head_dim,
                               window, sinks);
    if (st) return st;
    return 0;
}

extern "C" int noise_sink_decode(const noise_heads_t *q, const noise_heads_t *k, const noise_heads_t *v,
                                 const noise_heads_t *o, const void *start, int start_wide, int64_t batch,
                                 int64_t tokens, int64_t capacity, int64_t head_dim, int64_t window, int64_t sinks,
                                 float scale, void *workspace, int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_sink_decode";
    NOISE_CHECK_ARG(q && k && v && o && q->heads == o->heads && k->heads == v->heads, "%s: tensors missing or of other heads", fn);
    int st = check_sizes(fn, batch, tokens, capacity, q->heads, k->heads, head_dim, window, sinks);
    if (st) return st;
    NOISE_CHECK_ARG(tokens <= 16, "%s: at most 16 new tokens, got %lld", fn, (long long)tokens);
    if (batch == 0 || tokens == 0) return NOISE_OK;
    NOISE_CHECK_ARG(start && aligned(start, start_wide ? 8 : 4), "%s: start is required", fn);
    (void)workspace; (void)workspace_bytes;
    SinkArgs a;
    if ((st = check_heads(fn, "q", q, &a.q)) || (st = check_heads(fn, "k", k, &a.k)) ||
        (st = check_heads(fn, "v", v, &a.v)) || (st = check_heads(fn, "o", o, &a.o)))
        return st;
    fill_args(&a, nullptr, start, start_wide, tokens, capacity, q->heads, k->heads, window, sinks, scale);
    return launch_units(head_dim == 64 ? sink_fwd_kernel<64> : sink_fwd_kernel<128>, a, batch * q->heads * tokens,
                        (hipStream_t)stream, fn);
}
