// Norm of every head's queries and keys with the rotation in the same pass, its gradients, and its serving form that puts
// keys and values into a cache (utils/model.py:46-47, 55-58, 88-94, with learned weights and positions as options).
//
// A row of D elements is held by D / 16 lanes, each with 8 consecutive elements of either half (16 B loads), so that the
// rotation's pairs stay in a lane and the sum of squares needs log2(D / 16) exchanges. Rows are numbered token by token,
// heads innermost: neighbouring lanes read neighbouring memory, and all of a wave's rows share a few table rows.
// Memory bound: every element is read and written once (backward: two reads, one write). 8 x 2048 tokens, 8 + 8 heads of 64, bf16:
// 16 us forward (67 MB, 4.2 TB/s) and 20 us backward (101 MB, 5.1 TB/s; 3.8 us for the weights' sums); 16 prompts of 1500
// tokens, 32 + 8 heads of 128, into their cache: 124 us (591 MB, 4.8 TB/s). A large copy runs at 4.9 TB/s here.
#include "common.hpp"
#include "mfma.hpp"

namespace noise {
namespace {

constexpr int kThreads = 256;
constexpr int kPartials = 512;   // rows of partial weight gradients per tensor
constexpr int64_t kLaunchGroups = 1 << 22;  // a launch has fewer than 2^32 threads

struct Rows {
    void *ptr;
    int64_t s_b, s_t, s_h;
};

struct NormArgs {
    Rows x[2], y[2], v, v_out;     // backward: x, dy (y), and dx (v: of the queries, v_out: of the keys)
    const float *w[2];
    const float *cos, *sin;
    const void *start;
    float *partial;                // [2][kPartials][D]
    int64_t table_rows, capacity;
    int64_t first;                 // this launch's first workgroup
    uint32_t rows, tokens, heads[2], row_heads;  // row_heads: rows per token
    int start_wide, blocks;
    float eps;
};

__device__ __forceinline__ void load8(const float *p, float (&o)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
}
__device__ __forceinline__ void load8(const __bf16 *p, float (&o)[8]) {
    const bf16x8 v = load_bf16x8(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (float)v[e];
}
__device__ __forceinline__ void store8(float *p, const float (&o)[8]) {
    *reinterpret_cast<float4 *>(p) = float4{o[0], o[1], o[2], o[3]};
    *reinterpret_cast<float4 *>(p + 4) = float4{o[4], o[5], o[6], o[7]};
}
__device__ __forceinline__ void store8(__bf16 *p, const float (&o)[8]) {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (__bf16)o[e];
    store_bf16x8(p, v);
}

// sum over the LPR lanes of a row
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// (in unsigned numbers: a start near the end of its type wraps to a negative position, which is outside any table)
__device__ __forceinline__ int64_t position(const NormArgs &a, uint32_t b, uint32_t t) {
    if (!a.start) return t;
    const int64_t first = a.start_wide ? static_cast<const int64_t *>(a.start)[b] : (int64_t)static_cast<const int32_t *>(a.start)[b];
    return (int64_t)((uint64_t)first + t);
}

template <class E, int D>
__global__ __launch_bounds__(kThreads) void head_norm_kernel(NormArgs a) {
    constexpr int LPR = D / 16, kRows = kThreads / LPR, h2 = D / 2;
    const int64_t at = (a.first + blockIdx.x) * kRows + threadIdx.x / LPR;
    if (at >= a.rows) return;
    const uint32_t row = (uint32_t)at, c = 8 * (threadIdx.x % LPR);
    const uint32_t bt = row / a.row_heads, hh = row - bt * a.row_heads, b = bt / a.tokens, t = bt - b * a.tokens;
    const int64_t pos = position(a, b, t);
    const bool live = pos >= 0 && pos < a.table_rows && (a.capacity == 0 || pos < a.capacity);
    const int i = hh < a.heads[0] ? 0 : hh < a.heads[0] + a.heads[1] ? 1 : 2;
    const uint32_t h = i == 0 ? hh : i == 1 ? hh - a.heads[0] : hh - a.heads[0] - a.heads[1];
    // keys and values of a cache stand at their position and are not written without one
    if (i > 0 && a.capacity && !live) return;
    const int64_t to = i > 0 && a.capacity ? pos : t;
    if (i == 2) {
        const E *s = static_cast<const E *>(a.v.ptr) + b * a.v.s_b + t * a.v.s_t + h * a.v.s_h + c;
        E *d = static_cast<E *>(a.v_out.ptr) + b * a.v_out.s_b + to * a.v_out.s_t + h * a.v_out.s_h + c;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // the bits themselves, NaN payloads included
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int q = 0; q < (int)sizeof(E) / 2; ++q)
                reinterpret_cast<u32x4 *>(d + e * h2)[q] = reinterpret_cast<const u32x4 *>(s + e * h2)[q];
        }
        return;
    }
    const E *x = static_cast<const E *>(a.x[i].ptr) + b * a.x[i].s_b + t * a.x[i].s_t + h * a.x[i].s_h + c;
    E *y = static_cast<E *>(a.y[i].ptr) + b * a.y[i].s_b + to * a.y[i].s_t + h * a.y[i].s_h + c;
    float u[2][8];
    if (!live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[0][e] = 0.f;
        store8(y, u[0]);
        store8(y + h2, u[0]);
        return;
    }
    load8(x, u[0]);
    load8(x + h2, u[1]);
    float cs[8], sn[8];
    load8(a.cos + pos * h2 + c, cs);
    load8(a.sin + pos * h2 + c, sn);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += u[0][e] * u[0][e] + u[1][e] * u[1][e];
    const float r = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + a.eps);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[p][e] *= r;
        if (a.w[i]) {
            float w[8];
            load8(a.w[i] + p * h2 + c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[p][e] *= w[e];
        }
    }
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = u[0][e] * cs[e] + u[1][e] * sn[e];
    store8(y, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = u[1][e] * cs[e] - u[0][e] * sn[e];
    store8(y + h2, o);
}

// blockIdx.y: queries or keys. A workgroup takes every blocks-th batch of rows, so that its sums of the weights' gradients
// stay in registers until the end.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void head_norm_bwd_kernel(NormArgs a) {
    constexpr int LPR = D / 16, kRows = kThreads / LPR, h2 = D / 2;
    const int i = blockIdx.y;
    const uint32_t rows = a.rows / a.row_heads * a.heads[i], c = 8 * (threadIdx.x % LPR);
    const Rows &dst = i ? a.v_out : a.v;
    float w[2][8], dw[2][8];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[p][e] = a.w[i] ? a.w[i][p * h2 + c + e] : 1.f;
            dw[p][e] = 0.f;
        }
    for (int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / LPR; at < rows; at += (int64_t)a.blocks * kRows) {
        const uint32_t row = (uint32_t)at, bt = row / a.heads[i], h = row - bt * a.heads[i], b = bt / a.tokens,
                       t = bt - b * a.tokens;
        const int64_t pos = position(a, b, t);
        E *dx = static_cast<E *>(dst.ptr) + b * dst.s_b + t * dst.s_t + h * dst.s_h + c;
        float n[2][8], g[2][8];
        if (pos < 0 || pos >= a.table_rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[0][e] = 0.f;
            store8(dx, g[0]);
            store8(dx + h2, g[0]);
            continue;
        }
        const E *x = static_cast<const E *>(a.x[i].ptr) + b * a.x[i].s_b + t * a.x[i].s_t + h * a.x[i].s_h + c;
        const E *dy = static_cast<const E *>(a.y[i].ptr) + b * a.y[i].s_b + t * a.y[i].s_t + h * a.y[i].s_h + c;
        float cs[8], sn[8], d0[8], d1[8];
        load8(x, n[0]);
        load8(x + h2, n[1]);
        load8(dy, d0);
        load8(dy + h2, d1);
        load8(a.cos + pos * h2 + c, cs);
        load8(a.sin + pos * h2 + c, sn);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += n[0][e] * n[0][e] + n[1][e] * n[1][e];
        const float r = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + a.eps);
        float gn = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g[0][e] = d0[e] * cs[e] - d1[e] * sn[e];
            g[1][e] = d0[e] * sn[e] + d1[e] * cs[e];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                n[p][e] *= r;
                dw[p][e] += g[p][e] * n[p][e];
                g[p][e] *= w[p][e];
                gn += g[p][e] * n[p][e];
            }
        }
        gn = row_sum<LPR>(gn) * (1.0f / D);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[p][e] = r * (g[p][e] - n[p][e] * gn);
            store8(dx + p * h2, g[p]);
        }
    }
    if (!a.w[i]) return;
    __shared__ float sum[kRows][D + 1];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[threadIdx.x / LPR][p * h2 + c + e] = dw[p][e];
    __syncthreads();
    if (threadIdx.x < D) {
        float s = 0.f;
        for (int k = 0; k < kRows; ++k) s += sum[k][threadIdx.x];
        a.partial[((int64_t)i * kPartials + blockIdx.x) * D + threadIdx.x] = s;
    }
}

// dw[i] = the sum of its partial rows: a workgroup per 16 columns, 64 rows at a time
__global__ __launch_bounds__(1024) void head_norm_dw_kernel(const float *partial, float *dw0, float *dw1, int blocks, int D) {
    float *out = blockIdx.y ? dw1 : dw0;
    if (!out) return;
    __shared__ float sum[16][16];
    const int col = threadIdx.x & 15, wave = threadIdx.x >> 6;
    const float *p = partial + (int64_t)blockIdx.y * kPartials * D + 16 * blockIdx.x + col;
    float s = 0.f;
#pragma unroll 8
    for (int k = threadIdx.x >> 4; k < blocks; k += 64) s += p[(int64_t)k * D];
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if ((threadIdx.x & 63) < 16) sum[wave][col] = s;
    __syncthreads();
    if (threadIdx.x < 16) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += sum[w][col];
        out[16 * blockIdx.x + col] = s;
    }
}

// a tensor's strides and alignment for rows of 16 B accesses
int check_rows(const char *fn, const char *name, const noise_heads_t &h, int type, Rows *out) {
    const int64_t unit = type == NOISE_FP32 ? 4 : 8;
    NOISE_CHECK_ARG(h.ptr && aligned(h.ptr, 16), "%s: %s NULL or not 16 B aligned", fn, name);
    NOISE_CHECK_ARG(h.s_b % unit == 0 && h.s_t % unit == 0 && h.s_h % unit == 0,
                    "%s: %s strides must be multiples of %lld elements", fn, name, (long long)unit);
    *out = Rows{h.ptr, h.s_b, h.s_t, h.s_h};
    return NOISE_OK;
}

int check_norm(const char *fn, const noise_heads_t *x, const noise_heads_t *y, const float *const *w,
               const float *rope_cos, const float *rope_sin, int64_t table_rows, const void *start, int start_wide,
               int64_t batch, int64_t tokens, int64_t head_dim, int type, float eps, NormArgs *a) {
    NOISE_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128, got %lld", fn, (long long)head_dim);
    NOISE_CHECK_ARG(type == NOISE_BF16 || type == NOISE_FP32, "%s: unknown type %d", fn, type);
    NOISE_CHECK_ARG(x && y && w, "%s: NULL tensor table", fn);
    NOISE_CHECK_ARG(batch >= 0 && tokens >= 0 && x[0].heads > 0 && x[1].heads > 0 && x[0].heads < (1 << 20) &&
                        x[1].heads < (1 << 20), "%s: bad batch/tokens/heads", fn);
    NOISE_CHECK_ARG(y[0].heads == x[0].heads && y[1].heads == x[1].heads, "%s: x and y heads differ", fn);
    NOISE_CHECK_ARG(rope_cos && rope_sin && aligned(rope_cos, 16) && aligned(rope_sin, 16) && table_rows > 0,
                    "%s: rotation tables NULL, empty or not 16 B aligned", fn);
    NOISE_CHECK_ARG(start || tokens <= table_rows, "%s: %lld tokens but tables of %lld rows", fn, (long long)tokens,
                    (long long)table_rows);
    NOISE_CHECK_ARG(!start || aligned(start, start_wide ? 8 : 4), "%s: start misaligned", fn);
    NOISE_CHECK_ARG(eps >= 0.f, "%s: eps must not be negative", fn);
    for (int i = 0; i < 2; ++i) {
        NOISE_CHECK_ARG(!w[i] || aligned(w[i], 16), "%s: weights not 16 B aligned", fn);
        a->w[i] = w[i];
        a->heads[i] = (uint32_t)x[i].heads;
    }
    a->cos = rope_cos; a->sin = rope_sin; a->table_rows = table_rows;
    a->start = start; a->start_wide = start_wide; a->tokens = (uint32_t)tokens; a->eps = eps;
    a->partial = nullptr; a->capacity = 0; a->first = 0; a->blocks = 0;
    return NOISE_OK;
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int noise_qk_norm_rotary(const noise_heads_t x[2], const noise_heads_t y[2], const float *const w[2],
                                    const noise_heads_t *v, const noise_heads_t *v_out, const float *rope_cos,
                                    const float *rope_sin, int64_t table_rows, const void *start, int start_wide,
                                    int64_t batch, int64_t tokens, int64_t capacity, int64_t head_dim, int type,
                                    float eps, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_qk_norm_rotary";
    NormArgs a;
    int st = check_norm(fn, x, y, w, rope_cos, rope_sin, table_rows, start, start_wide, batch, tokens, head_dim, type,
                        eps, &a);
    if (st) return st;
    NOISE_CHECK_ARG(capacity >= 0 && (capacity > 0) == (v != nullptr) && (v != nullptr) == (v_out != nullptr),
                    "%s: a cache needs its capacity, v and v_out", fn);
    NOISE_CHECK_ARG(!v || (v->heads == x[1].heads && v_out->heads == x[1].heads), "%s: k and v heads differ", fn);
    const int64_t per = x[0].heads + x[1].heads * (v ? 2 : 1);
    if (batch == 0 || tokens == 0) return NOISE_OK;
    NOISE_CHECK_ARG(batch <= INT32_MAX / tokens && batch * tokens <= INT32_MAX / per, "%s: too many rows", fn);
    if ((st = check_rows(fn, "q", x[0], type, &a.x[0])) || (st = check_rows(fn, "k", x[1], type, &a.x[1])) ||
        (st = check_rows(fn, "q's output", y[0], type, &a.y[0])) ||
        (st = check_rows(fn, "k's output", y[1], type, &a.y[1])))
        return st;
    if (v && ((st = check_rows(fn, "v", *v, type, &a.v)) || (st = check_rows(fn, "v's output", *v_out, type, &a.v_out))))
        return st;
    a.capacity = capacity; a.row_heads = (uint32_t)per; a.rows = (uint32_t)(batch * tokens * per);
    const int64_t per_group = kThreads / (head_dim / 16), groups = (a.rows + per_group - 1) / per_group;
    auto kernel = type == NOISE_BF16 ? (head_dim == 64 ? head_norm_kernel<__bf16, 64> : head_norm_kernel<__bf16, 128>)
                                     : (head_dim == 64 ? head_norm_kernel<float, 64> : head_norm_kernel<float, 128>);
    for (a.first = 0; a.first < groups; a.first += kLaunchGroups) {
        const int64_t n = groups - a.first < kLaunchGroups ? groups - a.first : kLaunchGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(kThreads), 0, (hipStream_t)stream, a);
    }
    return launch_status(fn);
}

extern "C" int64_t noise_qk_norm_rotary_bwd_workspace_bytes(int64_t head_dim) {
    clear_error();
    NOISE_CHECK_ARG(head_dim == 64 || head_dim == 128, "noise_qk_norm_rotary_bwd_workspace_bytes: head_dim must be 64 or 128");
    return 2 * kPartials * head_dim * 4;
}

extern "C" int noise_qk_norm_rotary_bwd(const noise_heads_t x[2], const noise_heads_t dy[2], const noise_heads_t dx[2],
                                        const float *const w[2], float *const dw[2], const float *rope_cos,
                                        const float *rope_sin, int64_t table_rows, const void *start, int start_wide,
                                        int64_t batch, int64_t tokens, int64_t head_dim, int type, float eps,
                                        void *workspace, int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_qk_norm_rotary_bwd";
    NormArgs a;
    int st = check_norm(fn, x, dy, w, rope_cos, rope_sin, table_rows, start, start_wide, batch, tokens, head_dim, type,
                        eps, &a);
    if (st) return st;
    NOISE_CHECK_ARG(dx && dw && dx[0].heads == x[0].heads && dx[1].heads == x[1].heads, "%s: dx or dw missing", fn);
    const int64_t per = x[0].heads + x[1].heads;
    NOISE_CHECK_ARG(tokens == 0 || (batch <= INT32_MAX / tokens && batch * tokens <= INT32_MAX / per),
                    "%s: too many rows", fn);
    const bool weights = w[0] || w[1];
    NOISE_CHECK_ARG((!w[0] || dw[0]) && (!w[1] || dw[1]), "%s: a weight without its gradient", fn);
    NOISE_CHECK_ARG(!weights || (workspace && aligned(workspace, 16) &&
                                 workspace_bytes >= noise_qk_norm_rotary_bwd_workspace_bytes(head_dim)),
                    "%s: workspace NULL, misaligned or too small", fn);
    if (batch * tokens > 0 &&
        ((st = check_rows(fn, "q", x[0], type, &a.x[0])) || (st = check_rows(fn, "k", x[1], type, &a.x[1])) ||
         (st = check_rows(fn, "dq", dy[0], type, &a.y[0])) || (st = check_rows(fn, "dk", dy[1], type, &a.y[1])) ||
         (st = check_rows(fn, "q's gradient", dx[0], type, &a.v)) ||
         (st = check_rows(fn, "k's gradient", dx[1], type, &a.v_out))))
        return st;
    a.partial = static_cast<float *>(workspace);
    a.row_heads = (uint32_t)per; a.rows = (uint32_t)(batch * tokens * per);
    const int64_t most = batch * tokens * (x[0].heads > x[1].heads ? x[0].heads : x[1].heads);
    const int64_t per_group = kThreads / (head_dim / 16), groups = (most + per_group - 1) / per_group;
    a.blocks = (int)(groups < kPartials ? groups : kPartials);
    if (a.blocks) {
        auto kernel = type == NOISE_BF16
                          ? (head_dim == 64 ? head_norm_bwd_kernel<__bf16, 64> : head_norm_bwd_kernel<__bf16, 128>)
                          : (head_dim == 64 ? head_norm_bwd_kernel<float, 64> : head_norm_bwd_kernel<float, 128>);
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.blocks, 2), dim3(kThreads), 0, (hipStream_t)stream, a);
    }
    if (weights)
        hipLaunchKernelGGL(head_norm_dw_kernel, dim3((unsigned)(head_dim / 16), 2), dim3(1024), 0, (hipStream_t)stream,
                           a.partial, w[0] ? dw[0] : nullptr, w[1] ? dw[1] : nullptr, a.blocks, (int)head_dim);
    return launch_status(fn);
}
