// The gradients of the vocabulary's cross entropy for few rows (up to 64), where the weight's bytes count: it is read once for dx and
// dW is written once, straight from and to memory, through v_mfma_f32_16x16x32_bf16 or, exact products, v_mfma_f32_16x16x4_f32.
// A lane holds N consecutive columns (16 B) of a matrix's rows; product e of N takes the e-th of each lane's columns, so that rows
// are read and written in runs of 256 B. Every row of dZ takes part, with zeros in those without a target, whose x is taken as
// zeros too. Of up to 32 rows dZ is a sum of two bf16 values beside bf16 operands: so few rows' roundings would not average out,
// and the products are free. (Of 64 rows it would take 20 % longer at 131072 x 2048.) Bound by HBM: at 131072 x 2048 and 4 rows in
// bf16, dx takes 109 us (4.9 TB/s of weight read) and dW 109 (4.9 TB/s written).
#pragma once
#include "vocab_gemm.hpp"

namespace noise {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct FewGradArgs {
    const void *x, *w, *targets;
    int64_t x_ld, w_ld;
    const void *dz;        // [parts][16 RB][z_ld], zeros where nothing stands
    const void *dzt;       // [parts][z_ld][rows, up to whole steps]
    float *slabs;          // dx's sums of each workgroup (splits), as its lanes hold them
    void *dx, *dw;
    int64_t z_ld;
    int rows, vocab, dim, wide, blocks, splits, per;   // blocks: of 16 N columns; per: entries of a workgroup
    int across, stream;    // dW: a workgroup's waves take 4 blocks of columns (else entries in turn); stores that pass the caches by
};

// dZ's parts: the value in its type, and the rest of it
template <class E>
constexpr int parts_of(int rows) { return sizeof(E) == 2 && rows <= 32 ? 2 : 1; }

__device__ __forceinline__ bool has_target(const void *targets, int wide, int64_t vocab, int r) {
    const int64_t t = wide ? static_cast<const int64_t *>(targets)[r] : (int64_t)static_cast<const int32_t *>(targets)[r];
    return t >= 0 && t < vocab;
}

// From a lane's 8 columns of 8 rows: column e's 8 rows, an operand of 8 k
__device__ __forceinline__ void columns_of(const u32x4 (&in)[8], bf16x8 (&out)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            o[j] = __builtin_amdgcn_perm(in[2 * j + 1][e / 2], in[2 * j][e / 2], e % 2 ? 0x07060302 : 0x05040100);
        out[e] = __builtin_bit_cast(bf16x8, o);
    }
}

// Rows 0 .. N - 1 of a lane's columns as operands, and acc[e] += (column e's products with z, N values of k)
template <class E>
struct FewOperand {
    static constexpr int N = 16 / sizeof(E);
    bf16x8 v[8];
    __device__ __forceinline__ void set(const u32x4 (&rows)[N]) { columns_of(rows, v); }
    // FIRST: the columns are the product's rows (else its columns)
    template <bool FIRST>
    __device__ __forceinline__ f32x4 times(int e, const u32x4 &z, f32x4 acc) const {
        const bf16x8 b = __builtin_bit_cast(bf16x8, z);
        return FIRST ? mfma16x16x32(v[e], b, acc) : mfma16x16x32(b, v[e], acc);
    }
};
template <>
struct FewOperand<float> {
    static constexpr int N = 4;
    u32x4 v[4];
    __device__ __forceinline__ void set(const u32x4 (&rows)[4]) {
#pragma unroll
        for (int s = 0; s < 4; ++s) v[s] = rows[s];
    }
    template <bool FIRST>
    __device__ __forceinline__ f32x4 times(int e, const u32x4 &z, f32x4 acc) const {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float a = __uint_as_float(v[s][e]), b = __uint_as_float(z[s]);
            acc = FIRST ? __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0) : __builtin_amdgcn_mfma_f32_16x16x4f32(b, a, acc, 0, 0, 0);
        }
        return acc;
    }
};

// The first of a lane's columns. Past the end of the row it takes the last N again (dim >= N): the same values, kept once or twice.
template <int N>
__device__ __forceinline__ int column_of(int block, int i, int dim) {
    const int c = block * 16 * N + N * i;
    return c < dim - N ? c : dim - N;
}

// dx: the product's rows are columns, its columns rows r. blockIdx.y: a block of columns; the workgroup's entries go to its waves in
// turn, whose sums meet in LDS.
template <class E, int RB>
__global__ __launch_bounds__(256) void vocab_few_dx_kernel(FewGradArgs a) {
    constexpr int N = FewOperand<E>::N, K = 4 * N, PARTS = parts_of<E>(16 * RB);
    __shared__ f32x4 sums[4][4][RB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const E *w = static_cast<const E *>(a.w) + column_of<N>(blockIdx.y, i, a.dim);
    const E *dz = static_cast<const E *>(a.dz) + i * a.z_ld + N * g;
    const int begin = blockIdx.x * a.per, end = (int)(begin + a.per < a.z_ld ? begin + a.per : a.z_ld);
    f32x4 acc[N][RB] = {};
    for (int v0 = begin + K * wave; v0 < end; v0 += 4 * K) {
        u32x4 rows[N], z[PARTS][RB];
#pragma unroll
        for (int s = 0; s < N; ++s) {
            const int v = v0 + N * g + s;
            __builtin_memcpy(&rows[s], w + (int64_t)(v < a.vocab ? v : a.vocab - 1) * a.w_ld, 16);
        }
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
#pragma unroll
            for (int b = 0; b < RB; ++b) __builtin_memcpy(&z[q][b], __builtin_assume_aligned(dz + 16 * (q * RB + b) * a.z_ld + v0, 16), 16);
        FewOperand<E> op;
        op.set(rows);
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q)
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e][b] = op.template times<true>(e, z[q][b], acc[e][b]);
    }
    f32x4 *slab = reinterpret_cast<f32x4 *>(a.slabs) + ((int64_t)blockIdx.x * a.blocks + blockIdx.y) * (N * RB * 64);
#pragma unroll
    for (int h = 0; h < N; h += 4) {
        if (h) __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int b = 0; b < RB; ++b) sums[wave][e][b][lane] = acc[h + e][b];
        __syncthreads();
#pragma unroll
        for (int b = 0; b < RB; ++b)
            slab[((h + wave) * RB + b) * 64 + lane] =
                sums[0][wave][b][lane] + sums[1][wave][b][lane] + sums[2][wave][b][lane] + sums[3][wave][b][lane];
    }
}

// dx from the workgroups' sums, in order: a thread takes what one lane held of one product
template <class E, int RB>
__global__ __launch_bounds__(256) void vocab_few_dx_join_kernel(FewGradArgs a) {
    constexpr int N = FewOperand<E>::N;
    const int unit = blockIdx.x * 256 + threadIdx.x, units = a.blocks * N * RB * 64;
    if (unit >= units) return;
    const int lane = unit & 63, b = unit / 64 % RB, e = unit / (64 * RB) % N, block = unit / (64 * RB * N);
    const int r = 16 * b + (lane & 15);
    if (r >= a.rows) return;
    const f32x4 *p = reinterpret_cast<const f32x4 *>(a.slabs) + unit;
    f32x4 v = {};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) v += p[(int64_t)s * units];
    const bool in = has_target(a.targets, a.wide, a.vocab, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int q = 4 * (lane >> 4) + j;
        const int c = block * 16 * N + N * q, at = column_of<N>(block, q, a.dim) + e;
        if (c < a.dim && at >= c) static_cast<E *>(a.dx)[(int64_t)r * a.dim + at] = (E)(in ? v[j] : 0.f);
    }
}

// dW: the product's rows are entries, its columns columns. The operands of x stay in registers; the workgroup's waves take four
// blocks of columns, so that 1 KB of a row is written at a time, or where there are too few blocks its entries in turn, 16 at a
// time. Rows of whole 128 B of a dW larger than the caches are stored past them. (131072 x 2048 bf16: 180 us without either, 147
// with the latter.)
template <class E, int KB>
__global__ __launch_bounds__(256) void vocab_few_dw_kernel(FewGradArgs a) {
    constexpr int N = FewOperand<E>::N, KP = KB * 4 * N, PARTS = parts_of<E>(KP);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int block = a.across ? 4 * blockIdx.y + wave : blockIdx.y;
    const int c = column_of<N>(block, i, a.dim);
    const bool mine = block * 16 * N + N * i < a.dim;
    if (block >= a.blocks) return;
    FewOperand<E> op[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        u32x4 rows[N];
#pragma unroll
        for (int s = 0; s < N; ++s) {
            const int r = 4 * N * b + N * g + s;
            rows[s] = u32x4{0, 0, 0, 0};
            if (r < a.rows && has_target(a.targets, a.wide, a.vocab, r))
                __builtin_memcpy(&rows[s], static_cast<const E *>(a.x) + r * a.x_ld + c, 16);
        }
        op[b].set(rows);
    }
    const int begin = blockIdx.x * a.per, end = (int)(begin + a.per < a.z_ld ? begin + a.per : a.z_ld);
    for (int v0 = begin + (a.across ? 0 : 16 * wave); v0 < end; v0 += a.across ? 16 : 64) {
        const E *dz = static_cast<const E *>(a.dzt) + (int64_t)(v0 + i) * KP + N * g;
        u32x4 z[PARTS][KB];
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
#pragma unroll
            for (int b = 0; b < KB; ++b) __builtin_memcpy(&z[q][b], __builtin_assume_aligned(dz + q * a.z_ld * KP + 4 * N * b, 16), 16);
        f32x4 acc[N] = {};
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q)
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] = op[b].template times<false>(e, z[q][b], acc[e]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            E o[N];
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = (E)acc[e][j];
            const int v = v0 + 4 * g + j;
            if (!mine || v >= a.vocab) continue;
            E *to = static_cast<E *>(a.dw) + (int64_t)v * a.dim + c;
            if (a.stream) {
                u32x4 bits;
                __builtin_memcpy(&bits, o, 16);
                __builtin_nontemporal_store(bits, reinterpret_cast<u32x4 *>(to));
            } else {
                __builtin_memcpy(to, o, 16);
            }
        }
    }
}

}  // namespace
}  // namespace noise
