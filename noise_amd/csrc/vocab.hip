// Cross entropy of a linear head over a vocabulary, with its gradients, without the logits in memory: for each row x_r with a target
// t_r in 0 .. V - 1, z = cap(x W^T),
//   loss_r = lse_r - z_{r,t_r},  dZ_rv = w_r (exp(z_rv - lse_r) - [v = t_r]) cap'(z_rv),  dx = dZ W,  dW = dZ^T x,
// cap(z) = softcap tanh(z / softcap), cap' = 1 - (cap / softcap)^2. (The head is utils/model.py:204-206 and train/val/run.py:89-94.)
//
// Rows without a target take no part: live_kernel numbers the others and pack_kernel packs them one after the other (and zeroes what
// stands between them and the end of a tile); all counts of rows are read on the device. Rows are worked on in pieces, so that dZ
// takes at most kPieceBytes (but no fewer than kPad rows). Per piece:
//   loss_kernel    a tile of logits in registers, its rows' maxima and sums of exponentials left per 128 vocabulary entries, which
//                  lse_kernel adds up. Where bf16 gradients are asked for in the same call, the exponentials stay as well, and
//                  lse_dz_kernel makes dZ of them: a pass over 2 R V bytes instead of another product
//   dz_kernel      otherwise: the logits once more, and dZ from them, in bf16 or, beside fp32 operands, two times fp16
//   grad_kernel    dx and dW in one launch, k split over workgroups where there are few tiles; sum_kernel joins the splits' fp32 sums
// fp32 operands are held as sums of two fp16 values, scaled by a power of two per tensor (hi carries 11 bits of a value, lo the next
// 11), and each product is hi hi + hi lo + lo hi: what is left out is 2^-22 of a term, and 2^-38 of the tensors' largest values.
// A bf16 weight is read where it is if its rows are whole 16 B: what its last stage of k lacks comes from the zeros behind a row of x
// (losses of 300 rows of 131072 x 1000: 243 -> 153 us).
// dZ beside bf16 operands is rounded to bf16, 2^-8 of each term, so that the gradients' products run at bf16's rate: at 16384 x
// 4096 x 512 the results are off by 2.3e-3 of themselves, where fp32 inside and their own rounding leave 1.7e-3. A second part,
// which up to 32 rows have, would double the gradients' products, 144 of that call's 290 us. For few rows few_kernel forms the
// logits (few_rows says when), and z_dz_kernel makes dZ of them; up to 64 rows have gradients of their own too (few_grad_rows).
//
// Bound by the matrix units, and there by power at large sizes: the loss pass of 8192 x 131072 x 2048 in bf16 takes 3.65 ms (1.2
// PFLOP/s), on an x of zeros 2.96; a plain large product on this card reaches 1.35. Alone on the GPU, in us:
//                                  live   pack   loss   lse or lse_dz   dz    grad   sum
//   16384 x 4096 x 512 bf16, cap     10     9    124         45          -     144     9    (in one call)
//   8192 x 131072 x 2048 bf16        8     15   4025        922          -    7305     -    (in one call)
//   16384 x 4096 x 512 fp32          9     19    224          7         265    374    11    (through autograd; largest values 14)
//   the same in one call             10    19    224          7         262    377    11    (the logits twice as well; 15)
//   3333 x 50021 x 776 bf16, 2/3     6      7    209          5         234    487     9    (through autograd)
// At widths like 512, 8 stages of k, a tile's epilogue shows: two exponentials, a reciprocal and some 12 other operations per
// capped logit.
#include "vocab_few.hpp"
#include "vocab_gemm.hpp"

#include <type_traits>

namespace noise {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int64_t kPieceBytes = 1ll << 31;   // of dZ
constexpr int kSegment = 128;                // vocabulary entries per partial maximum and sum
constexpr int kPad = 256;                    // rows of the packed matrices and of dZ come in these

using Tile = Tiling<256, 256, 2, 4, 64, 2>;
using HalfTile = Tiling<128, 256, 2, 4, 64, 2>;

// What the kernels share. Row indices are those of the packed rows.
struct HeadArgs {
    Operand x, w, dz;
    const int *count;            // packed rows
    const int *live;             // packed row -> row
    const int *target;           // of a packed row
    const float *scales;         // 2^ex, 2^ew, 2^ed of fp32 operands (x, w, dZ), else 1
    const float *weight;         // of a packed row's loss
    float *lse, *zt;             // of a packed row
    float2 *partial;             // [rows of the piece][segments]: a segment's largest logit, and the sum of exponentials from there
    int64_t row0;                // the piece's first packed row
    int64_t piece;               // rows of the piece, at most
    int vocab, dim, nk, segments;  // nk: stages of k over dim
    int64_t w_k;                 // columns that w has in memory, if fewer than the stages (x's are zeros from dim on)
    int tiles_m;
    float softcap;
};

// A gradient: dx (of rows) or dW (of vocabulary entries)
struct Result {
    void *out;                   // NULL: not asked for, or (with sum) not yet
    float *slabs;                // [splits][n][m] where k is split
    float *sum;                  // dW over several pieces: fp32 [vocab][dim]
    uint32_t groups;             // workgroups of its product, at most
    uint32_t sums;               // workgroups that join its splits (0: it has none)
};
struct GradArgs {
    Result dx, dw;
    const uint2 *cut;            // the piece's (shares_of)
    int add, fp32, tiles_m;      // add: to dw.sum's values; fp32: the results' type
};

__device__ __forceinline__ int64_t piece_rows(const HeadArgs &a) {
    const int64_t n = *a.count - a.row0;
    return n < 0 ? 0 : n < a.piece ? n : a.piece;
}

// softcap tanh(z / softcap), k = 2 log2(e) / softcap, with an error of 2^-22 softcap: what enters exp(z) is absolute. Past
// kWideCap, where that would be more than 2^-17, WIDE: below 0.35 of the cap tanh's odd series up to the 11th power (the next term
// is 1.2e-8 of the value there), which leaves an error relative to the logit.
constexpr float kWideCap = 32.f;
template <bool WIDE>
__device__ __forceinline__ float cap_of(float z, float cap, float k) {
    const float far = cap - 2.f * cap * __builtin_amdgcn_rcpf(exp2_fast(z * k) + 1.f);
    if constexpr (!WIDE) return far;
    const float u = z * (k * 0.34657359f), u2 = u * u;   // (z / cap: log(2) / 2)
    float s = __builtin_fmaf(u2, -1382.f / 155925.f, 62.f / 2835.f);
    s = __builtin_fmaf(u2, s, -17.f / 315.f);
    s = __builtin_fmaf(u2, s, 2.f / 15.f);
    s = __builtin_fmaf(u2, s, -1.f / 3.f);
    return u2 < 0.1225f ? __builtin_fmaf(z * u2, s, z) : far;
}

// --- rows with a target, packed ---

// Up to kLiveParts workgroups with `chunk` rows each: how many rows before them have a target they count themselves
constexpr int kLiveParts = 64;
__global__ __launch_bounds__(1024) void vocab_live_kernel(const void *targets, int wide, int64_t rows, int64_t chunk, int64_t vocab,
                                                          const float *weight, const float *lse, int *count, int *live, int *place,
                                                          int *target, float *live_weight, float *live_lse, float *weight_max) {
    __shared__ int sums[2][16];
    __shared__ float tops[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto at = [&](int64_t r) {
        return wide ? static_cast<const int64_t *>(targets)[r] : (int64_t)static_cast<const int32_t *>(targets)[r];
    };
    const int64_t begin = blockIdx.x * chunk, end = begin + chunk < rows ? begin + chunk : rows;
    int n = 0;
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < begin; r += 1024) {
        const int64_t t = at(r);
        n += t >= 0 && t < vocab;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (lane == 0) sums[1][wave] = n;
    __syncthreads();
    int base = 0;
    for (int w = 0; w < 16; ++w) base += sums[1][w];
    float top = 0.f;
    for (int64_t r0 = begin; r0 < end; r0 += 1024) {
        const int64_t r = r0 + threadIdx.x;
        const int64_t t = r < end ? at(r) : -1;
        const float w = weight && r < end ? weight[r] : 1.f, l = lse && r < end ? lse[r] : 0.f;
        const bool in = t >= 0 && t < vocab;
        const uint64_t mask = __ballot(in);
        if (lane == 0) sums[0][wave] = __popcll(mask);
        __syncthreads();
        int to = base + __popcll(mask & ((1ull << lane) - 1));
        for (int k = 0; k < 16; ++k) {
            if (k < wave) to += sums[0][k];
            base += sums[0][k];
        }
        __syncthreads();
        if (r < end) place[r] = in ? to : -1;
        if (!in) continue;
        live[to] = (int)r;
        target[to] = (int)t;
        if (lse) live_lse[to] = l;
        if (weight) live_weight[to] = w;
        if (fabsf(w) < __builtin_inff()) top = fmaxf(top, fabsf(w));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) top = fmaxf(top, tops[w]);
        weight_max[blockIdx.x] = top;
        if (blockIdx.x + 1 == gridDim.x) *count = base;
    }
}

// --- operands ---

// x and the weight as they come, and where they go
struct PackArgs {
    const void *src[2];
    int64_t src_ld[2], rows[2], padded[2];   // padded: rows of the packed matrix (0: not packed)
    Operand to[2];
    int64_t dim;
    const int *place, *count;
    const float *max, *weight_max;           // fp32: kMaxParts values of x's and of the weight's largest, and of the tokens' weights'
    int live_parts;
    float *scales;
    void *dx;
    float *loss, *lse;
    uint2 *cuts;                             // of each piece's gradients (NULL: none are asked for)
    int64_t piece, pieces;
    uint32_t tiles_m;
    bool need_dx, need_dw;
};

constexpr int kMaxParts = 512;

// 8 values of 4 or 2 B at any address of their type; n of them exist
template <class E>
__device__ __forceinline__ void load8(const E *p, int64_t n, E (&v)[8]) {
    if (n >= 8) __builtin_memcpy(v, p, sizeof v);
    else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (E)0.f;
}

// Largest finite |v| of a matrix's rows (x: of those with a target), one value per workgroup; a wave takes a row
__global__ __launch_bounds__(256) void vocab_max_kernel(PackArgs a, float *to) {
    __shared__ float tops[4];
    const int which = blockIdx.y, lane = threadIdx.x & 63;
    const float *src = static_cast<const float *>(a.src[which]);
    float top = 0.f;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows[which]; r += 4 * kMaxParts) {
        if (which == 0 && a.place[r] < 0) continue;
        for (int64_t c = 8 * lane; c < a.dim; c += 512) {
            float v[8];
            load8(src + r * a.src_ld[which] + c, a.dim - c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = fabsf(v[e]);
                if (f < __builtin_inff()) top = fmaxf(top, f);
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (lane == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) to[which * kMaxParts + blockIdx.x] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
}

// The power of two that takes `top` to 2^14 .. 2^15 (within the normal ones)
__device__ __forceinline__ float scale_of(float top) {
    if (!(top > 0.f)) return 1.f;
    int e = 14 - ilogbf(top);
    e = e < -126 ? -126 : e > 126 ? 126 : e;
    return ldexpf(1.f, e);
}

// f as a sum of two fp16 values, as bits. An infinity is the second one: it meets the first of the other operand's alone, whose
// sign is that of the value (the second may be 0, which would make a NaN of it, or of the other sign).
__device__ __forceinline__ void halves(float f, uint16_t &hi, uint16_t &lo) {
    const bool far = fabsf(f) == __builtin_inff();
    const _Float16 h = far ? (_Float16)copysignf(65504.f, f) : (_Float16)f;
    const _Float16 l = (_Float16)(far ? f : f - (float)h);
    __builtin_memcpy(&hi, &h, 2);
    __builtin_memcpy(&lo, &l, 2);
}

// In how many shares workgroups take the stages of k of a tile of dx (x) and of dW (y), whose fp32 sums are then joined. Both
// products run in one launch. Of no shares, and shares of one, a half and a third of what all stages take on 256 CUs, those that
// come out best by what was measured: a workgroup takes 2.2 us per stage (3.3 where operands are sums of two) and 3 us more, 256
// run at a time, and joining costs 5 us and 0.09 us of the whole chip's time per tile's share. At most kSplitTiles shares of tiles,
// at least 4 stages each. (At 16384 x 4096 x 512 dx then has 1 share and dW 4, and both take 153 us with the join; in two launches,
// with 2 and 8, it was 195.)
constexpr uint32_t kSplitTiles = 512;
template <class T, bool SPLIT>
__device__ uint2 shares_of(int64_t rows, int64_t vocab, uint32_t tiles_m, bool dx, bool dw) {
    constexpr uint32_t kStage = SPLIT ? 33 : 22;   // in 100 ns
    uint32_t tiles[2] = {dx ? tiles_m * (uint32_t)((rows + T::NT - 1) / T::NT) : 0, dw ? tiles_m * (uint32_t)((vocab + T::NT - 1) / T::NT) : 0};
    uint32_t stages[2] = {(uint32_t)((vocab + kStep<T, SPLIT> - 1) / kStep<T, SPLIT>), (uint32_t)((rows + kStep<T, SPLIT> - 1) / kStep<T, SPLIT>)};
    const uint64_t work = (uint64_t)tiles[0] * stages[0] + (uint64_t)tiles[1] * stages[1];
    uint2 take = {1, 1};
    if (work == 0) return take;
    uint64_t best = 0;
    for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t each = k ? (uint32_t)((work + 256 * k - 1) / (256 * k)) : 0;
        uint32_t s[2], groups = 0, longest = 0, sums = 0;
        uint64_t all = 0;
        for (int w = 0; w < 2; ++w) {
            s[w] = each ? (stages[w] + each - 1) / each : 1;
            if (s[w] > stages[w] / 4) s[w] = stages[w] / 4;
            if (tiles[w] && s[w] > kSplitTiles / tiles[w]) s[w] = kSplitTiles / tiles[w];
            if (s[w] < 1) s[w] = 1;
            const uint32_t n = (stages[w] + s[w] - 1) / s[w];
            groups += tiles[w] * s[w];
            all += (uint64_t)tiles[w] * s[w] * n;
            if (tiles[w] && n > longest) longest = n;
            if (s[w] > 1) sums += tiles[w] * s[w];
        }
        const uint32_t rounds = (groups + 255) / 256;
        uint64_t time = all * rounds / groups;
        if (time < longest) time = longest;
        time = time * kStage + rounds * 30 + (sums ? 50 + sums * 9 / 10 : 0);
        if (k == 0 || time < best) best = time, take = uint2{s[0], s[1]};
    }
    return take;
}

// The packed matrices: x's rows at their places (zeros behind the last) and the weight's where it is packed, with zeros from dim to
// the packed row's end. Rows of x without a place: their losses, lse and rows of dx to zero. A wave takes a row; blockIdx.y: x or
// the weight.
template <class E, bool SPLIT>
__global__ __launch_bounds__(256) void vocab_pack_kernel(PackArgs a) {
    const int which = blockIdx.y, lane = threadIdx.x & 63;
    const int64_t rows = a.rows[which], padded = a.padded[which], ld = a.to[which].ld, waves = (int64_t)gridDim.x * 4;
    float scale = 1.f;
    if constexpr (SPLIT) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxParts / 64; ++i) top = fmaxf(top, a.max[which * kMaxParts + lane + 64 * i]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        scale = scale_of(top);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.scales[which] = scale;
            if (which == 0) {
                float most = 0.f;
                for (int i = 0; i < a.live_parts; ++i) most = fmaxf(most, a.weight_max[i]);
                a.scales[2] = scale_of(most);
            }
        }
    }
    if (a.cuts && blockIdx.x == 0 && which == 0)
        for (int64_t i = threadIdx.x; i < a.pieces; i += 256) {
            const int64_t left = *a.count - i * a.piece, there = left < 0 ? 0 : left < a.piece ? left : a.piece;
            a.cuts[i] = shares_of<Tile, SPLIT>(there, a.rows[1], a.tiles_m, a.need_dx, a.need_dw);
        }
    if (!padded) return;
    const E *src = static_cast<const E *>(a.src[which]);
    uint16_t *dst = reinterpret_cast<uint16_t *>(const_cast<__bf16 *>(a.to[which].ptr));
    const int64_t behind = which == 0 ? *a.count : rows;
    uint16_t none[8] = {};
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < (rows > padded ? rows : padded); r += waves) {
        if (r >= behind && r < padded)
            for (int64_t c = 8 * lane; c < ld; c += 512) {
                __builtin_memcpy(__builtin_assume_aligned(dst + r * ld + c, 16), none, 16);
                if (SPLIT) __builtin_memcpy(__builtin_assume_aligned(dst + a.to[which].lo + r * ld + c, 16), none, 16);
            }
        if (r >= rows) continue;
        const int64_t at = which == 0 ? a.place[r] : r;
        if (at < 0) {
            if (a.dx)
                for (int64_t c = lane; c < a.dim; c += 64) static_cast<E *>(a.dx)[r * a.dim + c] = (E)0.f;
            if (lane == 0) {
                if (a.loss) a.loss[r] = 0.f;
                if (a.lse) a.lse[r] = 0.f;
            }
            continue;
        }
        for (int64_t c = 8 * lane; c < ld; c += 512) {
            E v[8];
            load8(src + r * a.src_ld[which] + c, a.dim - c, v);
            uint16_t hi[8], lo[8];
            if constexpr (SPLIT) {
#pragma unroll
                for (int e = 0; e < 8; ++e) halves(v[e] * scale, hi[e], lo[e]);
                __builtin_memcpy(__builtin_assume_aligned(dst + a.to[which].lo + at * ld + c, 16), lo, 16);
            } else {
                __builtin_memcpy(hi, v, 16);
            }
            __builtin_memcpy(__builtin_assume_aligned(dst + at * ld + c, 16), hi, 16);
        }
    }
}

// --- logits ---

// The tile's logits, unscaled and capped. Past the vocabulary: -inf, or under the cap (where they are multiplied by cap') a value
// whose exponential vanishes beside any other's. CAP: 0 none, 2 past kWideCap.
template <class T, bool SPLIT, int CAP>
__device__ __forceinline__ void to_logits(const HeadArgs &a, int m0, int lane, f32x16 (&acc)[T::FB][T::NB]) {
    const float unit = SPLIT ? 1.f / a.scales[0] / a.scales[1] : 1.f, k = CAP ? 2.f * kLog2e / a.softcap : 0.f;
#pragma unroll
    for (int i = 0; i < T::FB; ++i)
#pragma unroll
        for (int j = 0; j < T::NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float z = SPLIT ? acc[i][j][r] * unit : acc[i][j][r];
                if (CAP) z = cap_of<CAP == 2>(z, a.softcap, k);
                acc[i][j][r] = z;
            }
    if (m0 + T::FB * 32 > a.vocab) {
        const float none = CAP ? -8.f * a.softcap - 200.f : -__builtin_inff();
#pragma unroll
        for (int i = 0; i < T::FB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (m0 + 32 * i + 16 * (r / 8) + 8 * (lane >> 5) + r % 8 >= a.vocab)
#pragma unroll
                    for (int j = 0; j < T::NB; ++j) acc[i][j][r] = none;
    }
}

// u of 0 .. 2^kUnits in 16 bits, two to a word: the 6 bits of its exponent that may be set and 10 of its mantissa. Off by 2^-11,
// before dZ's own 2^-8, and 0 below 2^-62 of the largest: fp16 has as many bits down to 2^-29 only, and none below 2^-39, where an
// improbable entry's gradients (logits 27 below the largest of its 128) would be 0 beside those that backward() gives.
constexpr int kUnits = -64;
__device__ __forceinline__ uint32_t two_units(float a, float b) {
    return __builtin_amdgcn_perm((__float_as_uint(b) << 3) + 0x8000u, (__float_as_uint(a) << 3) + 0x8000u, 0x07060302);
}
// 2^-kUnits u
__device__ __forceinline__ float unit_of(uint32_t word, int i) {
    return __uint_as_float(i ? word >> 3 & 0x1fffe000u : (word & 0xffffu) << 13) * 0x1p64f;
}

// STORE: 2^kUnits exp(z - the segment's maximum) cap'(z) as two_units in dZ's place, which vocab_lse_dz_kernel turns into dZ
template <class T, bool SPLIT, int CAP, bool STORE>
__global__ __launch_bounds__(64 * T::NW, 2) void vocab_loss_kernel(HeadArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[T::kLds];
    const int64_t rows = piece_rows(a);
    const int tiles_n = (int)((rows + T::NT - 1) / T::NT);   // (of the rows that there are: XCDs share those evenly)
    if ((int)blockIdx.x >= a.tiles_m * tiles_n) return;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, tiles_n, tm, tn);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x16 acc[T::FB][T::NB];
    product<T, false, false, SPLIT, SPLIT>(a.w, (int64_t)tm * T::MT, a.vocab - 1 - tm * T::MT, a.x, a.row0 + (int64_t)tn * T::NT,
                                           T::NT - 1, 0, a.nk, a.w_k, a.x.ptr + a.dim, lds, acc);
    const int m0 = tm * T::MT + T::wm(wave);
    if (m0 >= a.vocab) return;
    to_logits<T, SPLIT, CAP>(a, m0, lane, acc);
    const float bend = CAP ? -1.f / a.softcap / a.softcap : 0.f;   // of cap'
    static_assert(T::FB * 32 == kSegment, "a wave's entries are a segment");
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int64_t at = (int64_t)tn * T::NT + T::wn(wave) + 32 * j + (lane & 31), row = a.row0 + at;
        const bool there = at < rows;
        float top = kLowest;
#pragma unroll
        for (int i = 0; i < T::FB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
        top = fmaxf(top, swap_halves(top));
        const int t = there ? a.target[row] - m0 - 8 * (lane >> 5) : -1;
        const bool mine = t >= 0 && t < kSegment && !(t & 8);
        if (__any(mine)) {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < T::FB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) z = t == 32 * i + 16 * (r / 8) + r % 8 ? acc[i][j][r] : z;
            if (mine) a.zt[row] = z;
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < T::FB; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = acc[i][j][8 * h + e];
                    // (the difference first: the rounding of a product with log2(e) would stay in the exponent, 2^-24 of it, and
                    // the lowest values' would be infinite; where all are -inf, top is finite and z - top is not)
                    v[e] = STORE ? exp2_fast(__builtin_fmaf(z - top, kLog2e, (float)kUnits)) : exp2_fast((z - top) * kLog2e);
                    s += v[e];
                    if (STORE && CAP) v[e] *= fmaxf(__builtin_fmaf(z * bend, z, 1.f), 0.f);
                }
                if constexpr (STORE) {
                    uint16_t *to = reinterpret_cast<uint16_t *>(const_cast<__bf16 *>(a.dz.ptr)) + at * a.dz.ld + m0 + 32 * i +
                                   16 * h + 8 * (lane >> 5);
                    uint32_t words[4];
                    // (rows behind the last one are multiplied by zeros)
#pragma unroll
                    for (int e = 0; e < 4; ++e) words[e] = there ? two_units(v[2 * e], v[2 * e + 1]) : 0;
                    __builtin_memcpy(__builtin_assume_aligned(to, 16), words, 16);
                }
            }
        s += swap_halves(s);
        if (STORE) s *= 0x1p64f;
        if (lane < 32 && there) a.partial[at * a.segments + m0 / kSegment] = float2{top, s};
    }
}

// Sum over the wave of sums s with maxima top, which every lane gets: the same bits (the lower lane's first in each pair)
__device__ __forceinline__ void wave_sums(float &top, float &s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(top, o, 64), s2 = __shfl_xor(s, o, 64);
        const float m = fmaxf(top, m2), a = s * exp2_fast((top - m) * kLog2e), b = s2 * exp2_fast((m2 - m) * kLog2e);
        s = threadIdx.x & o ? b + a : a + b;
        top = m;
    }
}
// The same over the workgroup
__device__ __forceinline__ void join_sums(float &top, float &s, float2 (&slots)[4]) {
    wave_sums(top, s);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = float2{top, s};
    __syncthreads();
    top = slots[0].x, s = slots[0].y;
    for (int w = 1; w < 4; ++w) {
        const float m = fmaxf(top, slots[w].x);
        s = s * exp2_fast((top - m) * kLog2e) + slots[w].y * exp2_fast((slots[w].x - m) * kLog2e);
        top = m;
    }
}

// This thread's share of a row's segments
__device__ __forceinline__ void row_sums(const float2 *part, int segments, float &top, float &s) {
    for (int g = threadIdx.x; g < segments; g += 256) {
        const float2 p = part[g];
        const float m = fmaxf(top, p.x);
        s = s * exp2_fast((top - m) * kLog2e) + p.y * exp2_fast((p.x - m) * kLog2e);
        top = m;
    }
}

// Rows' lse and losses from their segments, a wave per row
__global__ __launch_bounds__(256) void vocab_lse_kernel(HeadArgs a, float *loss, float *lse) {
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), row = a.row0 + at;
    if (at >= piece_rows(a)) return;
    const int lane = threadIdx.x & 63;
    const float2 *part = a.partial + at * a.segments;
    float top = kLowest, s = 0.f;
    for (int g = lane; g < a.segments; g += 64) {
        const float2 p = part[g];
        const float m = fmaxf(top, p.x);
        s = s * exp2_fast((top - m) * kLog2e) + p.y * exp2_fast((p.x - m) * kLog2e);
        top = m;
    }
    wave_sums(top, s);
    if (lane) return;
    const float l = top + logf(s);
    const int to = a.live[row];
    a.lse[row] = l;
    loss[to] = l - a.zt[row];
    if (lse) lse[to] = l;
}

// A row's lse and loss from its segments, and dZ from what vocab_loss_kernel left, at the rate of a copy (134 MB read and written
// in 45 us): dZ_v = weight exp(top - lse) stored_v, and at the target weight (exp(z - lse) - 1) cap'(z) from its logit
__global__ __launch_bounds__(256) void vocab_lse_dz_kernel(HeadArgs a, float *loss) {
    __shared__ float2 slots[4];
    const int64_t at = blockIdx.x, row = a.row0 + at;
    if (at >= piece_rows(a)) return;
    const float2 *part = a.partial + at * a.segments;
    float top = kLowest, s = 0.f;
    row_sums(part, a.segments, top, s);
    join_sums(top, s, slots);
    const float l = top + logf(s), z = a.zt[row];
    if (threadIdx.x == 0) loss[a.live[row]] = l - z;
    const float w = a.weight ? a.weight[row] : 1.f, u = a.softcap > 0.f ? z / a.softcap : 0.f;
    const float own = w * (exp2_fast((z - l) * kLog2e) - 1.f) * (1.f - u * u);
    const int t = a.target[row], end = a.segments * kSegment;
    uint16_t *dz = reinterpret_cast<uint16_t *>(const_cast<__bf16 *>(a.dz.ptr)) + at * a.dz.ld;
#pragma unroll 4
    for (int c = 8 * threadIdx.x; c < (int)a.dz.ld; c += 2048) {
        __bf16 o[8];
        if (c < end) {
            uint32_t v[4];
            __builtin_memcpy(v, __builtin_assume_aligned(dz + c, 16), 16);
            const float f = w * exp2_fast((part[c / kSegment].x - l) * kLog2e);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (__bf16)(c + e == t ? own : unit_of(v[e / 2], e % 2) * f);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (__bf16)0.f;
        }
        __builtin_memcpy(__builtin_assume_aligned(dz + c, 16), o, 16);
    }
}

// --- the losses of a few rows ---

// What is read is the weight: a workgroup takes 16 VB vocabulary entries for 16 RB rows (blockIdx.y counts those), its four waves a
// quarter of dim each, straight from memory into v_mfma_f32_16x16x32_bf16's (fp32: v_mfma_f32_16x16x4_f32's, exact products)
// operands: 16 lanes on 16 rows of the weight, and the rows of x from the caches. The waves' sums meet in LDS; wave v takes entries
// 16 v on from there.
//
// Bound by HBM: 4 rows of 65536 x 2048 in bf16, 268 MB, take 53 us (5.1 TB/s) with 8 loads of 16 B per lane and block under way;
// loads that bypass the caches were slower. With WRITE the logits themselves are left, fp32, for vocab_z_dz_kernel or
// vocab_few_dz_kernel (and partial may be NULL).
struct FewArgs {
    const void *x, *w, *targets;
    int64_t x_ld, w_ld;
    float2 *partial;
    float *zt, *z;
    int64_t z_ld;
    int rows, vocab, dim, segments, wide;
    float softcap;
};

template <class E, int VB, int RB, bool CAP, bool WRITE>
__global__ __launch_bounds__(256) void vocab_few_kernel(FewArgs a) {
    constexpr int N = sizeof(E) == 2 ? 8 : 4;   // elements per load
    __shared__ float sums[4][VB][RB][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int v0 = blockIdx.x * 16 * VB, r0 = blockIdx.y * 16 * RB;
    const E *w[VB], *x[RB];
#pragma unroll
    for (int b = 0; b < VB; ++b) {
        const int v = v0 + 16 * b + i;
        w[b] = static_cast<const E *>(a.w) + (int64_t)(v < a.vocab ? v : a.vocab - 1) * a.w_ld;
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int r = r0 + 16 * b + i;
        x[b] = static_cast<const E *>(a.x) + (int64_t)(r < a.rows ? r : a.rows - 1) * a.x_ld;
    }
    f32x4 acc[VB][RB] = {};
    auto multiply = [&](const E (&vw)[N], const E (&vx)[N], f32x4 &c) {
        if constexpr (sizeof(E) == 2) {
            bf16x8 p, q;
            __builtin_memcpy(&p, vw, 16);
            __builtin_memcpy(&q, vx, 16);
            c = mfma16x16x32(p, q, c);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(vw[e], vx[e], c, 0, 0, 0);
        }
    };
    // steps of 4 N consecutive elements of dim, wave after wave; the last one may be cut
    const int steps = (a.dim + 4 * N - 1) / (4 * N), whole = a.dim / (4 * N);
    const int first = steps * wave / 4, last = steps * (wave + 1) / 4;
    int s = first;
    auto run = [&](auto count) {
        constexpr int U = decltype(count)::value;
        for (; s + U <= (last < whole ? last : whole); s += U) {
            E vw[VB][U][N];
#pragma unroll
            for (int b = 0; b < VB; ++b)
#pragma unroll
                for (int u = 0; u < U; ++u) __builtin_memcpy(vw[b][u], w[b] + (s + u) * 4 * N + g * N, 16);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int r = 0; r < RB; ++r) {
                    E vx[N];
                    __builtin_memcpy(vx, x[r] + (s + u) * 4 * N + g * N, 16);
#pragma unroll
                    for (int b = 0; b < VB; ++b) multiply(vw[b][u], vx, acc[b][r]);
                }
            }
        }
    };
    run(std::integral_constant<int, 8>{});
    run(std::integral_constant<int, 2>{});
    run(std::integral_constant<int, 1>{});
    for (; s < last; ++s) {
        const int at = s * 4 * N + g * N, n = a.dim - at;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            E vx[N];
#pragma unroll
            for (int e = 0; e < N; ++e) vx[e] = e < n ? x[r][at + e] : (E)0.f;
#pragma unroll
            for (int b = 0; b < VB; ++b) {
                E vw[N];
#pragma unroll
                for (int e = 0; e < N; ++e) vw[e] = e < n ? w[b][at + e] : (E)0.f;
                multiply(vw, vx, acc[b][r]);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int r = 0; r < RB; ++r) __builtin_memcpy(sums[wave][b][r][lane], &acc[b][r], 16);
    __syncthreads();
    // entries v0 + 16 wave + 4 g + e of row r0 + 16 r + i
    __shared__ float2 tops[4][RB][16];
    if (wave < VB) {
        const float k = CAP ? 2.f * kLog2e / a.softcap : 0.f;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            const int row = r0 + 16 * r + i, v = v0 + 16 * wave + 4 * g;
            float z[4], top = kLowest, t = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                z[e] = sums[0][wave][r][lane][e] + sums[1][wave][r][lane][e] + sums[2][wave][r][lane][e] + sums[3][wave][r][lane][e];
                if (CAP) z[e] = cap_of<true>(z[e], a.softcap, k);
                if (v + e >= a.vocab) z[e] = -__builtin_inff();
                top = fmaxf(top, z[e]);
            }
            if constexpr (WRITE) {
                // (rows of the logits are whole 16 entries)
                if (row < a.rows) __builtin_memcpy(__builtin_assume_aligned(a.z + row * a.z_ld + v, 16), z, 16);
                if (!a.partial) continue;
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
#pragma unroll
            for (int e = 0; e < 4; ++e) t += exp2_fast((z[e] - top) * kLog2e);
            t += __shfl_xor(t, 16, 64);
            t += __shfl_xor(t, 32, 64);
            if (g == 0) tops[wave][r][i] = float2{top, t};
            if (row < a.rows) {
                const int64_t target = a.wide ? static_cast<const int64_t *>(a.targets)[row]
                                              : (int64_t)static_cast<const int32_t *>(a.targets)[row];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (target == v + e && v + e < a.vocab) a.zt[row] = z[e];
            }
        }
    }
    if (WRITE && !a.partial) return;
    __syncthreads();
    for (int row = threadIdx.x; row < 16 * RB; row += 256) {
        if (r0 + row >= a.rows) continue;
        float2 p = tops[0][row / 16][row % 16];
#pragma unroll
        for (int b = 1; b < VB; ++b) {
            const float2 q = tops[b][row / 16][row % 16];
            const float m = fmaxf(p.x, q.x);
            p = float2{m, p.y * exp2_fast((p.x - m) * kLog2e) + q.y * exp2_fast((q.x - m) * kLog2e)};
        }
        a.partial[(int64_t)(r0 + row) * a.segments + blockIdx.x] = p;
    }
}

__global__ __launch_bounds__(256) void vocab_few_join_kernel(FewArgs a, float *loss, float *lse) {
    __shared__ float2 slots[4];
    const int row = blockIdx.x;
    const int64_t t = a.wide ? static_cast<const int64_t *>(a.targets)[row] : (int64_t)static_cast<const int32_t *>(a.targets)[row];
    const bool in = t >= 0 && t < a.vocab;
    float top = kLowest, s = 0.f;
    if (in) row_sums(a.partial + (int64_t)row * a.segments, a.segments, top, s);
    join_sums(top, s, slots);
    if (threadIdx.x) return;
    const float l = top + logf(s);
    loss[row] = in ? l - a.zt[row] : 0.f;
    if (lse) lse[row] = in ? l : 0.f;
}

// dZ of up to 64 rows from their logits and lse: by rows (dz, which may be z's place) and by entries (dzt). A thread takes an entry
// of N rows; zeros where there is no row, target or entry.
template <class E>
__global__ __launch_bounds__(256) void vocab_few_dz_kernel(FewArgs a, const float *lse, const float *weight, E *dz, E *dzt, int dz_rows, int kp) {
    constexpr int N = 16 / sizeof(E);
    const int parts = parts_of<E>(kp);
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int r0 = blockIdx.y * N;
    if (v >= a.z_ld) return;
    E o[N], rest[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int r = r0 + e;
        float d = 0.f;
        if (r < a.rows && v < a.vocab) {
            const int64_t t = a.wide ? static_cast<const int64_t *>(a.targets)[r] : (int64_t)static_cast<const int32_t *>(a.targets)[r];
            if (t >= 0 && t < a.vocab) {
                const float z = a.z[r * a.z_ld + v], w = weight ? weight[r] : 1.f, u = a.softcap > 0.f ? z / a.softcap : 0.f;
                d = exp2_fast((z - lse[r]) * kLog2e);
                if (v == t) d -= 1.f;
                d *= w * (1.f - u * u);
            }
        }
        o[e] = (E)d;
        rest[e] = (E)(d - (float)o[e]);
        if (r < dz_rows) {
            dz[r * a.z_ld + v] = o[e];
            if (parts > 1) dz[(dz_rows + r) * a.z_ld + v] = rest[e];
        }
    }
    __builtin_memcpy(__builtin_assume_aligned(dzt + v * kp + r0, 16), o, 16);
    if (parts > 1) __builtin_memcpy(__builtin_assume_aligned(dzt + (a.z_ld + v) * kp + r0, 16), rest, 16);
}

// dZ of packed rows from their logits and lse, which are by row; zeros in the rows behind the last. blockIdx.y: a share of the
// entries
constexpr int kDzEntries = 4096;
template <bool SPLIT>
__global__ __launch_bounds__(256) void vocab_z_dz_kernel(HeadArgs a, const float *logits, int64_t z_ld, const float *lse) {
    const int64_t at = blockIdx.x;
    const bool there = at < *a.count;
    const int row = there ? a.live[at] : 0, t = there ? a.target[at] : 0;
    const float *z = logits + row * z_ld;
    const float l = lse[row], w = (a.weight ? a.weight[at] : 1.f) * (SPLIT ? a.scales[2] : 1.f);
    const bool cap = a.softcap > 0.f;
    const float bend = cap ? -w / a.softcap / a.softcap : 0.f;   // of w cap'
    uint16_t *dz = reinterpret_cast<uint16_t *>(const_cast<__bf16 *>(a.dz.ptr)) + at * a.dz.ld;
    const int begin = blockIdx.y * kDzEntries, end = begin + kDzEntries < (int)a.dz.ld ? begin + kDzEntries : (int)a.dz.ld;
    for (int c = begin + 8 * threadIdx.x; c < end; c += 2048) {
        uint16_t hi[8] = {}, lo[8] = {};
        if (there && c < a.vocab) {
            float v[8];
            __builtin_memcpy(v, __builtin_assume_aligned(z + c, 16), 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float d = exp2_fast((v[e] - l) * kLog2e);
                if (c + e == t) d -= 1.f;
                d *= cap ? __builtin_fmaf(v[e] * bend, v[e], w) : w;
                if (c + e >= a.vocab) d = 0.f;
                if constexpr (SPLIT) halves(d, hi[e], lo[e]);
                else {
                    const __bf16 b = (__bf16)d;
                    __builtin_memcpy(&hi[e], &b, 2);
                }
            }
        }
        __builtin_memcpy(__builtin_assume_aligned(dz + c, 16), hi, 16);
        if constexpr (SPLIT) __builtin_memcpy(__builtin_assume_aligned(dz + a.dz.lo + c, 16), lo, 16);
    }
}

template <class E, int VB, bool WRITE>
void (*few_of(int64_t rows, bool cap))(FewArgs) {
    return rows <= 16   ? (cap ? vocab_few_kernel<E, VB, 1, true, WRITE> : vocab_few_kernel<E, VB, 1, false, WRITE>)
           : rows <= 32 ? (cap ? vocab_few_kernel<E, VB, 2, true, WRITE> : vocab_few_kernel<E, VB, 2, false, WRITE>)
                        : (cap ? vocab_few_kernel<E, VB, 4, true, WRITE> : vocab_few_kernel<E, VB, 4, false, WRITE>);
}
unsigned few_blocks(int64_t rows) { return (unsigned)((rows + 63) / 64); }
template <bool WRITE>
void (*few_of(int type, int blocks, int64_t rows, bool cap))(FewArgs) {
    return type == NOISE_FP32 ? (blocks == 2 ? few_of<float, 2, WRITE>(rows, cap) : few_of<float, 1, WRITE>(rows, cap))
                              : (blocks == 2 ? few_of<__bf16, 2, WRITE>(rows, cap) : few_of<__bf16, 1, WRITE>(rows, cap));
}

// zeros: rows of dW past the vocabulary
__global__ __launch_bounds__(256) void vocab_fill_kernel(uint16_t *p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

template <class T, bool SPLIT, int CAP>
__global__ __launch_bounds__(64 * T::NW, 2) void vocab_dz_kernel(HeadArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[T::kLds];
    const int64_t rows = piece_rows(a);
    const int tiles_n = (int)((rows + T::NT - 1) / T::NT);   // (of the rows that there are: XCDs share those evenly)
    if ((int)blockIdx.x >= a.tiles_m * tiles_n) return;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, tiles_n, tm, tn);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x16 acc[T::FB][T::NB];
    product<T, false, false, SPLIT, SPLIT>(a.w, (int64_t)tm * T::MT, a.vocab - 1 - tm * T::MT, a.x, a.row0 + (int64_t)tn * T::NT,
                                           T::NT - 1, 0, a.nk, a.w_k, a.x.ptr + a.dim, lds, acc);
    const int m0 = tm * T::MT + T::wm(wave);
    to_logits<T, SPLIT, CAP>(a, m0, lane, acc);
    uint16_t *dz = reinterpret_cast<uint16_t *>(const_cast<__bf16 *>(a.dz.ptr));
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int64_t at = (int64_t)tn * T::NT + T::wn(wave) + 32 * j + (lane & 31), row = a.row0 + at;
        const bool there = at < rows;
        const float w = there ? (a.weight ? a.weight[row] : 1.f) * (SPLIT ? a.scales[2] : 1.f) : 0.f;
        const float bend = CAP ? -w / a.softcap / a.softcap : 0.f;   // of w cap'
        const float lse = there ? a.lse[row] : 0.f;
        const int t = there ? a.target[row] - m0 - 8 * (lane >> 5) : -1;
#pragma unroll
        for (int i = 0; i < T::FB; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint16_t hi[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = acc[i][j][8 * h + e];
                    float d = exp2_fast((z - lse) * kLog2e);
                    if (t == 32 * i + 16 * h + e) d -= 1.f;
                    d *= CAP ? __builtin_fmaf(z * bend, z, w) : w;
                    if (!there) d = 0.f;
                    if constexpr (SPLIT) halves(d, hi[e], lo[e]);
                    else {
                        const __bf16 b = (__bf16)d;
                        __builtin_memcpy(&hi[e], &b, 2);
                    }
                }
                uint16_t *to = dz + at * a.dz.ld + m0 + 32 * i + 16 * h + 8 * (lane >> 5);
                __builtin_memcpy(__builtin_assume_aligned(to, 16), hi, 16);
                if constexpr (SPLIT) __builtin_memcpy(__builtin_assume_aligned(to + a.dz.lo, 16), lo, 16);
            }
    }
}

// --- gradients ---

// 8 consecutive results, of which n exist, in their type at any address of it
__device__ __forceinline__ void put_out(void *out, int fp32, int64_t at, int n, const float (&v)[8]) {
    if (fp32) {
        float *p = static_cast<float *>(out) + at;
        if (n >= 8) __builtin_memcpy(p, v, 32);
        else
            for (int e = 0; e < 8; ++e)
                if (e < n) p[e] = v[e];
    } else {
        __bf16 o[8], *p = static_cast<__bf16 *>(out) + at;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (__bf16)v[e];
        if (n >= 8) __builtin_memcpy(p, o, 16);
        else
            for (int e = 0; e < 8; ++e)
                if (e < n) p[e] = o[e];
    }
}

// Columns m .. m + 7 of result n: added to the pieces before, and stored as its row
template <bool DX>
__device__ __forceinline__ void finish(const HeadArgs &a, const GradArgs &g, int64_t n, int m, float (&v)[8]) {
    const Result &r = DX ? g.dx : g.dw;
    if (!DX && r.sum) {
        float *p = r.sum + n * a.x.ld + m;
        if (g.add)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += p[e];
        if (!r.out) __builtin_memcpy(__builtin_assume_aligned(p, 16), v, 32);
    }
    if (r.out) put_out(r.out, g.fp32, (DX ? (int64_t)a.live[a.row0 + n] : n) * a.dim + m, a.dim - m, v);
}

// How a gradient's product is cut, from the rows that there are
struct Cut {
    int64_t n_end;             // results along n: packed rows (dx) or vocabulary entries (dW)
    uint32_t tiles_n, tiles, stages, splits;
};
template <class T, bool DX, bool SPLIT>
__device__ __forceinline__ Cut cut_of(const HeadArgs &a, const GradArgs &g, int64_t rows) {
    Cut c;
    c.n_end = DX ? rows : a.vocab;
    c.tiles_n = (uint32_t)((c.n_end + T::NT - 1) / T::NT);
    c.tiles = g.tiles_m * c.tiles_n;
    c.stages = (uint32_t)(((DX ? a.vocab : rows) + kStep<T, SPLIT> - 1) / kStep<T, SPLIT>);
    c.splits = DX ? g.cut->x : g.cut->y;
    return c;
}

// A tile from column m0 and row or entry n0 on, over the stages first .. last - 1 of k
template <class T, bool DX, bool SPLIT>
__device__ __forceinline__ void gradient_tile(const HeadArgs &a, const GradArgs &g, const Cut &c, uint32_t split, int m0, int64_t n0, int first,
                                              int last, char *lds) {
    const Result &res = DX ? g.dx : g.dw;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dim8 = (a.dim + 7) / 8;   // chunks of a row
    f32x16 acc[T::FB][T::NB];
    if (DX)
        product<T, true, false, SPLIT, SPLIT>(a.w, m0, dim8 - m0 / 8 - 1, a.dz, n0, T::NT - 1, first, last, a.vocab, nullptr, lds, acc);
    else {
        Operand x = a.x;
        x.ptr += a.row0 * x.ld;
        product<T, true, true, SPLIT, SPLIT>(x, m0, dim8 - m0 / 8 - 1, a.dz, n0, (int)(a.dz.ld - n0) / 8 - 1, first, last, 1ll << 40,
                                             nullptr, lds, acc);
    }
    const float unit = SPLIT ? 1.f / a.scales[2] / a.scales[DX ? 1 : 0] : 1.f;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int64_t n = n0 + T::wn(wave) + 32 * j + (lane & 31);
        if (n >= c.n_end) continue;
#pragma unroll
        for (int i = 0; i < T::FB; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int m = m0 + T::wm(wave) + 32 * i + 16 * h + 8 * (lane >> 5);
                if (m >= a.dim) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = SPLIT ? acc[i][j][8 * h + e] * unit : acc[i][j][8 * h + e];
                if (c.splits > 1)
                    __builtin_memcpy(__builtin_assume_aligned(res.slabs + ((int64_t)split * c.n_end + n) * a.x.ld + m, 16), v, 32);
                else
                    finish<DX>(a, g, n, m, v);
            }
    }
}

// n: packed rows (DX) or vocabulary entries; m: columns of dim. What is left of dim in the last tile takes half a tile where that
// is enough.
template <class T, bool DX, bool SPLIT>
__device__ __forceinline__ void gradient(const HeadArgs &a, const GradArgs &g, uint32_t group, char *lds) {
    const Cut c = cut_of<T, DX, SPLIT>(a, g, piece_rows(a));
    if (group >= c.tiles * c.splits) return;
    const uint32_t split = group / c.tiles;
    int tm, tn;
    tile_of(group - split * c.tiles, g.tiles_m, c.tiles_n, tm, tn);
    const int first = (int)((int64_t)c.stages * split / c.splits), last = (int)((int64_t)c.stages * (split + 1) / c.splits);
    static_assert(HalfTile::NT == T::NT && HalfTile::BK == T::BK && HalfTile::kLds <= T::kLds, "the same stages and columns of tiles");
    if (a.dim - tm * T::MT <= HalfTile::MT)
        gradient_tile<HalfTile, DX, SPLIT>(a, g, c, split, tm * T::MT, (int64_t)tn * T::NT, first, last, lds);
    else
        gradient_tile<T, DX, SPLIT>(a, g, c, split, tm * T::MT, (int64_t)tn * T::NT, first, last, lds);
}

// Both gradients in one launch: neither waits for the other's last workgroups (16384 x 4096 x 512: 144 us, 0.95 PFLOP/s; 8192 x
// 131072 x 2048: 7.4 ms, 1.19)
template <class T, bool SPLIT>
__global__ __launch_bounds__(64 * T::NW, 2) void vocab_grad_kernel(HeadArgs a, GradArgs g) {
    __shared__ __attribute__((aligned(1024))) char lds[T::kLds];
    if (blockIdx.x < g.dx.groups) gradient<T, true, SPLIT>(a, g, blockIdx.x, lds);
    else gradient<T, false, SPLIT>(a, g, blockIdx.x - g.dx.groups, lds);
}

// The splits' sums, in order
template <class T, bool DX, bool SPLIT>
__device__ __forceinline__ void join_splits(const HeadArgs &a, const GradArgs &g, uint32_t group) {
    const Cut k = cut_of<T, DX, SPLIT>(a, g, piece_rows(a));
    if (k.splits == 1) return;   // (the product has written its results)
    const int64_t i = (int64_t)group * 256 + threadIdx.x;
    const uint32_t per = (uint32_t)(a.x.ld / 8);
    const int64_t n = i / per;
    const int m = (int)(i - n * per) * 8;
    if (n >= k.n_end || m >= a.dim) return;
    float v[8] = {};
    for (uint32_t s = 0; s < k.splits; ++s) {
        const float *p = (DX ? g.dx : g.dw).slabs + ((int64_t)s * k.n_end + n) * a.x.ld + m;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += p[e];
    }
    finish<DX>(a, g, n, m, v);
}
template <class T, bool SPLIT>
__global__ __launch_bounds__(256) void vocab_sum_kernel(HeadArgs a, GradArgs g) {
    if (blockIdx.x < g.dx.sums) join_splits<T, true, SPLIT>(a, g, blockIdx.x);
    else join_splits<T, false, SPLIT>(a, g, blockIdx.x - g.dx.sums);
}

// --- host ---

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// The workspace's parts, and how the work is cut
struct Plan {
    int64_t ld, rows, piece, pieces, vocab_ld, segments;
    int nk;
    bool split, pack_w, few;   // few: the logits of all rows are kept (at most 1 GiB)
    int64_t dx_groups, dw_groups, dx_slabs, dw_slabs;
    int64_t at_int, at_float, at_cuts, at_z, at_few, at_partial, at_x, at_w, at_dz, at_dx, at_dw, at_sum, bytes;
};

// For any number of rows up to the piece's: the most workgroups of a gradient's product, and the fp32 values of its splits' sums.
// rows: whether the results are rows (dx), of which there may be fewer than n_end
void most_of(bool rows, int64_t n_end, int64_t stages, int64_t ld, int64_t *groups, int64_t *slabs) {
    const int64_t tiles_m = (ld + Tile::MT - 1) / Tile::MT, tiles = tiles_m * ((n_end + Tile::NT - 1) / Tile::NT);
    *groups = tiles > kSplitTiles ? tiles : kSplitTiles;
    // s parts where s tiles <= kSplitTiles and 4 s <= stages
    const int64_t least = rows ? tiles_m : tiles, s = stages / 4 < kSplitTiles / least ? stages / 4 : kSplitTiles / least;
    int64_t n = s * n_end;
    if (rows && kSplitTiles / tiles_m * Tile::NT < n) n = kSplitTiles / tiles_m * Tile::NT;
    *slabs = s < 2 ? 0 : n * ld;
}

// Whether the logits come from vocab_few_kernel, whose every workgroup forms its own, or from the tiles of vocab_loss_kernel and
// vocab_dz_kernel, which share operands but are few and long where there are few entries or rows. By what was measured, in ns: the
// former read 5 TB/s of weight for each 64 rows and then multiply at 268 TFLOP/s (fp32: 119); a tile takes 1.5 us per stage of 64
// of dim when it is one of the only 256 and 2.3 otherwise (twice that in fp32, whose gradients have two such passes in one call and
// whose losses alone need x and the weight packed, 12 B read and written per value), and 15 us in all. 131072 x 2048 bf16, losses
// of 16, 32 and 64 rows: 132, 157 and 233 us against 165; 4096 x 512: 6, 7 and 9 against 27; 131072 x 2048 fp32: 257, 322 and 478
// against 970. Many rows of few entries are alike: 793 x 119 x 4096, loss and gradients, bf16 67 us against 125, fp32 103 against
// 499; past some thousand rows the tiles are as fast (4000 x 300 x 2048 bf16: 122 against 130).
bool few_rows(const noise_vocab_t *v, bool grad) {
    if (v->rows > 1 << 20 || v->rows * v->vocab > 1 << 28) return false;
    const double R = (double)v->rows, VD = (double)v->vocab * (double)v->dim, size = v->type == NOISE_FP32 ? 4 : 2;
    double few = VD * size * (double)((v->rows + 63) / 64) / 5e3 + 2 * R * VD / (size == 4 ? 119e3 : 268e3);
    const double rounds = (double)(((v->vocab + 255) / 256 * ((v->rows + 255) / 256) + 255) / 256), stages = (double)((v->dim + 63) / 64);
    double tiles = 15e3 + rounds * stages * (rounds > 1 ? 2300 : 1500) * (size == 4 ? (grad ? 4 : 2) : 1);
    if (size == 4 && !grad) tiles += (VD + R * (double)v->dim) * 12 / 5e3;
    // rows of x, read from far; the logits written and read, or their exponentials
    few += R * (double)v->dim / 250;
    if (grad) few += R * (double)v->vocab * 8 / 5e3, tiles += size == 4 ? 0 : R * (double)v->vocab * 6 / 5e3;
    return few < tiles;
}

template <bool SPLIT, bool STORE>
void (*loss_of(float softcap))(HeadArgs) {
    return softcap > kWideCap ? vocab_loss_kernel<Tile, SPLIT, 2, STORE>
           : softcap > 0.f    ? vocab_loss_kernel<Tile, SPLIT, 1, STORE>
                              : vocab_loss_kernel<Tile, SPLIT, 0, STORE>;
}
template <bool SPLIT>
void (*dz_of(float softcap))(HeadArgs) {
    return softcap > kWideCap ? vocab_dz_kernel<Tile, SPLIT, 2>
           : softcap > 0.f    ? vocab_dz_kernel<Tile, SPLIT, 1>
                              : vocab_dz_kernel<Tile, SPLIT, 0>;
}

// Gradients of rows this few have kernels of their own (vocab_few.hpp), whose columns come in 16 B. Tiles waste 192 of 256 rows or
// more, store dW in short runs, and need fp32 weights split: 131072 x 2048 bf16, loss and gradients of 4, 16 and 64 rows: 336, 373
// and 503 us against 667, 692 and 660; fp32: 641, 696 and 1291 against 1665, 1717 and 1939; 4096 x 512 bf16: 20, 22 and 30 against
// 40, 40 and 44.
bool few_grad_rows(const noise_vocab_t *v) { return v->rows <= 64 && v->dim >= 8; }

struct FewPlan {
    int blocks;   // of 16 entries per workgroup
    int64_t segments, at_partial, bytes;
};
FewPlan few_plan(const noise_vocab_t *v) {
    FewPlan p;
    // 32 entries per workgroup, or 16 where that leaves fewer than two workgroups per CU
    p.blocks = v->vocab >= 32 * 512 ? 2 : 1;
    p.segments = (v->vocab + 16 * p.blocks - 1) / (16 * p.blocks);
    p.at_partial = up(4 * v->rows, 1024);
    p.bytes = p.at_partial + 8 * p.segments * v->rows;
    return p;
}

// The gradients of up to 64 rows: where their workspace's parts are, behind the losses' (few_plan)
struct FewGradPlan {
    int64_t z_ld, at_lse, at_z, at_dz, at_dzt, at_slabs, bytes;
    int rb, kb, kp, dz_rows;   // blocks of 16 rows (dx) and of 4 N rows (dW), rows in those
    int columns, dx_per, dx_splits, dw_per, dw_chunks, across;
};
FewGradPlan few_grad_plan(const noise_vocab_t *v) {
    FewGradPlan p;
    const int size = v->type == NOISE_FP32 ? 4 : 2, n = 16 / size;
    p.z_ld = up(v->vocab, 32);
    p.rb = v->rows <= 16 ? 1 : v->rows <= 32 ? 2 : 4;
    p.dz_rows = 16 * p.rb;
    p.kb = size == 4 ? p.rb : p.rb == 4 ? 2 : 1;
    p.kp = p.kb * 4 * n;
    p.columns = (int)((v->dim + 16 * n - 1) / (16 * n));
    // workgroups: two per CU for dx, whose sums are then joined, and four for dW, whose waves hold x (half as many or
    // twice as many: up to 10 % more)
    auto cut = [&](int64_t groups, int64_t columns, int64_t step, int *per) {
        const int64_t want = groups / columns > 1 ? groups / columns : 1;
        *per = (int)up((p.z_ld + want - 1) / want, step);
        return (int)((p.z_ld + *per - 1) / *per);
    };
    p.dx_splits = cut(512, p.columns, 128, &p.dx_per);
    p.across = p.columns % 4 == 0 || p.columns >= 12;
    p.dw_chunks = cut(1024, p.across ? (p.columns + 3) / 4 : p.columns, p.across ? 16 : 64, &p.dw_per);
    int64_t at = up(few_plan(v).bytes, 1024);
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += up(bytes, 1024);
        return here;
    };
    p.at_lse = take(4 * v->rows);
    p.at_z = take(4 * p.dz_rows * p.z_ld);
    // (dZ in one or two bf16 parts, or one of fp32)
    const int64_t each = size == 4 ? 4 : 2 * parts_of<__bf16>(p.kp);
    p.at_dz = size == 4 ? p.at_z : take(each * p.dz_rows * p.z_ld);
    p.at_dzt = take(each * p.z_ld * p.kp);
    p.at_slabs = take(16ll * 64 * n * p.rb * p.columns * p.dx_splits);
    p.bytes = at;
    return p;
}

Plan plan_of(const noise_vocab_t *v, bool grad) {
    Plan p = {};
    p.split = v->type == NOISE_FP32;
    p.ld = up(v->dim, Tile::BK);
    const int64_t step = p.split ? kStep<Tile, true> : kStep<Tile, false>;
    p.nk = (int)(p.ld / step);
    p.rows = up(v->rows, kPad);
    p.vocab_ld = up(v->vocab, Tile::MT);
    p.segments = (v->vocab + kSegment - 1) / kSegment;
    const int64_t parts = p.split ? 2 : 1;
    int64_t most = kPieceBytes / (2 * parts * p.vocab_ld) / kPad * kPad;
    if (most < kPad) most = kPad;
    p.piece = p.rows < most ? p.rows : most;
    // pieces of one size
    p.pieces = (p.rows + p.piece - 1) / p.piece;
    p.piece = up((p.rows + p.pieces - 1) / p.pieces, kPad);
    p.pieces = (p.rows + p.piece - 1) / p.piece;
    // the weight is read where it is if its rows are whole 16 B at 16 B addresses
    p.pack_w = p.split || v->dim % 8 || v->weight_stride % 8 || !aligned(v->weight, 16) || v->weight_stride >= (1 << 23);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += up(bytes, 1024);
        return here;
    };
    p.at_int = take(4 * (3 * p.rows + 1));
    p.at_float = take(4 * (3 * p.rows + 4 + kLiveParts + 2 * kMaxParts));
    p.at_partial = take(8 * p.segments * p.piece);
    p.at_x = take(2 * parts * p.rows * p.ld);
    if (p.pack_w) p.at_w = take(2 * parts * v->vocab * p.ld);
    if (grad) {
        p.few = few_rows(v, true) && p.pieces == 1;
        if (p.few) {
            p.at_z = take(4 * v->rows * up(v->vocab, 32));
            p.at_few = take(up(few_plan(v).bytes, 16) + 4 * v->rows);
        }
        p.at_cuts = take(8 * p.pieces);
        p.at_dz = take(2 * parts * p.piece * p.vocab_ld);
        most_of(true, p.piece, (v->vocab + step - 1) / step, p.ld, &p.dx_groups, &p.dx_slabs);
        most_of(false, v->vocab, p.piece / step, p.ld, &p.dw_groups, &p.dw_slabs);
        p.at_dx = take(4 * p.dx_slabs);
        p.at_dw = take(4 * p.dw_slabs);
        if (p.pieces > 1) p.at_sum = take(4 * v->vocab * p.ld);
    }
    p.bytes = at;
    return p;
}

int check(const char *fn, const noise_vocab_t *v, float softcap) {
    NOISE_CHECK_ARG(v, "%s: NULL pointer", fn);
    NOISE_CHECK_ARG(v->type == NOISE_BF16 || v->type == NOISE_FP32, "%s: unknown type %lld", fn, (long long)v->type);
    NOISE_CHECK_ARG(v->rows >= 0 && v->rows <= (1 << 30) && v->dim > 0 && v->dim <= (1 << 16) && v->vocab > 0 && v->vocab <= (1 << 22),
                    "%s: rows 0 .. 2^30, dim 1 .. 65536 and vocab 1 .. 2^22 required", fn);
    NOISE_CHECK_ARG(softcap == 0.f || (softcap >= 1e-6f && softcap <= 1e6f), "%s: softcap must be 1e-6 .. 1e6, or 0 for none", fn);
    if (v->rows == 0) return NOISE_OK;
    NOISE_CHECK_ARG(v->x_stride >= 0 && v->weight_stride >= 0, "%s: strides must be 0 or more", fn);
    const size_t size = v->type == NOISE_BF16 ? 2 : 4;
    NOISE_CHECK_ARG(v->x && v->weight && v->targets && aligned(v->x, size) && aligned(v->weight, size) &&
                        aligned(v->targets, v->targets_wide ? 8 : 4),
                    "%s: a pointer is NULL or not aligned to its type", fn);
    return NOISE_OK;
}

int run_few(const char *fn, const noise_vocab_t *v, float softcap, float *loss, float *lse, void *workspace, int64_t workspace_bytes,
            hipStream_t stream) {
    const FewPlan p = few_plan(v);
    NOISE_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes,
                    "%s: workspace of %lld bytes (16 B aligned) required", fn, (long long)p.bytes);
    FewArgs a;
    a.x = v->x, a.w = v->weight, a.targets = v->targets, a.x_ld = v->x_stride, a.w_ld = v->weight_stride;
    a.zt = static_cast<float *>(workspace);
    a.partial = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + p.at_partial);
    a.rows = (int)v->rows, a.vocab = (int)v->vocab, a.dim = (int)v->dim, a.segments = (int)p.segments, a.wide = (int)v->targets_wide;
    a.softcap = softcap, a.z = nullptr, a.z_ld = 0;
    auto kernel = few_of<false>(v->type, p.blocks, v->rows, softcap > 0.f);
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.segments, few_blocks(v->rows)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(vocab_few_join_kernel, dim3((unsigned)v->rows), dim3(256), 0, stream, a, loss, lse);
    return launch_status(fn);
}

template <class E>
void few_grad_kernels(const FewGradPlan &p, const FewArgs &f, const FewGradArgs &g, const float *lse, const float *weight, hipStream_t stream) {
    constexpr int N = 16 / sizeof(E);
    E *dz = static_cast<E *>(const_cast<void *>(g.dz)), *dzt = static_cast<E *>(const_cast<void *>(g.dzt));
    hipLaunchKernelGGL(vocab_few_dz_kernel<E>, dim3((unsigned)((p.z_ld + 255) / 256), p.kp / N), dim3(256), 0, stream, f, lse, weight, dz, dzt,
                       p.dz_rows, p.kp);
    if (g.dx) {
        FewGradArgs d = g;
        d.per = p.dx_per;
        auto kernel = p.rb == 1 ? vocab_few_dx_kernel<E, 1> : p.rb == 2 ? vocab_few_dx_kernel<E, 2> : vocab_few_dx_kernel<E, 4>;
        auto join = p.rb == 1   ? vocab_few_dx_join_kernel<E, 1>
                    : p.rb == 2 ? vocab_few_dx_join_kernel<E, 2>
                                : vocab_few_dx_join_kernel<E, 4>;
        hipLaunchKernelGGL(kernel, dim3(p.dx_splits, p.columns), dim3(256), 0, stream, d);
        hipLaunchKernelGGL(join, dim3((p.columns * N * p.rb * 64 + 255) / 256), dim3(256), 0, stream, d);
    }
    if (g.dw) {
        FewGradArgs d = g;
        d.per = p.dw_per, d.across = p.across;
        d.stream = d.dim * sizeof(E) % 128 == 0 && aligned(d.dw, 16) && (int64_t)d.vocab * d.dim * (int64_t)sizeof(E) > 1 << 28;
        auto kernel = p.kb == 1 ? vocab_few_dw_kernel<E, 1> : p.kb == 2 ? vocab_few_dw_kernel<E, 2> : vocab_few_dw_kernel<E, 4>;
        hipLaunchKernelGGL(kernel, dim3(p.dw_chunks, p.across ? (p.columns + 3) / 4 : p.columns), dim3(256), 0, stream, d);
    }
}

void fill_behind(const noise_vocab_t *v, void *dw, int64_t width, hipStream_t stream) {
    if (!dw || width <= v->vocab) return;
    const int64_t halves = v->type == NOISE_FP32 ? 2 : 1, n = (width - v->vocab) * v->dim * halves;
    hipLaunchKernelGGL(vocab_fill_kernel, dim3(n < 256 * 1024 ? (unsigned)((n + 255) / 256) : 1024), dim3(256), 0, stream,
                       static_cast<uint16_t *>(dw) + v->vocab * v->dim * halves, n);
}

int run_few_grad(const char *fn, const noise_vocab_t *v, float softcap, const float *weight, float *loss, const float *given, void *dx,
                 void *dw, int64_t width, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    const FewPlan q = few_plan(v);
    const FewGradPlan p = few_grad_plan(v);
    NOISE_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes,
                    "%s: workspace of %lld bytes (16 B aligned) required", fn, (long long)p.bytes);
    char *ws = static_cast<char *>(workspace);
    FewArgs f = {};
    f.x = v->x, f.w = v->weight, f.targets = v->targets, f.x_ld = v->x_stride, f.w_ld = v->weight_stride;
    f.zt = reinterpret_cast<float *>(ws);
    f.partial = given ? nullptr : reinterpret_cast<float2 *>(ws + q.at_partial);
    f.rows = (int)v->rows, f.vocab = (int)v->vocab, f.dim = (int)v->dim, f.segments = (int)q.segments, f.wide = (int)v->targets_wide;
    f.softcap = softcap, f.z = reinterpret_cast<float *>(ws + p.at_z), f.z_ld = p.z_ld;
    float *lse = reinterpret_cast<float *>(ws + p.at_lse);
    auto kernel = few_of<true>(v->type, q.blocks, v->rows, softcap > 0.f);
    hipLaunchKernelGGL(kernel, dim3((unsigned)q.segments, few_blocks(v->rows)), dim3(256), 0, stream, f);
    if (!given) hipLaunchKernelGGL(vocab_few_join_kernel, dim3((unsigned)v->rows), dim3(256), 0, stream, f, loss, lse);
    FewGradArgs g = {};
    g.x = v->x, g.w = v->weight, g.targets = v->targets, g.x_ld = v->x_stride, g.w_ld = v->weight_stride;
    g.dz = ws + p.at_dz, g.dzt = ws + p.at_dzt, g.slabs = reinterpret_cast<float *>(ws + p.at_slabs), g.dx = dx, g.dw = dw;
    g.z_ld = p.z_ld, g.rows = f.rows, g.vocab = f.vocab, g.dim = f.dim, g.wide = f.wide, g.blocks = p.columns, g.splits = p.dx_splits;
    if (v->type == NOISE_FP32) few_grad_kernels<float>(p, f, g, given ? given : lse, weight, stream);
    else few_grad_kernels<__bf16>(p, f, g, given ? given : lse, weight, stream);
    fill_behind(v, dw, width, stream);
    return launch_status(fn);
}

// loss and lse (out, or with `given` lse in); dx and dw where grad
int run(const char *fn, const noise_vocab_t *v, float softcap, const float *weight, float *loss, float *lse, const float *given,
        void *dx, void *dw, int64_t width, bool grad, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    const Plan p = plan_of(v, grad);
    NOISE_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes,
                    "%s: workspace of %lld bytes (16 B aligned) required", fn, (long long)p.bytes);
    char *ws = static_cast<char *>(workspace);
    int *place = reinterpret_cast<int *>(ws + p.at_int), *live = place + p.rows, *target = live + p.rows, *count = target + p.rows;
    float *f = reinterpret_cast<float *>(ws + p.at_float);
    float *packed_weight = f, *packed_lse = f + p.rows, *zt = f + 2 * p.rows, *scales = f + 3 * p.rows,
          *weight_max = scales + 4, *maxima = weight_max + kLiveParts;
    const int64_t rows = v->rows;
    const int64_t parts = (rows + 1023) / 1024 < kLiveParts ? (rows + 1023) / 1024 : kLiveParts, chunk = up((rows + parts - 1) / parts, 1024);
    const int live_parts = (int)((rows + chunk - 1) / chunk);
    hipLaunchKernelGGL(vocab_live_kernel, dim3(live_parts), dim3(1024), 0, stream, v->targets, (int)v->targets_wide, rows, chunk,
                       v->vocab, weight, given, count, live, place, target, packed_weight, packed_lse, weight_max);
    HeadArgs a = {};
    a.x = Operand{reinterpret_cast<__bf16 *>(ws + p.at_x), p.ld, p.rows * p.ld};
    a.w = p.pack_w ? Operand{reinterpret_cast<__bf16 *>(ws + p.at_w), p.ld, v->vocab * p.ld}
                   : Operand{static_cast<const __bf16 *>(v->weight), v->weight_stride, 0};
    PackArgs k = {};
    k.src[0] = v->x, k.src[1] = v->weight, k.src_ld[0] = v->x_stride, k.src_ld[1] = v->weight_stride;
    k.rows[0] = rows, k.rows[1] = v->vocab, k.padded[0] = p.rows, k.padded[1] = p.pack_w ? v->vocab : 0;
    k.to[0] = a.x, k.to[1] = a.w, k.dim = v->dim, k.place = place, k.count = count;
    k.max = maxima, k.weight_max = weight_max, k.live_parts = live_parts, k.scales = scales, k.dx = dx, k.loss = loss, k.lse = lse;
    k.piece = p.piece, k.pieces = p.pieces, k.tiles_m = (uint32_t)((p.ld + Tile::MT - 1) / Tile::MT);
    k.cuts = grad ? reinterpret_cast<uint2 *>(ws + p.at_cuts) : nullptr, k.need_dx = dx != nullptr, k.need_dw = dw != nullptr;
    if (p.split) hipLaunchKernelGGL(vocab_max_kernel, dim3(kMaxParts, 2), dim3(256), 0, stream, k, maxima);
    const int64_t most = p.rows > k.padded[1] ? p.rows : k.padded[1], packs = (most + 3) / 4;
    hipLaunchKernelGGL((p.split ? vocab_pack_kernel<float, true> : vocab_pack_kernel<__bf16, false>),
                       dim3((unsigned)(packs < 4096 ? packs : 4096), p.pack_w ? 2 : 1), dim3(256), 0, stream, k);
    a.count = count, a.live = live, a.target = target, a.scales = scales;
    a.weight = weight ? packed_weight : nullptr;
    a.lse = packed_lse, a.zt = zt, a.partial = reinterpret_cast<float2 *>(ws + p.at_partial);
    a.segments = (int)p.segments, a.vocab = (int)v->vocab, a.dim = (int)v->dim, a.nk = p.nk, a.softcap = softcap;
    a.w_k = p.pack_w ? p.ld : v->dim;
    fill_behind(v, dw, width, stream);
    const int threads = 64 * Tile::NW;
    const bool cap = softcap > 0.f;
    for (int64_t i = 0; i < p.pieces; ++i) {
        a.row0 = i * p.piece, a.piece = p.rows - a.row0 < p.piece ? p.rows - a.row0 : p.piece;
        a.tiles_m = (int)((v->vocab + Tile::MT - 1) / Tile::MT);
        const dim3 tiles((unsigned)(a.tiles_m * (a.piece / Tile::NT)));
        a.dz = Operand{reinterpret_cast<__bf16 *>(ws + p.at_dz), p.vocab_ld, p.piece * p.vocab_ld};
        const bool store = grad && !p.split, few = p.few;
        if (few) {
            const FewPlan q = few_plan(v);
            FewArgs f = {};
            f.x = v->x, f.w = v->weight, f.targets = v->targets, f.x_ld = v->x_stride, f.w_ld = v->weight_stride;
            f.z = reinterpret_cast<float *>(ws + p.at_z), f.z_ld = up(v->vocab, 32);
            f.zt = reinterpret_cast<float *>(ws + p.at_few);
            f.partial = given ? nullptr : reinterpret_cast<float2 *>(ws + p.at_few + q.at_partial);
            float *own = reinterpret_cast<float *>(ws + p.at_few + up(q.bytes, 16));
            f.rows = (int)rows, f.vocab = (int)v->vocab, f.dim = (int)v->dim, f.segments = (int)q.segments, f.softcap = softcap;
            f.wide = (int)v->targets_wide;
            auto kernel = few_of<true>(v->type, q.blocks, rows, cap);
            hipLaunchKernelGGL(kernel, dim3((unsigned)q.segments, few_blocks(rows)), dim3(256), 0, stream, f);
            if (!given) hipLaunchKernelGGL(vocab_few_join_kernel, dim3((unsigned)rows), dim3(256), 0, stream, f, loss, own);
            // (dW's product reads whole stages of rows)
            hipLaunchKernelGGL((p.split ? vocab_z_dz_kernel<true> : vocab_z_dz_kernel<false>),
                               dim3((unsigned)up(rows, Tile::BK), (unsigned)((p.vocab_ld + kDzEntries - 1) / kDzEntries)), dim3(256), 0, stream, a,
                               f.z, f.z_ld, given ? given : own);
        } else if (!given) {
            auto kernel = p.split ? loss_of<true, false>(softcap) : store ? loss_of<false, true>(softcap) : loss_of<false, false>(softcap);
            hipLaunchKernelGGL(kernel, tiles, dim3(threads), 0, stream, a);
            if (store) hipLaunchKernelGGL(vocab_lse_dz_kernel, dim3((unsigned)a.piece), dim3(256), 0, stream, a, loss);
            else hipLaunchKernelGGL(vocab_lse_kernel, dim3((unsigned)(a.piece / 4)), dim3(256), 0, stream, a, loss, lse);
        }
        if (!grad) continue;
        if (!few && (given || !store)) {
            auto kernel = p.split ? dz_of<true>(softcap) : dz_of<false>(softcap);
            hipLaunchKernelGGL(kernel, tiles, dim3(threads), 0, stream, a);
        }
        GradArgs g = {};
        const int64_t per = p.ld / 8;
        g.tiles_m = (int)k.tiles_m, g.cut = k.cuts + i;
        g.add = i > 0, g.fp32 = p.split;
        if (dx) {
            g.dx.out = dx, g.dx.slabs = reinterpret_cast<float *>(ws + p.at_dx), g.dx.groups = (uint32_t)p.dx_groups;
            // (past kSplitTiles / 2 tiles nothing is split)
            const int64_t most = kSplitTiles / 2 / g.tiles_m * Tile::NT;
            if (p.dx_slabs) g.dx.sums = (uint32_t)(((a.piece < most ? a.piece : most) * per + 255) / 256);
        }
        if (dw) {
            g.dw.out = i + 1 == p.pieces ? dw : nullptr, g.dw.slabs = reinterpret_cast<float *>(ws + p.at_dw);
            g.dw.sum = p.pieces > 1 ? reinterpret_cast<float *>(ws + p.at_sum) : nullptr;
            g.dw.groups = (uint32_t)p.dw_groups;
            if (p.dw_slabs) g.dw.sums = (uint32_t)((v->vocab * per + 255) / 256);
        }
        if (g.dx.groups + g.dw.groups)
            hipLaunchKernelGGL((p.split ? vocab_grad_kernel<Tile, true> : vocab_grad_kernel<Tile, false>),
                               dim3(g.dx.groups + g.dw.groups), dim3(threads), 0, stream, a, g);
        if (g.dx.sums + g.dw.sums)
            hipLaunchKernelGGL((p.split ? vocab_sum_kernel<Tile, true> : vocab_sum_kernel<Tile, false>),
                               dim3(g.dx.sums + g.dw.sums), dim3(256), 0, stream, a, g);
    }
    return launch_status(fn);
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int64_t noise_vocab_workspace_bytes(const noise_vocab_t *v, int with_grad) {
    clear_error();
    if (check("noise_vocab_workspace_bytes", v, 0.f)) return -1;
    if (v->rows == 0) return 0;
    if (with_grad) return few_grad_rows(v) ? few_grad_plan(v).bytes : plan_of(v, true).bytes;
    return few_rows(v, false) ? few_plan(v).bytes : plan_of(v, false).bytes;
}

extern "C" int noise_vocab_loss(const noise_vocab_t *v, float softcap, float *loss, float *lse, void *workspace,
                                int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_vocab_loss";
    if (int e = check(fn, v, softcap)) return e;
    if (v->rows == 0) return NOISE_OK;
    NOISE_CHECK_ARG(loss && aligned(loss, 4) && aligned(lse, 4), "%s: loss NULL or not 4 B aligned", fn);
    if (few_rows(v, false)) return run_few(fn, v, softcap, loss, lse, workspace, workspace_bytes, (hipStream_t)stream);
    return run(fn, v, softcap, nullptr, loss, lse, nullptr, nullptr, nullptr, 0, false, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int noise_vocab_grad(const noise_vocab_t *v, float softcap, const float *weight, const float *lse, float *loss, void *dx,
                                void *dweight, int64_t width, void *workspace, int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_vocab_grad";
    if (int e = check(fn, v, softcap)) return e;
    const size_t size = v->type == NOISE_BF16 ? 2 : 4;
    NOISE_CHECK_ARG((lse != nullptr) != (loss != nullptr) || v->rows == 0, "%s: either lse in or loss out", fn);
    NOISE_CHECK_ARG(aligned(weight, 4) && aligned(lse, 4) && aligned(loss, 4) && aligned(dx, size) && aligned(dweight, size),
                    "%s: a pointer is not aligned to its type", fn);
    NOISE_CHECK_ARG(!dweight || (width >= v->vocab && width <= (1 << 30)), "%s: dweight needs vocab <= width", fn);
    if (v->rows == 0) return NOISE_OK;
    if (few_grad_rows(v))
        return run_few_grad(fn, v, softcap, weight, loss, lse, dx, dweight, width, workspace, workspace_bytes, (hipStream_t)stream);
    return run(fn, v, softcap, weight, loss, nullptr, lse, dx, dweight, width, true, workspace, workspace_bytes, (hipStream_t)stream);
}
