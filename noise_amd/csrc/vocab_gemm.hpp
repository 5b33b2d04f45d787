// The matrix products of the vocabulary's cross entropy: C[m][n] = sum_k A(m, k) B(n, k) in fp32 for a tile of MT x NT, on
// v_mfma_f32_32x32x16 in bf16 or fp16. Either operand lies in memory with k along its rows ("plain") or with k across them
// ("crossed": the tile is then read by columns, with transposing LDS reads), so that no operand is transposed in memory.
// NW = WM x WN waves; a wave owns FB x NB blocks of 32 x 32. The tiles of BK steps of k go through NS stages in LDS by direct
// global -> LDS copies; the fragments of the next 16 steps are read while the present ones are multiplied.
//
// The rows of a 32-row block of A are taken in the order sigma (bits 2 and 3 of the index swapped), which makes register r of a
// lane's block stand for m = 16 (r / 8) + 8 (lane / 32) + r % 8, n = lane % 32: eight consecutive m, 16 B of 16-bit results.
//
// The tile is 256 x 256 with 8 waves of 128 x 64, 64 of k per stage and two stages (128 KB of LDS): 12 fragments read per 32
// products of 32 x 32 x 16, two waves per SIMD. It reaches 1.1 to 1.27 PFLOP/s in large products (2048 wide), a library's product
// 1.35; where k is short the start and end of a tile show: 0.95 in the gradients of 16384 x 4096 x 512, 0.72 and 0.58 in the losses
// of 776 and 512 columns, with their exponentials. Measured and slower: 4 waves of 128 x 128 (by 8 to 12 %); 256 x 128 with stages
// of 32 and two workgroups per CU (the same at k = 512, 15 % slower at 2048); the same: wave priorities, persistent workgroups
// whose next tile begins under the epilogue (1 to 2 % faster, which is not worth its code).
#pragma once
#include "common.hpp"
#include "mfma.hpp"

namespace noise {
namespace {

// A matrix of 16-bit values; values held as a sum of two have their second ones `lo` elements further
struct Operand {
    const __bf16 *ptr;
    int64_t ld, lo;
};

__device__ __forceinline__ int sigma32(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

template <bool F16>
__device__ __forceinline__ f32x16 mfma16bit(bf16x8 a, bf16x8 b, f32x16 c) {
    if constexpr (F16) {
        typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        return mfma32x32x16(a, b, c);
    }
}

// As lds_dma16_at, with an address of its own for each lane
__device__ __forceinline__ void lds_dma16_from(uint64_t at, unsigned la) {
    const unsigned l = (unsigned)__builtin_amdgcn_readfirstlane((int)la);
    unsigned save;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(save)
                 : "v"(at), "s"(l)
                 : "memory");
}

// One operand's tile of ROWS x BK in LDS and its copies by NW waves
template <int ROWS, int BK, int NW, bool CROSSED>
struct Side {
    static constexpr int kBytes = ROWS * BK * 2;
    static constexpr int RB = CROSSED ? ROWS * 2 : BK * 2;    // bytes per LDS row
    static constexpr int CPR = RB / 16, RPC = 1024 / RB;      // 16 B chunks per row, rows per wave-wide copy
    static constexpr int N = kBytes / 1024 / NW;              // copies per wave
    static constexpr int RPB = RB < 256 ? 256 / RB : 1;       // rows per 256 B of banks
    static_assert(kBytes % (1024 * NW) == 0 && N > 0, "whole copies per wave");
    // plain: 32 rows of a fragment read must lie on distinct banks; crossed: the four rows of a transposing read
    __device__ static int swz(int r, int c) { return CROSSED ? c ^ (4 * (r & 3)) : c ^ ((r / RPB) % CPR); }
    static_assert(CROSSED ? (CPR >= 16 && NW * RPC % 4 == 0) : (NW * RPC % (RPB * CPR) == 0 && 32 % (RPB * CPR) == 0), "uniform swizzle");

    uint64_t base;       // of the tile's first element
    unsigned off[N];     // this lane's byte offset of each copy
    int row, chunk;      // this lane's row of the first copy and its chunk
    int64_t ld;

    // last: the last row that exists (plain), or the last chunk of 8 columns (crossed), from the tile's first
    __device__ __forceinline__ void init(const Operand &o, int64_t first, int last, int wave, int lane) {
        ld = o.ld;
        base = (uint64_t)(o.ptr + (CROSSED ? first : first * o.ld));
        row = wave * RPC + lane / CPR;
        chunk = swz(row, lane % CPR);
        if (CROSSED && chunk > last) chunk = last;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row + i * NW * RPC;
            off[i] = (unsigned)((CROSSED || r < last ? r : last) * (uint32_t)ld * 2 + chunk * 16);
        }
    }
    // k: the stage's first; left: how many k from there on are in memory. Crossed: rows past them repeat the last one (the other
    // operand is zero there). Plain: chunks past them are read from `zeros`.
    __device__ __forceinline__ void copy(int64_t k, int64_t lo, int left, const void *zeros, unsigned to, int wave) const {
        const __bf16 *p = reinterpret_cast<const __bf16 *>(base) + lo + (CROSSED ? k * ld : k);
        to += wave * 1024;
        if (CROSSED && left < BK) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row + i * NW * RPC;
                lds_dma16_at(p, (unsigned)((r < left ? r : left - 1) * (uint32_t)ld * 2 + chunk * 16), to + i * NW * 1024);
            }
            return;
        }
        if (!CROSSED && left < BK) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds_dma16_from(8 * chunk < left ? (uint64_t)p + off[i] : (uint64_t)zeros, to + i * NW * 1024);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) lds_dma16_at(p, off[i], to + i * NW * 1024);
    }
};

// The fragments of B blocks of 32 rows from row r0 of a tile
template <int ROWS, int BK, int NW, bool CROSSED, bool SIGMA, int B>
struct Fragments {
    using S = Side<ROWS, BK, NW, CROSSED>;
    int at[CROSSED ? B : BK / 16];
    __device__ __forceinline__ void init(int r0, int lane) {
        if constexpr (CROSSED) {
            const int g = lane >> 4, q = (lane >> 2) & 3;
            int block = lane & 3;                     // this lane's 4 columns of the group's 16
            if (SIGMA) block = ((block & 1) << 1) | (block >> 1);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int col = r0 + 32 * b + 16 * (g & 1) + 4 * block;
                at[b] = (8 * (g >> 1) + q) * S::RB + S::swz(q, col >> 3) * 16 + 2 * (col & 7);
            }
        } else {
            const int j = SIGMA ? sigma32(lane & 31) : lane & 31;
#pragma unroll
            for (int s = 0; s < BK / 16; ++s) at[s] = (r0 + j) * S::RB + S::swz(j, 2 * s + (lane >> 5)) * 16;
        }
    }
    __device__ __forceinline__ bf16x8 get(const char *tile, int s, int b) const {
        if constexpr (CROSSED) {
            const char *p = tile + at[b] + s * 16 * S::RB;
            return cat(lds_read_tr16(p), lds_read_tr16(p + 4 * S::RB));
        } else {
            return *reinterpret_cast<const bf16x8 *>(tile + at[s] + b * 32 * S::RB);
        }
    }
};

template <int MT_, int NT_, int WM_, int WN_, int BK_, int NS_>
struct Tiling {
    static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, BK = BK_, NS = NS_, NW = WM * WN;
    static constexpr int FB = MT / WM / 32, NB = NT / WN / 32;
    static constexpr int kStage = (MT + NT) * BK * 2, kLds = NS * kStage;
    __device__ static int wm(int wave) { return wave % WM * (MT / WM); }
    __device__ static int wn(int wave) { return wave / WM * (NT / WN); }
};

// k per stage. Operands that are sums of two values have both in a stage, for half the k.
template <class T, bool SPLIT>
constexpr int kStep = SPLIT ? T::BK / 2 : T::BK;

// acc = the product over the stages first .. last - 1 of k. With SPLIT, operands are sums of two, multiplied hi hi + hi lo + lo hi
// from one reading of each. a_k: how many k A has in memory (plain: whole chunks of 8). Ends with a barrier.
template <class T, bool CA, bool CB, bool F16, bool SPLIT>
__device__ __forceinline__ void product(const Operand &a, int64_t a0, int a_last, const Operand &b, int64_t b0, int b_last, int first,
                                        int last, int64_t a_k, const void *zeros, char *lds, f32x16 (&acc)[T::FB][T::NB]) {
    constexpr int BK = kStep<T, SPLIT>, NS = T::NS, SPK = BK / 16, P = SPLIT ? 2 : 1;
    using SA = Side<T::MT, BK, T::NW, CA>;
    using SB = Side<T::NT, BK, T::NW, CB>;
    constexpr int G = P * (SA::N + SB::N);
    static_assert(NS >= 2 && NS <= 4 && G * (NS - 1) < 64 && SPK % 2 == 0, "pipeline depth");
    static_assert(P * (SA::kBytes + SB::kBytes) == T::kStage, "a stage");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned lbase = lds_addr(lds);
    SA sa;
    SB sb;
    sa.init(a, a0, a_last, wave, lane);
    sb.init(b, b0, b_last, wave, lane);
    Fragments<T::MT, BK, T::NW, CA, true, T::FB> fa;
    Fragments<T::NT, BK, T::NW, CB, false, T::NB> fb;
    fa.init(T::wm(wave), lane);
    fb.init(T::wn(wave), lane);
#pragma unroll
    for (int i = 0; i < T::FB; ++i)
#pragma unroll
        for (int j = 0; j < T::NB; ++j) acc[i][j] = f32x16{};
    const int n = last - first;
    auto issue = [&](int p) {
        const unsigned st = lbase + (p % NS) * T::kStage;
        const int64_t k = (int64_t)(first + p) * BK;
#pragma unroll
        for (int q = 0; q < P; ++q) {
            sa.copy(k, q ? a.lo : 0, a_k - k < BK ? (int)(a_k - k) : BK, zeros, st + q * SA::kBytes, wave);
            sb.copy(k, q ? b.lo : 0, BK, nullptr, st + P * SA::kBytes + q * SB::kBytes, wave);
        }
    };
    bf16x8 va[2][P][T::FB], vb[2][P][T::NB];
    auto fetch = [&](int buf, const char *st, int s) {
#pragma unroll
        for (int q = 0; q < P; ++q) {
#pragma unroll
            for (int i = 0; i < T::FB; ++i) va[buf][q][i] = fa.get(st + q * SA::kBytes, s, i);
#pragma unroll
            for (int j = 0; j < T::NB; ++j) vb[buf][q][j] = fb.get(st + P * SA::kBytes + q * SB::kBytes, s, j);
        }
    };
#pragma unroll
    for (int p = 0; p < NS; ++p)
        if (p < n) issue(p);
    vm_wait_groups<G, NS - 1>(n - 1 < NS - 1 ? n - 1 : NS - 1);
    __syncthreads();
    fetch(0, lds, 0);
#pragma unroll 1
    for (int p = 0; p < n; ++p) {
        const char *st = lds + (p % NS) * T::kStage;
#pragma unroll
        for (int s = 0; s < SPK; ++s) {
            const int cur = s & 1;
            if (s + 1 < SPK) {
                fetch(cur ^ 1, st, s + 1);
            } else if (p + 1 < n) {
                // stage p + 1 has landed for every wave, and every wave has its last fragments of stage p, whose slot
                // takes stage p + NS
                vm_wait_groups<G, NS - 2>(n - 2 - p < NS - 2 ? n - 2 - p : NS - 2);
                __syncthreads();
                if (p + NS < n) issue(p + NS);
                fetch(cur ^ 1, lds + ((p + 1) % NS) * T::kStage, 0);
            }
#pragma unroll
            for (int q = 0; q < 2 * P - 1; ++q)
#pragma unroll
                for (int i = 0; i < T::FB; ++i)
#pragma unroll
                    for (int j = 0; j < T::NB; ++j)
                        acc[i][j] = mfma16bit<F16>(va[cur][q == 2][i], vb[cur][q == 1][j], acc[i][j]);
        }
    }
    __syncthreads();
}

// Which tile workgroup wg of tiles_m x tiles_n takes. Workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles, within
// which 8 tiles of m follow one another before the next of n, so that the tiles that an XCD works on at a time share operands in
// its L2. (Groups of 4 or 16 took the same time.)
__device__ __forceinline__ void tile_of(int wg, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int tiles = tiles_m * tiles_n, x = wg & 7, each = tiles >> 3, more = tiles & 7;
    const int t = x * each + (x < more ? x : more) + (wg >> 3);
    const int group = t / (8 * tiles_n), m0 = group * 8, wide = tiles_m - m0 < 8 ? tiles_m - m0 : 8;
    const int u = t - group * 8 * tiles_n;
    tm = m0 + u % wide;
    tn = u / wide;
}

}  // namespace
}  // namespace noise
