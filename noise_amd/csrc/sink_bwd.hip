// Backward pass of the attention with a sliding window and first tokens that stay visible, without atomics:
//   delta_i = sum_d dO_id (o + o_rest)_id,  p_ij = 2^(c s_ij - lse_i),  dS = p (dO V^T - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// Two kernels recompute the scores. sink_dq_kernel walks the key tiles of 128 queries (4 waves of 32) with transposed scores, as
// the forward pass does, and leaves delta and lse as the second kernel wants them. sink_dkv_kernel walks the query tiles of
// 128 keys (4 waves of 32, keys and values in registers) over all query heads of the key head. In both a lane's scores and
// their gradients are the operand of the product that adds them up, so neither passes through LDS; the tiles that walk
// by are copied into two LDS stages and read by rows and by columns. The lists of query tiles of the first tokens' keys reach
// to the end of the sequence, far past the window: a list is cut into parts of a fixed length, each part's sums go to the
// workspace in fp32 and sink_join_kernel adds them in order.
//
// Recomputing the scores in both kernels costs 8 products per pair where 5 would do (dQ's takes two); it keeps dQ's partial
// sums out of memory and their order fixed. Heads of 128 hold 250 registers, two waves per SIMD. 16384 tokens, 16 heads of 128
// on 4, window 2048, 4 first tokens: sink_dq_kernel 510 us (1.0 PFLOP/s), sink_dkv_kernel 510 us (1.0 PFLOP/s), matrix
// cores busy 0.52 and 0.49 of the time and the waves waiting for LDS reads between the products. 8 x 2048 tokens, 8 heads of
// 64, window 1024: 67 us (770 TFLOP/s) and 62 us (830), with the vector work on the scores (0.58 and 0.42 of the cycles) beside
// the products (0.40 and 0.41).
#include "sink_common.hpp"

namespace noise {
namespace {

constexpr int kTileRows = 64;  // rows of the tiles that walk by
constexpr int kOwnQ = 128;     // queries of a workgroup (dq)

struct BwdArgs {
    Rows q, k, v, o, rest, d_o, dq, dk, dv;
    const float *lse;
    float *nlse, *ndelta;    // -lse / c and -delta, [batch * heads][tokens]
    float *parts;
    const void *lengths;
    int64_t first;
    int wide, tokens, heads, kv_heads, group, window, sinks;
    int tiles;                       // of queries (dq) or keys (dk, dv)
    int rows;                        // batch * heads (dq) or batch * kv_heads (dk, dv)
    int sink_tiles, sink_parts, band_parts;  // key tiles with first tokens; most parts of each kind
    int sink_part, part;             // query tiles per part of each kind
    float scale, scale_log2;
};

__device__ __forceinline__ int seq_len(const BwdArgs &a, int b) {
    int len = a.tokens;
    if (a.lengths) {
        const int64_t n = at_wide(a.lengths, a.wide, b);
        len = n < 0 ? 0 : n < len ? (int)n : len;
        len = __builtin_amdgcn_readfirstlane(len);
    }
    return len;
}

// A tile's copies into its half of a stage by 4 waves; `rows` of its rows are there (1 or more), past them the last one is taken
template <int D>
struct Copies {
    using TL = Tile<D>;
    static constexpr int kTile = kTileRows * TL::RB, kStage = 2 * kTile;
    static constexpr int CPW = kTile / 1024 / 4;  // copies per wave and tensor
    static_assert(4 * TL::RPC % 16 == 0, "uniform swizzle");
    int r0, chunk, wave;
    __device__ Copies(int wave_, int lane) : wave(wave_) {
        r0 = TL::RPC * wave + lane / TL::CPR;
        chunk = TL::swb(r0, lane % TL::CPR);
    }
    __device__ __forceinline__ void one(const Rows &t, const __bf16 *tile, int rows, unsigned st) const {
        if (rows < kTileRows) {
#pragma unroll
            for (int i = 0; i < CPW; ++i) {
                const int r = i * 4 * TL::RPC + r0;
                lds_dma16_at(tile, (unsigned)(r < rows ? r : rows - 1) * (unsigned)t.s_t * 2 + chunk * 16,
                             st + (4 * i + wave) * 1024);
            }
        } else {
            const unsigned off = (unsigned)(r0 * (int)t.s_t * 2 + chunk * 16);
            const int64_t step = 4 * TL::RPC * t.s_t;
#pragma unroll
            for (int i = 0; i < CPW; ++i, tile += step) lds_dma16_at(tile, off, st + (4 * i + wave) * 1024);
        }
    }
};

// Fragments of a tile (a stage's half): rows in the order sigma, and columns (as a source, lane 16 g + i addresses row
// 8 (g / 2) + i / 4 (+ 16 s, + 4), columns 16 (g % 2) + 4 (i % 4) .. + 4 (+ 32 db: offset ^ 64 db))
template <int D>
struct Frags {
    using TL = Tile<D>;
    int rows, cols;
    __device__ Frags(int lane) {
        const int sj = sigma(lane & 31), hf = lane >> 5, r = 8 * hf + ((lane & 15) >> 2);
        rows = sj * TL::RB + (TL::swb(sj, hf) << 4);
        cols = r * TL::RB + (TL::swb(r, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + 8 * (lane & 1);
    }
    // rows 32 blk + sigma(j), k-step s
    __device__ __forceinline__ bf16x8 row(const char *tile, int blk, int s) const {
        return *reinterpret_cast<const bf16x8 *>(tile + (rows ^ (32 * s)) + blk * 32 * TL::RB);
    }
    // columns 32 db .., rows 16 s .. of the tile (the second read's four rows differ in the chunk's lowest bit)
    __device__ __forceinline__ bf16x8 col(const char *tile, int db, int s) const {
        const char *p = tile + 16 * TL::RB * s;
        return cat(lds_read_tr16(p + (cols ^ (64 * db))), lds_read_tr16(p + 4 * TL::RB + (cols ^ (64 * db) ^ 16)));
    }
};

// a wave's 32 x D block, held as [D / 32] transposed 32 x 32 results, times mul, stored as rows of bf16 through its own LDS:
// rows [r0, end) of the tensor, those from `zero` on as zeros
template <int D>
__device__ __forceinline__ void store_block(const f32x16 (&acc)[D / 32], float mul, const Rows &t, __bf16 *base, int r0,
                                            int end, int zero, char *lds, int lane) {
    using TL = Tile<D>;
    constexpr int kPitch = D + 8;
    __bf16 *stg = reinterpret_cast<__bf16 *>(lds);
    const int j = lane & 31, hf = lane >> 5;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (__bf16)(r0 + j < zero ? acc[db][4 * g + e] * mul : 0.f);
            store_bf16x4(stg + j * kPitch + 32 * db + 8 * g + 4 * hf, v);
        }
    wave_lds_sync();
#pragma unroll
    for (int it = 0; it < TL::CPR / 2; ++it) {
        const int c = it * 64 + lane, r = c / TL::CPR, ch = c % TL::CPR;
        if (r0 + r < end) store_bf16x8(base + (int64_t)(r0 + r) * t.s_t + ch * 8, load_bf16x8(stg + r * kPitch + ch * 8));
    }
    wave_lds_sync();
}

// SPLIT: 8 waves, every second key tile by either half, whose sums are added in LDS
template <int D, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 512 : 256, 2) void sink_dq_kernel(BwdArgs a) {
    using TL = Tile<D>;
    using CP = Copies<D>;
    constexpr int KS = D / 16, DB = D / 32, HALVES = SPLIT ? 2 : 1;
    __shared__ __attribute__((aligned(16))) char lds[2 * HALVES * CP::kStage];
    const int64_t wg = a.first + blockIdx.x;
    const int round = (int)(wg / a.rows), qt = a.tiles - 1 - round;
    const int row = row_of((int)(wg % a.rows), round, a.rows, a.lengths != nullptr);
    const int b = row / a.heads, h = row - b * a.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    const int len = seq_len(a, b), last = len - 1, q_lo = qt * kOwnQ;
    const int half = wave >> 2, q0w = q_lo + 32 * (wave & 3);
    __bf16 *dqb = a.dq.ptr + b * a.dq.s_b + h * a.dq.s_h;
    if (q_lo > last) {
        const int n = (a.tokens - q_lo < kOwnQ ? a.tokens - q_lo : kOwnQ) * TL::CPR;
        for (int c = tid; c < n; c += 256 * HALVES)
            store_bf16x8(dqb + (int64_t)(q_lo + c / TL::CPR) * a.dq.s_t + 8 * (c % TL::CPR), zero_bf16x8());
        return;
    }
    const __bf16 *Kb = a.k.ptr + b * a.k.s_b + (h / a.group) * a.k.s_h;
    const __bf16 *Vb = a.v.ptr + b * a.v.s_b + (h / a.group) * a.v.s_h;
    bf16x8 qf[KS], df[KS];
    float nd = 0.f, lse;
    {
        const int q = q0w + j < last ? q0w + j : last;
        const __bf16 *qp = a.q.ptr + b * a.q.s_b + h * a.q.s_h + (int64_t)q * a.q.s_t + 8 * hf;
        const __bf16 *dp = a.d_o.ptr + b * a.d_o.s_b + h * a.d_o.s_h + (int64_t)q * a.d_o.s_t + 8 * hf;
        const __bf16 *op = a.o.ptr + b * a.o.s_b + h * a.o.s_h + (int64_t)q * a.o.s_t + 8 * hf;
        const __bf16 *rp = a.rest.ptr + b * a.rest.s_b + h * a.rest.s_h + (int64_t)q * a.rest.s_t + 8 * hf;
        const int64_t li = (int64_t)row * a.tokens + q;
        lse = a.lse[li];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = load_bf16x8(qp + 16 * s);
            df[s] = load_bf16x8(dp + 16 * s);
            const bf16x8 o = load_bf16x8(op + 16 * s), rest = load_bf16x8(rp + 16 * s);
#pragma unroll
            for (int e = 0; e < 8; ++e) nd -= (float)df[s][e] * ((float)o[e] + (float)rest[e]);
        }
        nd += swap_halves(nd);
        if (hf == 0 && half == 0 && q0w + j <= last) {
            a.nlse[li] = -lse / a.scale_log2;
            a.ndelta[li] = nd;
        }
    }
    vm_wait<0>();
    const int W = a.window, n_sinks = a.sinks;
    const int q_hi = q_lo + kOwnQ - 1 < last ? q_lo + kOwnQ - 1 : last;
    const int band = (q_lo > W ? q_lo - W : 0) / kTileRows;
    const int sunk = (n_sinks + kTileRows - 1) / kTileRows < band ? (n_sinks + kTileRows - 1) / kTileRows : band;
    const int nt = sunk + q_hi / kTileRows - band + 1;
    auto tile_k0 = [&](int t) { return (t < sunk ? t : t - sunk + band) * kTileRows; };
    const CP cp(wave & 3, lane);
    const Frags<D> frags(lane);
    const unsigned lb = lds_addr(lds);
    auto issue = [&](int i) {
        const int t = i * HALVES + half;
        if (t >= nt) return;
        const unsigned st = lb + ((i & 1) * HALVES + half) * CP::kStage;
        const int k0 = tile_k0(t);
        cp.one(a.k, Kb + k0 * a.k.s_t, len - k0, st);
        cp.one(a.v, Vb + k0 * a.v.s_t, len - k0, st + CP::kTile);
    };
    f32x16 dq[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) dq[db] = f32x16{};
    const int wq_lo = q0w, wq_hi = q0w > last ? -1 : q0w + 31 < last ? q0w + 31 : last;
    const float c2 = a.scale_log2;
    const int rounds = (nt + HALVES - 1) / HALVES;
    issue(0);
#pragma unroll 1
    for (int i = 0; i < rounds; ++i) {
        vm_wait<0>();
        __syncthreads();   // round i's tiles landed, and every wave is past round i - 1
        if (i + 1 < rounds) issue(i + 1);
        const int t = i * HALVES + half;
        if (t >= nt) continue;
        const int k0 = tile_k0(t);
        if (k0 > wq_hi || (k0 + kTileRows - 1 < wq_lo - W && k0 >= n_sinks)) continue;
        const char *kt = lds + ((i & 1) * HALVES + half) * CP::kStage, *vt = kt + CP::kTile;
        const bool causal_edge = k0 + kTileRows - 1 > wq_lo, window_edge = k0 < wq_hi - W;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            // (the fragments' addresses are formed anew in each block: kept over the loop, they would push registers out to memory)
            Frags<D> fr = frags;
            asm volatile("" : "+v"(fr.rows), "+v"(fr.cols));
            f32x16 sc = f32x16{}, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = nd;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                sc = mfma32x32x16(fr.row(kt, kb, s), qf[s], sc);
                dp = mfma32x32x16(fr.row(vt, kb, s), df[s], dp);
            }
            if (causal_edge || window_edge) {
                // as in the forward pass: key c = 16 (r / 8) + r % 8 from here
                int d0 = q0w + j - k0 - 32 * kb - 8 * hf, ds = n_sinks - k0 - 32 * kb - 8 * hf;
                unsigned wd = (unsigned)(d0 - W > ds ? d0 - W - ds : 0);
                asm volatile("" : "+v"(d0), "+v"(wd), "+v"(ds));
                if (causal_edge)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[r] = 16 * (r >> 3) + (r & 7) <= d0 ? sc[r] : -__builtin_inff();
                if (window_edge)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sc[r] = (unsigned)(16 * (r >> 3) + (r & 7) - ds) >= wd ? sc[r] : -__builtin_inff();
            }
            // the scores' gradients as two bf16 each, of 16 bits together: a row's add up to zero, and with keys that have much in
            // common the roundings of a single one (up to 2^-8 each) would outweigh the result's own (dq's error against 64 bits, 300
            // keys and 70 first tokens: 3.1e-3 with one, 2.2e-3 with two, 1.7e-3 the rounding of the result alone; a third
            // more products, 55 -> 67 us at 8 x 2048 tokens, 8 heads of 64)
            bf16x8 g[2], rest[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = exp2_fast(__builtin_fmaf(sc[r], c2, -lse)) * dp[r];
                g[r >> 3][r & 7] = (__bf16)x;
                rest[r >> 3][r & 7] = (__bf16)(x - (float)(__bf16)x);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int d0 = 0; d0 < DB; d0 += 2) {
                    const bf16x8 x = fr.col(kt, d0, 2 * kb + s), y = fr.col(kt, d0 + 1, 2 * kb + s);
                    dq[d0] = mfma32x32x16(x, g[s], dq[d0]);
                    dq[d0 + 1] = mfma32x32x16(y, g[s], dq[d0 + 1]);
                    dq[d0] = mfma32x32x16(x, rest[s], dq[d0]);
                    dq[d0 + 1] = mfma32x32x16(y, rest[s], dq[d0 + 1]);
                }
        }
    }
    __syncthreads();
    constexpr int kPart = SPLIT ? DB * 16 * 64 * 4 : 32 * (D + 8) * 2;   // bytes of a wave's sums, or of its staged rows
    static_assert(32 * (D + 8) * 2 <= kPart && 4 * kPart <= 2 * HALVES * CP::kStage, "staging fits");
    char *mine = lds + (wave & 3) * kPart;
    if constexpr (SPLIT) {
        float *x = reinterpret_cast<float *>(mine) + 4 * lane;
        if (half) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4 *>(x + (db * 4 + g) * 256) =
                        f32x4{dq[db][4 * g], dq[db][4 * g + 1], dq[db][4 * g + 2], dq[db][4 * g + 3]};
        }
        __syncthreads();
        if (half) return;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(x + (db * 4 + g) * 256);
#pragma unroll
                for (int e = 0; e < 4; ++e) dq[db][4 * g + e] += v[e];
            }
        wave_lds_sync();
    }
    store_block<D>(dq, a.scale, a.dq, dqb, q0w, a.tokens, len, mine, lane);
}

// query tiles of key tile kt: first, and how many (of one query head)
__device__ __forceinline__ int query_tiles(const BwdArgs &a, int kt, int own, int len, int *first) {
    const int k_lo = kt * own, last = len - 1;
    *first = k_lo / kTileRows;
    if (k_lo > last) return 0;
    const int k_hi = k_lo + own - 1 + a.window;
    const int end = k_lo < a.sinks || k_hi > last ? last : k_hi;
    return end / kTileRows - *first + 1;
}

// KW: waves along the keys; with 2, two waves share each 32 keys, one for either half of the query tiles, and add up in LDS
template <int D, int KW>
__global__ __launch_bounds__(256, 2) void sink_dkv_kernel(BwdArgs a) {
    using TL = Tile<D>;
    using CP = Copies<D>;
    constexpr int KS = D / 16, DB = D / 32, kOwn = 32 * KW;
    __shared__ __attribute__((aligned(16))) char lds[2 * CP::kStage + 2 * 2 * kTileRows * 4];
    const int64_t wg = a.first + blockIdx.x;
    const int item = (int)(wg / a.rows), row = row_of((int)(wg % a.rows), item, a.rows, a.lengths != nullptr);
    // the first parts of all key tiles, then the second ones: the workgroups of an XCD go to its engines in turn, and one that
    // got all long parts would hold up the ones that follow
    const int ns = a.sink_tiles * a.sink_parts, bands = a.tiles - a.sink_tiles;
    const int kt = item < ns ? item % a.sink_tiles : a.sink_tiles + (item - ns) % bands;
    const int part = item < ns ? item / a.sink_tiles : (item - ns) / bands, size = item < ns ? a.sink_part : a.part;
    const int b = row / a.kv_heads, hk = row - b * a.kv_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    const int kw = wave % KW;
    const int len = seq_len(a, b), last = len - 1, k0w = kt * kOwn + 32 * kw;
    int first;
    const int nq = query_tiles(a, kt, kOwn, len, &first), total = a.group * nq, parts = (total + size - 1) / size;
    __bf16 *dkb = a.dk.ptr + b * a.dk.s_b + hk * a.dk.s_h, *dvb = a.dv.ptr + b * a.dv.s_b + hk * a.dv.s_h;
    if (part >= parts) {
        if (parts == 0 && part == 0) {
            const int n = (a.tokens - kt * kOwn < kOwn ? a.tokens - kt * kOwn : kOwn) * TL::CPR;
            for (int c = tid; c < n; c += 256) {
                const int64_t t = kt * kOwn + c / TL::CPR;
                store_bf16x8(dkb + t * a.dk.s_t + 8 * (c % TL::CPR), zero_bf16x8());
                store_bf16x8(dvb + t * a.dv.s_t + 8 * (c % TL::CPR), zero_bf16x8());
            }
        }
        return;
    }
    const int i0 = part * size, i1 = i0 + size < total ? i0 + size : total;
    bf16x8 kf[KS], vf[KS];
    {
        const int key = k0w + j < last ? k0w + j : last;
        const __bf16 *kp = a.k.ptr + b * a.k.s_b + hk * a.k.s_h + (int64_t)key * a.k.s_t + 8 * hf;
        const __bf16 *vp = a.v.ptr + b * a.v.s_b + hk * a.v.s_h + (int64_t)key * a.v.s_t + 8 * hf;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[s] = load_bf16x8(kp + 16 * s);
            vf[s] = load_bf16x8(vp + 16 * s);
        }
    }
    vm_wait<0>();
    const CP cp(wave, lane);
    const Frags<D> frags(lane);
    const unsigned lb = lds_addr(lds);
    // the list: query tiles first .. first + nq - 1 of the first head, then of the next; the copies are one tile ahead
    const int64_t q_step = kTileRows * a.q.s_t, d_step = kTileRows * a.d_o.s_t;
    int head, tile, q_next;
    const __bf16 *qp, *dop;
    const float *sp;
    auto seek = [&](int g, int t) {
        head = g;
        tile = t;
        q_next = (first + t) * kTileRows;
        const int h = hk * a.group + g;
        qp = a.q.ptr + b * a.q.s_b + h * a.q.s_h + (first + t) * q_step;
        dop = a.d_o.ptr + b * a.d_o.s_b + h * a.d_o.s_h + (first + t) * d_step;
        // waves 0 and 1: -lse / c and -delta of the tile's queries
        sp = (wave ? a.ndelta : a.nlse) + (int64_t)(b * a.heads + h) * a.tokens + q_next;
    };
    auto issue = [&](int i) {
        const unsigned st = lb + (i & 1) * CP::kStage;
        const int rows = len - q_next;
        cp.one(a.q, qp, rows, st);
        cp.one(a.d_o, dop, rows, st + CP::kTile);
        if (wave < 2)
            lds_dma4_at(sp, (unsigned)(lane < rows ? lane : rows - 1) * 4,
                        lb + 2 * CP::kStage + ((i & 1) * 2 + wave) * kTileRows * 4);
        if (tile + 1 == nq) {
            seek(head + 1, 0);
        } else {
            ++tile;
            q_next += kTileRows;
            qp += q_step;
            dop += d_step;
            sp += kTileRows;
        }
    };
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = dv[db] = f32x16{};
    const int W = a.window, n_sinks = a.sinks;
    // the queries that see this lane's key: key .. key + span (none: span -1)
    const int key = k0w + j;
    const int span = key > last ? -1 : (key < n_sinks || key + W > last ? last : key + W) - key;
    // ... and that see all of the wave's keys, or any
    const int all_lo = k0w + 31, all_hi = k0w + 31 > last ? -1 : k0w + W < last ? k0w + W : last;
    const int any_hi = k0w > last ? -1 : k0w < n_sinks || k0w + 31 + W > last ? last : k0w + 31 + W;
    const float c2 = a.scale_log2;
    seek(i0 / nq, i0 % nq);
    int q0 = q_next;
    issue(i0);
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        vm_wait<0>();
        __syncthreads();   // tile i landed, and every wave is past tile i - 1
        const int q_then = q_next;
        if (i + 1 < i1) issue(i + 1);
        const char *qt = lds + (i & 1) * CP::kStage, *dt = qt + CP::kTile;
        const float *stats = reinterpret_cast<const float *>(lds + 2 * CP::kStage) + (i & 1) * 2 * kTileRows;
#pragma unroll
        for (int x = 0; x < KW / 2; ++x) {
            const int qb = KW == 4 ? x : wave / KW, q = q0 + 32 * qb;
            if (q + 31 < k0w || q > any_hi) continue;
            // (as in sink_dq_kernel)
            Frags<D> fr = frags;
            asm volatile("" : "+v"(fr.rows), "+v"(fr.cols));
            // register r: query 16 (r / 8) + 8 hf + r % 8. The products accumulate onto -lse / c and -delta
            f32x16 sc, dp;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int at = 32 * qb + 16 * (r >> 3) + 8 * hf + (r & 7);
                const f32x4 x = *reinterpret_cast<const f32x4 *>(stats + at);
                const f32x4 y = *reinterpret_cast<const f32x4 *>(stats + kTileRows + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[r + e] = x[e], dp[r + e] = y[e];
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                sc = mfma32x32x16(fr.row(qt, qb, s), kf[s], sc);
                dp = mfma32x32x16(fr.row(dt, qb, s), vf[s], dp);
            }
            if (q < all_lo || q + 31 > all_hi) {
                // seen iff 0 <= query - key <= span: queries from q + 8 hf are c = 16 (r / 8) + r % 8
                int lo = key - q - 8 * hf;
                unsigned n = (unsigned)(span + 1);
                asm volatile("" : "+v"(lo), "+v"(n));
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sc[r] = (unsigned)(16 * (r >> 3) + (r & 7) - lo) < n ? sc[r] : -__builtin_inff();
            }
            bf16x8 p[2], g[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = exp2_fast(sc[r] * c2);
                p[r >> 3][r & 7] = (__bf16)e;
                g[r >> 3][r & 7] = (__bf16)(e * dp[r]);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    dv[db] = mfma32x32x16(fr.col(dt, db, 2 * qb + s), p[s], dv[db]);
                    dk[db] = mfma32x32x16(fr.col(qt, db, 2 * qb + s), g[s], dk[db]);
                }
        }
        q0 = q_then;
    }
    if constexpr (KW == 2) {
        // the second wave's sums onto the first's, through LDS
        __syncthreads();
        float *x = reinterpret_cast<float *>(lds) + kw * (DB * 16 * 64) + 4 * lane;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x16 &s = half ? dv[db] : dk[db];
                    f32x4 *at = reinterpret_cast<f32x4 *>(x + (db * 4 + g) * 256);
                    if (wave >= KW) *at = f32x4{s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
                }
            __syncthreads();
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x16 &s = half ? dv[db] : dk[db];
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(x + (db * 4 + g) * 256);
                    if (wave < KW) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * g + e] += v[e];
                    }
                }
            __syncthreads();
        }
        if (wave >= KW) return;
    }
    if (parts > 1) {
        // [dk, dv][db][g][lane][4] of each wave: whole lines
        float *out = a.parts + ((int64_t)(item * (int64_t)a.rows + row) * KW + kw) * (2 * DB * 16 * 64) + 4 * lane;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x16 &s = x ? dv[db] : dk[db];
                    *reinterpret_cast<f32x4 *>(out + ((x * DB + db) * 4 + g) * 256) =
                        f32x4{s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
                }
        return;
    }
    if constexpr (KW == 4) __syncthreads();
    char *stg = lds + kw * 32 * (D + 8) * 2;
    store_block<D>(dk, a.scale, a.dk, dkb, k0w, a.tokens, len, stg, lane);
    store_block<D>(dv, 1.f, a.dv, dvb, k0w, a.tokens, len, stg, lane);
}

// Adds the parts of key tiles that have several, in order. grid: (key tiles times rows, blocks of 32 dims of dk, then of dv), a
// wave per 32 keys, the same registers as above
template <int D, int KW>
__global__ __launch_bounds__(64 * KW) void sink_join_kernel(BwdArgs a, int band) {
    constexpr int DB = D / 32, kOwn = 32 * KW;
    const int kt = (band ? a.sink_tiles : 0) + blockIdx.x / a.rows, row = blockIdx.x % a.rows;
    const int b = row / a.kv_heads, hk = row - b * a.kv_heads;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = blockIdx.y / DB, db = blockIdx.y % DB;
    const int len = seq_len(a, b);
    int first;
    const int total = a.group * query_tiles(a, kt, kOwn, len, &first), size = band ? a.part : a.sink_part;
    const int parts = (total + size - 1) / size;
    if (parts < 2) return;
    const int ns = a.sink_tiles * a.sink_parts;
    const int item = kt < a.sink_tiles ? kt : ns + kt - a.sink_tiles;
    const int next = kt < a.sink_tiles ? a.sink_tiles : a.tiles - a.sink_tiles;   // items from part to part
    const int key = kt * kOwn + 32 * wave + (lane & 31);
    if (key >= a.tokens) return;
    const float *src = a.parts + ((int64_t)(item * (int64_t)a.rows + row) * KW + wave) * (2 * DB * 16 * 64) +
                       (x * DB + db) * 1024 + 4 * lane;
    f32x4 s[4] = {};
    for (int p = 0; p < parts; ++p)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            s[g] += *reinterpret_cast<const f32x4 *>(src + (int64_t)p * next * a.rows * KW * (2 * DB * 16 * 64) + g * 256);
    const Rows &t = x ? a.dv : a.dk;
    const float mul = x ? 1.f : a.scale;
    __bf16 *out = t.ptr + b * t.s_b + hk * t.s_h + (int64_t)key * t.s_t + 32 * db + 4 * (lane >> 5);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (__bf16)(s[g][e] * mul);
        store_bf16x4(out + 8 * g, v);
    }
}

// How the lists of query tiles are cut: a key tile with first tokens into at most sink_parts of sink_part tiles, the others into
// at most band_parts of `part`.
struct Plan {
    int64_t own, tiles, rows, sink_tiles, sink_parts, band_parts, sink_part, part, items;
    int64_t stats, bytes;
};
Plan plan(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t window, int64_t sinks) {
    Plan p;
    const int64_t group = heads / kv_heads, q_tiles = (tokens + kTileRows - 1) / kTileRows;
    window = window < tokens ? window : tokens;
    sinks = sinks < tokens ? sinks : tokens;
    p.rows = batch * kv_heads;
    // 64 keys (two waves on each 32, the queries halved between them) where 128 would leave the CUs without a second workgroup:
    // one sequence of 8192 tokens, 8 heads of 128 on 2, 290 us against 350 for the whole pass; 8 heads of 64, 8 x 2048
    // tokens (1024 of 128), 127 us with 128 keys, and no less with 64
    p.own = p.rows * ((tokens + 127) / 128) < 1024 ? 64 : 128;
    p.tiles = (tokens + p.own - 1) / p.own;
    p.sink_tiles = (sinks + p.own - 1) / p.own;
    const int64_t reach = (window + p.own - 1) / kTileRows + 1;
    const int64_t band = group * (reach < q_tiles ? reach : q_tiles);
    // the others' lists in all: whole ones, then the last tiles' shorter ones, step by step
    const int64_t step = p.own / kTileRows, whole = q_tiles > reach ? (q_tiles - reach) / step + 1 : 0;
    const int64_t full = whole < p.tiles ? whole : p.tiles, tail = p.tiles - full;
    const int64_t steps = p.rows * group * (full * reach + tail * (q_tiles - full * step) - step * (tail * (tail - 1) / 2));
    // as many parts as make 512 workgroups (two per CU) of them, six tiles or more each: 4096 tokens, 8 heads of 128 on 2,
    // window 1024 (128 lists): 185 us for the whole pass uncut, 104 in four. Each part's sums are written and read once more,
    // so lists that come near 512 (544: an odd few over do not matter) stay whole: 280 lists, 121 us whole, 135 in two
    int64_t cut = 544 * band / (steps > 0 ? steps : 1);
    cut = cut < band / 6 ? cut : band / 6;
    cut = cut > 1 ? cut : 1;
    p.part = (band + cut - 1) / cut;
    p.band_parts = p.sink_tiles < p.tiles ? (band + p.part - 1) / p.part : 0;
    // as long as the others' parts, or longer where many first tokens would make more than 1024 of them
    const int64_t least = (p.rows * p.sink_tiles * group * q_tiles + 1023) / 1024;
    p.sink_part = p.part > least ? p.part : least;
    p.sink_parts = p.sink_tiles ? (group * q_tiles + p.sink_part - 1) / p.sink_part : 0;
    p.items = p.sink_tiles * p.sink_parts + (p.tiles - p.sink_tiles) * p.band_parts;
    p.stats = (batch * heads * tokens * 4 + 15) / 16 * 16;
    p.bytes = 2 * p.stats;
    // (the first tokens' items come first: whole lists after them need no room)
    const int64_t held = p.band_parts > 1 ? p.items : p.sink_parts > 1 ? p.sink_tiles * p.sink_parts : 0;
    p.bytes += held * p.rows * p.own * head_dim * 2 * 4;
    return p;
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int64_t noise_sink_attention_bwd_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads,
                                                            int64_t kv_heads, int64_t head_dim, int64_t window,
                                                            int64_t sinks) {
    clear_error();
    const int st = check_sizes("noise_sink_attention_bwd_workspace_bytes", batch, tokens, tokens, heads, kv_heads,
                               head_dim, window, sinks);
    if (st) return st;
    if (batch == 0 || tokens == 0) return 0;
    return plan(batch, tokens, heads, kv_heads, head_dim, window, sinks).bytes;
}

extern "C" int noise_sink_attention_bwd(const noise_heads_t *q, const noise_heads_t *k, const noise_heads_t *v,
                                        const noise_heads_t *o, const noise_heads_t *o_rest, const noise_heads_t *d_o,
                                        const float *lse,
                                        const noise_heads_t *dq, const noise_heads_t *dk, const noise_heads_t *dv,
                                        const void *lengths, int lengths_wide, int64_t batch, int64_t tokens,
                                        int64_t head_dim, int64_t window, int64_t sinks, float scale, void *workspace,
                                        int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_sink_attention_bwd";
    NOISE_CHECK_ARG(q && k && v && o && o_rest && d_o && dq && dk && dv && q->heads == o->heads &&
                        q->heads == o_rest->heads && q->heads == d_o->heads &&
                        q->heads == dq->heads && k->heads == v->heads && k->heads == dk->heads && k->heads == dv->heads,
                    "%s: tensors missing or of other heads", fn);
    int st = check_sizes(fn, batch, tokens, tokens, q->heads, k->heads, head_dim, window, sinks);
    if (st || (st = check_scale(fn, scale))) return st;
    if (batch == 0 || tokens == 0) return NOISE_OK;
    NOISE_CHECK_ARG(lse && aligned(lse, 4), "%s: lse is required", fn);
    NOISE_CHECK_ARG(!lengths || aligned(lengths, lengths_wide ? 8 : 4), "%s: lengths misaligned", fn);
    const Plan p = plan(batch, tokens, q->heads, k->heads, head_dim, window, sinks);
    NOISE_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes,
                    "%s: workspace NULL, misaligned or below %lld bytes", fn, (long long)p.bytes);
    BwdArgs a;
    if ((st = check_heads(fn, "q", q, &a.q)) || (st = check_heads(fn, "k", k, &a.k)) ||
        (st = check_heads(fn, "v", v, &a.v)) || (st = check_heads(fn, "o", o, &a.o)) ||
        (st = check_heads(fn, "o_rest", o_rest, &a.rest)) || (st = check_heads(fn, "d_o", d_o, &a.d_o)) || (st = check_heads(fn, "dq", dq, &a.dq)) ||
        (st = check_heads(fn, "dk", dk, &a.dk)) || (st = check_heads(fn, "dv", dv, &a.dv)))
        return st;
    for (const Rows *t : {&a.q, &a.k, &a.v, &a.d_o})
        NOISE_CHECK_ARG(t->s_t >= 0 && t->s_t < kMaxStride, "%s: token strides of q, k, v and d_o must be below 2^25", fn);
    NOISE_CHECK_ARG(p.rows * p.items < (1 << 30), "%s: too many key tiles", fn);
    a.lse = lse;
    a.nlse = static_cast<float *>(workspace);
    a.ndelta = a.nlse + p.stats / 4;
    a.parts = a.ndelta + p.stats / 4;
    a.lengths = lengths; a.wide = lengths_wide;
    a.tokens = (int)tokens; a.heads = (int)q->heads; a.kv_heads = (int)k->heads; a.group = a.heads / a.kv_heads;
    a.window = (int)(window < tokens ? window : tokens);
    a.sinks = (int)(sinks < tokens ? sinks : tokens);
    a.sink_tiles = (int)p.sink_tiles; a.sink_parts = (int)p.sink_parts; a.band_parts = (int)p.band_parts;
    a.part = (int)p.part; a.sink_part = (int)(p.sink_part < INT32_MAX / 2 ? p.sink_part : INT32_MAX / 2);
    a.scale = scale; a.scale_log2 = scale * kLog2e;
    const bool narrow = head_dim == 64;
    auto launch = [&](void (*kernel)(BwdArgs), int64_t rows, int64_t items, int threads) {
        a.rows = (int)rows;
        for (a.first = 0; a.first < rows * items; a.first += kLaunchGroups) {
            const int64_t n = rows * items - a.first < kLaunchGroups ? rows * items - a.first : kLaunchGroups;
            hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3((unsigned)threads), 0, (hipStream_t)stream, a);
        }
    };
    a.tiles = (int)((tokens + kOwnQ - 1) / kOwnQ);
    // no more workgroups than CUs: two halves of the keys for each (4096 tokens, 4 heads of 64, causal: the whole pass 91 us
    // against 107)
    const bool split = batch * q->heads * a.tiles <= 256;
    launch(narrow ? (split ? sink_dq_kernel<64, true> : sink_dq_kernel<64, false>)
                  : (split ? sink_dq_kernel<128, true> : sink_dq_kernel<128, false>), batch * q->heads, a.tiles, split ? 512 : 256);
    const bool small = p.own == 64;
    a.tiles = (int)p.tiles;
    launch(narrow ? (small ? sink_dkv_kernel<64, 2> : sink_dkv_kernel<64, 4>)
                  : (small ? sink_dkv_kernel<128, 2> : sink_dkv_kernel<128, 4>), p.rows, p.items, 256);
    for (int band = 0; band < 2; ++band) {
        const int64_t n = band ? (p.band_parts > 1 ? p.tiles - p.sink_tiles : 0) : p.sink_parts > 1 ? p.sink_tiles : 0;
        if (n)
            hipLaunchKernelGGL(narrow ? (small ? sink_join_kernel<64, 2> : sink_join_kernel<64, 4>)
                                      : (small ? sink_join_kernel<128, 2> : sink_join_kernel<128, 4>),
                               dim3((unsigned)(n * p.rows), (unsigned)(head_dim / 32 * 2)),
                               dim3(small ? 128 : 256), 0, (hipStream_t)stream, a, band);
    }
    return launch_status(fn);
}
