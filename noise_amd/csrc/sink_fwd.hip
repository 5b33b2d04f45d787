// Forward pass of the attention with a sliding window and first tokens that stay visible.
//
// One pass over the visible key tiles with a running maximum and sum. A workgroup takes 256 queries of one head (8 waves of
// 32) and walks its list of 64-key tiles: those of the first tokens that lie before the window, then the window's. Per
// tile S^T = K Q^T, so that a lane holds 32 scores of one query and a row's maximum needs one exchange between the
// wave's halves, and O^T += V^T P^T with P straight from those registers (the K rows of each 32-key block are read in the
// order sigma, which makes a lane's 16 scores two runs of eight keys). Tiles are copied global -> LDS into a ring of four
// stages; V^T fragments come from transposing reads of the V tile. The waves work in two groups half a tile apart, one of each
// on every SIMD, so that one group's softmax (VALU) runs beside the other's products (matrix cores): per barrier group A
// does S, softmax and O of tile t, group B softmax and O of tile t - 1, then S of tile t.
//
// Heads of 128: bound by the matrix products (16384 tokens, 16 heads on 4, window 2048, 4 first tokens: 290 us, 890 TFLOP/s
// of the visible pairs, 1 PFLOP/s with the tiles' edges; a large bf16 product runs at 1250 here; matrix cores busy 0.44 of the
// time, vector units 0.45). Heads of 64: by the vector work on the scores and the products together, 64 and 34 % of the cycles
// (8 x 2048 tokens, 8 heads, window 1024, which 128-query workgroups take: 44 us, 590 TFLOP/s; 47 us with what the backward
// pass needs).
#include "sink_common.hpp"

namespace noise {
namespace {

constexpr int kBK = 64;    // keys per tile

enum { kPaired, kFour, kSplit };

struct FwdArgs {
    Rows q, k, v, o, rest;
    float *lse;
    const void *lengths;
    int64_t first;        // this launch's first workgroup
    int wide, tokens, heads, group, window, sinks, qtiles, rows;  // group: query heads per key head; rows: batch * heads
    float scale_log2;
};

// FORM: kPaired, as above, 256 queries by 8 waves, for long windows; kFour, 128 queries by 4 waves and two stages; for no more
// workgroups than there are CUs, kSplit, 128 queries by 8 waves, every second tile by either half, which are joined in LDS.
// TRAIN: with what the backward pass needs beside o, the rows' lse and o's own rounding error. The backward pass forms
// dP - dO.o, which nearly cancels where one weight is close to 1: there o's rounding (up to 2^-8 of o) would drown it. With o
// and its error, and with a running maximum that is exact (so that the largest weight is 1 and its rounding nothing), what is
// left is up to 2^-8 of the other weights' terms of dO.o, which vanish with them.
template <int D, int FORM, bool TRAIN>
__global__ __launch_bounds__(FORM == kFour ? 256 : 512) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 2, D == 64 ? 4 : 2)))
void sink_fwd_kernel(FwdArgs a) {
    using TL = Tile<D>;
    constexpr int RB = TL::RB, KS = D / 16, DB = D / 32, NW = FORM == kFour ? 4 : 8, NS = FORM == kPaired ? 4 : 2;
    constexpr int kBQ = FORM == kPaired ? 256 : 128, HALVES = FORM == kSplit ? 2 : 1;
    constexpr int kTile = kBK * RB, kStage = 2 * kTile;
    constexpr int CPW = kStage / 1024 / 4;   // copies per wave of group A and tile
    __shared__ __attribute__((aligned(16))) char lds[NS * HALVES * kStage];

    // the last query tiles (those with the most keys) of all heads first
    const int64_t wg = a.first + blockIdx.x;
    const int round = (int)(wg / a.rows), qt = a.qtiles - 1 - round;
    const int row = row_of((int)(wg % a.rows), round, a.rows, a.lengths != nullptr);
    const int b = row / a.heads, h = row - b * a.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    int len = a.tokens;
    if (a.lengths) {
        const int64_t n = at_wide(a.lengths, a.wide, b);
        len = n < 0 ? 0 : n < len ? (int)n : len;
        len = __builtin_amdgcn_readfirstlane(len);
    }
    const int wg_q_lo = qt * kBQ, last = len - 1;
    __bf16 *ob = a.o.ptr + b * a.o.s_b + h * a.o.s_h;
    if (wg_q_lo > last) {
        // queries past the length: zeros
        const int n = (a.tokens - wg_q_lo < kBQ ? a.tokens - wg_q_lo : kBQ) * TL::CPR;
        for (int c = tid; c < n; c += 64 * NW)
            store_bf16x8(ob + (int64_t)(wg_q_lo + c / TL::CPR) * a.o.s_t + 8 * (c % TL::CPR), zero_bf16x8());
        return;
    }
    const int W = a.window, n_sinks = a.sinks;
    const int half = FORM == kSplit ? wave >> 2 : 0, q0w = wg_q_lo + 32 * (FORM == kSplit ? wave & 3 : wave);
    const __bf16 *Qb = a.q.ptr + b * a.q.s_b + h * a.q.s_h;
    const __bf16 *Kb = a.k.ptr + b * a.k.s_b + (h / a.group) * a.k.s_h;
    const __bf16 *Vb = a.v.ptr + b * a.v.s_b + (h / a.group) * a.v.s_h;

    // rows past the last token are the last token's: such queries are not stored and such keys are seen by no query
    bf16x8 qf[KS];
    {
        const int q = q0w + j < last ? q0w + j : last;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_bf16x8(Qb + (int64_t)q * a.q.s_t + 16 * s + 8 * hf);
    }
    vm_wait<0>();  // (the compiler's own wait for them in the tile loop would also drain the copies in flight)

    const int wg_q_hi = wg_q_lo + kBQ - 1 < last ? wg_q_lo + kBQ - 1 : last;
    const int band = (wg_q_lo > W ? wg_q_lo - W : 0) / kBK;
    const int sunk = (n_sinks + kBK - 1) / kBK < band ? (n_sinks + kBK - 1) / kBK : band;
    const int nt = sunk + wg_q_hi / kBK - band + 1;
    auto tile_k0 = [&](int t) { return (t < sunk ? t : t - sunk + band) * kBK; };

    // copies of 1 KB: c = 4 i + wave % 4 of K's and of V's, by group A (kPaired) or a tile's four waves
    const int crow = lane / TL::CPR, cslot = lane % TL::CPR;
    const bool group_a = wave < 4;
    const unsigned lb = lds_addr(lds);
    // this lane's chunk: row R = RPC c + crow, whose swizzle does not depend on i (RPC 4 i is a multiple
    // of the swizzles' period of 16 rows)
    static_assert(4 * TL::RPC % 16 == 0, "uniform swizzle");
    const int r0 = TL::RPC * (wave & 3) + crow;
    const int kchunk = TL::swz(r0, cslot), vchunk = TL::swt(r0, cslot);
    const unsigned koff = (unsigned)(r0 * a.k.s_t * 2 + kchunk * 16), voff = (unsigned)(r0 * a.v.s_t * 2 + vchunk * 16);
    const int64_t kstep = 4 * TL::RPC * a.k.s_t, vstep = 4 * TL::RPC * a.v.s_t;
    auto issue = [&](int k0, unsigned st) {
        const __bf16 *kp = Kb + k0 * a.k.s_t, *vp = Vb + k0 * a.v.s_t;
        st += (wave & 3) * 1024;
        if (k0 + kBK > len) {
            // the tile with the last token: each lane's row is clamped
#pragma unroll
            for (int i = 0; i < CPW / 2; ++i) {
                const int r = i * 4 * TL::RPC + r0;
                const unsigned rr = (unsigned)(k0 + r > last ? last - k0 : r);
                lds_dma16_at(kp, rr * (unsigned)a.k.s_t * 2 + kchunk * 16, st + 4 * i * 1024);
                lds_dma16_at(vp, rr * (unsigned)a.v.s_t * 2 + vchunk * 16, st + kTile + 4 * i * 1024);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < CPW / 2; ++i, kp += kstep) lds_dma16_at(kp, koff, st + 4 * i * 1024);
#pragma unroll
        for (int i = 0; i < CPW / 2; ++i, vp += vstep) lds_dma16_at(vp, voff, st + kTile + 4 * i * 1024);
    };
    // fragment offsets in a stage: K row sigma(j) (+ 32 kb), k-step s; V^T by columns: as a source, lane 16 g + i addresses key
    // 8 (g / 2) + i / 4 (+ 16 s, + 4), dims 16 (g % 2) + 4 (i % 4) .. + 4 (+ 32 db: offset ^ 64 db)
    const int sj = sigma(j);
    const int kfo = sj * RB + (TL::swz(sj, hf) << 4);
    const int vnr = 8 * hf + ((lane & 15) >> 2);
    const int vnb = kTile + vnr * RB + (TL::swt(vnr, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + 8 * (lane & 1);

    float m = kLowest, l = 0.f;
    f32x16 o[DB], sc[2];
    bf16x8 pf[4];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
    // (a wave whose queries all lie past the last token has no active tile)
    const int wq_lo = q0w, wq_hi = q0w > last ? -1 : q0w + 31 < last ? q0w + 31 : last;
    const float c2 = a.scale_log2;

    auto active = [&](int t) {
        const int k0 = tile_k0(t);
        return k0 <= wq_hi && (k0 + kBK - 1 >= wq_lo - W || k0 < n_sinks);
    };
    auto qk = [&](int t) {
        const char *st = lds + ((t / HALVES & (NS - 1)) * HALVES + half) * kStage;
        sc[0] = f32x16{};
        sc[1] = f32x16{};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                sc[kb] = mfma32x32x16(*reinterpret_cast<const bf16x8 *>(st + (kfo ^ (32 * s)) + kb * 32 * RB), qf[s], sc[kb]);
    };
    auto softmax = [&](int t) {
        const int k0 = tile_k0(t);
        const bool causal_edge = k0 + kBK - 1 > wq_lo, window_edge = k0 < wq_hi - W;
        if (causal_edge || window_edge) {
            // key of register r in block kb: k0 + 8 hf + c, c = 32 kb + 16 (r / 8) + r % 8; seen iff c <= d0 and
            // not ds <= c < d0 - W, with d0 = q - k0 - 8 hf and ds = n - k0 - 8 hf (one unsigned compare)
            int d0 = q0w + j - k0 - 8 * hf, ds = n_sinks - k0 - 8 * hf;
            unsigned wd = (unsigned)(d0 - W > ds ? d0 - W - ds : 0);
            // (pinned here: compares hoisted above the products would each hold a 64-bit lane mask)
            asm volatile("" : "+v"(d0), "+v"(wd), "+v"(ds));
            auto mask = [&](auto visible) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int c = 32 * kb + 16 * (r >> 3) + (r & 7);
                        sc[kb][r] = visible(c) ? sc[kb][r] : -__builtin_inff();
                    }
            };
            if (causal_edge) mask([&](int c) { return c <= d0; });
            if (window_edge) mask([&](int c) { return (unsigned)(c - ds) >= wd; });
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kb][r]);
        mx = fmaxf(mx, swap_halves(mx));
        // the reference maximum moves (TRAIN: with every larger score) only where some row's maximum passes it by more than 8 (log2 units): the weights stay
        // below 2^8, and sums and outputs share the stale maximum, so that the rescale runs in few tiles
        const float mc = mx * c2;
        if (__builtin_amdgcn_ballot_w64(mc > m + (TRAIN ? 0.f : 8.0f))) {
            const float m_new = fmaxf(m, mc);
            const float alpha = exp2_fast(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] *= alpha;
        }
        float rs = 0.f;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = exp2_fast(__builtin_fmaf(sc[kb][r], c2, -m));
                sc[kb][r] = p;
                rs += p;
            }
        l += rs;
        // the weights rounded to bf16 (half a step of 2^-8 each) for the product on the matrix cores; the row sum is theirs before it
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) pf[s][e] = (__bf16)sc[s >> 1][8 * (s & 1) + e];
    };
    auto pv = [&](int t) {
        const char *st = lds + ((t / HALVES & (NS - 1)) * HALVES + half) * kStage;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const char *p = st + (vnb ^ (64 * db)) + 16 * RB * s;
                o[db] = mfma32x32x16(cat(lds_read_tr16(p), lds_read_tr16(p + 4 * RB)), pf[s], o[db]);
            }
    };

    if constexpr (FORM != kPaired) {
        // round t0 works on tiles HALVES t0 + half
        const int rounds = (nt + HALVES - 1) / HALVES;
        auto copy = [&](int i) {
            const int t = i * HALVES + half;
            if (t < nt) issue(tile_k0(t), lb + ((i & (NS - 1)) * HALVES + half) * kStage);
        };
        copy(0);
#pragma unroll 1
        for (int i0 = 0; i0 < rounds; i0 += NS) {
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                const int i = i0 + u, t = i * HALVES + half;
                if (i < rounds) {
                    vm_wait<0>();
                    __syncthreads();  // round i's tiles landed, and every wave is past round i - 1
                    if (i + 1 < rounds) copy(i + 1);
                    if (t < nt && active(t)) {
                        qk(t);
                        softmax(t);
                        pv(t);
                    }
                }
            }
        }
    } else {
    if (group_a) {
#pragma unroll
        for (int t = 0; t < 3; ++t)
            if (t < nt) issue(tile_k0(t), lb + t * kStage);
        vm_wait_groups<CPW, 2>(nt - 1 < 2 ? nt - 1 : 2);
    }
    __syncthreads();  // barrier 0: tile 0 landed
    if (group_a) {
#pragma unroll 1
        for (int t0 = 0; t0 < nt; t0 += NS) {
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                const int t = t0 + u;
                if (t < nt) {
                    if (active(t)) {
                        qk(t);
                        softmax(t);
                        pv(t);
                    }
                    if (t + 1 < nt) {
                        // tile t + 1 landed; of those after it, min(t + 2, nt - 1) - (t + 1) may be in flight
                        vm_wait_groups<CPW, 1>(nt - 2 - t < 1 ? nt - 2 - t : 1);
                        __syncthreads();  // barrier t + 1: every wave is past tile t - 1
                        if (t + 3 < nt) issue(tile_k0(t + 3), lb + ((t + 3) & (NS - 1)) * kStage);
                    }
                }
            }
        }
    } else {
        if (active(0)) qk(0);
#pragma unroll 1
        for (int t0 = 0; t0 < nt; t0 += NS) {
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                const int t = t0 + u;
                if (t >= 1 && t < nt) {
                    __syncthreads();  // barrier t: tile t landed
                    if (active(t - 1)) {
                        softmax(t - 1);
                        pv(t - 1);
                    }
                    if (active(t)) qk(t);
                }
            }
        }
        if (active(nt - 1)) {
            softmax(nt - 1);
            pv(nt - 1);
        }
    }
    }

    // O^T through LDS (the ring, free once both groups are past their last tile), stored as whole rows; queries past the
    // length get zeros
    if constexpr (FORM == kSplit) {
        // the second half's maximum, sum and outputs (l and o still as the lanes hold them) onto the first's
        constexpr int kPart = DB * 16 * 64;
        static_assert((4 * kPart + 8 * 64) * 4 <= NS * HALVES * kStage, "one half's outputs fit");
        float *x = reinterpret_cast<float *>(lds) + (wave & 3) * kPart + 4 * lane;
        float *ml = reinterpret_cast<float *>(lds) + 4 * kPart + (wave & 3) * 128 + lane;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4 *>(x + (db * 4 + g) * 256) =
                        f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
            ml[0] = m;
            ml[64] = l;
        }
        __syncthreads();
        if (half) return;
        const float m2 = ml[0], top = fmaxf(m, m2), f = exp2_fast(m - top), f2 = exp2_fast(m2 - top);
        l = l * f + ml[64] * f2;
        m = top;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(x + (db * 4 + g) * 256);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[db][4 * g + e] = o[db][4 * g + e] * f + v[e] * f2;
            }
    }
    constexpr int kPitch = D + 8;
    static_assert(NW / HALVES * 32 * kPitch * 2 <= NS * HALVES * kStage, "staging fits the ring");
    l += swap_halves(l);
    const int q = q0w + j;
    const float inv = q <= last ? 1.0f / l : 0.f;   // (a token sees itself: l > 0)
    if constexpr (FORM != kSplit) __syncthreads();
    else wave_lds_sync();
    __bf16 *stg = reinterpret_cast<__bf16 *>(lds) + wave * (FORM == kSplit ? DB * 16 * 64 * 2 : 32 * kPitch);
    auto store = [&](const Rows &t, __bf16 *base, auto rounded) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                bf16x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = rounded(q <= last ? o[db][4 * g + e] * inv : 0.f);
                store_bf16x4(stg + j * kPitch + 32 * db + 8 * g + 4 * hf, v);
            }
        wave_lds_sync();
#pragma unroll
        for (int it = 0; it < TL::CPR / 2; ++it) {
            const int c = it * 64 + lane, r = c / TL::CPR, ch = c % TL::CPR;
            if (q0w + r < a.tokens)
                store_bf16x8(base + (int64_t)(q0w + r) * t.s_t + ch * 8, load_bf16x8(stg + r * kPitch + ch * 8));
        }
    };
    store(a.o, ob, [](float x) { return (__bf16)x; });
    if constexpr (TRAIN) {
        wave_lds_sync();
        store(a.rest, a.rest.ptr + b * a.rest.s_b + h * a.rest.s_h, [](float x) { return (__bf16)(x - (float)(__bf16)x); });
        if (hf == 0 && q <= last) a.lse[(int64_t)row * a.tokens + q] = m + __builtin_amdgcn_logf(l);
    }
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int noise_sink_attention_fwd(const noise_heads_t *q, const noise_heads_t *k, const noise_heads_t *v,
                                        const noise_heads_t *o, const noise_heads_t *o_rest, float *lse,
                                        const void *lengths, int lengths_wide,
                                        int64_t batch, int64_t tokens, int64_t head_dim, int64_t window,
                                        int64_t sinks, float scale, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_sink_attention_fwd";
    NOISE_CHECK_ARG(q && k && v && o && q->heads == o->heads && k->heads == v->heads, "%s: tensors missing or of other heads", fn);
    int st = check_sizes(fn, batch, tokens, tokens, q->heads, k->heads, head_dim, window, sinks);
    if (st || (st = check_scale(fn, scale))) return st;
    if (batch == 0 || tokens == 0) return NOISE_OK;
    FwdArgs a;
    if ((st = check_heads(fn, "q", q, &a.q)) || (st = check_heads(fn, "k", k, &a.k)) ||
        (st = check_heads(fn, "v", v, &a.v)) || (st = check_heads(fn, "o", o, &a.o)))
        return st;
    NOISE_CHECK_ARG((lse == nullptr) == (o_rest == nullptr) && aligned(lse, 4) && (!o_rest || o_rest->heads == q->heads),
                    "%s: o_rest and lse go together", fn);
    if (o_rest && (st = check_heads(fn, "o_rest", o_rest, &a.rest))) return st;
    NOISE_CHECK_ARG(a.k.s_t >= 0 && a.k.s_t < kMaxStride && a.v.s_t >= 0 && a.v.s_t < kMaxStride,
                    "%s: token strides of k and v must be below 2^25", fn);
    NOISE_CHECK_ARG(!lengths || aligned(lengths, lengths_wide ? 8 : 4), "%s: lengths misaligned", fn);
    a.lse = lse; a.lengths = lengths; a.wide = lengths_wide;
    a.tokens = (int)tokens; a.heads = (int)q->heads; a.group = (int)(q->heads / k->heads);
    a.window = (int)(window < tokens ? window : tokens);
    a.sinks = (int)(sinks < tokens ? sinks : tokens);
    a.rows = (int)(batch * q->heads);
    // 256-query workgroups where they fill the CUs twice and their windows are long, else smaller ones, which have less to do
    // past the window's edges. kPaired and kFour (us, TRAIN), 16 heads of 128 on 4, 4 x 4096 tokens: window 1024 182 and 167,
    // 1536 216 and 208, 2048 249 and 244, 4096 302 and 303; 16384 tokens: 1024 195 and 184, 2048 319 and 315, 3000 434 and
    // 419; 8 heads of 64, 8 x 2048 tokens: 1024 49.4 and 46.4, 1536 55.7 and 53.1, causal 57.6 and 55.0; 16 x 2048 tokens:
    // 1024 84.7 and 85.7, causal 95.3 and 98.8; 16384 tokens: 1024 58.0 and 58.4, 2048 93 and 98, 4000 162 and 170, 8000 288
    // and 271. So from 1536 on the two lie within 5 % of one another, on either side, and the border is not a sharp one.
    // With fewer workgroups: 8 heads of 64, 4 x 2048 tokens, window 1024 (256 of 256), kPaired 32.9, kFour 28.3; 8 heads of
    // 128, 4096 tokens (256 of 128), kFour 33.0, kSplit 28.3; 4 heads of 64, 4096 tokens, causal (128 of 128), kPaired 76,
    // kFour 61, kSplit 41
    const int64_t paired = (tokens + 255) / 256 * a.rows, fours = (tokens + 127) / 128 * a.rows;
    const int form = paired >= 512 && a.window >= 2048 ? kPaired : fours > 256 ? kFour : kSplit;
    a.qtiles = (int)(form == kPaired ? (tokens + 255) / 256 : (tokens + 127) / 128);
    a.scale_log2 = scale * kLog2e;
    auto pick = [&](auto... kernels) {   // [head_dim 64, 128][form][lse]
        void (*all[])(FwdArgs) = {kernels...};
        return all[(head_dim == 64 ? 0 : 6) + 2 * form + (lse ? 1 : 0)];
    };
    auto kernel = pick(sink_fwd_kernel<64, kPaired, false>, sink_fwd_kernel<64, kPaired, true>,
                       sink_fwd_kernel<64, kFour, false>, sink_fwd_kernel<64, kFour, true>,
                       sink_fwd_kernel<64, kSplit, false>, sink_fwd_kernel<64, kSplit, true>,
                       sink_fwd_kernel<128, kPaired, false>, sink_fwd_kernel<128, kPaired, true>,
                       sink_fwd_kernel<128, kFour, false>, sink_fwd_kernel<128, kFour, true>,
                       sink_fwd_kernel<128, kSplit, false>, sink_fwd_kernel<128, kSplit, true>);
    const int64_t groups = (int64_t)a.qtiles * a.rows;
    for (a.first = 0; a.first < groups; a.first += kLaunchGroups) {
        const int64_t n = groups - a.first < kLaunchGroups ? groups - a.first : kLaunchGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(form == kFour ? 256 : 512), 0, (hipStream_t)stream, a);
    }
    return launch_status(fn);
}
