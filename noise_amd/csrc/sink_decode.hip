// A few new tokens against a cache, with a sliding window and first tokens that stay visible.
//
// Bound by the reading of the visible keys and values, once for every 32 rows (tokens times query heads) of a key head. The slots that a sequence's tokens see between them
// are listed without gaps (the first tokens, then the window's), cut into tiles of 32 and dealt out to the waves of the
// workgroups that share the list. A wave keeps two tiles of its own in LDS, one being copied (whole lines, straight to
// LDS) while the other is worked on, and needs no barrier before the end: four waves of a CU have 64 KB in flight. The
// products are the forward pass's, S^T = K Q^T and O^T += V^T P^T, with up to 32 rows (tokens times query heads of the
// key head) as the columns. The waves join their sums in LDS; the parts of a list over several workgroups go to the workspace
// in fp32 and sink_decode_join_kernel adds them up.
//
// 64 sequences, 32 heads of 128 on 8, 4101 visible slots each: 184 us, 5.9 TB/s (a large copy runs at 4.9 TB/s here, read and
// write together); with 8 new tokens (32 rows) 190 us, with 9 or 16, which read everything twice, 311 and 315. One sequence of
// 8 heads of 64, 1029 slots: 5.4 us over 72 workgroups and 4.8 us for the join, where the
// call's host part takes 12 us.
#include "sink_common.hpp"

namespace noise {
namespace {

constexpr int kKeys = 32;      // slots per tile
constexpr int kRows = 32;      // rows per workgroup
constexpr int kWaves = 4;

struct DecodeArgs {
    Rows q, k, v, o;
    const void *start;
    float *parts;               // [units][splits][kRows][D + 2]: sums, maximum, weight
    int64_t window, sinks, first;
    int wide, tokens, slots, heads, kv_heads, group, splits, blocks;   // blocks: of kRows rows per key head
    int64_t units;              // batch * kv_heads * blocks
    float scale_log2;
};

// The list of slots that the tokens of a sequence see: u < sunk -> slot u, else u - sunk + lo
struct List {
    int sunk, lo, n;
};
__device__ __forceinline__ List slots_of(const DecodeArgs &a, int64_t start) {
    List s{0, 0, 0};
    const int64_t end = start + a.tokens;                     // past the last token's position
    if (end <= 0) return s;
    const int64_t p0 = start > 0 ? start : 0, lo = p0 > a.window ? p0 - a.window : 0;
    s.lo = (int)(lo < a.slots ? lo : a.slots);
    s.sunk = (int)(a.sinks < s.lo ? a.sinks : s.lo);
    s.n = s.sunk + (int)(end < a.slots ? end : a.slots) - s.lo;
    return s;
}

// Direct global -> LDS copy as lds_dma16_at, from a 64-bit address per lane
__device__ __forceinline__ void lds_dma16_lane(const void *src, unsigned la) {
    const unsigned l = (unsigned)__builtin_amdgcn_readfirstlane((int)la);
    unsigned save;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(save)
                 : "v"(src), "s"(l)
                 : "memory");
}

template <int D>
__global__ __launch_bounds__(64 * kWaves) void sink_decode_kernel(DecodeArgs a) {
    using TL = Tile<D>;
    constexpr int RB = TL::RB, KS = D / 16, DB = D / 32;
    constexpr int kTile = kKeys * RB, kStage = 2 * kTile, CPT = kTile / 1024;
    constexpr int kPitch = D + 4;
    static_assert(kWaves * kRows * kPitch * 4 + 2 * kWaves * kRows * 4 <= kWaves * 2 * kStage, "the waves' sums fit");
    __shared__ __attribute__((aligned(16))) char lds[kWaves * 2 * kStage];
    const int64_t wg = a.first + blockIdx.x;
    const int64_t unit = wg / a.splits;
    const int split = (int)(wg % a.splits);
    const int64_t bk = unit / a.blocks;
    const int blk = (int)(unit % a.blocks), hk = (int)(bk % a.kv_heads);
    const int64_t b = bk / a.kv_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    const int rows = a.tokens * a.group - blk * kRows < kRows ? a.tokens * a.group - blk * kRows : kRows;
    int64_t start = at_wide(a.start, a.wide, b);
    start = start < -kFar ? -kFar : start > kFar ? kFar : start;  // (sums with it stay in 64 bits)
    const List list = slots_of(a, start);
    const int tiles = (list.n + kKeys - 1) / kKeys, per = (tiles + a.splits - 1) / a.splits;
    const int t_end = (split + 1) * per < tiles ? (split + 1) * per : tiles;

    const int rr = blk * kRows + (j < rows ? j : 0), tok = rr / a.group, h = hk * a.group + rr % a.group;
    bf16x8 qf[KS];
    {
        const __bf16 *qp = a.q.ptr + b * a.q.s_b + tok * a.q.s_t + h * a.q.s_h + 8 * hf;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_bf16x8(qp + 16 * s);
    }
    // in the list's numbering this lane's token sees u < u_end without us <= u < ul
    const int64_t pos = start + tok;
    int u_end, us, ul;
    {
        const int64_t e = (pos + 1 < a.slots ? pos + 1 : a.slots) - list.lo + list.sunk;
        const int64_t s = (a.sinks > list.lo ? (a.sinks < a.slots ? a.sinks : a.slots) - list.lo : 0) + list.sunk;
        const int64_t l = pos - a.window - list.lo + list.sunk;
        u_end = pos < 0 ? 0 : (int)e;
        us = (int)s;
        ul = (int)(l < us ? us : l < list.n ? l : list.n > us ? list.n : us);
    }
    vm_wait<0>();

    const __bf16 *Kb = a.k.ptr + b * a.k.s_b + hk * a.k.s_h, *Vb = a.v.ptr + b * a.v.s_b + hk * a.v.s_h;
    const unsigned lw = lds_addr(lds) + wave * 2 * kStage;
    const char *mine = lds + wave * 2 * kStage;
    auto issue = [&](int t, int slot) {
        const unsigned st = lw + slot * kStage;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int r = c * TL::RPC + lane / TL::CPR;
            int u = t * kKeys + r;
            u = u < list.n ? u : list.n - 1;
            const int64_t key = u < list.sunk ? u : u - list.sunk + list.lo;
            lds_dma16_lane(Kb + key * a.k.s_t + 8 * TL::swz(r, lane % TL::CPR), st + c * 1024);
            lds_dma16_lane(Vb + key * a.v.s_t + 8 * TL::swt(r, lane % TL::CPR), st + kTile + c * 1024);
        }
    };
    const int sj = sigma(j), vnr = 8 * hf + ((lane & 15) >> 2);
    const int kfo = sj * RB + (TL::swz(sj, hf) << 4);
    const int vnb = kTile + vnr * RB + (TL::swt(vnr, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + 8 * (lane & 1);

    float m = kLowest, l = 0.f;
    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
    int t = split * per + wave;
    if (t < t_end) issue(t, 0);
#pragma unroll 1
    for (int slot = 0; t < t_end; t += kWaves, slot ^= 1) {
        if (t + kWaves < t_end) {
            // (this wave's reads of the stage's last tile have returned)
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
            issue(t + kWaves, slot ^ 1);
            vm_wait<2 * CPT>();
        } else {
            vm_wait<0>();
        }
        wave_lds_sync();
        const char *st = mine + slot * kStage;
        f32x16 sc = f32x16{};
#pragma unroll
        for (int s = 0; s < KS; ++s)
            sc = mfma32x32x16(*reinterpret_cast<const bf16x8 *>(st + (kfo ^ (32 * s))), qf[s], sc);
        const int u0 = t * kKeys;
        if (a.tokens > 1 || u0 + kKeys > list.n) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int u = u0 + 16 * (r >> 3) + 8 * hf + (r & 7);
                sc[r] = u < u_end && (unsigned)(u - us) >= (unsigned)(ul - us) ? sc[r] : -__builtin_inff();
            }
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[r]);
        mx = fmaxf(mx, swap_halves(mx)) * a.scale_log2;
        if (__builtin_amdgcn_ballot_w64(mx > m + 8.0f)) {
            const float m_new = fmaxf(m, mx), alpha = exp2_fast(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] *= alpha;
        }
        // (the weights rounded to bf16 for the product on the matrix cores; their sum is the unrounded ones')
        bf16x8 pf[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = exp2_fast(__builtin_fmaf(sc[r], a.scale_log2, -m));
            l += p;
            pf[r >> 3][r & 7] = (__bf16)p;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const char *p = st + (vnb ^ (64 * db)) + 16 * RB * s;
                o[db] = mfma32x32x16(cat(lds_read_tr16(p), lds_read_tr16(p + 4 * RB)), pf[s], o[db]);
            }
    }
    // the waves' maxima, then their sums at the common one
    __syncthreads();
    l += swap_halves(l);
    float *sums = reinterpret_cast<float *>(lds), *ms = sums + kWaves * kRows * kPitch, *ls = ms + kWaves * kRows;
    if (hf == 0) {
        ms[wave * kRows + j] = m;
        ls[wave * kRows + j] = l;
    }
    __syncthreads();
    float top = m;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ms[w * kRows + j]);
    const float f = exp2_fast(m - top);
    if (j < rows) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4 *>(sums + (wave * kRows + j) * kPitch + 32 * db + 8 * g + 4 * hf) =
                    f32x4{o[db][4 * g] * f, o[db][4 * g + 1] * f, o[db][4 * g + 2] * f, o[db][4 * g + 3] * f};
    }
    __syncthreads();
    for (int c = tid; c < rows * (D / 8); c += 64 * kWaves) {
        const int r = c / (D / 8), d = 8 * (c % (D / 8));
        float top_r = ms[r], weight = 0.f, s[8] = {};
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top_r = fmaxf(top_r, ms[w * kRows + r]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            weight += ls[w * kRows + r] * exp2_fast(ms[w * kRows + r] - top_r);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += sums[(w * kRows + r) * kPitch + d + e];
        }
        if (a.splits > 1) {
            float *out = a.parts + ((unit * a.splits + split) * kRows + r) * (D + 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) out[d + e] = s[e];
            if (d == 0) {
                out[D] = top_r;
                out[D + 1] = weight;
            }
        } else {
            const int row = blk * kRows + r;
            const float inv = 1.f / weight;
            bf16x8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (__bf16)(weight != 0.f ? s[e] * inv : 0.f);
            store_bf16x8(a.o.ptr + b * a.o.s_b + row / a.group * a.o.s_t + (hk * a.group + row % a.group) * a.o.s_h + d, v);
        }
    }
}

// The parts of a row, one wave per row
template <int D>
__global__ __launch_bounds__(256) void sink_decode_join_kernel(DecodeArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (a.first + blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int per = a.tokens * a.group;
    const int64_t bk = at / per, b = bk / a.kv_heads;
    if (at >= a.units / a.blocks * per) return;
    const int row = (int)(at % per), hk = (int)(bk % a.kv_heads);
    const float *p = a.parts + ((bk * a.blocks + row / kRows) * a.splits * kRows + row % kRows) * (D + 2);
    const int64_t step = (int64_t)kRows * (D + 2);
    // a lane per part (and every 64th from there): maxima and weights at once, then the sums, several parts in flight
    float top = kLowest, weight = 0.f, s[D / 64] = {};
    for (int i = lane; i < a.splits; i += 64) top = fmaxf(top, p[i * step + D]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    for (int i0 = 0; i0 < a.splits; i0 += 64) {
        const int n = a.splits - i0 < 64 ? a.splits - i0 : 64;
        const float f = lane < n ? exp2_fast(p[(i0 + lane) * step + D] - top) : 0.f;
        weight += lane < n ? p[(i0 + lane) * step + D + 1] * f : 0.f;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float fi = __shfl(f, i, 64);
#pragma unroll
            for (int e = 0; e < D / 64; ++e) s[e] += p[(i0 + i) * step + lane + 64 * e] * fi;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) weight += __shfl_xor(weight, o, 64);
    const float inv = 1.f / weight;
    __bf16 *out = a.o.ptr + b * a.o.s_b + row / a.group * a.o.s_t + (hk * a.group + row % a.group) * a.o.s_h;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) out[lane + 64 * e] = (__bf16)(weight != 0.f ? s[e] * inv : 0.f);
}

// Workgroups that share a list: enough for two on each of the 256 CUs, of four tiles (one per wave) or more. One workgroup for
// each list of 1029 slots, 8 in all, took 15 us. 32 heads of 128 on 8 (8 lists a sequence, one workgroup on a CU at a time), 4101
// slots, in us: 32 sequences in two parts (as here) 100, whole 96; 33 sequences 124 and 141; 64 sequences whole (as here) 185,
// in two 191; 128 sequences 362 and 373. Whole lists a little past a full round of workgroups are the costly case: 65
// sequences 229 (in three 199), 97 sequences 316 (in three 287). 8 heads of 64 (two workgroups on a CU): 64 sequences 107 whole,
// 102 in eight; 65 sequences 135 and 103.
int64_t splits_of(int64_t units, int64_t tokens, int64_t slots, int64_t window, int64_t sinks) {
    int64_t most = window < slots && sinks < slots && window + sinks + tokens < slots ? window + sinks + tokens : slots;
    const int64_t useful = (most + kWaves * kKeys - 1) / (kWaves * kKeys), wanted = (512 + units - 1) / units;
    const int64_t n = useful < wanted ? useful : wanted;
    return n > 1 ? n : 1;
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int64_t noise_sink_decode_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                     int64_t capacity, int64_t head_dim, int64_t window,
                                                     int64_t sinks) {
    clear_error();
    const char *fn = "noise_sink_decode_workspace_bytes";
    const int st = check_sizes(fn, batch, tokens, capacity, heads, kv_heads, head_dim, window, sinks);
    if (st) return st;
    NOISE_CHECK_ARG(tokens <= 16, "%s: at most 16 new tokens, got %lld", fn, (long long)tokens);
    if (batch == 0 || tokens == 0 || capacity == 0) return 0;
    const int64_t units = batch * kv_heads * ((tokens * (heads / kv_heads) + kRows - 1) / kRows);
    const int64_t splits = splits_of(units, tokens, capacity, window, sinks);
    return splits > 1 ? units * splits * kRows * (head_dim + 2) * 4 : 0;
}

extern "C" int noise_sink_decode(const noise_heads_t *q, const noise_heads_t *k, const noise_heads_t *v,
                                 const noise_heads_t *o, const void *start, int start_wide, int64_t batch,
                                 int64_t tokens, int64_t capacity, int64_t head_dim, int64_t window, int64_t sinks,
                                 float scale, void *workspace, int64_t workspace_bytes, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_sink_decode";
    NOISE_CHECK_ARG(q && k && v && o && q->heads == o->heads && k->heads == v->heads, "%s: tensors missing or of other heads", fn);
    int st = check_sizes(fn, batch, tokens, capacity, q->heads, k->heads, head_dim, window, sinks);
    if (st || (st = check_scale(fn, scale))) return st;
    NOISE_CHECK_ARG(tokens <= 16, "%s: at most 16 new tokens, got %lld", fn, (long long)tokens);
    if (batch == 0 || tokens == 0) return NOISE_OK;
    NOISE_CHECK_ARG(capacity > 0, "%s: the cache has no slots", fn);
    NOISE_CHECK_ARG(start && aligned(start, start_wide ? 8 : 4), "%s: start is required", fn);
    DecodeArgs a;
    if ((st = check_heads(fn, "q", q, &a.q)) || (st = check_heads(fn, "k", k, &a.k)) ||
        (st = check_heads(fn, "v", v, &a.v)) || (st = check_heads(fn, "o", o, &a.o)))
        return st;
    a.start = start; a.wide = start_wide;
    a.window = window < kFar ? window : kFar;
    a.sinks = sinks < kFar ? sinks : kFar;
    a.tokens = (int)tokens; a.slots = (int)capacity; a.heads = (int)q->heads; a.kv_heads = (int)k->heads;
    a.group = a.heads / a.kv_heads;
    a.blocks = (a.tokens * a.group + kRows - 1) / kRows;
    a.units = batch * a.kv_heads * a.blocks;
    a.splits = (int)splits_of(a.units, tokens, capacity, window, sinks);
    a.scale_log2 = scale * kLog2e;
    const int64_t need = a.splits > 1 ? a.units * a.splits * kRows * (head_dim + 2) * 4 : 0;
    NOISE_CHECK_ARG(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need),
                    "%s: workspace NULL, misaligned or below %lld bytes", fn, (long long)need);
    a.parts = static_cast<float *>(workspace);
    const bool narrow = head_dim == 64;
    auto launch = [&](void (*kernel)(DecodeArgs), int64_t groups) {
        for (a.first = 0; a.first < groups; a.first += kLaunchGroups) {
            const int64_t n = groups - a.first < kLaunchGroups ? groups - a.first : kLaunchGroups;
            hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, a);
        }
    };
    launch(narrow ? sink_decode_kernel<64> : sink_decode_kernel<128>, a.units * a.splits);
    if (a.splits > 1)
        launch(narrow ? sink_decode_join_kernel<64> : sink_decode_join_kernel<128>,
               (batch * a.kv_heads * a.tokens * a.group + 3) / 4);
    return launch_status(fn);
}
