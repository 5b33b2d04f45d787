// The residual stream between two blocks: a block's output, through a norm if asked, times its gate onto the scaled stream, and
// the norm that the next block reads; and the gradients (utils/model.py:46-47 and the mixing of the forward that
// train/val/eggroll.py:77-94 repeats, with learned weights, a gate and a norm of the block's output as options). Per row of D:
//   b = y  or  y ry wy, ry = 1 / sqrt(mean y^2 + eps);  t = x + g b;  x' = s t + s0 x0;  n = x' r;  h = n w
//   backward, G = dx' + r (u - n mean(u n)), u = dh w:  dx = s G,  dx0 = s0 G,  dg = s G b,  db = s G g,
//   dy = db  or  ry (e - ny mean(e ny)), e = db wy, ny = y ry;  ds = sum G t, ds0 = sum G x0, dw = sum dh n, dwy = sum db ny
// The backward pass forms x' again from x, y and x0 in fp32, so that n carries none of x's rounding to its stored type (and
// reads what ds, ds0 and dg need anyway).
//
// Memory bound. TEAM lanes hold a row, 8 consecutive elements each, as raw 16 B words that are unpacked where used (single bf16
// values take a register each, and the backward pass 1.6 times as long); sums over a row are lane swaps for teams of up to a wave,
// and one exchange through LDS per sum for larger ones, which are a workgroup. Workgroups of the backward pass take a run of rows
// of one gate each, hold the weights and the sums over rows in registers, and leave one row of partial sums; a second kernel adds
// those up in a fixed order. Measured, in us (and TB/s of what has to be read and written):
//                                                                        forward      backward     join
//   16384 x 512, fp32 stream, bf16 branch, x0                            30 (4.4)     37 (5.9)       4
//   3333 x 1001, fp32, both norms, weights, a gate per sequence          18 (3.0)     25 (3.2)       6
//   8192 x 4096, bf16, both norms, weights, a gate per channel           54 (5.0)     98 (4.1)       4
//   2048 x 8192, fp32, both norms, weights, a gate per channel           63 (4.3)     90 (4.5)       6
// (of one call after another; the first two are in the caches in part). Rows that are not whole 8 elements have tail code and, in
// fp32, 4 B alignment: 3333 x 1000 takes 12, 19 and 5. The backward pass of 4096 holds 200 registers per lane, so one workgroup of
// 8 waves per CU: the loads of a row wait for the sums of the one before. Loading a row ahead, or 128 registers, costs more
// (spills). Past 4096 a row has 16 waves and 128 registers are all there are: with y's norm and x0, or with y's norm and tail code,
// 6 to 32 of them go to memory (2048 x 8192 fp32 with x0: 119 us, 4.5 TB/s as without; 8191 wide, both: 168 us, 3.2).
#include "common.hpp"
#include "mfma.hpp"

#include <type_traits>

namespace noise {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kLaunchGroups = 1 << 20;   // a launch has fewer than 2^32 threads
constexpr int kMaxDim = 8192;

struct ResArgs {
    const void *x, *y, *x0, *gate, *dout, *dh;
    const float *scale, *x0_scale, *wy, *w;
    void *out, *h;                   // backward: dx, dy
    void *dx0, *dgate;               // dgate: of a gate per row only
    float *part_w, *part_wy, *part_g;   // [parts][D] partial sums
    double *part_s;                  // [parts][2]
    int64_t rows, gate_rows, s_x, s_y, s_x0, first;
    int64_t gates, gates_per_part, parts_per_gate, part_rows;  // backward: how the rows are cut (Cut)
    int D, gate_bf16;
    float eps;
};

// 8 elements at any address of their type; n: how many of them exist (zeros for the others). FULL: 8 or none do
template <class E, bool FULL>
struct Eight {
    static constexpr int W = sizeof(E) / 2;   // 16 B words
    u32x4 v[W];
    __device__ __forceinline__ void load(const E *p, int n) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = u32x4{0, 0, 0, 0};
        if (n >= 8) {
            __builtin_memcpy(v, p, sizeof v);
        } else if (!FULL && n > 0) {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < n) {
                    if constexpr (W == 2) v[e / 4][e % 4] = __float_as_uint(p[e]);
                    else v[0][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[e] << (16 * (e % 2));
                }
        }
    }
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (W == 2) return __uint_as_float(v[e / 4][e % 4]);
        return __uint_as_float(e % 2 ? v[0][e / 2] & 0xffff0000u : v[0][e / 2] << 16);
    }
};
template <bool FULL, class E>
__device__ __forceinline__ void put8(E *p, int n, const float (&o)[8]) {
    if (n >= 8) {
        E v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (E)o[e];
        __builtin_memcpy(p, v, 8 * sizeof(E));
    } else if constexpr (!FULL) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = (E)o[e];
    }
}

// v + the value of the lane that `control` (a DPP one) pairs this lane with
template <int CONTROL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}

// N sums over a team of TEAM lanes. Within a wave by DPP (lanes 1, 2, 4 and 8 apart: pairs and halves of four swapped, halves of 8
// and 16 lanes mirrored) and lane swaps: a sixth of the time of shuffles, which go through LDS. Teams larger than a wave are the
// workgroup: their waves' sums go through LDS, in two alternating sets of slots, so that one barrier per call is enough.
template <int TEAM, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float *slots, int &turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = add_dpp<0xb1>(v[i]);    // quad_perm 1 0 3 2
        v[i] = add_dpp<0x4e>(v[i]);    // quad_perm 2 3 0 1
        v[i] = add_dpp<0x141>(v[i]);   // row_half_mirror
        v[i] = add_dpp<0x140>(v[i]);   // row_mirror
        if constexpr (TEAM >= 64) v[i] = sum_lanes_16_32(v[i]);
    }
    if constexpr (TEAM > 64) {
        constexpr int NW = TEAM / 64;
        float *s = slots + 2 * NW * turn;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i * NW + (threadIdx.x >> 6)] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = s[i * NW];
#pragma unroll
            for (int w = 1; w < NW; ++w) v[i] += s[i * NW + w];
        }
    }
}

template <int TEAM>
constexpr int group_threads() { return TEAM > 64 ? TEAM : 256; }

// 8 values of a gate's row at `at`, of a weight from c on: ones where there is none
template <bool FULL>
__device__ __forceinline__ void get_gate(const ResArgs &a, int64_t at, int n, float (&o)[8]) {
    if (a.gate_bf16) {
        Eight<__bf16, FULL> v;
        v.load(static_cast<const __bf16 *>(a.gate) + at, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e];
    } else {
        Eight<float, FULL> v;
        v.load(static_cast<const float *>(a.gate) + at, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e];
    }
}
template <bool FULL>
__device__ __forceinline__ void get_weight(const float *w, int c, int n, float (&o)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 1.f;
    if (!w) return;
    Eight<float, FULL> v;
    v.load(w + c, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = v[e];
}

template <class EX, class EY, int TEAM, bool POST, bool FULL>
__global__ __launch_bounds__(group_threads<TEAM>()) void residual_kernel(ResArgs a) {
    constexpr int NT = group_threads<TEAM>(), TEAMS = NT / TEAM;
    __shared__ float slots[4 * (TEAM > 64 ? TEAM / 64 : 1)];
    int turn = 0;
    const int64_t row = (a.first + blockIdx.x) * TEAMS + threadIdx.x / TEAM;
    if (row >= a.rows) return;   // (whole teams: a team larger than a wave is the workgroup)
    const int c = 8 * (threadIdx.x % TEAM), D = a.D, n = D - c;
    Eight<EX, FULL> x, x0;
    Eight<EY, FULL> y;
    x.load(static_cast<const EX *>(a.x) + row * a.s_x + c, n);
    if (a.y) y.load(static_cast<const EY *>(a.y) + row * a.s_y + c, n);
    if (a.x0) x0.load(static_cast<const EX *>(a.x0) + row * a.s_x0 + c, n);
    float g[8], w[8], wy[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = 1.f;
    if (a.gate) get_gate<FULL>(a, row / a.gate_rows * D + c, n, g);
    get_weight<FULL>(a.w, c, n, w);
    if (POST) get_weight<FULL>(a.wy, c, n, wy);
    const float inv = 1.f / (float)D, scale = a.scale ? *a.scale : 1.f, x0_scale = a.x0_scale ? *a.x0_scale : 1.f;
    float ry = 1.f;
    if constexpr (POST) {
        float s[1] = {0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) s[0] += y[e] * y[e];
        team_sum<TEAM>(s, slots, turn);
        ry = rsqrtf(s[0] * inv + a.eps);
    }
    float t[8], s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = x[e];
    if (a.y) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += g[e] * (POST ? y[e] * ry * wy[e] : y[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] *= scale;
    if (a.x0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += x0_scale * x0[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += t[e] * t[e];
    team_sum<TEAM>(s, slots, turn);
    const float r = rsqrtf(s[0] * inv + a.eps);
    put8<FULL>(static_cast<EX *>(a.out) + row * D + c, n, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = t[e] * r * w[e];
    put8<FULL>(static_cast<EY *>(a.h) + row * D + c, n, t);
}

// MIX: with x0. (Loading the next row before working on the present one was slower, by 5 to 10 %: it takes registers from other
// rows.)
template <class EX, class EY, int TEAM, bool POST, bool MIX, bool FULL>
__global__ __launch_bounds__(group_threads<TEAM>()) void residual_bwd_kernel(ResArgs a) {
    constexpr int NT = group_threads<TEAM>(), TEAMS = NT / TEAM;
    __shared__ float slots[4 * (TEAM > 64 ? TEAM / 64 : 1)];
    __shared__ double scalars[2][NT / 64];
    __shared__ float fold[TEAMS > 1 ? TEAMS * TEAM * 8 : 1];
    int turn = 0;
    const int64_t part = a.first + blockIdx.x;
    const bool row_gate = a.gate_rows == 1;   // (a gate per row is not summed: all rows are one unit)
    const int64_t unit_rows = row_gate ? a.rows : a.gate_rows, at = part % a.parts_per_gate;
    const int64_t first_unit = part / a.parts_per_gate * a.gates_per_part;
    const int64_t last_unit = first_unit + a.gates_per_part < a.gates ? first_unit + a.gates_per_part : a.gates;
    const int lane = threadIdx.x % TEAM, D = a.D, c = 8 * lane, n = D - c;
    const float inv = 1.f / (float)D, scale = a.scale ? *a.scale : 1.f, x0_scale = MIX && a.x0_scale ? *a.x0_scale : 1.f;
    float sw[8] = {}, swy[8] = {}, sg[8] = {};
    // the weights and the gate: in registers, or in LDS where 16 waves leave 128 registers to each
    constexpr bool SHARED = TEAM == 1024;
    constexpr int W = 0, WY = 1, GATE = 2;
    __shared__ __attribute__((aligned(16))) float shared[SHARED ? 3 : 1][SHARED ? 8 * TEAM : 1];
    float own[SHARED ? 1 : 3][8];
    auto hold = [&](int which, const float (&v)[8]) {
        if constexpr (SHARED) __builtin_memcpy(&shared[which][c], v, 32);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) own[which][e] = v[e];
    };
    auto take = [&](int which, float (&v)[8]) {
        if constexpr (SHARED) __builtin_memcpy(v, &shared[which][c], 32);   // (each lane its own: no barrier)
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = own[which][e];
    };
    {
        float v[8];
        get_weight<FULL>(a.w, c, n, v);
        hold(W, v);
        if (POST) get_weight<FULL>(a.wy, c, n, v), hold(WY, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 1.f;
        hold(GATE, v);
    }
    double ds = 0., ds0 = 0.;
    // the teams' sums, added in LDS
    auto leave = [&](float *to, float (&v)[8]) {
        if constexpr (TEAMS > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) fold[(threadIdx.x / TEAM * 8 + e) * TEAM + lane] = v[e];
            __syncthreads();
            if (threadIdx.x < TEAM) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    for (int k = 1; k < TEAMS; ++k) v[e] += fold[(k * 8 + e) * TEAM + lane];
            }
        }
        if (threadIdx.x < TEAM) put8<FULL>(to + c, n, v);
    };
    for (int64_t unit = first_unit; unit < last_unit; ++unit) {
        const int64_t begin = unit * unit_rows + at * a.part_rows, end = (unit + 1) * unit_rows;
        const int64_t stop = begin + a.part_rows < end ? begin + a.part_rows : end, from = begin + threadIdx.x / TEAM;
        float w[8], wy[8], g[8];
        if (a.gate && !row_gate) get_gate<FULL>(a, unit * D + c, n, g), hold(GATE, g);
        // this lane's elements of the row, of the contiguous tensors and of the others
        int64_t o = from * D + c;
        const EX *x = static_cast<const EX *>(a.x) + from * a.s_x + c, *x0 = static_cast<const EX *>(a.x0) + from * a.s_x0 + c;
        const EY *y = static_cast<const EY *>(a.y) + from * a.s_y + c;
        for (int64_t row = from; row < stop; row += TEAMS, o += TEAMS * D, x += TEAMS * a.s_x, y += TEAMS * a.s_y, x0 += TEAMS * a.s_x0) {
            Eight<EX, FULL> vx, vx0, vdo;
            Eight<EY, FULL> vy, vdh;
            vx.load(x, n);
            if (a.y) vy.load(y, n);
            if (MIX) vx0.load(x0, n);
            vdo.load(static_cast<const EX *>(a.dout) + o, a.dout ? n : 0);
            if (a.dh) vdh.load(static_cast<const EY *>(a.dh) + o, n);
            if (a.gate && row_gate) get_gate<FULL>(a, o, n, g), hold(GATE, g);
            float ry = 1.f;
            if constexpr (POST) {
                float s[1] = {0.f};
#pragma unroll
                for (int e = 0; e < 8; ++e) s[0] += vy[e] * vy[e];
                team_sum<TEAM>(s, slots, turn);
                ry = rsqrtf(s[0] * inv + a.eps);
            }
            // t and x' (out), G
            float t[8], out[8], G[8], ls = 0.f, ls0 = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = vx[e], G[e] = vdo[e];
            if (a.y) {
                take(GATE, g);
                if (POST) take(WY, wy);
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] += g[e] * (POST ? vy[e] * ry * wy[e] : vy[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = MIX ? t[e] * scale + x0_scale * vx0[e] : t[e] * scale;
            if (a.dh) {
                float s[2] = {0.f, 0.f};   // of x'^2 and u x'
                take(W, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[0] += out[e] * out[e], s[1] += vdh[e] * w[e] * out[e];
                team_sum<TEAM>(s, slots, turn);
                const float r = rsqrtf(s[0] * inv + a.eps), m = s[1] * r * inv * r;   // (r mean(u n): n = x' r)
                take(W, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    G[e] += r * (vdh[e] * w[e] - out[e] * m);
                    sw[e] += vdh[e] * (out[e] * r);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ls += G[e] * t[e];
                if (MIX) ls0 += G[e] * vx0[e];
            }
            ds += (double)ls, ds0 += (double)ls0;
            if (MIX && a.dx0) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = x0_scale * G[e];
                put8<FULL>(static_cast<EX *>(a.dx0) + o, n, v);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) G[e] *= scale;
            if (a.out) put8<FULL>(static_cast<EX *>(a.out) + o, n, G);
            if (!a.y) continue;
            // of y: G becomes db, then e
            float dg[8], s3[1] = {0.f};
            take(GATE, g);
            if (POST) take(WY, wy);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float ny = vy[e] * ry;
                dg[e] = G[e] * (POST ? ny * wy[e] : vy[e]);
                sg[e] += dg[e];
                G[e] *= g[e];
                if constexpr (POST) {
                    swy[e] += G[e] * ny;
                    G[e] *= wy[e];
                    s3[0] += G[e] * ny;
                }
            }
            if (a.dgate) {
                if (a.gate_bf16) put8<FULL>(static_cast<__bf16 *>(a.dgate) + o, n, dg);
                else put8<FULL>(static_cast<float *>(a.dgate) + o, n, dg);
            }
            if (!a.h) continue;
            if constexpr (POST) {
                team_sum<TEAM>(s3, slots, turn);
                const float m3 = s3[0] * inv * ry;
#pragma unroll
                for (int e = 0; e < 8; ++e) G[e] = ry * (G[e] - vy[e] * m3);
            }
            put8<FULL>(static_cast<EY *>(a.h) + o, n, G);
        }
        if (a.part_g) {
            leave(a.part_g + (unit * a.parts_per_gate + at) * D, sg);
#pragma unroll
            for (int e = 0; e < 8; ++e) sg[e] = 0.f;
        }
    }
    if (a.part_s) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            ds += __shfl_xor(ds, o, 64);
            ds0 += __shfl_xor(ds0, o, 64);
        }
        if ((threadIdx.x & 63) == 0) scalars[0][threadIdx.x >> 6] = ds, scalars[1][threadIdx.x >> 6] = ds0;
        __syncthreads();
        if (threadIdx.x < 2) {
            double s = 0.;
            for (int k = 0; k < NT / 64; ++k) s += scalars[threadIdx.x][k];
            a.part_s[2 * part + threadIdx.x] = s;
        }
    }
    if (a.part_w) leave(a.part_w + part * D, sw);
    if constexpr (POST) {
        if (a.part_wy) leave(a.part_wy + part * D, swy);
    }
}

struct JoinArgs {
    const float *part[3];            // of w, wy (all parts together) and the gate (each gate's parts)
    float *to[2];
    void *dgate;
    const double *part_s;
    float *ds, *ds0;
    int64_t parts, parts_per_gate, gates;
    int D, gate_bf16;
};

// 32 columns of one sum, 32 runs of parts after one another
__global__ __launch_bounds__(1024) void residual_join_kernel(JoinArgs a) {
    __shared__ float s[32][33];
    const int which = blockIdx.z, col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    if (which < 3) {
        if (!a.part[which]) return;
        const int64_t n = which < 2 ? a.parts : a.parts_per_gate, sums = which < 2 ? 1 : a.gates;
        for (int64_t g = blockIdx.y; g < sums; g += gridDim.y) {
            float v = 0.f;
            if (col < a.D) {
#pragma unroll 8
                for (int64_t p = slice; p < n; p += 32) v += a.part[which][(g * n + p) * a.D + col];
            }
            s[slice][threadIdx.x & 31] = v;
            __syncthreads();
            if (slice == 0 && col < a.D) {
                for (int k = 1; k < 32; ++k) v += s[k][threadIdx.x & 31];
                if (which < 2) a.to[which][col] = v;
                else if (a.gate_bf16) static_cast<__bf16 *>(a.dgate)[g * a.D + col] = (__bf16)v;
                else static_cast<float *>(a.dgate)[g * a.D + col] = v;
            }
            __syncthreads();
        }
        return;
    }
    if (!a.part_s || blockIdx.x > 0 || blockIdx.y > 0) return;
    __shared__ double d[2][16];
    double v[2] = {0., 0.};
    for (int64_t p = threadIdx.x; p < a.parts; p += 1024) v[0] += a.part_s[2 * p], v[1] += a.part_s[2 * p + 1];
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o, 64);
        if ((threadIdx.x & 63) == 0) d[k][threadIdx.x >> 6] = v[k];
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        double t = 0.;
        for (int w = 0; w < 16; ++w) t += d[threadIdx.x][w];
        float *to = threadIdx.x == 0 ? a.ds : a.ds0;
        if (to) *to = (float)t;
    }
}

// lanes of a row, and threads of a workgroup
int team_of(int64_t D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }
int threads_of(int team) { return team > 64 ? team : 256; }

// FULL: rows of whole 8 elements
template <class EX, class EY, bool POST, bool FULL>
void (*forward_of(int team))(ResArgs) {
    return team == 16    ? residual_kernel<EX, EY, 16, POST, FULL>
           : team == 64  ? residual_kernel<EX, EY, 64, POST, FULL>
           : team == 128 ? residual_kernel<EX, EY, 128, POST, FULL>
           : team == 256 ? residual_kernel<EX, EY, 256, POST, FULL>
           : team == 512 ? residual_kernel<EX, EY, 512, POST, FULL>
                         : residual_kernel<EX, EY, 1024, POST, FULL>;
}
template <class EX, class EY, bool POST, bool MIX, bool FULL>
void (*backward_of(int team))(ResArgs) {
    return team == 16    ? residual_bwd_kernel<EX, EY, 16, POST, MIX, FULL>
           : team == 64  ? residual_bwd_kernel<EX, EY, 64, POST, MIX, FULL>
           : team == 128 ? residual_bwd_kernel<EX, EY, 128, POST, MIX, FULL>
           : team == 256 ? residual_bwd_kernel<EX, EY, 256, POST, MIX, FULL>
           : team == 512 ? residual_bwd_kernel<EX, EY, 512, POST, MIX, FULL>
                         : residual_bwd_kernel<EX, EY, 1024, POST, MIX, FULL>;
}
// f.operator()<EX, EY> for a pair of types
template <class F>
auto of_types(int64_t x, int64_t y, F f) {
    return x == NOISE_FP32 ? (y == NOISE_FP32 ? f(0.f, 0.f) : f(0.f, (__bf16)0.f)) : f((__bf16)0.f, (__bf16)0.f);
}

// How the backward pass cuts the rows into the parts of its workgroups: several gates' rows each, or a gate's rows (all rows where
// no gate is summed) in several parts. Eight waves per CU, which is what the registers leave room for (twice as many parts cost the
// join 6 us more at a width of 4096).
struct Cut {
    int64_t gates, gates_per_part, parts_per_gate, rows, parts;
};
Cut cut_of(int64_t rows, int64_t gate_rows, int64_t D) {
    const int team = team_of(D);
    const int64_t teams = threads_of(team) / team, want = threads_of(team) > 512 ? 256 : 131072 / threads_of(team);
    const int64_t unit = gate_rows > 1 ? gate_rows : rows;
    Cut c;
    c.gates = rows / unit;
    const int64_t most = (unit + teams - 1) / teams;
    int64_t per = (want + c.gates - 1) / c.gates;
    if (per > most) per = most;
    c.rows = ((unit + per - 1) / per + teams - 1) / teams * teams;
    c.parts_per_gate = (unit + c.rows - 1) / c.rows;
    c.gates_per_part = c.parts_per_gate > 1 ? 1 : (c.gates + want - 1) / want;
    c.parts = (c.gates + c.gates_per_part - 1) / c.gates_per_part * c.parts_per_gate;
    return c;
}

int check(const char *fn, const noise_residual_t *a, float eps) {
    NOISE_CHECK_ARG(a && a->rows >= 0 && a->dim > 0 && a->dim <= kMaxDim, "%s: rows >= 0 and dim 1 .. %d required", fn, kMaxDim);
    const bool types = (a->x_type == NOISE_FP32 && (a->y_type == NOISE_FP32 || a->y_type == NOISE_BF16)) ||
                       (a->x_type == NOISE_BF16 && a->y_type == NOISE_BF16);
    NOISE_CHECK_ARG(types, "%s: types %lld and %lld", fn, (long long)a->x_type, (long long)a->y_type);
    NOISE_CHECK_ARG(eps >= 0.f && eps < 3e38f, "%s: eps must be 0 or more", fn);
    if (a->rows == 0) return NOISE_OK;
    const size_t sx = a->x_type == NOISE_BF16 ? 2 : 4, sy = a->y_type == NOISE_BF16 ? 2 : 4;
    NOISE_CHECK_ARG(a->x && aligned(a->x, sx) && aligned(a->y, sy) && aligned(a->x0, sx), "%s: x NULL or a pointer not aligned", fn);
    NOISE_CHECK_ARG(a->rows <= INT64_MAX / 8 / kMaxDim, "%s: too many rows", fn);
    NOISE_CHECK_ARG(a->y || (!a->gate && !a->norm_y), "%s: a gate or norm of y without y", fn);
    NOISE_CHECK_ARG(a->norm_y || !a->y_weight, "%s: a weight of y's norm without the norm", fn);
    NOISE_CHECK_ARG(a->x0 || !a->x0_scale, "%s: x0_scale without x0", fn);
    NOISE_CHECK_ARG(aligned(a->scale, 4) && aligned(a->x0_scale, 4) && aligned(a->y_weight, 4) && aligned(a->weight, 4),
                    "%s: a pointer is not aligned to its type", fn);
    if (a->gate) {
        NOISE_CHECK_ARG(a->gate_type == NOISE_BF16 || a->gate_type == NOISE_FP32, "%s: unknown gate type", fn);
        NOISE_CHECK_ARG(a->gate_rows > 0 && a->rows % a->gate_rows == 0 && aligned(a->gate, a->gate_type == NOISE_BF16 ? 2 : 4),
                        "%s: rows must be a multiple of gate_rows", fn);
    }
    return NOISE_OK;
}

ResArgs args_of(const noise_residual_t *r, float eps) {
    ResArgs a = {};
    a.x = r->x, a.y = r->y, a.x0 = r->x0, a.gate = r->gate;
    a.scale = r->scale, a.x0_scale = r->x0_scale, a.wy = r->y_weight, a.w = r->weight;
    a.rows = r->rows, a.gate_rows = r->gate ? r->gate_rows : r->rows;
    a.s_x = r->x_stride, a.s_y = r->y_stride, a.s_x0 = r->x0_stride;
    a.D = (int)r->dim, a.gate_bf16 = r->gate_type == NOISE_BF16, a.eps = eps;
    return a;
}

}  // namespace
}  // namespace noise

using namespace noise;

extern "C" int noise_residual_norm(const noise_residual_t *r, void *out, void *h, float eps, noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_residual_norm";
    if (int e = check(fn, r, eps)) return e;
    if (r->rows == 0) return NOISE_OK;
    NOISE_CHECK_ARG(out && h && aligned(out, r->x_type == NOISE_BF16 ? 2 : 4) && aligned(h, r->y_type == NOISE_BF16 ? 2 : 4),
                    "%s: an output is NULL or not aligned to its type", fn);
    ResArgs a = args_of(r, eps);
    a.out = out, a.h = h;
    const int team = team_of(r->dim), threads = threads_of(team);
    auto kernel = of_types(r->x_type, r->y_type, [&](auto x, auto y) {
        using X = decltype(x);
        using Y = decltype(y);
        const bool full = r->dim % 8 == 0;
        return r->norm_y ? (full ? forward_of<X, Y, true, true>(team) : forward_of<X, Y, true, false>(team))
                         : (full ? forward_of<X, Y, false, true>(team) : forward_of<X, Y, false, false>(team));
    });
    const int64_t teams = threads / team, groups = (r->rows + teams - 1) / teams;
    for (a.first = 0; a.first < groups; a.first += kLaunchGroups) {
        const int64_t n = groups - a.first < kLaunchGroups ? groups - a.first : kLaunchGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads), 0, (hipStream_t)stream, a);
    }
    return launch_status(fn);
}

extern "C" int64_t noise_residual_norm_bwd_workspace_bytes(int64_t rows, int64_t gate_rows, int64_t dim) {
    clear_error();
    NOISE_CHECK_ARG(rows > 0 && rows <= INT64_MAX / 8 / kMaxDim && gate_rows > 0 && rows % gate_rows == 0 && dim > 0 && dim <= kMaxDim,
                    "noise_residual_norm_bwd_workspace_bytes: rows a multiple of gate_rows and dim 1 .. %d required", kMaxDim);
    const Cut c = cut_of(rows, gate_rows, dim);
    return c.parts * (2 * 4 * dim + 16) + c.gates * c.parts_per_gate * 4 * dim;
}

extern "C" int noise_residual_norm_bwd(const noise_residual_t *r, const void *dout, const void *dh,
                                       const noise_residual_grads_t *d, float eps, void *workspace, int64_t workspace_bytes,
                                       noise_stream_t stream) {
    clear_error();
    const char *fn = "noise_residual_norm_bwd";
    if (int e = check(fn, r, eps)) return e;
    NOISE_CHECK_ARG(d, "%s: NULL pointer", fn);
    const size_t sx = r->x_type == NOISE_BF16 ? 2 : 4, sy = r->y_type == NOISE_BF16 ? 2 : 4;
    NOISE_CHECK_ARG(aligned(dout, sx) && aligned(dh, sy) && aligned(d->dx, sx) && aligned(d->dy, sy) && aligned(d->dx0, sx) &&
                        aligned(d->dgate, r->gate_type == NOISE_BF16 ? 2 : 4) && aligned(d->dscale, 4) &&
                        aligned(d->dx0_scale, 4) && aligned(d->dy_weight, 4) && aligned(d->dweight, 4),
                    "%s: a pointer is not aligned to its type", fn);
    NOISE_CHECK_ARG((r->y || !d->dy) && (r->x0 || (!d->dx0 && !d->dx0_scale)) && (r->gate || !d->dgate) &&
                        (r->norm_y || !d->dy_weight),
                    "%s: a gradient of an absent tensor", fn);
    ResArgs a = args_of(r, eps);
    const bool row_gate = r->gate && r->gate_rows == 1 && r->rows > 1;
    const bool sums = d->dweight || d->dy_weight || (d->dgate && !row_gate);
    const bool scalars = d->dscale || d->dx0_scale;
    a.dout = dout, a.dh = dh, a.out = d->dx, a.h = d->dy, a.dx0 = d->dx0;
    a.dgate = row_gate ? d->dgate : nullptr;
    if (r->rows == 0) return NOISE_OK;
    const Cut c = cut_of(r->rows, a.gate_rows, r->dim);
    const int64_t parts = c.parts;
    if (sums || scalars) {
        const int64_t need = noise_residual_norm_bwd_workspace_bytes(r->rows, a.gate_rows, r->dim);
        NOISE_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= need,
                        "%s: workspace of %lld bytes (16 B aligned) required", fn, (long long)need);
        char *w = static_cast<char *>(workspace);
        if (scalars) a.part_s = reinterpret_cast<double *>(w);
        w += 16 * parts;
        if (d->dweight) a.part_w = reinterpret_cast<float *>(w);
        w += 4 * parts * r->dim;
        if (d->dy_weight) a.part_wy = reinterpret_cast<float *>(w);
        w += 4 * parts * r->dim;
        if (d->dgate && !row_gate) a.part_g = reinterpret_cast<float *>(w);
    }
    const int team = team_of(r->dim);
    auto kernel = of_types(r->x_type, r->y_type, [&](auto x, auto y) {
        using X = decltype(x);
        using Y = decltype(y);
        auto of = [&](auto full) {
            constexpr bool F = decltype(full)::value;
            return r->norm_y ? (r->x0 ? backward_of<X, Y, true, true, F>(team) : backward_of<X, Y, true, false, F>(team))
                             : (r->x0 ? backward_of<X, Y, false, true, F>(team) : backward_of<X, Y, false, false, F>(team));
        };
        return r->dim % 8 ? of(std::false_type{}) : of(std::true_type{});
    });
    a.gates = c.gates, a.gates_per_part = c.gates_per_part, a.parts_per_gate = c.parts_per_gate, a.part_rows = c.rows;
    for (a.first = 0; a.first < parts; a.first += kLaunchGroups) {
        const int64_t n = parts - a.first < kLaunchGroups ? parts - a.first : kLaunchGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads_of(team)), 0, (hipStream_t)stream, a);
    }
    if (sums || scalars) {
        JoinArgs j;
        j.part[0] = a.part_w, j.part[1] = a.part_wy, j.part[2] = a.part_g, j.part_s = a.part_s;
        j.to[0] = d->dweight, j.to[1] = d->dy_weight, j.dgate = d->dgate, j.ds = d->dscale, j.ds0 = d->dx0_scale;
        j.parts = parts, j.parts_per_gate = c.parts_per_gate, j.gates = c.gates, j.D = (int)r->dim, j.gate_bf16 = a.gate_bf16;
        const unsigned gates = !a.part_g ? 1 : c.gates < 4096 ? (unsigned)c.gates : 4096;
        hipLaunchKernelGGL(residual_join_kernel, dim3((unsigned)(r->dim + 31) / 32, gates, 4), dim3(1024), 0,
                           (hipStream_t)stream, j);
    }
    return launch_status(fn);
}
