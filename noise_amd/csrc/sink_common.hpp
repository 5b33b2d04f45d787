// Shared pieces of the attention kernels with a sliding window and first tokens that stay visible (sink_*.hip): the
// arguments, the layout of key and value tiles in LDS, and the host's checks.
//
// Query i sees the keys j <= i with i - j <= W or j < n. All products run on v_mfma_f32_32x32x16_bf16 with the scores
// transposed or not so that a lane's 16 results of a 32 x 32 block are the operand of the next product (mfma.hpp gives
// the lane layout).
#pragma once
#include "common.hpp"
#include "mfma.hpp"

namespace noise {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;  // a running maximum before the first score
constexpr int64_t kFar = 1ll << 62;         // sums of a position and a window stay in 64 bits
constexpr int64_t kLaunchGroups = 1 << 22;  // a launch has fewer than 2^32 threads (a multiple of 8: XCDs do not move)
constexpr int64_t kMaxStride = 1 << 25;     // token strides that a tile's 32-bit copy offsets span

struct Rows {
    __bf16 *ptr;
    int64_t s_b, s_t, s_h;
};

__device__ __forceinline__ int64_t at_wide(const void *p, int wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
}

// Which row (of heads of sequences) workgroup u of a round of `rows` workgroups takes. Workgroups go to the 8 XCDs in turn. With
// rows in eighths each XCD takes neighbouring rows, whose heads share keys in its L2; in padded batches that would leave the
// XCDs of short sequences idle, so there the rounds are shifted against each other.
__device__ __forceinline__ int row_of(int u, int round, int rows, bool padded) {
    if (padded) return (u + round) % rows;
    return rows % 8 ? u : (u & 7) * (rows / 8) + (u >> 3);
}

// bits 2 and 3 of a row index swapped: with a block's rows read in this order, register r of a lane's 32 x 32 result
// stands for row 16 (r / 8) + 8 (lane / 32) + r % 8, eight consecutive ones per operand of the next product
__device__ __forceinline__ int sigma(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

// A tile of rows of D bf16 in LDS, filled by 1 KB wave-wide copies. It is read in two ways: 16 B of each lane's own row
// (16 lanes on 16 consecutive rows must lie on distinct banks), and by columns, with transposing reads of four rows for
// each group of 16 lanes (the four rows of two neighbouring groups must). The 16 B chunks of a row are XOR-swizzled by
// swz for the first, swt for the second and swb for both.
template <int D>
struct Tile {
    static constexpr int RB = 2 * D;             // bytes per row
    static constexpr int CPR = D / 8;            // 16 B chunks per row
    static constexpr int RPC = 1024 / RB;        // rows per copy
    __device__ static int swz(int r, int c) { return D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); }
    __device__ static int swt(int r, int c) { return D == 64 ? c ^ (2 * (r & 3)) : c ^ (4 * (r & 3)); }
    // bits 2 (and 3) from the row's lowest differing bits, as swt; the others from the next two, so that 16 rows differ
    __device__ static int swb(int r, int c) {
        return D == 64 ? c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3)) : c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    }
};

int check_heads(const char *fn, const char *name, const noise_heads_t *h, Rows *out) {
    NOISE_CHECK_ARG(h && h->ptr && aligned(h->ptr, 16), "%s: %s NULL or not 16 B aligned", fn, name);
    NOISE_CHECK_ARG(h->s_b % 8 == 0 && h->s_t % 8 == 0 && h->s_h % 8 == 0, "%s: %s strides must be multiples of 8", fn, name);
    *out = Rows{static_cast<__bf16 *>(h->ptr), h->s_b, h->s_t, h->s_h};
    return NOISE_OK;
}

// Hidden scores are -inf before the scale is applied, and maxima are taken there: it has to be positive. Within these limits its
// product with log2 e and the backward pass's quotient of a log-sum-exp by it are normal numbers.
int check_scale(const char *fn, float scale) {
    NOISE_CHECK_ARG(scale >= 1e-30f && scale <= 1e30f, "%s: scale must be positive, 1e-30 .. 1e30", fn);
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
    NOISE_CHECK_ARG(batch <= INT32_MAX / heads && (tokens == 0 || batch * heads <= INT64_MAX / 1024 / tokens),
                    "%s: too many rows", fn);
    return NOISE_OK;
}

}  // namespace
}  // namespace noise
