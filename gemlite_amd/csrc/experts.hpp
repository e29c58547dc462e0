// Products grouped by expert: what the streaming kernel (experts_stream.hip), the tiled GEMM (experts_gemm.hip), the
// finishing kernel and the host side (experts.hip) share.
//
// The R rows of a call are sorted by expert: rows offsets[e] .. offsets[e + 1] - 1 meet the weights of expert e, rows in front
// of offsets[0] and from offsets[E] on meet none.  offsets lives on the device, so the host knows only R and E: a launch has as many row tiles
// as any distribution can need, and a workgroup finds its tile (expert, first row, last row) from offsets itself.
#pragma once

#include "common.hpp"

namespace gla {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// Waits until at most N of the wave's vector memory operations are in flight.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// weight formats
enum ExpertFormat { kEW4 = 0, kEF8 = 1, kE16 = 2 };

struct ExpertArgs {
    const unsigned char* x;         // activation rows: fp16 / bf16, or e4m3 bytes (F8, tiled GEMM)
    const unsigned char* w;         // expert 0's weights
    const unsigned char* scales;    // W4: [E][G][N] 16-bit; F8: [E][K/128][ceil(N/128)] fp32
    const unsigned char* zeros;     // W4: as scales, or NULL
    const unsigned char* sums;      // W4, tiled GEMM: [rows of x][groups] sums of a group's activations, as 16-byte operand pieces
    const float* scales_x;          // F8, tiled GEMM: [rows of x][K/128] (the streaming kernel quantises 16-bit rows itself)
    const float* bias;              // [E][N] fp32 or NULL
    void* out;                      // 16-bit rows (rows / gated)
    float* partials;                // [S][R][N] fp32 (combined, or S > 1)
    const int32_t* offsets;         // [E + 1]
    const int32_t* order;           // gated: sorted row -> flat (token, slot) index
    int64_t w_stride_e, meta_stride_e;  // bytes per expert of w / of scales (and zeros)
    int64_t xsm;                    // bytes per row of x
    int64_t osm;                    // elements per row of out
    int R, E, N, K;
    int top_k;                      // gated: flat index / top_k = row of x
    int half;                       // gated: N / 2 (gate columns 0 .. half - 1, up columns half ..), else 0
    int S;                          // K splits
    int to_partials;                // raw fp32 sums to `partials` instead of finished rows to `out`
    int group;                      // W4: K-values per group (scales and zeros have the activations' type)
    uint32_t group_mul, top_k_mul;  // n / (group / 32) and n / top_k as the high half of n * this (0: see divide_by)
    int top_k_divides;              // R * top_k passes 2^32, where top_k_mul is not exact: divide
    int groups;                     // W4: K / group
    int stream_waves;               // streaming kernel: waves of a workgroup, 4 (W4: or 2)
    int chunk;                      // streaming kernel: units of 128 K-values per wave; tiled GEMM: stages per split
    float c1, c2;                   // W4: zero-point term of a weight = zero * (c1 + c2 * scale)
};

// Sum of the row tiles of all experts for BM-row tiles, at most (host): a experts with rows need a + floor((R - a) / BM).
inline int64_t max_row_tiles(int64_t R, int E, int BM) {
    const int64_t a = R < (int64_t)E + 2 ? R : (int64_t)E + 2;  // rows without an expert count as two more: in front, behind
    return a + (R - a) / BM;
}

// Inclusive sum over the wave's lanes (row shifts inside 16 lanes, then the two row broadcasts; lanes outside a shift add 0).
__device__ __forceinline__ int wave_inclusive_sum(int v) {
#define GLA_DPP0(ctrl, rm) __builtin_amdgcn_update_dpp(0, v, (ctrl), (rm), 0xf, false)
    v += GLA_DPP0(0x111, 0xf);  // row_shr:1
    v += GLA_DPP0(0x112, 0xf);  // row_shr:2
    v += GLA_DPP0(0x114, 0xf);  // row_shr:4
    v += GLA_DPP0(0x118, 0xf);  // row_shr:8
    v += GLA_DPP0(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    v += GLA_DPP0(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef GLA_DPP0
    return v;
}

struct ExpertTile {
    int expert;   // E: the rows without an expert (they become zeros); -1: no such tile
    int row0, row_end;
    int total;    // row tiles in all
};

// The row tile `pick(total)` of the call's `total` ones, computed by every wave for itself: lane l counts the tiles of
// experts l C .. l C + C - 1 (C = 1 up to 63 experts), an inclusive sum over the lanes finds the lane, that lane the
// expert; the tiles of the rows in front of offsets[0] come last.  Offsets are clamped to 0 .. R and an expert whose end
// is not behind its begin has no tiles, so no tile leaves the R rows whatever they hold (where they do not rise, rows may have
// several tiles or none).  One round trip to memory and about a hundred vector instructions; a table written by the routing kernel would cost the same round
// trip.
template <int BM, typename Pick>
__device__ __forceinline__ ExpertTile find_tile(const int32_t* offsets, int E, int R, bool with_rest, Pick pick) {
    const int lane = threadIdx.x & 63;
    const int C = (E + 1 + 63) / 64;
    auto at = [&](int e) __attribute__((always_inline)) {
        const int v = e > E ? R : offsets[e];
        return v < 0 ? 0 : (v > R ? R : v);
    };
    auto tiles_of = [&](int e, int lo, int hi) __attribute__((always_inline)) {
        return e > E || (e == E && !with_rest) || hi <= lo ? 0 : (hi - lo + BM - 1) / BM;
    };
    int mine = 0;
    {
        int lo = at(lane * C);
        for (int c = 0; c < C; ++c) {
            const int e = lane * C + c;
            const int hi = at(e + 1);
            mine += tiles_of(e, lo, hi);
            lo = hi;
        }
    }
    const int upto = wave_inclusive_sum(mine);
    ExpertTile r;
    const int first = with_rest ? __builtin_amdgcn_readfirstlane(at(0)) : 0, of_experts = __builtin_amdgcn_readlane(upto, 63);
    r.total = of_experts + (first + BM - 1) / BM;
    const int t = pick(r.total);
    if (t < 0 || t >= r.total) {
        r.expert = -1;
        r.row0 = r.row_end = 0;
        return r;
    }
    if (t >= of_experts) {
        r.expert = E;
        r.row0 = (t - of_experts) * BM;
        r.row_end = r.row0 + BM < first ? r.row0 + BM : first;
        return r;
    }
    const int owner = __builtin_ctzll(__ballot(upto > t));
    int left = t - (upto - mine), found = -1, row0 = 0, row_end = 0;
    int lo = at(lane * C);
    for (int c = 0; c < C; ++c) {
        const int e = lane * C + c;
        const int hi = at(e + 1);
        const int n = tiles_of(e, lo, hi);
        if (found < 0 && left >= 0 && left < n) {
            found = e;
            row0 = lo + left * BM;
            row_end = hi;
        }
        left -= n;
        lo = hi;
    }
    r.expert = __builtin_amdgcn_readlane(found, owner);
    r.row0 = __builtin_amdgcn_readlane(row0, owner);
    r.row_end = __builtin_amdgcn_readlane(row_end, owner);
    if (r.row_end > r.row0 + BM) r.row_end = r.row0 + BM;
    return r;
}

// n / d as the high half of n * mul, mul = ceil(2^32 / d): exact while n d < 2^32.  mul = 0 stands for d = 1 (it would be
// 2^32).
inline uint32_t divide_mul(uint32_t d) { return d <= 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); }
__device__ __forceinline__ uint32_t divide_by(uint32_t n, uint32_t mul) { return mul == 0 ? n : __umulhi(n, mul); }

// Row of x that sorted row r reads.
__device__ __forceinline__ int64_t source_row(const ExpertArgs& a, int r) {
    if (a.order == nullptr) return r;
    int v = a.order[r];
    v = v < 0 ? 0 : (v > a.R - 1 ? a.R - 1 : v);
    return a.top_k_divides ? (int64_t)(v / a.top_k) : (int64_t)divide_by((uint32_t)v, a.top_k_mul);
}

// Column of the weights that column c of the W columns of unit u stands for: u W + c, or (gated) W / 2 gate columns
// followed by the same up columns, so that whoever computes the unit holds both factors of an output.
template <int W>
__device__ __forceinline__ int unit_column(int half, int u, int c) {
    if (half == 0) return u * W + c;
    return u * (W / 2) + (c % (W / 2)) + (c < W / 2 ? 0 : half);
}
// The same for a run of 4 columns that starts at c, moved back inside its half where it would begin past the end (N and
// half are multiples of 8).
template <int W>
__device__ __forceinline__ int unit_column_inside(int half, int N, int u, int c) {
    const int in = half == 0 ? u * W + c : u * (W / 2) + (c % (W / 2));
    const int top = (half == 0 ? N : half) - 4;
    return (in > top + 3 ? top : in) + (half != 0 && c >= W / 2 ? half : 0);
}

__device__ __forceinline__ float silu_mul(float gate, float up) { return gate / (1.0f + __expf(-gate)) * up; }

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (BF16) return pack_bf16x2(lo, hi);
    else return pack_half2(lo, hi);
}

// Larger magnitudes of two pairs of fp16 / bf16 values, as 15-bit integers (their order is the values', NaN above infinity:
// a NaN is never lost).
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t magnitude_max(uint32_t m, uint32_t v) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, v & 0x7fff7fffu)));
}

// The scale and the reciprocal that a block of 128 activations of amax is quantised with (NaN if it holds one).  (The
// constant's reciprocal, not a division: the codes of values that lie on a border between two depend on it.)  An infinity
// would be the code of inf * (1 / inf), a NaN, which the clamp to the codes' range loses: the scale is NaN in its place.
__device__ __forceinline__ void block_scale(float amax, float& s, float& inv) {
    s = amax * (1.0f / 448.0f);
    s = s < 1e-6f ? 1e-6f : s;
    s = s < __builtin_inff() ? s : __builtin_nanf("");
    inv = 1.0f / s;
}

// Four values of such a block -> four e4m3 codes.
__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d, float inv) {
    auto lim = [](float v) __attribute__((always_inline)) { return __builtin_amdgcn_fmed3f(v, -448.0f, 448.0f); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(lim(a * inv), lim(b * inv), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lim(c * inv), lim(d * inv), r, true);
}

template <bool BF16>
__device__ __forceinline__ float low16(uint32_t v) {
    if constexpr (BF16) return __builtin_bit_cast(float, v << 16);
    else return half_bits_to_float((uint16_t)v);
}
template <bool BF16>
__device__ __forceinline__ float high16(uint32_t v) {
    if constexpr (BF16) return __builtin_bit_cast(float, v & 0xffff0000u);
    else return half_bits_to_float((uint16_t)(v >> 16));
}

// A float as three bf16 values in the high halves of t: 8 bits of its significand each, so that their sum is exact (but for
// underflow).
__device__ __forceinline__ void bf16_terms(float v, uint32_t (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        t[i] = __builtin_bit_cast(uint32_t, v) & 0xffff0000u;
        v -= __builtin_bit_cast(float, t[i]);
    }
}
__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// 16-bit rows -> sums of every group of `group` values, in fp32, as the activations' side of eight products of bf16 terms
// [rows][K / group][8] (experts_quant.hip)
int launch_experts_sums(const void* x, bool bf16, int64_t xsm, int rows, int K, int group, unsigned char* sums, hipStream_t stream);

// 16-bit rows -> e4m3 codes [rows][K] and scales [rows][K/128] (experts_quant.hip)
int launch_experts_quantise(const void* x, bool bf16, int64_t xsm, int rows, int K, unsigned char* codes, float* scales, hipStream_t stream);

int launch_experts_stream(const ExpertArgs& a, int format, bool bf16, int rows, hipStream_t stream);
int launch_experts_gemm(const ExpertArgs& a, int format, bool bf16, int bm, hipStream_t stream);

// logits NULL: the ids are given and only sorted.  counts: route_counts() integers of scratch (select: not for given ids).
int64_t route_counts(int T, int E, int top_k, bool select);
int launch_route(const void* logits, int dtype, int64_t stride, int T, int E, int top_k, int sigmoid, int renormalize, float scale,
                 float* weights, int32_t* ids, int32_t* offsets, int32_t* order, int32_t* places, int32_t* counts, hipStream_t stream);

}  // namespace gla
