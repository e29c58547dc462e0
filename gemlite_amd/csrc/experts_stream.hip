// Products grouped by expert, few rows per expert: every weight is read once and meets one 16-row MFMA tile that holds MR
// (4 or 16) activation rows.  Bound by the bytes of the experts that have rows.
//
//  * A workgroup owns WC columns (64; 16-bit weights 32) of one expert for one tile of MR rows; gated calls take half of
//    them from the gate and the same ones of the up projection.  Its 4 (2) waves split K and meet once in LDS at the end, so
//    a launch with few column tiles still has thousands of loads in flight; gridDim.z splits K further where even that
//    leaves the chip empty (fp32 sums to the workspace, added in order by the finishing kernel).
//  * A wave walks its K range in units of 128 values and shares nothing with the others on the way: the load unit copies a
//    unit's weights, activation rows and scales straight into the wave's own ring of D slots in LDS (global_load_lds), so
//    what is in flight costs no registers and no barrier stands in the loop; the wave waits on its own copy counter.
//    (With the same units in registers, 150 to 220 of them per lane, one token took 46 us where this takes 29.)
//  * W4: a 16-byte piece is the packed words of 4 adjacent columns of one word row; a word is 8 K-values of one column =
//    the lane's share of the B operand of v_mfma_f32_16x16x32.  The codes go into the MFMA as they are (bf16 128 + q, fp16
//    1024 + q: one shift and one masked OR per pair) and the group's scale and zero are applied to the sums:
//    w = s q + z  =>  sum(x w) = s sum(x (off + q)) + (z - off s) sum(x), with sum(x) from one more MFMA against ones.
//    Per code that is 1 vector instruction against 3 for dequantising in front of the MFMA, which at 4 bits would be as
//    slow as the memory, and the weights are never rounded.
//  * F8: 16-bit rows are quantised on the way into the MFMA, 4 lanes to a row's 128 values; the e4m3 bytes of a 128-block
//    go into one v_mfma_f32_16x16x128 that starts from zero, and its result joins the fp32 sum times the two scales.
//  * 16-bit weights: plain MFMAs.
//
// Measured (calls in a captured graph, copies of the weights in turn that make 700 MB together / the same weights again, which the
// 256 MB cache keeps in part): 4-bit, E = 8, top 2, 4096 -> 2 x 14336, one token 29.5 / 28.4 us for 117 MB; 14336 -> 4096, 16 tokens 48 / 48 us
// with the finishing kernel's 4 for 247 MB (5.5 TB/s); E = 64, top 6, 2048 -> 2 x 1408, 61 tokens 50 / 51 us for 208 MB (a workgroup's K
// range is 4 to 8 units there and its start weighs as much as its stream); 16-bit, 16 experts of 2048 x 1000, 129 rows 14.1 / 12.6 us
// for 66 MB; fp8, E = 128, top 8, 768 -> 2048, one token 11.1 / 10.0 us with the finishing kernel's 4.
#include <type_traits>

#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

__device__ __align__(16) unsigned char g_zero_piece[16];  // what activations past the end of K are read from

template <int N>
__device__ __forceinline__ void wait_copies() {
    wait_vmcnt<N>();
    asm volatile("" ::: "memory");
}

template <bool BF16>
__device__ __forceinline__ float4_t mfma16(const u32x4& a, const u32x4& b, float4_t c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// Eight consecutive K-values as registers (k, k + 4): the order of the packed codes.
__device__ __forceinline__ u32x4 pairs_of(const u32x4& v) {
    return u32x4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                 __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}

// FU: K-values between two folds of a W4 group's constants (the largest of 128, 64, 32 that divides the group).
// NW: waves of a workgroup.
template <int FMT, int MR, int FU, int NW>
struct StreamShape {
    static constexpr int WC = FMT == kE16 ? 32 : 64;
    static constexpr int NT = WC / 16;
    static constexpr int FOLDS = 128 / FU;
    static constexpr int W_OPS = FMT == kEW4 ? 4 : 8, M_OPS = FMT == kEW4 ? FOLDS : (FMT == kEF8 ? 1 : 0);
    static constexpr int W_BYTES = W_OPS * 1024;
    // XO: activation copies per unit, 4 rows each
    static constexpr int ops(int xo) { return W_OPS + xo + M_OPS; }
    static constexpr int slot(int xo) { return W_BYTES + xo * 1024 + M_OPS * 256; }
    static constexpr int depth(int xo) { return FMT == kEW4 && xo <= 2 ? 3 : 2; }
    static constexpr int ring(int xo) { return depth(xo) * slot(xo); }
    static constexpr int most(int a, int b) { return a > b ? a : b; }
    static constexpr int RING = most(ring(MR / 4), most(ring(1), MR > 4 ? ring(2) : 0));  // per wave
    static constexpr int LDS = NW * most(RING, 16 * WC * 4);
};

template <int FMT, bool BF16, int MR, int FU, int NW>
__global__ __launch_bounds__(NW * 64, 2) void experts_stream_kernel(ExpertArgs a) {
    using SH = StreamShape<FMT, MR, FU, NW>;
    constexpr int WC = SH::WC, NT = SH::NT;

    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cg = lane & 15, kb = lane >> 4;
    const int ct = blockIdx.x, split = blockIdx.z;
    const ExpertTile tile = find_tile<MR>(a.offsets, a.E, a.R, !a.to_partials, [](int) { return (int)blockIdx.y; });
    if (tile.expert < 0) return;
    float* red = (float*)smem;  // [NW][16][WC], when the ring is done

    // the K loop for a tile of up to 4 XO rows: only rows that are there are copied
    auto run = [&](auto xo_tag) __attribute__((always_inline)) {
        constexpr int XO = decltype(xo_tag)::value, D = SH::depth(XO), OPS = SH::ops(XO), SLOT = SH::slot(XO);
        constexpr int X_OFF = SH::W_BYTES, M_OFF = X_OFF + XO * 1024;
        unsigned char* ring = smem + wave * SH::RING;
        const unsigned char* we = a.w + (int64_t)tile.expert * a.w_stride_e;
        const unsigned char* se = a.scales + (int64_t)tile.expert * a.meta_stride_e;
        const unsigned char* ze = a.zeros == nullptr ? se : a.zeros + (int64_t)tile.expert * a.meta_stride_e;
        const int units = (a.K + 127) / 128;
        const int u0 = (split * NW + wave) * a.chunk, u1 = u0 + a.chunk < units ? u0 + a.chunk : units;

        // ---- copy plan: a wave-uniform base that advances per unit plus 32-bit lane offsets; activation rows have
        // 64-bit addresses of their own
        const unsigned char* x_src[XO];
        int x_piece[XO];
#pragma unroll
        for (int q = 0; q < XO; ++q) {
            const int row = 4 * q + kb;
            int r = tile.row0 + row;
            if (r > tile.row_end - 1) r = tile.row_end - 1;  // multiplied, never stored
            x_piece[q] = (cg ^ row) * 16;                    // piece p of row r lies at position p ^ r
            x_src[q] = a.x + source_row(a, r) * a.xsm + x_piece[q];
        }
        uint32_t w_off[FMT == kEW4 ? 1 : SH::W_OPS];
        if constexpr (FMT == kEW4) {
            w_off[0] = ((uint32_t)unit_column_inside<WC>(a.half, a.N, ct, 4 * cg) + (uint32_t)kb * (uint32_t)a.N) * 4u;
        } else {
            constexpr int BYTES = FMT == kE16 ? 256 : 128, LANES = BYTES / 16, ROWS = 64 / LANES;  // of a column per unit
#pragma unroll
            for (int q = 0; q < SH::W_OPS; ++q) {
                const int c = q * ROWS + lane / LANES;
                const int p = FMT == kE16 ? (lane & 15) ^ (c & 15) : (lane & 7) ^ ((c >> 1) & 7);
                w_off[q] = (uint32_t)unit_column_inside<WC>(a.half, a.N, ct, c) * (uint32_t)(a.K * (FMT == kE16 ? 2 : 1));
                w_off[q] += (uint32_t)(p * 16);
            }
        }
        uint32_t m_off = 0;
        const unsigned char* m_base = se;
        if constexpr (FMT == kEW4) {
            const int c = 2 * (lane & 31);  // a pair lies inside its run of 4
            m_off = (uint32_t)(unit_column_inside<WC>(a.half, a.N, ct, c & ~3) + (c & 3)) * 2u;
            m_base = lane < 32 ? se : ze;
        } else if constexpr (FMT == kEF8) {
            m_off = (uint32_t)(unit_column_inside<WC>(a.half, a.N, ct, lane & ~3) >> 7) * 4u;
        }
        const int groups = a.groups;
        const int Kb = a.K * 2;
        const unsigned char* zero_piece = g_zero_piece;
        asm volatile("" : "+s"(zero_piece));
        typedef const __attribute__((address_space(1))) void* gptr;
        typedef __attribute__((address_space(3))) void* lptr;
        auto issue = [&](int u, unsigned char* slot) __attribute__((always_inline)) {
            if constexpr (FMT == kEW4) {
                const unsigned char* base = we + (int64_t)u * 16 * a.N * 4;
                const int rows = a.K / 8 - u * 16;  // word rows past the end of K: the unit's first ones again (they meet zeros)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    __builtin_amdgcn_global_load_lds((gptr)(base + (int64_t)(4 * s < rows ? 4 * s : 0) * a.N * 4 + w_off[0]), (lptr)(slot + s * 1024), 16, 0, 2);
            } else {
                const unsigned char* base = we + (int64_t)u * (FMT == kE16 ? 256 : 128);
#pragma unroll
                for (int q = 0; q < SH::W_OPS; ++q) {
                    uint32_t off = w_off[q];
                    if constexpr (FMT == kE16) {
                        // a unit may end past K: those pieces are the column's first ones of the unit (they meet zeros)
                        const int p = ((lane & 15) ^ ((q * 4 + kb) & 15)) * 16;
                        if (u * 256 + p >= Kb) off -= (uint32_t)p;
                    }
                    __builtin_amdgcn_global_load_lds((gptr)(base + off), (lptr)(slot + q * 1024), 16, 0, 2);
                }
            }
#pragma unroll
            for (int q = 0; q < XO; ++q) {
                const unsigned char* p = x_src[q] + (int64_t)u * 256;
                if constexpr (FMT != kEF8) p = u * 256 + x_piece[q] < Kb ? p : zero_piece;
                __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(slot + X_OFF + q * 1024), 16, 0, 0);
            }
            if constexpr (FMT == kEW4) {
#pragma unroll
                for (int h = 0; h < SH::FOLDS; ++h) {
                    int g = (int)divide_by((uint32_t)(u * 4 + h * (FU / 32)), a.group_mul);
                    if (g > groups - 1) g = groups - 1;
                    __builtin_amdgcn_global_load_lds((gptr)(m_base + (int64_t)g * a.N * 2 + m_off), (lptr)(slot + M_OFF + h * 256), 4, 0, 0);
                }
            } else if constexpr (FMT == kEF8) {
                __builtin_amdgcn_global_load_lds((gptr)(se + (int64_t)u * ((a.N + 127) / 128) * 4 + m_off), (lptr)(slot + M_OFF), 4, 0, 0);
            }
        };

        float4_t acc[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
        const float4_t zero4 = float4_t{0.f, 0.f, 0.f, 0.f};
        uint32_t mask = 0x000f000fu, magic = BF16 ? 0x43004300u : 0x64006400u;
        asm volatile("" : "+s"(mask), "+v"(magic));  // registers, so that v_and_or_b32 is selected
        const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
        const u32x4 ones = u32x4{one, one, one, one};
        const int x_row = cg < 4 * XO ? cg : 4 * XO - 1;
        auto x_at = [&](const unsigned char* slot, int piece) __attribute__((always_inline)) {
            return *(const u32x4*)(slot + X_OFF + x_row * 256 + ((piece ^ x_row) & 15) * 16);
        };

        // one unit: its operands from LDS into registers, `refill` of the slot, then the arithmetic
        auto unit = [&](const unsigned char* slot, auto refill) __attribute__((always_inline)) {
            if constexpr (FMT == kEW4) {
                u32x4 w[4], x[4];
                u32x2 rs[SH::FOLDS], rz[SH::FOLDS];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    w[s] = *(const u32x4*)(slot + s * 1024 + lane * 16);
                    x[s] = x_at(slot, 4 * s + kb);
                }
#pragma unroll
                for (int h = 0; h < SH::FOLDS; ++h) {
                    rs[h] = *(const u32x2*)(slot + M_OFF + h * 256 + cg * 8);
                    rz[h] = *(const u32x2*)(slot + M_OFF + h * 256 + 128 + cg * 8);
                }
                refill();
#pragma unroll
                for (int h = 0; h < SH::FOLDS; ++h) {
                    float4_t dot[NT], sum;
#pragma unroll
                    for (int s2 = 0; s2 < FU / 32; ++s2) {
                        const int s = h * (FU / 32) + s2;
                        const u32x4 xa = pairs_of(x[s]);
                        sum = mfma16<BF16>(xa, ones, s2 == 0 ? zero4 : sum);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const uint32_t v = w[s][t];
                            const u32x4 q = u32x4{(v & mask) | magic, ((v >> 4) & mask) | magic, ((v >> 8) & mask) | magic, ((v >> 12) & mask) | magic};
                            dot[t] = mfma16<BF16>(xa, q, s2 == 0 ? zero4 : dot[t]);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float sc = t & 1 ? high16<BF16>(rs[h][t / 2]) : low16<BF16>(rs[h][t / 2]);
                        float zp = t & 1 ? high16<BF16>(rz[h][t / 2]) : low16<BF16>(rz[h][t / 2]);
                        zp = a.zeros == nullptr ? 0.0f : zp * __builtin_fmaf(a.c2, sc, a.c1);
                        const float off = __builtin_fmaf(BF16 ? -128.0f : -1024.0f, sc, zp);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[t][r] = __builtin_fmaf(off, sum[r], __builtin_fmaf(sc, dot[t][r], acc[t][r]));
                    }
                }
            } else if constexpr (FMT == kEF8) {
                typedef union {
                    int8_t_v v;
                    u32x4 c[2];
                } op_t;
                op_t wo[NT], xo;
                float sw[NT], f[32], sx, inv;
                uint32_t m = 0;
                const int swz = (cg >> 1) & 7;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    wo[t].c[0] = *(const u32x4*)(slot + (16 * t + cg) * 128 + ((2 * kb) ^ swz) * 16);
                    wo[t].c[1] = *(const u32x4*)(slot + (16 * t + cg) * 128 + ((2 * kb + 1) ^ swz) * 16);
                    sw[t] = *(const float*)(slot + M_OFF + (16 * t + 4 * kb) * 4);
                }
                u32x4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = x_at(slot, 4 * kb + i);
                refill();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t v = x[i / 4][i % 4];
                    f[2 * i] = low16<BF16>(v);
                    f[2 * i + 1] = high16<BF16>(v);
                    m = magnitude_max(m, v);
                }
                m = magnitude_max(m, wave_xor(m, 16));
                m = magnitude_max(m, wave_xor(m, 32));
                block_scale(low16<BF16>((m & 0xffffu) > (m >> 16) ? m & 0xffffu : m >> 16), sx, inv);
#pragma unroll
                for (int i = 0; i < 8; ++i) xo.c[i / 4][i % 4] = quantise4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], inv);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float4_t d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wo[t].v, xo.v, zero4, 0, 0, 0, 127, 0, 127);
                    const float sc = sx * sw[t];
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[t][r] = __builtin_fmaf(sc, d[r], acc[t][r]);
                }
            } else {
                u32x4 w[NT][4], x[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    x[s] = x_at(slot, 4 * s + kb);
#pragma unroll
                    for (int t = 0; t < NT; ++t) w[t][s] = *(const u32x4*)(slot + (16 * t + cg) * 256 + ((4 * s + kb) ^ cg) * 16);
                }
                refill();
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] = mfma16<BF16>(w[t][s], x[s], acc[t]);
            }
        };

#pragma unroll
        for (int d = 0; d < D; ++d)
            if (u0 + d < u1) issue(u0 + d, ring + d * SLOT);
        static_assert(D == 2 || D == 3, "waits of the last units");
        int u = u0, at = 0;
#pragma unroll 1
        for (; u + D < u1; ++u) {
            wait_copies<(D - 1) * OPS>();
            unsigned char* slot = ring + at * SLOT;
            unit(slot, [&]() __attribute__((always_inline)) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
                issue(u + D, slot);
            });
            at = at == D - 1 ? 0 : at + 1;
        }
#pragma unroll 1
        for (; u < u1; ++u) {
            // (the last D units: the counter cannot tell them apart by one constant)
            if (D > 2 && u + 2 < u1) wait_copies<(D - 1) * OPS>();
            else if (u + 1 < u1) wait_copies<OPS>();
            else wait_copies<0>();
            unit(ring + at * SLOT, []() __attribute__((always_inline)) {});
            at = at == D - 1 ? 0 : at + 1;
        }
        if constexpr (FMT == kEW4) {
            // A sum that is not finite may be so only because of the codes' offset (inf - inf, or an overflow of 128 x): such
            // sums are taken again from dequantised weights, rounded to 16 bits.
            bool odd = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) odd = odd || !(__builtin_fabsf(acc[t][r]) < __builtin_inff());
            if (__any(odd)) {
                const int col = unit_column_inside<WC>(a.half, a.N, ct, 4 * cg);
                int row = tile.row0 + cg;
                if (row > tile.row_end - 1) row = tile.row_end - 1;
                const unsigned char* x = a.x + source_row(a, row) * a.xsm + kb * 16;
                float4_t plain[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) plain[t] = zero4;
                const int k1 = u1 * 128 < a.K ? u1 * 128 : a.K;
#pragma unroll 1
                for (int k = u0 * 128; k < k1; k += 32) {
                    const u32x4 w = *(const u32x4*)(we + ((int64_t)(k / 8 + kb) * a.N + col) * 4);
                    const int64_t at = ((int64_t)(k / a.group) * a.N + col) * 2;
                    const u32x2 rs = *(const u32x2*)(se + at), rz = *(const u32x2*)(ze + at);
                    const u32x4 xa = pairs_of(*(const u32x4*)(x + (int64_t)k * 2));
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float sc = t & 1 ? high16<BF16>(rs[t / 2]) : low16<BF16>(rs[t / 2]);
                        float zp = t & 1 ? high16<BF16>(rz[t / 2]) : low16<BF16>(rz[t / 2]);
                        zp = a.zeros == nullptr ? 0.0f : zp * __builtin_fmaf(a.c2, sc, a.c1);
                        u32x4 q;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            q[j] = pack16<BF16>(__builtin_fmaf((float)((w[t] >> (4 * j)) & 15u), sc, zp),
                                                __builtin_fmaf((float)((w[t] >> (4 * j + 16)) & 15u), sc, zp));
                        plain[t] = mfma16<BF16>(xa, q, plain[t]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!(__builtin_fabsf(acc[t][r]) < __builtin_inff())) acc[t][r] = plain[t][r];
            }
        }
        __syncthreads();  // every ring is done

        // ---- the waves' sums.  W4: the lane holds rows 4 kb + r of columns 4 cg + t; else (weights were the row operand)
        // row cg of columns 16 t + 4 kb + r
        float* mine = red + wave * (16 * WC);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (FMT == kEW4)
                *(float4_t*)(mine + (4 * kb + i) * WC + 4 * cg) = float4_t{acc[0][i], acc[1][i], acc[2][i], acc[3][i]};
            else if (i < NT)
                *(float4_t*)(mine + cg * WC + 16 * i + 4 * kb) = acc[i < NT ? i : 0];
        }
    };
    if (tile.expert < a.E) {
        const int rows = tile.row_end - tile.row0;
        if constexpr (MR == 4) run(std::integral_constant<int, 1>{});
        else if (rows <= 4) run(std::integral_constant<int, 1>{});
        else if (rows <= 8) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, 4>{});
    }
    __syncthreads();

    // ---- a thread finishes 4 adjacent columns of a row (gated: 4 gate and 4 up columns)
    const bool none = tile.expert >= a.E;
    auto total = [&](int row, int c) __attribute__((always_inline)) {
        float4_t v = float4_t{0.f, 0.f, 0.f, 0.f};
        if (none) return v;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += *(const float4_t*)(red + w * (16 * WC) + row * WC + c);
        if (a.bias != nullptr && split == 0) v += *(const float4_t*)(a.bias + (int64_t)tile.expert * a.N + unit_column<WC>(a.half, ct, c));
        return v;
    };
    const bool pairs = a.half != 0 && !a.to_partials;
    const int per_row = pairs ? WC / 8 : WC / 4, width = a.half ? a.half : a.N;
    for (int i = tid; i < MR * per_row; i += NW * 64) {
        const int row = i / per_row, c = (i % per_row) * 4;
        const int r = tile.row0 + row;
        const int in_half = a.half ? ct * (WC / 2) + (c % (WC / 2)) : ct * WC + c;
        if (r >= tile.row_end || in_half >= width) continue;  // N (half) is a multiple of 8: whole vectors
        float4_t v = total(row, c);
        if (a.to_partials) {
            *(float4_t*)(a.partials + ((int64_t)split * a.R + r) * a.N + unit_column<WC>(a.half, ct, c)) = v;
            continue;
        }
        if (pairs) {
            const float4_t up = total(row, c + WC / 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = silu_mul(v[j], up[j]);
        }
        *(u32x2*)((uint16_t*)a.out + (int64_t)r * a.osm + in_half) = u32x2{pack16<BF16>(v[0], v[1]), pack16<BF16>(v[2], v[3])};
    }
}

template <int FMT, bool BF16, int MR, int FU, int NW>
int launch_one(const ExpertArgs& a, hipStream_t stream) {
    using SH = StreamShape<FMT, MR, FU, NW>;
    static_assert(SH::LDS <= 160 * 1024 && 3 * SH::ops(4) < 64, "ring does not fit LDS or the counter");
    const int64_t tiles = max_row_tiles(a.R, a.E, MR);
    if (tiles > 65535 || a.S > 65535) {
        set_error("experts: %lld row tiles exceed the grid", (long long)tiles);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    const auto kernel = experts_stream_kernel<FMT, BF16, MR, FU, NW>;
    static DeviceOnce once;
    if (once.first()) {
        const int rc = check_hip(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SH::LDS), "hipFuncSetAttribute");
        if (rc != GLA_OK) return rc;
    }
    const int cols = a.half ? SH::WC / 2 : SH::WC, width = a.half ? a.half : a.N;
    kernel<<<dim3((width + cols - 1) / cols, (unsigned)tiles, a.S), NW * 64, SH::LDS, stream>>>(a);
    return check_hip(hipGetLastError(), "experts_stream");
}

template <int FMT, bool BF16, int MR>
int launch_fold(const ExpertArgs& a, hipStream_t stream) {
    if constexpr (FMT == kEW4) {
        const bool two = a.stream_waves == 2;
        if (a.group % 128 == 0) return two ? launch_one<FMT, BF16, MR, 128, 2>(a, stream) : launch_one<FMT, BF16, MR, 128, 4>(a, stream);
        if (a.group % 64 == 0) return two ? launch_one<FMT, BF16, MR, 64, 2>(a, stream) : launch_one<FMT, BF16, MR, 64, 4>(a, stream);
        return two ? launch_one<FMT, BF16, MR, 32, 2>(a, stream) : launch_one<FMT, BF16, MR, 32, 4>(a, stream);
    } else {
        return launch_one<FMT, BF16, MR, 128, 4>(a, stream);
    }
}

template <int FMT>
int launch_format(const ExpertArgs& a, bool bf16, int rows, hipStream_t stream) {
    // (4-bit units are small enough for two workgroups per CU with room for 16 rows as well: no shorter tile)
    if constexpr (FMT != kEW4) {
        if (rows <= 4) return bf16 ? launch_fold<FMT, true, 4>(a, stream) : launch_fold<FMT, false, 4>(a, stream);
    }
    return bf16 ? launch_fold<FMT, true, 16>(a, stream) : launch_fold<FMT, false, 16>(a, stream);
}

}  // namespace

int launch_experts_stream(const ExpertArgs& a, int format, bool bf16, int rows, hipStream_t stream) {
    switch (format) {
        case kEW4: return launch_format<kEW4>(a, bf16, rows, stream);
        case kEF8: return launch_format<kEF8>(a, bf16, rows, stream);
        default: return launch_format<kE16>(a, bf16, rows, stream);
    }
}

}  // namespace gla
