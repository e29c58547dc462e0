// Products grouped by expert, few rows per expert: every weight is read once, straight into registers, and meets one or
// two 16-row MFMA tiles of activations.  Bound by the bytes of the experts that have rows.
//
//  * A workgroup owns 64 columns of one expert's weights (gated: 32 gate and the same 32 up columns) for one tile of
//    16 RT rows; its NW waves split K, so that a launch with few column tiles still has thousands of loads in flight,
//    and meet once in LDS at the end.  gridDim.z splits K further when even that leaves the chip empty; those sums go
//    to the workspace in fp32 and the finishing kernel adds them in order.
//  * A wave walks its K range in units of 128 values (16-bit weights: 64) with a ring of D units of weights,
//    activations and scales in registers, all loads issued D - 1 units ahead.  A unit past the end of the range loads
//    the same few bytes for every lane instead (one request), which keeps the loop free of branches around loads.
//  * W4: a lane's 128-bit load is the packed words of 4 adjacent columns of one word row; a word is 8 K-values of one
//    column = the lane's share of the B operand of v_mfma_f32_16x16x32.  The codes go into the MFMA as they are (bf16
//    128 + q, fp16 1024 + q: one shift and one masked OR per pair) and the group's scale and zero are applied to the
//    sums: w = s q + z  =>  sum(x w) = s sum(x (off + q)) + (z - off s) sum(x), with sum(x) from one more MFMA against
//    ones.  Per code that is 1 vector instruction against 2.5 for dequantising in front of the MFMA, which at 4 bits
//    would be as slow as the memory, and the weights are never rounded.
//  * F8: the e4m3 bytes of a 128-block go into one v_mfma_f32_16x16x128 that starts from zero; its result joins the fp32
//    sum times the block's two scales.
//  * 16-bit weights: plain MFMAs.
#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

template <bool BF16>
__device__ __forceinline__ float4_t mfma16(const u32x4& a, const u32x4& b, float4_t c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ u32x4 load16(const unsigned char* p) { return *(const u32x4*)p; }
__device__ __forceinline__ u32x4 load16_streaming(const unsigned char* p) { return __builtin_nontemporal_load((const u32x4*)p); }

// Four consecutive K-values and the four after them as registers (k, k + 4): the order of the packed codes.
__device__ __forceinline__ u32x4 pairs_of(const u32x4& v) {
    return u32x4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                 __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}

// FU: K-values between two folds of a W4 group's constants (the largest of 128, 64, 32 that divides the group).
// QX (F8): x holds 16-bit rows and every wave quantises its share of a unit itself, 4 lanes to a row's 128 values (decode:
// one launch less; the work is repeated by every column tile, which is why more rows are quantised by a launch in front).
template <int FMT, bool BF16, int RT, int FU, int NW, int D, bool QX>
__global__ __launch_bounds__(NW * 64) void experts_stream_kernel(ExpertArgs a) {
    constexpr int KU = FMT == kE16 ? 64 : 128;            // K-values per unit
    constexpr int NT = 4;                                 // 16-column MFMA tiles per wave
    constexpr int WL = FMT == kEW4 ? 4 : 2 * NT;          // weight loads per lane and unit
    constexpr int XL = FMT == kEW4 || QX ? 4 : 2;         // activation loads per lane, row tile and unit
    constexpr int FOLDS = KU / FU;
    constexpr int GL = FMT == kEW4 ? FOLDS : 1;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cg = lane & 15, kb = lane >> 4;
    const ExpertTile tile = find_tile<16 * RT>(a.offsets, a.E, a.R, !a.to_partials, [](int) { return (int)blockIdx.y; });
    if (tile.expert < 0) return;
    const int ct = blockIdx.x, split = blockIdx.z;
    extern __shared__ __align__(16) float red[];  // [NW][16 RT][64]

    if (tile.expert < a.E) {
        const unsigned char* we = a.w + (int64_t)tile.expert * a.w_stride_e;
        const unsigned char* se = a.scales + (int64_t)tile.expert * a.meta_stride_e;
        const unsigned char* ze = a.zeros == nullptr ? se : a.zeros + (int64_t)tile.expert * a.meta_stride_e;
        const int units = (a.K + KU - 1) / KU;
        const int slots = a.S * NW, slot = split * NW + wave;
        const int u0 = units * slot / slots, u1 = units * (slot + 1) / slots;

        // ---- addresses
        const unsigned char* xr[RT];
        const float* sxr[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            int r = tile.row0 + 16 * rt + cg;
            if (r > tile.row_end - 1) r = tile.row_end - 1;  // computed, never stored
            const int64_t src = source_row(a, r);
            xr[rt] = a.x + src * a.xsm;
            if constexpr (FMT == kEF8 && !QX) sxr[rt] = a.scales_x + src * (a.K / 128);
        }
        uint32_t w_off[FMT == kEW4 ? 1 : NT];
        uint32_t m_off[NT];
        auto column = [&](int c) __attribute__((always_inline)) { return unit_column_inside<64>(a.half, a.N, ct, c); };
        if constexpr (FMT == kEW4) {
            w_off[0] = (uint32_t)column(4 * cg) * 4u + (uint32_t)kb * (uint32_t)a.N * 4u;
            m_off[0] = (uint32_t)column(4 * cg) * 2u;
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int n = column(16 * t + cg);
                w_off[t] = FMT == kEF8 ? (uint32_t)n * (uint32_t)a.K + (uint32_t)kb * 32u : ((uint32_t)n * (uint32_t)a.K + (uint32_t)kb * 16u) * 2u;
                m_off[t] = (uint32_t)(column(16 * t + 4 * kb) >> 7) * 4u;
            }
        }
        const int groups = FMT == kEW4 ? a.K / a.group : 0;
        const int nblk = (a.N + 127) / 128;

        struct Unit {
            u32x4 w[WL];
            u32x4 x[RT][XL];
            u32x2 s[GL], z[GL];           // W4
            float sx[RT], sw[NT];         // F8
        };
        Unit buf[D];
        auto group_at = [&](int k) __attribute__((always_inline)) {
            const int g = a.group == FU ? k / FU : k / a.group;
            return g > groups - 1 ? groups - 1 : g;
        };
        auto load = [&](Unit& b, int u) __attribute__((always_inline)) {
            const uint32_t on = u < u1 ? 0xffffffffu : 0u;
            const int uc = u < u1 ? u : u0;
            if constexpr (FMT == kEW4) {
                const uint32_t row = (uint32_t)a.N * 4u;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    // (a unit may end past K: its last steps read the unit's first ones again and meet zeros)
                    const int step = uc * 128 + s * 32 < a.K ? s : 0;
                    b.w[s] = load16_streaming(we + (int64_t)(uc * 16 + 4 * step) * row + (w_off[0] & on));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) b.x[rt][s] = load16(xr[rt] + (int64_t)(uc * 256 + step * 64) + (((uint32_t)kb * 16u) & on));
                }
#pragma unroll
                for (int h = 0; h < GL; ++h) {
                    const int64_t g = (int64_t)group_at(uc * 128 + h * FU) * (a.N * 2);
                    b.s[h] = *(const u32x2*)(se + g + (m_off[0] & on));
                    b.z[h] = *(const u32x2*)(ze + g + (m_off[0] & on));
                }
            } else if constexpr (FMT == kEF8) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const unsigned char* p = we + (int64_t)uc * 128 + (w_off[t] & on);
                    b.w[2 * t] = load16_streaming(p);
                    b.w[2 * t + 1] = load16_streaming(p + 16);
                    b.sw[t] = *(const float*)(se + (int64_t)uc * nblk * 4 + m_off[t]);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const unsigned char* p = xr[rt] + (int64_t)uc * (QX ? 256 : 128) + (((uint32_t)kb * (QX ? 64u : 32u)) & on);
#pragma unroll
                    for (int i = 0; i < XL; ++i) b.x[rt][i] = load16(p + 16 * i);
                    if constexpr (!QX) b.sx[rt] = sxr[rt][uc];
                }
            } else {
                const bool in = uc * 64 + kb * 16 < a.K;  // the last unit may be half one
                const int64_t k = (int64_t)uc * 128;
                const uint32_t back = in ? 0u : (uint32_t)kb * 32u;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const unsigned char* p = we + k + ((w_off[t] - back) & on);
                    b.w[2 * t] = load16_streaming(p);
                    b.w[2 * t + 1] = load16_streaming(p + 16);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const unsigned char* p = xr[rt] + k + (((uint32_t)kb * 32u - back) & on);
                    b.x[rt][0] = load16(p);
                    b.x[rt][1] = load16(p + 16);
                }
            }
        };

        float4_t acc[RT][NT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[rt][t] = float4_t{0.f, 0.f, 0.f, 0.f};
        const float4_t zero4 = float4_t{0.f, 0.f, 0.f, 0.f};
        uint32_t mask = 0x000f000fu, magic = BF16 ? 0x43004300u : 0x64006400u;
        asm volatile("" : "+s"(mask), "+v"(magic));  // registers, so that v_and_or_b32 is selected
        const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
        const u32x4 ones = u32x4{one, one, one, one};

        auto compute = [&](Unit& b, int u) __attribute__((always_inline)) {
            if constexpr (FMT == kEW4) {
#pragma unroll
                for (int h = 0; h < FOLDS; ++h) {
                    float4_t dot[RT][NT], sum[RT];
#pragma unroll
                    for (int s2 = 0; s2 < FU / 32; ++s2) {
                        const int s = h * (FU / 32) + s2;
                        u32x4 xa[RT];
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            xa[rt] = pairs_of(b.x[rt][s]);
                            if (u * 128 + s * 32 >= a.K) xa[rt] = u32x4{0, 0, 0, 0};
                            sum[rt] = mfma16<BF16>(xa[rt], ones, s2 == 0 ? zero4 : sum[rt]);
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const uint32_t w = b.w[s][t];
                            const u32x4 q = u32x4{(w & mask) | magic, ((w >> 4) & mask) | magic, ((w >> 8) & mask) | magic, ((w >> 12) & mask) | magic};
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) dot[rt][t] = mfma16<BF16>(xa[rt], q, s2 == 0 ? zero4 : dot[rt][t]);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint32_t rs = b.s[h][t / 2] >> (16 * (t & 1)), rz = b.z[h][t / 2] >> (16 * (t & 1));
                        const float sc = a.meta_bf16 ? bf16_bits_to_float((uint16_t)rs) : half_bits_to_float((uint16_t)rs);
                        float zp = a.meta_bf16 ? bf16_bits_to_float((uint16_t)rz) : half_bits_to_float((uint16_t)rz);
                        zp = a.zeros == nullptr ? 0.0f : zp * __builtin_fmaf(a.c2, sc, a.c1);
                        const float off = __builtin_fmaf(BF16 ? -128.0f : -1024.0f, sc, zp);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                acc[rt][t][r] = __builtin_fmaf(off, sum[rt][r], __builtin_fmaf(sc, dot[rt][t][r], acc[rt][t][r]));
                    }
                }
            } else if constexpr (FMT == kEF8) {
                typedef union {
                    int8_t_v v;
                    u32x4 c[2];
                } op_t;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    op_t xo;
                    if constexpr (QX) {
                        float f[32], amax = 0.0f, inv;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint32_t v = b.x[rt][i / 4][i % 4];
                            f[2 * i] = low16<BF16>(v);
                            f[2 * i + 1] = high16<BF16>(v);
                            amax = fmaxf(amax, fmaxf(fabsf(f[2 * i]), fabsf(f[2 * i + 1])));
                        }
                        amax = fmaxf(amax, wave_xor(amax, 16));
                        amax = fmaxf(amax, wave_xor(amax, 32));
                        block_scale(amax, b.sx[rt], inv);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            xo.c[i / 4][i % 4] = quantise4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], inv);
                    } else {
                        xo.c[0] = b.x[rt][0];
                        xo.c[1] = b.x[rt][1];
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        op_t wo;
                        wo.c[0] = b.w[2 * t];
                        wo.c[1] = b.w[2 * t + 1];
                        const float4_t d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wo.v, xo.v, zero4, 0, 0, 0, 127, 0, 127);
                        const float sc = b.sx[rt] * b.sw[t];
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[rt][t][r] = __builtin_fmaf(sc, d[r], acc[rt][t][r]);
                    }
                }
            } else {
                const bool in = u * 64 + kb * 16 < a.K;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        u32x4 xa = b.x[rt][h];
                        if (!in) xa = u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[rt][t] = mfma16<BF16>(b.w[2 * t + h], xa, acc[rt][t]);
                    }
                }
            }
        };

        if (u0 < u1) {
#pragma unroll
            for (int d = 0; d < D - 1; ++d) load(buf[d], u0 + d);
#pragma unroll 1
            for (int u = u0; u < u1; u += D) {
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    load(buf[(d + D - 1) % D], u + d + D - 1);
                    if (u + d < u1) compute(buf[d], u + d);
                }
            }
        }
        // ---- the waves' sums meet in LDS.  W4: the lane holds rows 4 kb + r of columns 4 cg + t; else (weights were the
        // row operand) row cg of columns 16 t + 4 kb + r
        float* mine = red + wave * (16 * RT * 64);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (FMT == kEW4)
                    *(float4_t*)(mine + (16 * rt + 4 * kb + i) * 64 + 4 * cg) = float4_t{acc[rt][0][i], acc[rt][1][i], acc[rt][2][i], acc[rt][3][i]};
                else
                    *(float4_t*)(mine + (16 * rt + cg) * 64 + 16 * i + 4 * kb) = acc[rt][i];
            }
    }
    __syncthreads();

    // ---- a thread finishes 4 adjacent columns of a row (gated: 4 gate and 4 up columns)
    const bool none = tile.expert >= a.E;
    auto total = [&](int row, int c) __attribute__((always_inline)) {
        float4_t v = float4_t{0.f, 0.f, 0.f, 0.f};
        if (none) return v;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += *(const float4_t*)(red + w * (16 * RT * 64) + row * 64 + c);
        if (a.bias != nullptr && split == 0) {
            const float* b = a.bias + (int64_t)tile.expert * a.N + unit_column<64>(a.half, ct, c);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += b[i];
        }
        return v;
    };
    const bool pairs = a.half != 0 && !a.to_partials;
    const int per_row = pairs ? 8 : 16, width = a.half ? a.half : a.N;
    for (int i = tid; i < 16 * RT * per_row; i += NW * 64) {
        const int row = i / per_row, c = (i % per_row) * 4;
        const int r = tile.row0 + row;
        const int in_half = a.half ? ct * 32 + (c & 31) : ct * 64 + c;
        if (r >= tile.row_end || in_half >= width) continue;  // N (half) is a multiple of 8: whole vectors
        float4_t v = total(row, c);
        if (a.to_partials) {
            *(float4_t*)(a.partials + ((int64_t)split * a.R + r) * a.N + unit_column<64>(a.half, ct, c)) = v;
            continue;
        }
        if (pairs) {
            const float4_t up = total(row, c + 32);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = silu_mul(v[j], up[j]);
        }
        *(u32x2*)((uint16_t*)a.out + (int64_t)r * a.osm + in_half) = u32x2{pack16<BF16>(v[0], v[1]), pack16<BF16>(v[2], v[3])};
    }
}

template <int FMT, bool BF16, int RT, int FU, bool QX = false>
int launch_one(const ExpertArgs& a, hipStream_t stream) {
    constexpr int NW = 8, D = 3;
    const int64_t tiles = max_row_tiles(a.R, a.E, 16 * RT);
    if (tiles > 65535 || a.S > 65535) {
        set_error("experts: %lld row tiles exceed the grid", (long long)tiles);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    const int lds = NW * 16 * RT * 64 * 4;
    const auto kernel = experts_stream_kernel<FMT, BF16, RT, FU, NW, D, QX>;
    static DeviceOnce once;
    if (once.first()) {
        const int rc = check_hip(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute");
        if (rc != GLA_OK) return rc;
    }
    const int tiles_n = a.half ? (a.half + 31) / 32 : (a.N + 63) / 64;
    kernel<<<dim3(tiles_n, (unsigned)tiles, a.S), NW * 64, lds, stream>>>(a);
    return check_hip(hipGetLastError(), "experts_stream");
}

template <int FMT, bool BF16, int RT>
int launch_fold(const ExpertArgs& a, hipStream_t stream) {
    if constexpr (FMT == kEW4) {
        if (a.group % 128 == 0) return launch_one<FMT, BF16, RT, 128>(a, stream);
        if (a.group % 64 == 0) return launch_one<FMT, BF16, RT, 64>(a, stream);
        return launch_one<FMT, BF16, RT, 32>(a, stream);
    } else if constexpr (FMT == kEF8) {
        if (a.scales_x == nullptr) return launch_one<FMT, BF16, RT, 128, true>(a, stream);
        return launch_one<FMT, BF16, RT, 128>(a, stream);
    } else {
        return launch_one<FMT, BF16, RT, 64>(a, stream);
    }
}

template <int FMT>
int launch_format(const ExpertArgs& a, bool bf16, int row_tiles, hipStream_t stream) {
    if (bf16) return row_tiles > 1 ? launch_fold<FMT, true, 2>(a, stream) : launch_fold<FMT, true, 1>(a, stream);
    return row_tiles > 1 ? launch_fold<FMT, false, 2>(a, stream) : launch_fold<FMT, false, 1>(a, stream);
}

}  // namespace

int launch_experts_stream(const ExpertArgs& a, int format, bool bf16, int row_tiles, hipStream_t stream) {
    switch (format) {
        case kEW4: return launch_format<kEW4>(a, bf16, row_tiles, stream);
        case kEF8: return launch_format<kEF8>(a, bf16, row_tiles, stream);
        default: return launch_format<kE16>(a, bf16, row_tiles, stream);
    }
}

}  // namespace gla
