// Products grouped by expert, many rows per expert: a tiled MFMA GEMM over ragged row blocks.
//
//  * Workgroup tile BM rows of one expert x 256 (BM = 64: 128) columns, 8 (4) waves; pipeline stage of 128 bytes of K per
//    activation row (64 16-bit values or 128 e4m3 codes).  Operand tiles and scales are copied global -> LDS by the load unit
//    (global_load_lds) into a ring of stages, all of them in flight; gated calls gather their activation rows on the
//    way.  16-byte chunk c of a 128-byte row r lies at position c ^ ((r >> 1) & 7), chosen on the global side of the copy,
//    so that the 16 lanes of an LDS read phase hit 16 different bank groups.
//  * The weights are the row operand of every MFMA: a lane holds 4 adjacent output columns of one row.
//  * 16-bit weights and W4: v_mfma_f32_32x32x16, four K-steps per stage, fragments of a K-step read during the one in
//    front of it.  The barrier of a stage stands before its last K-step, whose fragments are in registers by then: the
//    matrix pipe has work while the waves meet and the first fragments of the next stage arrive.
//  * W4: the packed words lie in LDS as they are in memory (a word = 8 K-values of a column = a lane's share of a
//    K-step's operand).  The codes go into the MFMA as they are (bf16 16 + q, fp16 64 + q: a byte select and a masked OR per
//    pair), so that no weight is rounded.  With w = s q + z on a group,
//        sum(x w) = s sum(x (off + q)) + (z - off s) sum(x).
//    First terms: the sums are kept divided by their column's current scale; where a group begins they are multiplied by the
//    old scale over the new one, which needs no second set of accumulators (128 rows: two workgroups on a CU).  Second
//    terms: a launch in front (experts_quant.hip) takes every group's sum of x; sum and constant are three bf16 terms
//    each (24 bits), and eight of the products of two groups fill one MFMA behind the K loop.  Sums that are not finite are
//    taken again from dequantised weights.  (Weights dequantised and rounded in front of the MFMA: the error of a result 1.7
//    times that of its own rounding; the bf16 call below 1010 us whatever the groups, where this takes 1070 for groups of
//    128, 1200 for 64 and 1550 for 32.)
//  * F8: v_mfma_f32_16x16x128 starts from zero on every 128-block and its result joins the fp32 sum times the block's two
//    scales.
//  * gridDim.y splits K where the tiles do not fill the chip (fp32 sums to the workspace, added in order by the
//    finishing kernel).
//  * A workgroup's tile is found from the offsets on the device; the tiles that exist are dealt to the 8 XCDs in
//    contiguous bands, and a band is walked in groups of 8 row tiles x all columns, so that the L2 of an XCD keeps a
//    weight panel for all row tiles of the group.
//
// Measured (calls in a row): 4-bit, E = 8, top 2, 4096 -> 2 x 14336, groups of 128, 2048 tokens 1060 to 1140 us
// by card (840 to 910 TFLOP/s; fp16 1180); fp8,
// E = 32, top 4, 4096 -> 2 x 2048, 4096 tokens 420 us (1310 TFLOP/s); 16-bit, 16 experts of 4096^2, 8200 rows 325 us (850; 1070 at 16000
// rows in 256-row tiles).  What the counters show on random operands, and on zeros, where the power limit does not lower the clock:
//  * 16-bit, 16000 rows: MFMA busy in 63 % of the clocks at 1.50 GHz (zeros: 54 % at 2.28 GHz, 422 for 502 us); LDS reads in 24 %,
//    no bank conflicts; waves spend 47 % of their time at a wait.  Power first, then the waits of a ring of two stages with one
//    workgroup per CU (the dense 16-bit kernel, four stages of half the K: 71 % at 1.55 GHz, 16384 rows in 469 us).
//  * fp8, 16384 rows: MFMA busy 39 % at 2.02 GHz (zeros 37 % at 2.33): not power; LDS reads in 33 %, two fifths of that conflicts.
//  * 4-bit: MFMA busy 52 %, vector instructions 63 % at 1.79 GHz (zeros 53 % and 64 % at 2.25, 870 for 1056 us).
// Without the copies of the K loop, and so without their waits, LDS writes and power, fp8 takes 324 us instead of 412 and 16-bit (16000
// rows) 444 instead of 576; the fold of the fp8 scales costs nothing.
// Measured and not kept: four waves with 128 x 128 wave tiles (a third less read from LDS, one wave per SIMD: 635 against 576
// us at 16000 rows), 256 x 128 tiles on four waves with two workgroups per CU (667), stages of 64 bytes of K in a ring of four
// (600; 128 rows 733 against 598).
#include <type_traits>

#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

__device__ __align__(16) unsigned char g_zero_chunk[16];  // what activations past the end of K are read from

__device__ __forceinline__ void bare_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int FMT, int BM, int BN>
struct GemmShape {
    static constexpr int WAVES = BN / 32, THREADS = 64 * WAVES;
    static constexpr int WC = FMT == kEW4 ? 32 : 64;               // wave columns (W4: no weight is dequantised twice)
    static constexpr int WN = BN / WC, WM = BM / (WAVES / WN);     // waves side by side, rows of a wave
    static constexpr int A_BYTES = BM * 128;
    static constexpr int B_BYTES = FMT == kEW4 ? 8 * BN * 4 : BN * 128;
    // W4: [32-half][column]; F8: rows, columns
    static constexpr int M_BYTES = FMT == kEW4 ? 4 * BN : (FMT == kEF8 ? (BM + BN) * 4 : 0);
    static constexpr int STAGE = A_BYTES + B_BYTES + M_BYTES;
    static constexpr int RING = FMT == kEW4 ? (BM == 128 ? 3 : 4) : (BM == 256 ? 2 : 3);  // (W4: two workgroups per CU)
    static constexpr int A_JOBS = BM / 8 / WAVES;                  // copies per wave and stage
    static constexpr int B_JOBS = B_BYTES / 1024 / WAVES;
    static constexpr int M_JOBS = FMT == kE16 ? 0 : 1;
    static constexpr int LPS = A_JOBS + B_JOBS + M_JOBS;
    static constexpr int X_OFF = RING * STAGE;                     // W4: 32 floats per wave, see `spread`
    static constexpr int LDS = X_OFF + (FMT == kEW4 ? WAVES * 128 : 0);
};

// One tile of up to BM rows x BN columns.
template <int FMT, bool BF16, int BM, int BN>
__device__ __forceinline__ void gemm_tile(const ExpertArgs& a, const ExpertTile& tile, int ct, unsigned char* smem) {
    using SH = GemmShape<FMT, BM, BN>;
    constexpr int WAVES = SH::WAVES;
    constexpr int RING = SH::RING, LPS = SH::LPS, WC = SH::WC, WM = SH::WM;
    constexpr bool F8 = FMT == kEF8, W4 = FMT == kEW4;
    constexpr int MT = F8 ? 16 : 32;                   // MFMA tile edge
    constexpr int TI = WM / MT, TJ = WC / MT;
    constexpr int KS = F8 ? 128 : 64;                  // K-values per stage
    constexpr int ES = F8 ? 1 : 2;                     // bytes per activation
    constexpr int B_OFF = SH::A_BYTES, M_OFF = SH::A_BYTES + SH::B_BYTES;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / SH::WN, wn = wave % SH::WN;
    const int expert = tile.expert;
    const int width = a.half ? a.half : a.N;

    // ---- copies
    const int Kb = a.K * ES;                                     // bytes of an activation row
    const int k_first = blockIdx.y * a.chunk;                    // first stage of this K split
    const int all_stages = (a.K + KS - 1) / KS;
    const int stages = all_stages - k_first < a.chunk ? all_stages - k_first : a.chunk;
    const unsigned char* a_src[SH::A_JOBS];
    int a_dst[SH::A_JOBS], a_chunk[SH::A_JOBS];
#pragma unroll
    for (int i = 0; i < SH::A_JOBS; ++i) {
        const int row = (wave + WAVES * i) * 8 + (lane >> 3);
        int r = tile.row0 + row;
        if (r > tile.row_end - 1) r = tile.row_end - 1;          // multiplied, never stored
        a_chunk[i] = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
        a_src[i] = a.x + source_row(a, r) * a.xsm + a_chunk[i] + (int64_t)k_first * 128;
        a_dst[i] = (wave + WAVES * i) * 1024;
    }
    const unsigned char* we = a.w + (int64_t)expert * a.w_stride_e;
    const unsigned char* se = a.scales + (int64_t)expert * a.meta_stride_e;
    const unsigned char* ze = a.zeros == nullptr ? se : a.zeros + (int64_t)expert * a.meta_stride_e;
    uint32_t b_off[SH::B_JOBS];
    int b_chunk = 0, w4_row = 0;
    if constexpr (W4) {
        const int c = (4 * lane) % BN;                           // of the tile: 4 columns per lane,
        w4_row = wave * (256 / BN) + 4 * lane / BN;              // 256 / BN word rows of the stage per wave
        b_off[0] = ((uint32_t)unit_column_inside<WC>(a.half, a.N, ct * SH::WN + c / WC, c % WC) + (uint32_t)w4_row * (uint32_t)a.N) * 4u;
    } else {
#pragma unroll
        for (int i = 0; i < SH::B_JOBS; ++i) {
            const int c = (wave + WAVES * i) * 8 + (lane >> 3);
            b_chunk = ((lane & 7) ^ ((c >> 1) & 7)) * 16;        // the same for all i (c advances by 8 WAVES)
            b_off[i] = (uint32_t)unit_column_inside<WC>(a.half, a.N, ct * SH::WN + c / WC, c % WC) * (uint32_t)(a.K * ES);
        }
    }
    // one 4-byte copy per wave and stage: W4: scales of 128 columns for one 32-half of the stage (four jobs, done twice: all
    // waves have the same number of copies in flight); F8: the activation scales of 64 rows, or the block scale of each of
    // 64 columns
    uint32_t m_off = 0;
    int64_t m_row = 0;
    int m_dst = 0, m_half = 0, m_step = (a.N + 127) / 128 * 4;
    const unsigned char* m_src = se;
    if constexpr (W4) {
        static_assert(BN == 256, "four copies of scales");
        const int part = wave & 1, c = part * 128 + 2 * lane;
        m_half = (wave >> 1) & 1;
        // (a pair lies inside the run of 4 it belongs to)
        m_off = (uint32_t)(unit_column_inside<WC>(a.half, a.N, ct * SH::WN + (c & ~3) / WC, (c & ~3) % WC) + (c & 3)) * 2u;
        m_dst = M_OFF + m_half * (BN * 2) + part * 256;
    } else if constexpr (F8) {
        constexpr int JOBS = BM / 64 + BN / 64;
        static_assert(JOBS <= WAVES, "one scale copy per wave");
        const int q = wave < JOBS ? wave : JOBS - 1;
        if (q < BM / 64) {
            int r = tile.row0 + q * 64 + lane;
            if (r > tile.row_end - 1) r = tile.row_end - 1;
            m_row = source_row(a, r) * (a.K / 128) * 4;
            m_src = (const unsigned char*)a.scales_x;
            m_step = 4;
        } else {
            const int c = (q - BM / 64) * 64 + lane;
            m_row = (unit_column_inside<WC>(a.half, a.N, ct * SH::WN + (c & ~3) / WC, (c & ~3) % WC) >> 7) * 4;
        }
        m_dst = M_OFF + q * 256;
    }
    const int groups = a.groups;
    const unsigned char* zero_chunk = g_zero_chunk;
    asm volatile("" : "+s"(zero_chunk));  // its address stays in registers
    typedef const __attribute__((address_space(1))) void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    // The weights' address of a stage is a wave-uniform base that advances per stage plus a 32-bit lane offset; the base
    // is made opaque, or the compiler keeps one 64-bit address per copy in vector registers, which the accumulators need.
    const int64_t b_step = W4 ? (int64_t)a.N * 32 : 128;
    const unsigned char* b_base = we + k_first * b_step;
    auto issue_one = [&](int k, int slot, int c) __attribute__((always_inline)) {
        unsigned char* base = smem + slot * SH::STAGE;
        if (c < SH::A_JOBS) {
            const unsigned char* p = a_src[c] + (int64_t)k * 128;
            if constexpr (!F8) p = (k_first + k) * 128 + a_chunk[c] < Kb ? p : zero_chunk;
            __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(base + a_dst[c]), 16, 0, 0);
        } else if (c < SH::A_JOBS + SH::B_JOBS) {
            const int i = c - SH::A_JOBS;
            if constexpr (W4) {
                // word rows past the end of K: the stage's first ones again (they meet zeros)
                const uint32_t back = (k_first + k) * 8 + w4_row < a.K / 8 ? 0u : (uint32_t)a.N * 16u;
                __builtin_amdgcn_global_load_lds((gptr)(b_base + (b_off[0] - back)), (lptr)(base + B_OFF + wave * 1024), 16, 0, 0);
            } else {
                const uint32_t chunk = F8 || (k_first + k) * 128 + b_chunk < Kb ? (uint32_t)b_chunk : 0u;
                __builtin_amdgcn_global_load_lds((gptr)(b_base + (b_off[i] + chunk)), (lptr)(base + B_OFF + (wave + WAVES * i) * 1024), 16, 0, 0);
            }
        } else if constexpr (W4) {
            int g = (int)divide_by((uint32_t)((k_first + k) * 2 + m_half), a.group_mul);
            if (g > groups - 1) g = groups - 1;
            __builtin_amdgcn_global_load_lds((gptr)(m_src + (int64_t)g * a.N * 2 + m_off), (lptr)(base + m_dst), 4, 0, 0);
        } else if constexpr (F8) {
            const unsigned char* p = m_src + (int64_t)(k_first + k) * m_step + m_row;
            __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(base + m_dst), 4, 0, 0);
        }
        if (c == LPS - 1) {
            b_base += b_step;
            asm volatile("" : "+s"(b_base));
        }
    };

    // ---- accumulators and fragment addresses
    typedef typename std::conditional<F8, float4_t, float16_t>::type acc_t;
    constexpr int AE = F8 ? 4 : 16;
    acc_t acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < AE; ++e) acc[i][j][e] = 0.0f;
    int fr = lane & (MT - 1), fk = lane / MT;        // row of a fragment, K part
    const int swz = (fr >> 1) & 7;                   // (tile offsets are multiples of 16 rows)
    const int a_row = (wm * WM + fr) * 128, b_row = B_OFF + (wn * WC + fr) * 128;

#pragma unroll
    for (int u = 0; u < RING; ++u)
        if (u < stages) {
#pragma unroll
            for (int c = 0; c < LPS; ++c) issue_one(u, u, c);
        }
    if (stages >= RING) wait_vmcnt<(RING - 1) * LPS>();
    else wait_vmcnt<0>();
    bare_barrier();

    if constexpr (F8) {
        typedef union {
            int8_t_v v;
            u32x4 c[2];
        } op_t;
        const int c0 = ((2 * fk) ^ swz) * 16, c1 = ((2 * fk + 1) ^ swz) * 16;
        // Tile (i, j) of the wave is slice q = i TJ + j of a stage: its MFMA, the fold of the slice three in front, and a
        // share of the LDS reads and copies, with the scheduler fenced between slices (left alone it reads every fragment
        // right in front of its MFMA).  The fragment of activation row tile i + 1 is read during tile i; the barrier
        // stands before the last row tile, and a column's weight fragment for the next stage is read behind the last MFMA
        // that uses the old one.
        op_t fa[2], fb[TJ];
        float sx[2], sw[TJ];
        float4_t d[4];
        float sc[4];
        const float4_t zero4 = float4_t{0.f, 0.f, 0.f, 0.f};
        auto read_a = [&](const unsigned char* base, int i, int buf) __attribute__((always_inline)) {
            fa[buf].c[0] = *(const u32x4*)(base + a_row + i * 2048 + c0);
            fa[buf].c[1] = *(const u32x4*)(base + a_row + i * 2048 + c1);
            sx[buf] = *(const float*)(base + M_OFF + (wm * WM + i * 16 + fr) * 4);
        };
        auto read_b = [&](const unsigned char* base, int j) __attribute__((always_inline)) {
            fb[j].c[0] = *(const u32x4*)(base + b_row + j * 2048 + c0);
            fb[j].c[1] = *(const u32x4*)(base + b_row + j * 2048 + c1);
            sw[j] = *(const float*)(base + M_OFF + (BM + wn * WC + j * 16 + 4 * fk) * 4);
        };
        constexpr int NS = TI * TJ;
        auto fold = [&](int q) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[q / TJ][q % TJ][e] = __builtin_fmaf(d[q % 4][e], sc[q % 4], acc[q / TJ][q % TJ][e]);
        };
        static_assert(TJ == 4 && TI % 2 == 0, "slices");
        read_a(smem, 0, 0);
#pragma unroll
        for (int j = 0; j < TJ; ++j) read_b(smem, j);
        const unsigned char* base = smem;
        int slot = 0;
        auto stage = [&](int k, auto refill_tag) __attribute__((always_inline)) {
            constexpr bool REFILL = decltype(refill_tag)::value;
            const int next_slot = slot == RING - 1 ? 0 : slot + 1;
            const unsigned char* next = smem + next_slot * SH::STAGE;
#pragma unroll
            for (int q = 0; q < NS; ++q) {
                const int i = q / TJ, j = q % TJ;
                if (q == (TI - 1) * TJ) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    wait_vmcnt<REFILL ? (RING - 2) * LPS : 0>();
                    bare_barrier();
                }
                d[q % 4] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j].v, fa[i & 1].v, zero4, 0, 0, 0, 127, 0, 127);
                sc[q % 4] = sx[i & 1] * sw[j];
                if (q >= 3) fold(q - 3);
                if (i + 1 < TI) {
                    if (j == 0) read_a(base, i + 1, (i + 1) & 1);
                } else {
                    if (j == 0) read_a(next, 0, 0);
                    read_b(next, j);
                    if constexpr (REFILL) {
#pragma unroll
                        for (int c = j * LPS / TJ; c < (j + 1) * LPS / TJ; ++c) issue_one(k + RING, slot, c);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            fold(NS - 3);
            fold(NS - 2);
            fold(NS - 1);
            slot = next_slot;
            base = next;
        };
        int k = 0;
#pragma unroll 1
        for (; k + RING < stages; ++k) stage(k, std::true_type{});
#pragma unroll 1
        for (; k < stages; ++k) stage(k, std::false_type{});
    } else if constexpr (W4) {
        static_assert(TJ == 1 && WM == BM, "a wave has 32 columns and every row");
        constexpr float OFF = BF16 ? 16.0f : 64.0f;                                     // of a code in the MFMA
        constexpr uint32_t CODE = BF16 ? 0x00780078u : 0x00f000f0u, BASE = BF16 ? 0x41804180u : 0x54005400u;
        float* const mine = (float*)(smem + SH::X_OFF) + wave * 32;
        u32x4 fa[TI], fb[2];         // (an activation fragment is read anew behind its one MFMA of a K-step)
        uint32_t word, scale;        // codes of the next K-step, the lane's column's scale of the 32-half it belongs to
        uint32_t mask = CODE, offset = BASE;  // 0 where that scale is 0: codes of such a group enter as zeros
        static_assert(SH::STAGE % 128 == 0, "rows of 128 bytes");
        uint32_t a_off = (uint32_t)(fr * 128 + (fk ^ swz) * 16);
        auto read_a = [&](const unsigned char* base, int s, int i) __attribute__((always_inline)) {
            fa[i] = *(const u32x4*)(base + (a_off ^ (32 * s)) + i * 32 * 128);  // chunk (2 s + fk) ^ swz of the row
        };
        auto read_word = [&](const unsigned char* base, int s) __attribute__((always_inline)) {
            word = *(const uint32_t*)(base + B_OFF + (2 * s + fk) * (BN * 4) + (wn * WC + fr) * 4);
        };
        auto read_scale = [&](const unsigned char* base, int h) __attribute__((always_inline)) {
            scale = *(const uint16_t*)(base + M_OFF + h * (BN * 2) + (wn * WC + fr) * 2);
        };
        // register q of the operand: OFF + codes 2q, 2q + 1, a shift each for the word and a byte select and a masked OR here
        auto convert = [&](int q) __attribute__((always_inline)) -> uint32_t {
            const uint32_t lo = BF16 ? word << 3 : word << 4, hi = BF16 ? word >> 1 : word;
            return (__builtin_amdgcn_perm(hi, lo, 0x0c000c00u | ((4 + q) << 16) | q) & mask) | offset;
        };
        auto choose = [&]() __attribute__((always_inline)) {
            const bool none = (scale & 0x7fffu) == 0;
            mask = none ? 0u : CODE;
            offset = none ? 0u : BASE;
        };
        auto mfma = [&](const u32x4& b, const u32x4& x, float16_t c) __attribute__((always_inline)) {
            if constexpr (BF16)
                return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, b), __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, b), __builtin_bit_cast(half8_t, x), c, 0, 0, 0);
        };
        // a factor of the lane's column, to the lanes that hold the column's sums: through LDS (one wave: in order)
        auto put = [&](float v) __attribute__((always_inline)) {
            mine[fr] = v;
            __builtin_amdgcn_wave_barrier();
        };
        auto times = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4_t f = *(const float4_t*)(mine + 8 * g + 4 * fk);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][0][4 * g + e] *= f[e];
            }
        };
        const int halves = a.group / 32;
        int left = halves;  // 32-halves to the next group (a split begins where a group does)
        bool enters = false;
        float unit = 1.0f;                           // the scale the column's sums are divided by
        // exponent of the column's first scale that is not 0 (-1: none yet): the others have to be within 2^60 of it, so that no
        // sum in their units leaves fp32's range
        int reference = -1;
        auto exponent = [](float s) __attribute__((always_inline)) { return (int)(__builtin_bit_cast(uint32_t, s) >> 23 & 255u); };
        auto enter_group = [&]() __attribute__((always_inline)) {
            const float s = low16<BF16>(scale);
            float r = 1.0f;
            if (s != 0.0f) {
                if (reference < 0) reference = exponent(s);  // (the sums are 0)
                else r = unit / s;
                const int off = exponent(s) - reference;
                if (off > 60 || off < -60) r = __builtin_nanf("");  // (taken again below)
                unit = s;
            }
            put(r);
        };

        const unsigned char* base = smem;
#pragma unroll
        for (int i = 0; i < TI; ++i) read_a(base, 0, i);
        read_scale(base, 0);
        read_word(base, 0);
        choose();
        if (low16<BF16>(scale) != 0.0f) {
            unit = low16<BF16>(scale);
            reference = exponent(unit);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) fb[0][q] = convert(q);
        int slot = 0;
        auto stage = [&](int k, auto refill_tag) __attribute__((always_inline)) {
            constexpr bool REFILL = decltype(refill_tag)::value;
            const int next_slot = slot == RING - 1 ? 0 : slot + 1;
            const unsigned char* next = smem + next_slot * SH::STAGE;
            asm volatile("" : "+v"(a_off));  // or one address per K-step stays in registers, which the sums need
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int cur = s & 1, nxt = cur ^ 1;
                if (s == 3) {  // as for 16-bit weights
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    wait_vmcnt<REFILL ? (RING - 2) * LPS : 0>();
                    bare_barrier();
                }
                const unsigned char* from = s == 3 ? next : base;
                const int s1 = (s + 1) & 3;
                if (s % 2 == 0 && enters) {
#pragma unroll
                    for (int i = 0; i < TI; ++i) times(i);
                }
                read_word(from, s1);
                if (s == 1) read_scale(base, 1);
                if (s == 3) read_scale(next, 0);
                // slices of one MFMA each, with the scheduler fenced between them
#pragma unroll
                for (int i = 0; i < TI; ++i) {
                    acc[i][0] = mfma(fb[cur], fa[i], acc[i][0]);
                    read_a(from, s1, i);
                    if (s % 2 == 1 && i == 0) choose();
#pragma unroll
                    for (int q = i * 4 / TI; q < (i + 1) * 4 / TI; ++q) fb[nxt][q] = convert(q);
                    if (s % 2 == 1 && i == TI - 1) {  // does the next 32-half begin a group?
                        enters = --left == 0 && (s == 1 || k + 1 < stages);
                        if (enters) {
                            enter_group();
                            left = halves;
                        }
                    }
                    if constexpr (REFILL) {
                        if (s == 3) {
#pragma unroll
                            for (int c = i * LPS / TI; c < (i + 1) * LPS / TI; ++c) issue_one(k + RING, slot, c);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            slot = next_slot;
            base = next;
        };
        int k = 0;
#pragma unroll 1
        for (; k + RING < stages; ++k) stage(k, std::true_type{});
#pragma unroll 1
        for (; k < stages; ++k) stage(k, std::false_type{});
        // (the lane's number anew: nothing but the sums, the unit and wave-uniform values stays in registers behind the loop)
        int fresh = 0;
        asm volatile("" : "+s"(fresh));
        fresh = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (uint32_t)fresh));
        put(unit);
        fr = fresh & 31;
        fk = fresh >> 5;
#pragma unroll
        for (int i = 0; i < TI; ++i) times(i);

        // ---- the groups' constants times their sums of activations, two groups to an MFMA
        const int k0 = k_first * 64, k1 = k0 + stages * 64 < a.K ? k0 + stages * 64 : a.K;
        const int g0 = k0 / a.group, g1 = (k1 + a.group - 1) / a.group;
        const int col = unit_column_inside<WC>(a.half, a.N, ct * SH::WN + wn, fr & ~3) + (fr & 3);
        constexpr int AT_ONCE = 16, PIECES = BM * AT_ONCE / SH::THREADS, STEPS = AT_ONCE / 2;  // groups, pieces per thread, MFMAs
        static_assert(BM * AT_ONCE * 16 <= SH::X_OFF, "sums of a chunk of groups fit the ring");
        const int piece = wave * 64 + (fk * 32 + fr);
        uint32_t x_off = (uint32_t)(fr * (AT_ONCE * 16) + (fk ^ (fr & (AT_ONCE - 1))) * 16);  // piece 2 j + fk of a row: ^ 32 j
        const unsigned char* from[PIECES];
        u32x4 held[PIECES];
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            int r = tile.row0 + (piece + q * SH::THREADS) / AT_ONCE;
            if (r > tile.row_end - 1) r = tile.row_end - 1;
            from[q] = a.sums + (source_row(a, r) * groups + piece % AT_ONCE) * 16;
        }
        auto hold = [&](int gc) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                held[q] = u32x4{0, 0, 0, 0};
                if (gc + piece % AT_ONCE < g1) held[q] = *(const u32x4*)(from[q] + (int64_t)gc * 16);
            }
        };
#pragma unroll 1
        for (int gc = g0; gc < g1; gc += AT_ONCE) {
            hold(gc);
            uint32_t sb[STEPS], zb[STEPS];  // (all in flight together)
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                const int g = gc + 2 * j + fk;
                const int64_t at = ((int64_t)(g < g1 ? g : g1 - 1) * a.N + col) * 2;
                sb[j] = *(const uint16_t*)(se + at);
                zb[j] = *(const uint16_t*)(ze + at);
            }
            __syncthreads();  // the ring (the chunk in front) has been read
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                const int row = (piece + q * SH::THREADS) / AT_ONCE;
                *(u32x4*)(smem + row * (AT_ONCE * 16) + (((piece % AT_ONCE) ^ (row & (AT_ONCE - 1))) * 16)) = held[q];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                if (gc + 2 * j >= g1) break;
                asm volatile("" : "+v"(x_off));  // (no address per step in registers)
                const float sc = low16<BF16>(sb[j]);
                float z = a.zeros == nullptr ? 0.0f : low16<BF16>(zb[j]) * __builtin_fmaf(a.c2, sc, a.c1);
                z = gc + 2 * j + fk < g1 ? __builtin_fmaf(-OFF, sc, z) : 0.0f;
                uint32_t t[3];
                bf16_terms(z, t);
                const u32x4 b = u32x4{high_halves(t[0], t[0]), high_halves(t[0], t[1]), high_halves(t[1], t[1]), high_halves(t[2], t[2])};
#pragma unroll
                for (int i = 0; i < TI; ++i) {
                    const u32x4 x = *(const u32x4*)(smem + (x_off ^ (32 * j)) + i * 32 * (AT_ONCE * 16));
                    acc[i][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, b), __builtin_bit_cast(bf16x8_t, x), acc[i][0], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);  // (or the fragments of all steps are read first, which takes the sums' registers)
            }
        }

        // ---- sums that are not finite, perhaps only because of the codes' offset (inf - inf, or an overflow of OFF x) or of scales
        // that are 2^60 apart: again from dequantised weights, rounded to 16 bits
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 16; ++e) odd = odd || !(__builtin_fabsf(acc[i][0][e]) < __builtin_inff());
            if (!__any(odd)) continue;
            int r = tile.row0 + i * 32 + fr;
            if (r > tile.row_end - 1) r = tile.row_end - 1;
            const unsigned char* x = a.x + source_row(a, r) * a.xsm + fk * 16;
            float16_t plain;
#pragma unroll
            for (int e = 0; e < 16; ++e) plain[e] = 0.0f;
#pragma unroll 1
            for (int k = k0; k < k1; k += 16) {
                const uint32_t w = *(const uint32_t*)(we + ((int64_t)(k / 8 + fk) * a.N + col) * 4);
                const int64_t at = ((int64_t)(k / a.group) * a.N + col) * 2;
                const float sc = low16<BF16>(*(const uint16_t*)(se + at));
                const float z = a.zeros == nullptr ? 0.0f : low16<BF16>(*(const uint16_t*)(ze + at)) * __builtin_fmaf(a.c2, sc, a.c1);
                u32x4 b;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    b[q] = pack16<BF16>(__builtin_fmaf((float)((w >> (8 * q)) & 15u), sc, z), __builtin_fmaf((float)((w >> (8 * q + 4)) & 15u), sc, z));
                plain = mfma(b, *(const u32x4*)(x + (int64_t)k * 2), plain);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!(__builtin_fabsf(acc[i][0][e]) < __builtin_inff())) acc[i][0][e] = plain[e];
        }
    } else {
        u32x4 fa[2][TI], fb[2][TJ];
        auto read_a = [&](const unsigned char* base, int s, int buf, int i) __attribute__((always_inline)) {
            fa[buf][i] = *(const u32x4*)(base + a_row + i * 32 * 128 + (((2 * s + fk) ^ swz) * 16));
        };
        auto read_b = [&](const unsigned char* base, int s, int buf, int j) __attribute__((always_inline)) {
            fb[buf][j] = *(const u32x4*)(base + b_row + j * 32 * 128 + (((2 * s + fk) ^ swz) * 16));
        };
        auto mfma = [&](int i, int j, int buf, const u32x4& b) __attribute__((always_inline)) {
            if constexpr (BF16)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, b), __builtin_bit_cast(bf16x8_t, fa[buf][i]), acc[i][j], 0, 0, 0);
            else
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, b), __builtin_bit_cast(half8_t, fa[buf][i]), acc[i][j], 0, 0, 0);
        };
        // the copies of the last K-step's slice q (the slot is free behind the stage's barrier)
        auto refill_slice = [&](int k, int slot, int q, bool on) __attribute__((always_inline)) {
            if (!on) return;
#pragma unroll
            for (int c = q * LPS / (TI * TJ); c < (q + 1) * LPS / (TI * TJ); ++c) issue_one(k + RING, slot, c);
        };

        // ---- prologue: fragments of K-step 0
        const unsigned char* base = smem;
#pragma unroll
        for (int i = 0; i < TI; ++i) read_a(base, 0, 0, i);
#pragma unroll
        for (int j = 0; j < TJ; ++j) read_b(base, 0, 0, j);
        int slot = 0;
        auto stage = [&](int k, auto refill_tag) __attribute__((always_inline)) {
            constexpr bool REFILL = decltype(refill_tag)::value;
            const int next_slot = slot == RING - 1 ? 0 : slot + 1;
            const unsigned char* next = smem + next_slot * SH::STAGE;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int cur = s & 1, nxt = cur ^ 1;
                if (s == 3) {
                    // the fragments of this K-step are in registers; the next stage's copies have landed, here and (behind the
                    // barrier) everywhere, and nobody reads this stage's slot any more
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    wait_vmcnt<REFILL ? (RING - 2) * LPS : 0>();
                    bare_barrier();
                }
                const unsigned char* from = s == 3 ? next : base;
                const int s1 = (s + 1) & 3;
                // slices of one MFMA each, with the scheduler fenced between them (left alone it reads every fragment
                // right in front of its MFMA)
#pragma unroll
                for (int q = 0; q < TI * TJ; ++q) {
                    const int i = q / TJ, j = q % TJ;
                    mfma(i, j, cur, fb[cur][j]);
                    if (q < TJ) read_b(from, s1, nxt, q);
                    if (j == 0) read_a(from, s1, nxt, i);
                    if (s == 3) refill_slice(k, slot, q, REFILL);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            slot = next_slot;
            base = next;
        };
        int k = 0;
#pragma unroll 1
        for (; k + RING < stages; ++k) stage(k, std::true_type{});
#pragma unroll 1
        for (; k < stages; ++k) stage(k, std::false_type{});
    }

    // ---- epilogue: the lane holds row fr of an MFMA tile and runs of 4 columns
    constexpr int RUNS = AE / 4;
    auto run_col = [&](int j, int g) __attribute__((always_inline)) { return F8 ? j * 16 + 4 * fk : j * 32 + 8 * g + 4 * fk; };  // of the wave tile
    auto get = [&](int i, int j, int g) __attribute__((always_inline)) {
        float4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
        if (a.bias != nullptr && blockIdx.y == 0) {
            const float4_t b = *(const float4_t*)(a.bias + (int64_t)expert * a.N + unit_column_inside<WC>(a.half, a.N, ct * SH::WN + wn, run_col(j, g)));
            v += b;
        }
        return v;
    };
    const bool pairs = a.half != 0 && !a.to_partials;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int r = tile.row0 + wm * WM + i * MT + fr;
        if (r >= tile.row_end) continue;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int g = 0; g < RUNS; ++g) {
                const int c = run_col(j, g);
                const bool second = c >= WC / 2;
                const int in = a.half ? (ct * SH::WN + wn) * (WC / 2) + (c % (WC / 2)) : (ct * SH::WN + wn) * WC + c;
                if (in >= width) continue;
                if (a.to_partials) {
                    *(float4_t*)(a.partials + ((int64_t)blockIdx.y * a.R + r) * a.N + in + (a.half && second ? a.half : 0)) = get(i, j, g);
                } else if (!pairs) {
                    const float4_t v = get(i, j, g);
                    *(u32x2*)((uint16_t*)a.out + (int64_t)r * a.osm + in) = u32x2{pack16<BF16>(v[0], v[1]), pack16<BF16>(v[2], v[3])};
                } else if (!second) {
                    // the up columns: WC / 2 further on, in the same lane
                    constexpr int HALF = WC / 2;
                    constexpr int DJ = F8 ? HALF / 16 : HALF / 32, DG = F8 || HALF >= 32 ? 0 : HALF / 8;
                    const int j2 = j + DJ < TJ ? j + DJ : j, g2 = g + DG < RUNS ? g + DG : g;
                    const float4_t v = get(i, j, g), up = get(i, j2, g2);
                    float h[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] = silu_mul(v[e], up[e]);
                    *(u32x2*)((uint16_t*)a.out + (int64_t)r * a.osm + in) = u32x2{pack16<BF16>(h[0], h[1]), pack16<BF16>(h[2], h[3])};
                }
            }
    }
}

// Workgroup tile of at most BM rows x BN columns.  A tile with fewer rows than a shorter tile has (an expert's last one)
// runs as that: 8200 rows on 16 experts of 4096^2, 16-bit, took 329 us when every tile cost as much as a full one.
template <int FMT, bool BF16, int BM, int BN>
__global__ __launch_bounds__((GemmShape<FMT, BM, BN>::THREADS), (FMT == kEW4 ? 4 : 1)) void experts_gemm_kernel(ExpertArgs a, int tiles_n) {
    extern __shared__ __align__(16) unsigned char smem[];
    int ct = 0;
    const ExpertTile tile = find_tile<BM>(a.offsets, a.E, a.R, !a.to_partials, [&](int total_m) {
        const int total = total_m * tiles_n, pid = blockIdx.x;
        if (pid >= total) return -1;
        const int xcd = pid & 7, q = total >> 3, r = total & 7;
        const int t = xcd * q + (xcd < r ? xcd : r) + (pid >> 3);
        constexpr int GROUP = 8;
        const int width = GROUP * tiles_n, group = t / width, first = group * GROUP;
        const int rows = total_m - first < GROUP ? total_m - first : GROUP;
        ct = (t - group * width) / rows;
        return first + (t - group * width) % rows;
    });
    if (tile.expert < 0) return;
    const int rows = tile.row_end - tile.row0;
    if (tile.expert >= a.E) {  // rows without an expert
        const int width = a.half ? a.half : a.N;
        const int c0 = a.half ? ct * (BN / 2) : ct * BN, cols = a.half ? BN / 2 : BN;
        for (int i = threadIdx.x; i < rows * (cols / 4); i += blockDim.x) {
            const int r = tile.row0 + i / (cols / 4), c = c0 + (i % (cols / 4)) * 4;
            if (c < width) *(u32x2*)((uint16_t*)a.out + (int64_t)r * a.osm + c) = u32x2{0, 0};
        }
        return;
    }
    if constexpr (BM >= 256) {
        if (rows > 128) {
            gemm_tile<FMT, BF16, 256, BN>(a, tile, ct, smem);
            return;
        }
    }
    if constexpr (BM >= 128) {
        if (rows > 64) {
            gemm_tile<FMT, BF16, 128, BN>(a, tile, ct, smem);
            return;
        }
    }
    gemm_tile<FMT, BF16, 64, BN>(a, tile, ct, smem);
}

template <int FMT, bool BF16, int BM, int BN>
int launch_one(const ExpertArgs& a, hipStream_t stream) {
    constexpr int L64 = GemmShape<FMT, 64, BN>::LDS, L128 = BM >= 128 ? GemmShape<FMT, 128, BN>::LDS : 0, L256 = BM >= 256 ? GemmShape<FMT, 256, BN>::LDS : 0;
    constexpr int LA = L64 > L128 ? L64 : L128, LDS = LA > L256 ? LA : L256;
    static_assert(LDS <= 160 * 1024, "ring does not fit LDS");
    const int cols = a.half ? BN / 2 : BN, width = a.half ? a.half : a.N;
    const int tiles_n = (width + cols - 1) / cols;
    const int64_t grid = max_row_tiles(a.R, a.E, BM) * tiles_n;
    if (grid >= (int64_t)1 << 31) {
        set_error("experts: %lld tiles exceed the grid", (long long)grid);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    const auto kernel = experts_gemm_kernel<FMT, BF16, BM, BN>;
    static DeviceOnce once;
    if (once.first()) {
        const int rc = check_hip(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS), "hipFuncSetAttribute");
        if (rc != GLA_OK) return rc;
    }
    kernel<<<dim3((unsigned)grid, a.S), GemmShape<FMT, BM, BN>::THREADS, LDS, stream>>>(a, tiles_n);
    return check_hip(hipGetLastError(), "experts_gemm");
}

// 64-row tiles (little arithmetic per weight: bound by memory) of fp8 and 16-bit weights: 4 waves on 128 columns, so that
// two workgroups share a CU and one starts while the other streams (256 tokens, 16 experts of 4096^2, 16-bit: 105 -> 98 us;
// 64 tokens top 8 of 128, fp8 2048 -> 2 x 768: 64 -> 57 us).  4-bit weights fill LDS less and do better on 256 columns
// (64 tokens top 2 of 8, 4096 -> 2 x 14336: 160 against 182 us), as do all taller tiles, which read least from LDS that way.
template <int FMT, bool BF16>
int launch_bm(const ExpertArgs& a, int bm, hipStream_t stream) {
    if constexpr (FMT != kEW4) {
        if (bm >= 256) return launch_one<FMT, BF16, 256, 256>(a, stream);
    }
    if (bm >= 128) return launch_one<FMT, BF16, 128, 256>(a, stream);
    return launch_one<FMT, BF16, 64, FMT == kEW4 ? 256 : 128>(a, stream);
}

}  // namespace

int launch_experts_gemm(const ExpertArgs& a, int format, bool bf16, int bm, hipStream_t stream) {
    switch (format) {
        case kEW4: return bf16 ? launch_bm<kEW4, true>(a, bm, stream) : launch_bm<kEW4, false>(a, bm, stream);
        case kEF8: return bf16 ? launch_bm<kEF8, true>(a, bm, stream) : launch_bm<kEF8, false>(a, bm, stream);
        default: return bf16 ? launch_bm<kE16, true>(a, bm, stream) : launch_bm<kE16, false>(a, bm, stream);
    }
}

}  // namespace gla
