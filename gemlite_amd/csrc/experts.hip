// C entry points of the mixture-of-experts operators: argument checks, the choice between the streaming kernel and the
// tiled GEMM, and the finishing kernel that joins K splits and the experts of a token.
#include <numeric>

#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

struct FinishArgs {
    const float* partials;   // [S][R][N]
    const int32_t* offsets;
    const int32_t* places;   // combined: [T][k]
    const float* weights;    // combined: [T][k]
    void* out;
    int64_t osm;
    int R, E, N, S, k, half;
};

// out[r] = sum of the splits (gated: silu(gate) * up of it), or zeros where the row has no expert; combined: out[t] =
// sum over the token's slots of weight * sum of the splits of its row.  All sums in fp32, in a fixed order; bound by the
// fp32 rows it reads (32008 rows of 2048 to 4001 tokens: 50 us for 278 MB).  The rows are not rounded to 16 bits on the way,
// which would halve that: it would add an error as large as that of rounding the result.  A thread takes 4 columns of one row.
template <bool BF16, bool COMBINED>
__global__ __launch_bounds__(256) void experts_finish_kernel(FinishArgs a) {
    const int64_t row = blockIdx.x;
    const int width = a.half ? a.half : a.N;
    const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (c >= width) return;
    const int from = a.offsets[0] > 0 ? a.offsets[0] : 0;  // rows outside from .. limit - 1 have no expert
    int limit = a.offsets[a.E];
    if (limit > a.R) limit = a.R;
    const int64_t slab = (int64_t)a.R * a.N;
    auto sum_at = [&](int64_t r, int col) __attribute__((always_inline)) {
        const float* p = a.partials + r * a.N + col;
        float4_t v = *(const float4_t*)p;
        for (int s = 1; s < a.S; ++s) v += *(const float4_t*)(p + s * slab);
        return v;
    };
    float4_t v = float4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (COMBINED) {
        for (int j = 0; j < a.k; ++j) {
            const int p = a.places[row * a.k + j];
            if (p < from || p >= limit) continue;
            const float w = a.weights[row * a.k + j];
            const float4_t y = sum_at(p, c);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(w, y[i], v[i]);
        }
    } else if (row >= from && row < limit) {
        v = sum_at(row, c);
        if (a.half) {
            const float4_t up = sum_at(row, c + a.half);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = silu_mul(v[i], up[i]);
        }
    }
    *(u32x2*)((uint16_t*)a.out + row * a.osm + c) = u32x2{pack16<BF16>(v[0], v[1]), pack16<BF16>(v[2], v[3])};
}

int format_of(const gla_experts_args& p) {
    if (p.W_nbits == 4 && p.elements_per_sample == 8 && p.channel_scale_mode == GLA_CSM_NONE &&
        (p.input_dtype == GLA_DT_FP16 || p.input_dtype == GLA_DT_BF16))
        return kEW4;
    if (p.W_nbits == 8 && p.elements_per_sample == 1 && p.channel_scale_mode == GLA_CSM_BLOCK && p.input_dtype == GLA_DT_FP8 &&
        p.W_group_mode == GLA_WGM_NONE)
        return kEF8;
    if (p.W_nbits == 16 && p.elements_per_sample == 1 && p.channel_scale_mode == GLA_CSM_NONE && p.W_group_mode == GLA_WGM_NONE &&
        (p.input_dtype == GLA_DT_FP16 || p.input_dtype == GLA_DT_BF16))
        return kE16;
    return -1;
}

bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

int validate(const gla_experts_args* p) {
    if (p == nullptr || p->struct_size != sizeof(gla_experts_args)) {
        set_error("experts: struct_size does not match this library");
        return GLA_ERR_INVALID_ARGUMENT;
    }
    if (p->mode < GLA_EXPERTS_ROWS || p->mode > GLA_EXPERTS_COMBINED) {
        set_error("experts: mode %d", p->mode);
        return GLA_ERR_UNSUPPORTED_MODE;
    }
    const bool combined = p->mode == GLA_EXPERTS_COMBINED, gated = p->mode == GLA_EXPERTS_GATED;
    if (p->R < 0 || p->R > GLA_EXPERTS_MAX_ROWS || p->T < 0 || p->E <= 0 || p->E > GLA_EXPERTS_MAX || p->N <= 0 || p->K <= 0 || p->K > (1 << 20)) {
        set_error("experts: R=%d T=%d E=%d (1..%d) N=%d K=%d (at most 2^20)", p->R, p->T, p->E, GLA_EXPERTS_MAX, p->N, p->K);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    if (p->output_dtype != GLA_DT_FP16 && p->output_dtype != GLA_DT_BF16) {
        set_error("experts: output type %d (fp16 and bf16 are built)", p->output_dtype);
        return GLA_ERR_UNSUPPORTED_DTYPE;
    }
    if ((gated || combined) && (p->R > 0 || p->T > 0) && (p->top_k <= 0 || (int64_t)p->T * p->top_k != p->R)) {
        set_error("experts: T=%d tokens of %d slots are not the plan's R=%d rows", p->T, p->top_k, p->R);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    const int fmt = format_of(*p);
    if (fmt < 0) {
        set_error("experts: W_nbits=%d elements_per_sample=%d input_dtype=%d output_dtype=%d channel_scale_mode=%d W_group_mode=%d is not built "
                  "(4-bit codes in 32-bit words with group scales, fp8 with 128 x 128 block scales, 16-bit weights)",
                  p->W_nbits, p->elements_per_sample, p->input_dtype, p->output_dtype, p->channel_scale_mode, p->W_group_mode);
        return GLA_ERR_UNSUPPORTED_MODE;
    }
    if (p->x_dtype != p->output_dtype || (fmt != kEF8 && p->input_dtype != p->x_dtype)) {
        set_error("experts: activations of type %d (input type %d) with output type %d", p->x_dtype, p->input_dtype, p->output_dtype);
        return GLA_ERR_UNSUPPORTED_DTYPE;
    }
    if (p->tile_config != -1) {
        const int rows = p->tile_config % 1000, splits = p->tile_config / 1000;
        if (p->tile_config < 0 || splits > 64 || (rows != 4 && rows != 16 && rows != 64 && rows != 128 && rows != 256) ) {
            set_error("experts: tile_config %d", p->tile_config);
            return GLA_ERR_INVALID_ARGUMENT;
        }
    }
    const int kstep = fmt == kEF8 ? 128 : 32;
    if (p->K % kstep != 0 || p->N % (gated ? 16 : 8) != 0) {
        set_error("experts: K=%d has to be a multiple of %d, N=%d of %d", p->K, kstep, p->N, gated ? 16 : 8);
        return GLA_ERR_MISALIGNED_SHAPE;
    }
    const int64_t expert_bytes = fmt == kEW4 ? (int64_t)p->K / 2 * p->N : (int64_t)p->K * p->N * (fmt == kE16 ? 2 : 1);
    if (expert_bytes >= (int64_t)1 << 31) {
        set_error("experts: one expert's weights take %lld bytes (2^31 or more)", (long long)expert_bytes);
        return GLA_ERR_UNSUPPORTED_MODE;
    }
    if (p->R > 0) {
        if (!p->x || !p->w || !p->out || !p->offsets || (gated && !p->order) || (combined && (!p->places || !p->weights))) {
            set_error("experts: NULL pointer");
            return GLA_ERR_INVALID_ARGUMENT;
        }
        if (p->x_stride_m < p->K || p->out_stride_m < (gated ? p->N / 2 : p->N)) {
            set_error("experts: row strides %lld / %lld are shorter than the rows", (long long)p->x_stride_m, (long long)p->out_stride_m);
            return GLA_ERR_INVALID_ARGUMENT;
        }
        if (!aligned(p->x, 16) || p->x_stride_m % 8 || !aligned(p->w, 16) || p->w_stride_e % 16 || !aligned(p->out, 8) || p->out_stride_m % 4 ||
            !aligned(p->scales, fmt == kEF8 ? 4 : 16) || !aligned(p->zeros, 16) || p->meta_stride_e % (fmt == kEF8 ? 4 : 16) ||
            !aligned(p->bias, 16)) {
            set_error("experts: x and its rows, w, scales, zeros and bias have to be 16-byte aligned (fp8: scales 4-byte), out and its rows 8-byte");
            return GLA_ERR_INVALID_ARGUMENT;
        }
        if (p->w_stride_e < expert_bytes) {
            set_error("experts: w_stride_e=%lld bytes is shorter than an expert's %lld", (long long)p->w_stride_e, (long long)expert_bytes);
            return GLA_ERR_INVALID_ARGUMENT;
        }
        if (fmt == kEF8 && (!p->scales || p->meta_dtype != GLA_DT_FP32)) {
            set_error("experts: fp8 experts need fp32 block scales");
            return GLA_ERR_INVALID_ARGUMENT;
        }
    }
    if (fmt == kEW4) {
        if (p->group_size <= 0 || p->group_size % 32 != 0 || p->K % p->group_size != 0) {
            set_error("experts: groups of %d K-values (multiples of 32 that divide K=%d)", p->group_size, p->K);
            return GLA_ERR_MISALIGNED_SHAPE;
        }
        if (p->W_group_mode != GLA_WGM_SCALE && p->W_group_mode != GLA_WGM_SHIFT_SCALE && p->W_group_mode != GLA_WGM_FMA) {
            set_error("experts: W_group_mode %d of 4-bit codes (scale, shift and scale, fma are built)", p->W_group_mode);
            return GLA_ERR_UNSUPPORTED_MODE;
        }
        if (p->meta_dtype != p->x_dtype) {
            set_error("experts: scales of type %d with activations of type %d (they have to be the same)", p->meta_dtype, p->x_dtype);
            return GLA_ERR_UNSUPPORTED_DTYPE;
        }
        if (p->R > 0 && (!p->scales || (p->W_group_mode != GLA_WGM_SCALE && !p->zeros))) {
            set_error("experts: NULL scales or zeros");
            return GLA_ERR_INVALID_ARGUMENT;
        }
    }
    return GLA_OK;
}

struct ExpertPlanHost {
    int format;
    int bm;      // rows per tile: 4, 16 (streaming kernel), 64, 128, 256 (tiled GEMM)
    int S, chunk, waves;
    bool to_partials;
    bool quantise;                       // F8: a launch in front writes codes and scales to the workspace
    bool sums;                           // W4: a launch in front writes the sums of the groups there
    int64_t partial_bytes, code_bytes, total_bytes;  // of the workspace: fp32 rows, codes, scales
};

// Rows per tile from the mean rows per expert with any (the distribution itself is on the device; rows without an expert count
// too, so a plan most of whose slots belong to other ranks gets taller tiles than its own rows need).  Times in us, both sides
// of each threshold, at the sizes named (E experts, k of them per token); up to 24 rows per expert with copies of the weights
// in turn, 700 MB together, so that each call finds its own in memory:
//  * 4-bit, 4096 -> 2 x 14336, E = 8, k = 2, groups of 128 (of 64 and 32 the same sides): 16-row streaming tiles against 64-row
//    ones at 8 rows per expert 112 / 171, at 16 154 / 175, at 20 192 / 177; 64 against 128 rows at 32 rows per expert 186 / 201, at
//    48 191 / 208, at 64 231 / 238, at 100 347 / 280; 14336 -> 4096 combined at 64 134 / 128.  (256-row tiles would leave one workgroup per CU,
//    128-row ones two.)
//  * 16-bit, 4096^2, E = 16: 4 against 16 at 2 rows per expert 53 / 58, at 3 76 / 58; 16 against 64 at 6 65 / 85, at 12 105 / 93; 64
//    against 128 at 28 112 / 116, at 57 125 / 114.  Above, 128- and 256-row tiles cost 1.0 to 1.7 and run in rounds of one per
//    CU: whichever needs less.
//  * fp8: the streaming kernel quantises in every wave and needs long K ranges.  4 / 16 / 64 rows: K = 4096 (-> 2 x 2048, E = 32,
//    k = 4) at 1 row per expert 54 / 61 / 83, at 4 94 / 84 / 114, at 8 154 / 110 / 122; 7168 there at 4 161 / 131 / 149, at 8 261 / 173 / 168;
//    3584 at 2 56 / 65 / 64, at 4 82 / 77 / 80; 2560 at 2 45 / 53 / 50, at 4 65 / 63 / 60, and 2560 -> 2 x 768, E = 128, k = 8 at 2 62 / 68 / 61;
//    2048 -> 2 x 768, E = 128, k = 8 at 1 41 / 53 / 43, at 2 53 / 61 / 51, at 4 84 / 78 / 64; 768 -> 2048 at 1 token 11.2 / 11.3 / 15.1, at 8 tokens
//    28 / 39 / 28.  64 against 128 at 62 rows per expert 119 / 121, at 125 168 / 147; 128 against 256 at 250 151 / 174 and 232 / 222,
//    at 512 449 / 404.
int choose_rows(int format, int K, int64_t R, int64_t active, int64_t width_of_128) {
    const int64_t per = active > 0 ? R / active : 0;
    if (format == kEF8) {
        if (K >= 4096 ? per <= 8 : K > 2048 ? per <= 2 : per <= 1 && active * width_of_128 <= 256) return per > 2 ? 16 : 4;
        return per <= 64 ? 64 : per <= 300 ? 128 : 256;
    }
    if (format == kE16) {
        if (per <= 9) return per <= 2 ? 4 : 16;
        if (per <= 32) return 64;
        const int64_t wide = (width_of_128 + 1) / 2;
        auto rounds = [&](int64_t bm) {
            const int64_t partly = (R + bm * active / 2) / bm;  // tiles, if the last one of an expert is half full
            return ((partly > active ? partly : active) * wide + 255) / 256;
        };
        return rounds(256) * 17 <= rounds(128) * 10 ? 256 : 128;
    }
    return per <= 16 ? 16 : per <= 48 ? 64 : 128;
}

ExpertPlanHost plan_of(const gla_experts_args& p) {
    ExpertPlanHost h;
    h.format = format_of(p);
    const int want_rows = p.tile_config < 0 ? 0 : p.tile_config % 1000, want_s = p.tile_config < 0 ? 0 : p.tile_config / 1000;
    const int64_t active = p.R < p.E ? p.R : p.E;
    // workgroups side by side for BN columns of weights (gated: half of them from either half)
    auto across = [&](int bn) { return (int64_t)(p.N + bn - 1) / bn; };
    h.bm = want_rows ? want_rows : choose_rows(h.format, p.K, p.R, active, across(128));
    if (h.format == kEW4) h.bm = h.bm == 4 ? 16 : h.bm == 256 ? 128 : h.bm;  // (not built for 4-bit weights: never better)
    // K splits until every CU has work: a finishing launch adds them (combined calls have one anyway; others split only
    // where that leaves most of the chip empty)
    const int steps = (p.K + 127) / 128;
    const bool stream = h.bm <= 16;
    const int64_t tiles = stream ? active * across(h.format == kE16 ? 32 : 64)
                                 : (p.R / h.bm + active) * across(h.bm == 64 && h.format != kEW4 ? 128 : 256);
    const int64_t enough = stream ? 256 : h.format == kEW4 ? 768 : h.bm == 64 ? 384 : 192;
    int s = 1;
    while (tiles * s < enough && s < 8 && steps >= 16 * s) s *= 2;
    if (p.mode != GLA_EXPERTS_COMBINED && (s < 4 || tiles > 96)) s = 1;
    h.S = want_s > 0 ? want_s : s;
    // 4-bit weights, many workgroups: two waves of twice the K range each, which start half as often (one token, 4096 -> 2 x
    // 14336, 896 workgroups, weights in memory: 32.2 -> 29.9 us; 16 tokens top 2 of 8: 109 -> 106; 61 tokens top 6 of 64, 2048 ->
    // 2 x 1408: 49 -> 46; 14336 -> 4096, 512 workgroups: 48 -> 64)
    h.waves = h.format == kEW4 && tiles * h.S >= 768 && steps >= 16 * h.S ? 2 : 4;
    const int unit = stream || h.format == kEF8 ? 128 : 64, parts = stream ? h.waves * h.S : h.S;
    const int n_units = (p.K + unit - 1) / unit;
    h.chunk = (n_units + parts - 1) / parts;
    if (!stream && h.format == kEW4) {
        // splits begin where groups do: a group's second term and all of its first belong to one of them
        const int m = p.group_size / std::gcd(p.group_size, unit);
        h.chunk = (h.chunk + m - 1) / m * m;
    }
    if (!stream) h.S = (n_units + h.chunk - 1) / h.chunk;  // every split has a stage
    h.to_partials = p.mode == GLA_EXPERTS_COMBINED || h.S > 1;
    h.partial_bytes = h.to_partials ? (int64_t)h.S * p.R * p.N * 4 : 0;
    const int64_t rows = p.mode == GLA_EXPERTS_GATED ? p.T : p.R;
    h.quantise = h.format == kEF8 && h.bm > 16;
    h.code_bytes = h.quantise ? rows * p.K : 0;
    h.sums = h.format == kEW4 && h.bm > 16;
    h.total_bytes = h.partial_bytes + h.code_bytes + (h.quantise ? rows * (p.K / 128) * 4 : 0) + (h.sums ? rows * (p.K / p.group_size) * 16 : 0);
    return h;
}

}  // namespace

}  // namespace gla

using namespace gla;

extern "C" {

int64_t gla_experts_workspace_bytes(const gla_experts_args* p) {
    const int rc = validate(p);
    if (rc != GLA_OK) return rc;
    return plan_of(*p).total_bytes;
}

int gla_experts_matmul(const gla_experts_args* p, void* stream) {
    const int rc = validate(p);
    if (rc != GLA_OK) return rc;
    if (p->R == 0) return GLA_OK;
    const ExpertPlanHost h = plan_of(*p);
    if (h.total_bytes > 0 && (p->workspace == nullptr || (int64_t)p->workspace_bytes < h.total_bytes || !aligned(p->workspace, 16))) {
        set_error("experts: a 16-byte aligned workspace of %lld bytes required, %llu given", (long long)h.total_bytes,
                  (unsigned long long)p->workspace_bytes);
        return GLA_ERR_WORKSPACE_TOO_SMALL;
    }
    const bool bf16 = p->output_dtype == GLA_DT_BF16;
    ExpertArgs a{};
    a.x = (const unsigned char*)p->x;
    a.w = (const unsigned char*)p->w;
    a.scales = (const unsigned char*)(p->scales != nullptr ? p->scales : p->w);
    a.zeros = p->W_group_mode == GLA_WGM_SCALE ? nullptr : (const unsigned char*)p->zeros;
    a.bias = p->bias;
    a.out = p->out;
    a.partials = (float*)p->workspace;
    a.offsets = p->offsets;
    a.order = p->mode == GLA_EXPERTS_GATED ? p->order : nullptr;
    a.w_stride_e = p->w_stride_e;
    a.meta_stride_e = p->meta_stride_e;
    a.xsm = p->x_stride_m * 2;
    a.osm = p->out_stride_m;
    a.R = p->R;
    a.E = p->E;
    a.N = p->N;
    a.K = p->K;
    a.top_k = p->top_k;
    a.half = p->mode == GLA_EXPERTS_GATED ? p->N / 2 : 0;
    a.S = h.S;
    a.to_partials = h.to_partials;
    a.group = p->group_size;
    a.groups = h.format == kEW4 ? p->K / p->group_size : 0;
    a.group_mul = divide_mul(h.format == kEW4 ? p->group_size / 32 : 1);
    a.top_k_mul = divide_mul(p->top_k);
    a.top_k_divides = (int64_t)p->R * p->top_k > (int64_t)1 << 32;
    a.chunk = h.chunk;
    a.stream_waves = h.waves;
    a.c1 = p->W_group_mode == GLA_WGM_FMA ? 1.0f : 0.0f;
    a.c2 = p->W_group_mode == GLA_WGM_SHIFT_SCALE ? -1.0f : 0.0f;
    hipStream_t s = (hipStream_t)stream;
    if (h.quantise) {
        unsigned char* codes = (unsigned char*)p->workspace + h.partial_bytes;
        float* scales_x = (float*)(codes + h.code_bytes);  // (K is a multiple of 128: aligned)
        const int rcq = launch_experts_quantise(p->x, bf16, a.xsm, p->mode == GLA_EXPERTS_GATED ? p->T : p->R, p->K, codes, scales_x, s);
        if (rcq != GLA_OK) return rcq;
        a.x = codes;
        a.xsm = p->K;
        a.scales_x = scales_x;
    }
    if (h.sums) {
        unsigned char* sums = (unsigned char*)p->workspace + h.partial_bytes;
        const int rcs = launch_experts_sums(p->x, bf16, a.xsm, p->mode == GLA_EXPERTS_GATED ? p->T : p->R, p->K, p->group_size, sums, s);
        if (rcs != GLA_OK) return rcs;
        a.sums = sums;
    }
    const int rc2 = h.bm > 16 ? launch_experts_gemm(a, h.format, bf16, h.bm, s) : launch_experts_stream(a, h.format, bf16, h.bm, s);
    if (rc2 != GLA_OK || !h.to_partials) return rc2;
    const bool combined = p->mode == GLA_EXPERTS_COMBINED;
    FinishArgs f{a.partials, p->offsets, p->places, p->weights, p->out, p->out_stride_m, p->R, p->E, p->N, h.S, p->top_k, a.half};
    const int width = a.half ? a.half : p->N;
    const dim3 grid(combined ? p->T : p->R, (width + 1023) / 1024);
    if (combined) {
        if (bf16) experts_finish_kernel<true, true><<<grid, 256, 0, s>>>(f);
        else experts_finish_kernel<false, true><<<grid, 256, 0, s>>>(f);
    } else {
        if (bf16) experts_finish_kernel<true, false><<<grid, 256, 0, s>>>(f);
        else experts_finish_kernel<false, false><<<grid, 256, 0, s>>>(f);
    }
    return check_hip(hipGetLastError(), "experts_finish");
}

static int check_route_sizes(int64_t T, int E, int top_k) {
    if (T < 0 || E <= 0 || E > GLA_EXPERTS_MAX || top_k <= 0 || top_k > 64 || T * top_k >= ((int64_t)1 << 31)) {
        set_error("route: T=%lld E=%d (1..%d) top_k=%d (1..64)", (long long)T, E, GLA_EXPERTS_MAX, top_k);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    return GLA_OK;
}

static int check_route(int64_t T, int E, int top_k, const void* ids, const void* offsets, const void* order, const void* places) {
    const int rc = check_route_sizes(T, E, top_k);
    if (rc != GLA_OK) return rc;
    if (offsets == nullptr || (T > 0 && (ids == nullptr || order == nullptr || places == nullptr))) {
        set_error("route: NULL pointer");
        return GLA_ERR_INVALID_ARGUMENT;
    }
    return GLA_OK;
}

int64_t gla_route_workspace_bytes(int T, int E, int top_k) {
    const int rc = check_route_sizes(T, E, top_k);
    return rc != GLA_OK ? rc : route_counts(T, E, top_k, true) * 4;
}

int64_t gla_plan_workspace_bytes(int T, int E, int top_k) {
    const int rc = check_route_sizes(T, E, top_k);
    return rc != GLA_OK ? rc : route_counts(T, E, top_k, false) * 4;
}

static int check_counts(int T, int E, int top_k, bool select, const void* workspace, int64_t bytes) {
    const int64_t need = route_counts(T, E, top_k, select) * 4;
    if (need > 0 && (workspace == nullptr || bytes < need || !aligned(workspace, 16))) {
        set_error("route: a 16-byte aligned workspace of %lld bytes required, %lld given", (long long)need, (long long)bytes);
        return GLA_ERR_WORKSPACE_TOO_SMALL;
    }
    return GLA_OK;
}

int gla_route_experts(const void* logits, int dtype, int64_t stride, int T, int E, int top_k, int scoring, int renormalize, float scale,
                      float* weights, int32_t* ids, int32_t* offsets, int32_t* order, int32_t* places, void* workspace,
                      int64_t workspace_bytes, void* stream) {
    int rc = check_route(T, E, top_k, ids, offsets, order, places);
    if (rc != GLA_OK) return rc;
    if (dtype != GLA_DT_FP32 && dtype != GLA_DT_FP16 && dtype != GLA_DT_BF16) {
        set_error("route: logits of type %d (fp32, fp16 and bf16 are built)", dtype);
        return GLA_ERR_UNSUPPORTED_DTYPE;
    }
    if (top_k > E || (scoring != GLA_SCORING_SOFTMAX && scoring != GLA_SCORING_SIGMOID)) {
        set_error("route: top_k=%d of %d experts, scoring %d", top_k, E, scoring);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    if (T > 0 && (logits == nullptr || weights == nullptr || (T > 1 && stride < E))) {
        set_error("route: NULL pointer, or rows %lld apart with %d logits", (long long)stride, E);
        return GLA_ERR_INVALID_ARGUMENT;
    }
    if ((rc = check_counts(T, E, top_k, true, workspace, workspace_bytes)) != GLA_OK) return rc;
    return launch_route(logits, T > 0 ? dtype : GLA_DT_FP32, stride, T, E, top_k, scoring == GLA_SCORING_SIGMOID, renormalize, scale, weights, ids,
                        offsets, order, places, (int32_t*)workspace, (hipStream_t)stream);
}

int gla_plan_experts(const int32_t* ids, int T, int E, int top_k, int32_t* offsets, int32_t* order, int32_t* places, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    int rc = check_route(T, E, top_k, ids, offsets, order, places);
    if (rc != GLA_OK) return rc;
    if ((rc = check_counts(T, E, top_k, false, workspace, workspace_bytes)) != GLA_OK) return rc;
    return launch_route(nullptr, 0, 0, T, E, top_k, 0, 0, 1.0f, nullptr, const_cast<int32_t*>(ids), offsets, order, places, (int32_t*)workspace,
                        (hipStream_t)stream);
}

}  // extern "C"
