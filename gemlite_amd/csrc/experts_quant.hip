// Rows of 16-bit activations -> e4m3 codes with one fp32 scale per 128 values, for the fp8 experts: what the streaming
// kernel does in registers for a few rows, as a launch of its own in front of it or of the tiled GEMM.
//
// 16 lanes share a block of 128 values (8 each, one 16-byte load), so a wave step is 4 blocks = 1 KB in, 512 bytes out.
// Bound by these bytes (32008 rows of 1408: 27 us for 135 MB).
#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

template <bool BF16>
__global__ __launch_bounds__(256) void experts_quantise_kernel(const unsigned char* x, int64_t xsm, int64_t blocks, int per_row, int K,
                                                               unsigned char* codes, float* scales) {
    const int lane = threadIdx.x & 15;
    const int64_t b = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (b >= blocks) return;  // whole groups of 16 lanes
    const int64_t row = b / per_row;
    const int k = (int)(b - row * per_row) * 128 + lane * 8;
    const u32x4 v = *(const u32x4*)(x + row * xsm + (int64_t)k * 2);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = low16<BF16>(v[i]);
        f[2 * i + 1] = high16<BF16>(v[i]);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = magnitude_max(m, v[i]);
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) m = magnitude_max(m, wave_xor(m, x));
    const float amax = low16<BF16>((m & 0xffffu) > (m >> 16) ? m & 0xffffu : m >> 16);
    float s, inv;
    block_scale(amax, s, inv);
    *(u32x2*)(codes + row * K + k) = u32x2{quantise4(f[0], f[1], f[2], f[3], inv), quantise4(f[4], f[5], f[6], f[7], inv)};
    if (lane == 0) scales[b] = s;
}

// Sums of the groups of a row, for the tiled GEMM of 4-bit experts: L lanes to a group, 8 values of a lane at a time, in a
// fixed order.  Bound by the bytes it reads.
template <bool BF16, int L>
__global__ __launch_bounds__(256) void experts_sums_kernel(const unsigned char* x, int64_t xsm, int64_t count, int groups, int group, unsigned char* sums) {
    const int lane = threadIdx.x & (L - 1);
    const int64_t q = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (q >= count) return;  // whole sets of L lanes
    const int64_t row = q / groups;
    const unsigned char* p = x + row * xsm + (q - row * groups) * group * 2;
    float s = 0.0f;
    for (int k = lane * 8; k < group; k += L * 8) {
        const u32x4 v = *(const u32x4*)(p + (int64_t)k * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) s += low16<BF16>(v[i]) + high16<BF16>(v[i]);
    }
#pragma unroll
    for (int m = 1; m < L; m <<= 1) s += wave_xor(s, m);
    uint32_t t[3];
    bf16_terms(s, t);
    if (lane == 0) *(u32x4*)(sums + q * 16) = u32x4{high_halves(t[0], t[1]), high_halves(t[2], t[0]), high_halves(t[1], t[2]), high_halves(t[0], t[1])};
}

template <bool BF16, int L>
void launch_sums(const void* x, int64_t xsm, int64_t count, int groups, int group, unsigned char* sums, hipStream_t stream) {
    experts_sums_kernel<BF16, L><<<(unsigned)((count * L + 255) / 256), 256, 0, stream>>>((const unsigned char*)x, xsm, count, groups, group, sums);
}

}  // namespace

int launch_experts_sums(const void* x, bool bf16, int64_t xsm, int rows, int K, int group, unsigned char* sums, hipStream_t stream) {
    const int groups = K / group;
    const int64_t count = (int64_t)rows * groups;
    // (long groups: a wave each, or few groups would leave the chip empty)
    if (group >= 1024) bf16 ? launch_sums<true, 64>(x, xsm, count, groups, group, sums, stream) : launch_sums<false, 64>(x, xsm, count, groups, group, sums, stream);
    else bf16 ? launch_sums<true, 4>(x, xsm, count, groups, group, sums, stream) : launch_sums<false, 4>(x, xsm, count, groups, group, sums, stream);
    return check_hip(hipGetLastError(), "experts_sums");
}

int launch_experts_quantise(const void* x, bool bf16, int64_t xsm, int rows, int K, unsigned char* codes, float* scales, hipStream_t stream) {
    const int64_t blocks = (int64_t)rows * (K / 128);
    const dim3 grid((unsigned)((blocks + 15) / 16));
    if (bf16) experts_quantise_kernel<true><<<grid, 256, 0, stream>>>((const unsigned char*)x, xsm, blocks, K / 128, K, codes, scales);
    else experts_quantise_kernel<false><<<grid, 256, 0, stream>>>((const unsigned char*)x, xsm, blocks, K / 128, K, codes, scales);
    return check_hip(hipGetLastError(), "experts_quantise");
}

}  // namespace gla
