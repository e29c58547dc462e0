// Rows of 16-bit activations -> e4m3 codes with one fp32 scale per 128 values, for the fp8 experts: what the streaming
// kernel does in registers for a few rows, as a launch of its own in front of it or of the tiled GEMM.
//
// 16 lanes share a block of 128 values (8 each, one 16-byte load), so a wave step is 4 blocks = 1 KB in, 512 bytes out.
// Bound by these bytes (32008 rows of 1408: 27 us for 135 MB).
#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

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

}  // namespace

int launch_experts_quantise(const void* x, bool bf16, int64_t xsm, int rows, int K, unsigned char* codes, float* scales, hipStream_t stream) {
    const int64_t blocks = (int64_t)rows * (K / 128);
    const dim3 grid((unsigned)((blocks + 15) / 16));
    if (bf16) experts_quantise_kernel<true><<<grid, 256, 0, stream>>>((const unsigned char*)x, xsm, blocks, K / 128, K, codes, scales);
    else experts_quantise_kernel<false><<<grid, 256, 0, stream>>>((const unsigned char*)x, xsm, blocks, K / 128, K, codes, scales);
    return check_hip(hipGetLastError(), "experts_quantise");
}

}  // namespace gla
