// Routing of tokens to experts: the k largest logits of every row with their weights, and the (token, slot) pairs sorted
// by expert.
//
//   selected   the k largest logits of a row, ties to the lower expert; NaN and -inf are never selected (id -1, weight 0)
//   weights    softmax or sigmoid of the logits in fp32; renormalised over the selected ones or not; times a factor
//   order      flat indices token * k + slot, sorted by expert, within an expert in rising order; slots without an expert
//              come last.  offsets[e] is where expert e's begin; places is the inverse of order
//
// A wave per token (32 tokens and 16 waves to a workgroup): lane l holds logits l, l + 64, ...; each of the k rounds is one
// wave-wide maximum and, where several lanes have it, one minimum of their indices (DPP, no LDS).  A small call
// (small_call()) is done by one workgroup in one launch.  Otherwise a first launch selects and counts each block's
// slots per expert, and a second one sorts: every block adds up the counts of the blocks in front of it for itself (they
// are a few kilobytes in L2), so no third launch has to.  Counting by ballots and integer sums only: the result does not
// depend on the order of execution.
//
// Bound by the selection's instructions and by latency: 8191 tokens of 128 fp32 logits, top 8 (4 MB): 9.2 + 6.6 us, 14.5 in a graph
// (with the rounds on floats and both reductions in each 3 us more); one token of 64: 3.7 us.  Sorting given ids alone: 8191 x 8 9.0
// us, 128 x 8 3.8.
#include "common.hpp"
#include "experts.hpp"

namespace gla {

namespace {

constexpr int kSmallSlots = 1024;  // (token, slot) pairs that one workgroup sorts, a thread each
constexpr int kSmallTokens = 40;   // tokens that one workgroup selects for
constexpr int kMaxBlocks = 256;
constexpr int kMinTokens = 32;  // tokens per block, at least
constexpr int kThreads = 1024;

struct RouteArgs {
    const void* logits;  // NULL: ids are given
    int64_t stride;
    int T, E, k;
    int sigmoid, renormalize;
    float scale;
    float* weights;
    int32_t* ids;
    int32_t *offsets, *order, *places;
    int32_t* counts;  // [E + 1][blocks]
    int blocks, tokens;  // tokens per block
};

// Logits as integers of the same order (both zeros the same, NaN as -inf): the wave-wide maximum of integers is one
// instruction per step, that of floats three.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v == v ? v + 0.0f : -__builtin_inff());
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, key ^ ((key & 0x80000000u) != 0 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kNoneKey = 0x007fffffu;  // of -inf

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define GLA_STEP(ctrl, rm)                                                                           \
    {                                                                                                \
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, (ctrl), (rm), 0xf, false); \
        v = o > v ? o : v;                                                                           \
    }
    GLA_STEP(0x111, 0xf);
    GLA_STEP(0x112, 0xf);
    GLA_STEP(0x114, 0xf);
    GLA_STEP(0x118, 0xf);
    GLA_STEP(0x142, 0xa);
    GLA_STEP(0x143, 0xc);
#undef GLA_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ int wave_min(int v) {
#define GLA_STEP(ctrl, rm)                                                            \
    {                                                                                 \
        const int o = __builtin_amdgcn_update_dpp(v, v, (ctrl), (rm), 0xf, false);    \
        v = o < v ? o : v;                                                            \
    }
    GLA_STEP(0x111, 0xf);
    GLA_STEP(0x112, 0xf);
    GLA_STEP(0x114, 0xf);
    GLA_STEP(0x118, 0xf);
    GLA_STEP(0x142, 0xa);
    GLA_STEP(0x143, 0xc);
#undef GLA_STEP
    return __builtin_amdgcn_readlane(v, 63);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += wave_xor(v, m);
    return v;
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* row, int i) {
    if constexpr (DT == GLA_DT_FP32) return ((const float*)row)[i];
    else if constexpr (DT == GLA_DT_FP16) return half_bits_to_float(((const uint16_t*)row)[i]);
    else return bf16_bits_to_float(((const uint16_t*)row)[i]);
}

constexpr float kNone = -__builtin_inff();

// The logits of token t, lane l those of experts l, l + 64, ..
template <int DT, int V>
__device__ __forceinline__ void load_token(const RouteArgs& a, int t, float (&v)[V]) {
    const int lane = threadIdx.x & 63;
    const int DTS = DT == GLA_DT_FP32 ? 4 : 2;
    const char* row = (const char*)a.logits + (int64_t)t * a.stride * DTS;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j * 64 + lane < a.E ? logit_at<DT>(row, j * 64 + lane) : kNone;
}

// One token by one wave: its id (or -1) in lane j < k; ids and weights stored.
template <int V>
__device__ __forceinline__ int select_token(const RouteArgs& a, int t, const float (&v)[V]) {
    const int lane = threadIdx.x & 63;
    uint32_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = key_of(v[j]);
    float top = 0.0f, denom = 0.0f;
    uint32_t val = kNoneKey;
    int id = -1;
    for (int r = 0; r < a.k; ++r) {
        uint32_t best = key[0];
        int at = lane;
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) {
                best = key[j];
                at = j * 64 + lane;
            }
        const uint32_t m = wave_max(best);
        if (r == 0) {
            top = value_of(m);
            if (!a.renormalize && !a.sigmoid) {  // softmax over all experts
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) s += key[j] == kNoneKey ? 0.0f : (key[j] == m ? 1.0f : expf(value_of(key[j]) - top));
                denom = wave_sum(s);
            }
        }
        if (m == kNoneKey) break;
        const unsigned long long has = __ballot(best == m);
        // the lane that has it; several: the lowest expert of theirs
        const int c = (has & (has - 1)) == 0 ? __builtin_amdgcn_readlane(at, __builtin_ctzll(has)) : wave_min(best == m ? at : 0x7fffffff);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c == j * 64 + lane) key[j] = kNoneKey;
        if (lane == r) {
            val = m;
            id = c;
        }
    }
    const float x = value_of(val);
    // (equal to the maximum: 1, also where that is infinite)
    float w = id < 0 ? 0.0f : (a.sigmoid ? 1.0f / (1.0f + expf(-x)) : (x == top ? 1.0f : expf(x - top)));
    if (a.renormalize) denom = wave_sum(w);
    if (a.renormalize || !a.sigmoid) w = denom > 0.0f ? w / denom : 0.0f;
    if (lane < a.k) {
        a.weights[(int64_t)t * a.k + lane] = w * a.scale;
        a.ids[(int64_t)t * a.k + lane] = id;
    }
    return id;
}

// Lanes with the same class: how many in front of this one, and how many in all (lanes that are off have class -1).
__device__ __forceinline__ void match_lanes(int cls, int bits, int& rank, int& count) {
    unsigned long long same = __ballot(cls >= 0);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((cls >> b) & 1);
        same &= ((cls >> b) & 1) ? set : ~set;
    }
    const int lane = threadIdx.x & 63;
    rank = __popcll(same & ((1ull << lane) - 1));
    count = __popcll(same);
}

__device__ __forceinline__ int class_of(int id, int E) { return id < 0 || id >= E ? E : id; }

// totals[0 .. E] -> their exclusive sums, by wave 0 (totals is overwritten); the caller synchronises around it.
__device__ __forceinline__ void scan_classes(int* totals, int classes) {
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    int base = 0;
    for (int e0 = 0; e0 < classes; e0 += 64) {
        const int mine = e0 + lane < classes ? totals[e0 + lane] : 0;
        const int upto = wave_inclusive_sum(mine);
        if (e0 + lane < classes) totals[e0 + lane] = base + upto - mine;
        base += __builtin_amdgcn_readlane(upto, 63);
    }
}

// Everything in one workgroup (small_call()).  DT < 0: the ids are given.
template <int DT, int V>
__global__ __launch_bounds__(1024) void route_small_kernel(RouteArgs a, int bits) {
    extern __shared__ int lds[];
    const int classes = a.E + 1, slots = a.T * a.k;
    int* ids = lds;                        // [kSmallSlots]
    int* totals = lds + kSmallSlots;       // [classes]
    int* counts = totals + classes;        // [waves][classes]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    for (int i = tid; i < waves * classes; i += blockDim.x) counts[i] = 0;
    if constexpr (DT >= 0) {
        for (int t = wave; t < a.T; t += waves) {
            float v[V];
            load_token<DT, V>(a, t, v);
            const int id = select_token<V>(a, t, v);
            if (lane < a.k) ids[t * a.k + lane] = id;
        }
    } else {
        if (tid < slots) ids[tid] = a.ids[tid];
    }
    __syncthreads();
    const int cls = tid < slots ? class_of(ids[tid], a.E) : -1;
    int rank, count;
    match_lanes(cls, bits, rank, count);
    if (cls >= 0 && rank == 0) counts[wave * classes + cls] = count;
    __syncthreads();
    for (int e = tid; e < classes; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < waves; ++w) {
            const int c = counts[w * classes + e];
            counts[w * classes + e] = sum;
            sum += c;
        }
        totals[e] = sum;
    }
    __syncthreads();
    scan_classes(totals, classes);
    __syncthreads();
    for (int e = tid; e < classes; e += blockDim.x) a.offsets[e] = totals[e];
    if (cls >= 0) {
        const int p = totals[cls] + counts[wave * classes + cls] + rank;
        a.order[p] = tid;
        a.places[tid] = p;
    }
}

// Block b: selects for its tokens (or reads their ids) and counts them per class.
template <int DT, int V>
__global__ __launch_bounds__(kThreads) void route_select_kernel(RouteArgs a) {
    extern __shared__ int lds[];  // [classes]
    const int classes = a.E + 1, b = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < classes; e += kThreads) lds[e] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)b * a.tokens;
    const int64_t t1 = t0 + a.tokens < a.T ? t0 + a.tokens : a.T;
    if constexpr (DT >= 0) {
        float v[V], ahead[V];  // the next token's logits arrive while this one's are selected from
        if (t0 + wave < t1) load_token<DT, V>(a, (int)(t0 + wave), v);
        for (int64_t t = t0 + wave; t < t1; t += kThreads / 64) {
            const int64_t next = t + kThreads / 64;
            load_token<DT, V>(a, (int)(next < t1 ? next : t), ahead);
            const int id = select_token<V>(a, (int)t, v);
            if (lane < a.k) atomicAdd(&lds[class_of(id, a.E)], 1);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = ahead[j];
        }
    } else {
        for (int64_t i = t0 * a.k + threadIdx.x; i < t1 * a.k; i += kThreads) atomicAdd(&lds[class_of(a.ids[i], a.E)], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < classes; e += kThreads) a.counts[(int64_t)e * a.blocks + b] = lds[e];
}

// Block b: where its slots go.
__global__ __launch_bounds__(kThreads) void route_sort_kernel(RouteArgs a, int bits) {
    extern __shared__ int lds[];
    constexpr int WAVES = kThreads / 64;
    const int classes = a.E + 1, b = blockIdx.x;
    int* totals = lds;             // [classes]: all slots of the class, then where the class begins
    int* next = lds + classes;     // [classes]: of this class in the blocks in front, then the next free place
    int* counts = next + classes;  // [WAVES][classes]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < WAVES * classes; i += kThreads) counts[i] = 0;
    // a wave per class: lane l has the counts of blocks 4 l .. 4 l + 3 (at most 256 blocks, a multiple of 4)
    constexpr int AHEAD = 8;  // classes whose counts a wave has in flight
    for (int e0 = wave; e0 < classes; e0 += AHEAD * WAVES) {
        int4 c[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int e = e0 + i * WAVES;
            c[i] = int4{0, 0, 0, 0};
            if (4 * lane < a.blocks && e < classes) c[i] = *(const int4*)(a.counts + (int64_t)e * a.blocks + 4 * lane);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int e = e0 + i * WAVES;
            const int4 v = c[i];
            const int upto = wave_inclusive_sum(v.x + v.y + v.z + v.w);
            if (e >= classes) continue;
            if (lane == 63) totals[e] = upto;
            if (lane == b >> 2) next[e] = upto - (v.x + v.y + v.z + v.w) + ((b & 3) > 0 ? v.x : 0) + ((b & 3) > 1 ? v.y : 0) + ((b & 3) > 2 ? v.z : 0);
        }
    }
    __syncthreads();
    scan_classes(totals, classes);
    __syncthreads();
    for (int e = tid; e < classes; e += kThreads) {
        if (b == 0) a.offsets[e] = totals[e];
        next[e] += totals[e];
    }
    __syncthreads();
    const int64_t t0 = (int64_t)b * a.tokens;
    const int64_t t1 = t0 + a.tokens < a.T ? t0 + a.tokens : a.T;
    for (int64_t i0 = t0 * a.k; i0 < t1 * a.k; i0 += kThreads) {
        const int64_t i = i0 + tid;
        const int cls = i < t1 * a.k ? class_of(a.ids[i], a.E) : -1;
        int rank, count;
        match_lanes(cls, bits, rank, count);
        if (cls >= 0 && rank == 0) counts[wave * classes + cls] = count;
        __syncthreads();
        if (cls >= 0) {
            int p = next[cls] + rank;
            for (int w = 0; w < wave; ++w) p += counts[w * classes + cls];
            a.order[p] = (int32_t)i;
            a.places[i] = p;
        }
        __syncthreads();
        if (cls >= 0 && rank == 0) {
            atomicAdd(&next[cls], count);
            counts[wave * classes + cls] = 0;
        }
        __syncthreads();
    }
}

int bits_of(int classes) {
    int b = 1;
    while ((1 << b) < classes) ++b;
    return b;
}

// One workgroup in one launch, or two launches over many.  Sorting given ids is faster in one up to the last thread (us, one
// launch / two: 1024 tokens top 1 of 64 3.5 / 7.0, 128 top 8 of 256 4.2 / 9.4).  Selecting is serial in the 16 waves: top 2 of 8 at
// 32 / 64 / 512 tokens 4.9 / 6.2, 7.0 / 6.5, 36 / 7.9; top 6 of 64 at 40 / 48 7.5 / 7.8, 8.5 / 8.1; top 8 of 128 at 32 / 40 / 128 8.4 / 9.0,
// 9.4 / 9.4, 22.9 / 12.6; top 8 of 256 at 40 / 48 10.9 / 11.8, 13.0 / 12.0; top 16 of 1024 at 24 / 40 23.6 / 29.3, 36.8 / 32.1.
bool small_call(int64_t T, int top_k, bool select) { return T * top_k <= kSmallSlots && (!select || T <= kSmallTokens); }

template <int DT, int V>
int launch_dt(RouteArgs a, hipStream_t stream) {
    const int classes = a.E + 1, bits = bits_of(classes);
    if (small_call(a.T, a.k, DT >= 0)) {
        const int slots = a.T * a.k;
        int waves = slots > 64 ? (slots + 63) / 64 : 1;
        if (DT >= 0 && waves < a.T) waves = a.T < 16 ? a.T : 16;
        const int lds = (kSmallSlots + classes + waves * classes) * 4;  // at most 73 KB
        static DeviceOnce once;
        if (once.first()) {
            const int rc = check_hip(hipFuncSetAttribute((const void*)route_small_kernel<DT, V>, hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024),
                                     "hipFuncSetAttribute");
            if (rc != GLA_OK) return rc;
        }
        route_small_kernel<DT, V><<<1, waves * 64, lds, stream>>>(a, bits);
        return check_hip(hipGetLastError(), "route_small");
    }
    static DeviceOnce once;
    if (once.first()) {
        const int rc = check_hip(hipFuncSetAttribute((const void*)route_sort_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024), "hipFuncSetAttribute");
        if (rc != GLA_OK) return rc;
    }
    route_select_kernel<DT, V><<<a.blocks, kThreads, classes * 4, stream>>>(a);
    route_sort_kernel<<<a.blocks, kThreads, (2 + kThreads / 64) * classes * 4, stream>>>(a, bits);
    return check_hip(hipGetLastError(), "route_sort");
}

template <int DT>
int launch_v(const RouteArgs& a, hipStream_t stream) {
    if (a.E <= 64) return launch_dt<DT, 1>(a, stream);
    if (a.E <= 128) return launch_dt<DT, 2>(a, stream);
    if (a.E <= 256) return launch_dt<DT, 4>(a, stream);
    if (a.E <= 512) return launch_dt<DT, 8>(a, stream);
    return launch_dt<DT, 16>(a, stream);
}

}  // namespace

static int route_blocks(int T) {
    int b = (T + kMinTokens - 1) / kMinTokens;
    if (b > kMaxBlocks) b = kMaxBlocks;
    return b < 4 ? 4 : (b + 3) / 4 * 4;
}

int64_t route_counts(int T, int E, int top_k, bool select) { return small_call(T, top_k, select) ? 0 : (int64_t)(E + 1) * route_blocks(T); }

int launch_route(const void* logits, int dtype, int64_t stride, int T, int E, int top_k, int sigmoid, int renormalize, float scale,
                 float* weights, int32_t* ids, int32_t* offsets, int32_t* order, int32_t* places, int32_t* counts, hipStream_t stream) {
    RouteArgs a{logits, stride, T, E, top_k, sigmoid, renormalize, scale, weights, ids, offsets, order, places, counts, route_blocks(T), 0};
    a.tokens = (T + a.blocks - 1) / a.blocks;
    if (logits == nullptr) return launch_dt<-1, 1>(a, stream);
    if (dtype == GLA_DT_FP32) return launch_v<GLA_DT_FP32>(a, stream);
    if (dtype == GLA_DT_FP16) return launch_v<GLA_DT_FP16>(a, stream);
    return launch_v<GLA_DT_BF16>(a, stream);
}

}  // namespace gla
