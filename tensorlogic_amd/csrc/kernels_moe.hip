// kernels_moe.hip -- a mixture-of-experts layer for a few tokens: router, the
// chosen experts' SwiGLU and their weighted sum.
//
//   l = R x,  p = softmax(l),  T = the `top` largest (ties: the first expert)
//   g_e = p_e, or p_e / sum_T p
//   y = sum_{e in T} Wd_e (g_e silu(Wg_e x) * (Wu_e x))
//
// Weights are the f16 values that their packed types stand for, as in
// linear(); everything between x and y is f32, rounded once.
#include <cmath>

#include "device_common.hpp"
#include "internal.hpp"

namespace tlhip {

namespace {

template <int WT>
__device__ __forceinline__ float weight(const void* w, const uint16_t* d, int64_t row, int K, int k) {
    if constexpr (WT == TLHIP_F16) return h2f(((const uint16_t*)w)[row * K + k]);
    const float s = h2f(d[row * (K / 32) + k / 32]);
    if constexpr (WT == TLHIP_Q8_0) return (float)(h16)((float)((const int8_t*)w)[row * K + k] * s);
    const uint8_t b = ((const uint8_t*)w)[row * (K / 2) + k / 32 * 16 + k % 16];
    return (float)(h16)((float)((k & 16 ? b >> 4 : b & 15) - 8) * s);
}

// A workgroup per token: the logits, the chosen experts and their weights.
__global__ __launch_bounds__(256) void moe_router_kernel(MoeArgs a) {
    __shared__ float lg[kMoeMaxExperts];
    const int m = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int e = wave; e < a.E; e += 4) {
        float s = 0.0f;
        for (int k = lane; k < a.K; k += 64) s = fmaf(h2f(a.x[(size_t)m * a.K + k]), h2f(a.router[(size_t)e * a.K + k]), s);
        s = wave_sum<64>(s);
        if (lane == 0) lg[e] = s;
    }
    __syncthreads();
    if (wave) return;
    float v[kMoeMaxExperts / 64], big = -INFINITY, z = 0.0f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < kMoeMaxExperts / 64; j++) {
        const int e = lane + 64 * j;
        v[j] = e < a.E ? lg[e] : -INFINITY;
        nan |= v[j] != v[j];
        big = fmaxf(big, v[j]);
    }
    nan = __any(nan);
    big = wave_max(big);
#pragma unroll
    for (int j = 0; j < kMoeMaxExperts / 64; j++) z += lane + 64 * j < a.E ? __builtin_amdgcn_exp2f((v[j] - big) * 1.44269504f) : 0.0f;
    z = wave_sum<64>(z);
    // rounds of the largest (value, lowest index); a chosen one leaves.  NaN
    // ranks below everything, so every round finds an expert.
    float chosen = 0.0f, mine = 0.0f;
    uint32_t gone = 0;
    int id = 0;
    for (int t = 0; t < a.top; t++) {
        uint64_t best = 0;
#pragma unroll
        for (int j = 0; j < kMoeMaxExperts / 64; j++) {
            const uint32_t e = lane + 64 * j, b = __float_as_uint(v[j] + 0.0f);
            const uint32_t o = v[j] != v[j] ? 1u : b & 0x80000000u ? ~b : b | 0x80000000u;
            const uint64_t k = e < (uint32_t)a.E && !(gone >> j & 1) ? (uint64_t)o << 32 | (0xFFFFFFFFu - e) : 0;
            best = k > best ? k : best;
        }
        for (int k = 32; k; k >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)best, k, 64);
            best = o > best ? o : best;
        }
        const int e = (int)(0xFFFFFFFFu - (uint32_t)best);
        if ((e & 63) == lane) gone |= 1u << (e >> 6);
        const float p = __builtin_amdgcn_exp2f((lg[e] - big) * 1.44269504f);
        chosen += p;
        if (lane == t) {
            id = e;
            mine = p;
        }
    }
    if (lane < a.top) {
        a.ids[(size_t)m * a.top + lane] = id;
        a.g[(size_t)m * a.top + lane] = nan ? NAN : mine / (a.normalize ? chosen : z);
    }
}

// A wave per (token and choice, row of gate and up).
template <int WT>
__global__ __launch_bounds__(256) void moe_gate_up_kernel(MoeArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)a.M * a.top * a.I) return;
    const int pair = (int)(at / a.I), i = (int)(at % a.I), lane = threadIdx.x & 63;
    const int64_t row = (int64_t)a.ids[pair] * a.I + i;
    const uint16_t* x = a.x + (size_t)(pair / a.top) * a.K;
    float gt = 0.0f, up = 0.0f;
    for (int k = lane; k < a.K; k += 64) {
        const float xv = h2f(x[k]);
        gt = fmaf(weight<WT>(a.gate, a.gate_d, row, a.K, k), xv, gt);
        up = fmaf(weight<WT>(a.up, a.up_d, row, a.K, k), xv, up);
    }
    gt = wave_sum<64>(gt);
    up = wave_sum<64>(up);
    if (lane == 0) a.h[(size_t)pair * a.I + i] = a.g[pair] * (gt / (1.0f + __expf(-gt)) * up);
}

// A wave per output.
template <int WT>
__global__ __launch_bounds__(256) void moe_down_kernel(MoeArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)a.M * a.K) return;
    const int m = (int)(at / a.K), n = (int)(at % a.K), lane = threadIdx.x & 63;
    float s = 0.0f;
    for (int t = 0; t < a.top; t++) {
        const int pair = m * a.top + t;
        const int64_t row = (int64_t)a.ids[pair] * a.K + n;
        for (int i = lane; i < a.I; i += 64) s = fmaf(weight<WT>(a.down, a.down_d, row, a.I, i), a.h[(size_t)pair * a.I + i], s);
    }
    s = wave_sum<64>(s);
    if (lane == 0) a.y[(size_t)m * a.K + n] = f2h(s);
}

}  // namespace

tlhip_status launch_moe(hipStream_t s, const MoeArgs& a) {
    moe_router_kernel<<<a.M, 256, 0, s>>>(a);
    const unsigned gu = (unsigned)(((int64_t)a.M * a.top * a.I + 3) / 4), dn = (unsigned)(((int64_t)a.M * a.K + 3) / 4);
    if (a.wt_gu == TLHIP_F16) moe_gate_up_kernel<TLHIP_F16><<<gu, 256, 0, s>>>(a);
    else if (a.wt_gu == TLHIP_Q4_0) moe_gate_up_kernel<TLHIP_Q4_0><<<gu, 256, 0, s>>>(a);
    else moe_gate_up_kernel<TLHIP_Q8_0><<<gu, 256, 0, s>>>(a);
    if (a.wt_down == TLHIP_F16) moe_down_kernel<TLHIP_F16><<<dn, 256, 0, s>>>(a);
    else if (a.wt_down == TLHIP_Q4_0) moe_down_kernel<TLHIP_Q4_0><<<dn, 256, 0, s>>>(a);
    else moe_down_kernel<TLHIP_Q8_0><<<dn, 256, 0, s>>>(a);
    return TLHIP_OK;
}

}  // namespace tlhip
