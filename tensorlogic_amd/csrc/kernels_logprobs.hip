// kernels_logprobs.hip -- token_logprobs: of each row of logits the log
// probability of a given token, the entropy, and the n most likely tokens.
//
// With m = max x, z = sum e^(x - m) and t = sum (x - m) e^(x - m):
//   log p_i = (x_i - m) - log z,   H = log z - t / z.
// One pass keeps m, z and t up to date: when m rises by -d, z becomes z e^d
// and t becomes (t + d z) e^d.  All in f32.
#include <cmath>

#include "device_common.hpp"
#include "internal.hpp"

namespace tlhip {

namespace {

constexpr float kLog2e = 1.44269504088896f, kLn2 = 0.693147180559945f;

struct Stat {
    float m, z, t;
    static __device__ __forceinline__ Stat none() { return Stat{-3.4028234663852886e38f, 0.0f, 0.0f}; }
    __device__ __forceinline__ void raise(float mn) {
        const float d = m - mn, f = __builtin_amdgcn_exp2f(d * kLog2e);
        t = f > 0.0f ? fmaf(d, z, t) * f : 0.0f;   // (d may be infinite where f is 0)
        z *= f;
        m = mn;
    }
    __device__ __forceinline__ void add(float x) {
        if (x > m) raise(x);
        const float d = x - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
        z += e;
        t += e > 0.0f ? d * e : 0.0f;              // (-inf: nothing)
    }
    __device__ __forceinline__ void join(Stat o) {
        const float mn = fmaxf(m, o.m);
        raise(mn);
        o.raise(mn);
        z += o.z;
        t += o.t;
    }
};

// Keys ordered as the pairs (value up, index down); -0 is 0.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

template <bool F32>
__device__ __forceinline__ float at(const LogprobArgs& a, int64_t i) {
    return F32 ? ((const float*)a.x)[i] : h2f(((const uint16_t*)a.x)[i]);
}

template <bool F32>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
    __shared__ Stat st[4];
    __shared__ uint64_t best[4];
    const int64_t row = blockIdx.x, base = row * a.V;
    const int tid = threadIdx.x, wave = tid >> 6;
    Stat s = Stat::none();
    for (int i = tid; i < a.V; i += 256) s.add(at<F32>(a, base + i));
    for (int k = 32; k; k >>= 1) {
        Stat o;
        o.m = __shfl_xor(s.m, k, 64);
        o.z = __shfl_xor(s.z, k, 64);
        o.t = __shfl_xor(s.t, k, 64);
        s.join(o);
    }
    if ((tid & 63) == 0) st[wave] = s;
    __syncthreads();
    s = st[0];
    for (int k = 1; k < 4; k++) s.join(st[k]);
    // a NaN or +inf among the logits, or nothing but -inf: no distribution
    const bool ok = s.z > 0.0f && s.z < INFINITY;
    const float lz = __builtin_amdgcn_logf(s.z) * kLn2;
    if (tid == 0) {
        if (a.logprob) {
            const int id = a.ids[row];
            a.logprob[row] = ok && id >= 0 && id < a.V ? at<F32>(a, base + id) - s.m - lz : NAN;
        }
        if (a.entropy) a.entropy[row] = ok ? lz - s.t / s.z : NAN;
    }
    uint64_t below = ~0ull;
    for (int n = 0; n < a.n_top; n++) {
        uint64_t b = 0;
        if (ok)
            for (int i = tid; i < a.V; i += 256) {
                const uint64_t k = key_of(at<F32>(a, base + i), i);
                if (k < below && k > b) b = k;
            }
        for (int k = 32; k; k >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)b, k, 64);
            b = o > b ? o : b;
        }
        __syncthreads();
        if ((tid & 63) == 0) best[wave] = b;
        __syncthreads();
        for (int k = 0; k < 4; k++) b = best[k] > b ? best[k] : b;
        if (tid == 0) {
            a.top_logprob[row * a.n_top + n] = ok ? key_value(b) - s.m - lz : NAN;
            a.top_ids[row * a.n_top + n] = ok ? (int32_t)(0xFFFFFFFFu - (uint32_t)b) : -1;
        }
        below = b;
    }
}

}  // namespace

tlhip_status launch_logprobs(hipStream_t s, const LogprobArgs& a) {
    if (a.f32) logprobs_kernel<true><<<a.rows, 256, 0, s>>>(a);
    else logprobs_kernel<false><<<a.rows, 256, 0, s>>>(a);
    return TLHIP_OK;
}

}  // namespace tlhip
