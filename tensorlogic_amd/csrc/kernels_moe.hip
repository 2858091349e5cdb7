// kernels_moe.hip -- a mixture-of-experts layer for a few tokens: router, the
// chosen experts' SwiGLU and their weighted sum.
//
//   l = R x,  p = softmax(l),  T = the `top` largest (ties: the first expert)
//   g_e = p_e, or p_e / sum_T p
//   y = sum_{e in T} Wd_e (g_e silu(Wg_e x) * (Wu_e x))
//
// Weights are the f16 values that their packed types stand for, as in
// linear(); everything between x and y is f32, rounded once.
//
// Four launches: the router (a workgroup per token); gate and up; down; the
// sum over a token's experts.  What bounds the middle two is reading the
// weights of the experts that some token chose, so each is read once: a
// workgroup takes 16 rows of one expert (of gate and of up both), finds that
// expert's tokens, and multiplies by all of them on the matrix cores
// (v_mfma_f32_16x16x32_f16, A = 16 weight rows x 32 k, B = 32 k x 16 columns;
// unused columns cost nothing that is scarce).  Its eight waves share out k
// and add up through LDS.
//
// A lane's 16-byte weight load is one Q4_0 block (half a Q8_0 block, eight f16
// values), from which it supplies A's 8-element pieces in whatever order the
// unpacking leaves them: the columns are laid out in LDS in that order.
//
// The product after the activation takes h, f32, as two f16 columns, h 2^-e =
// hi + lo, with the power of two that puts the token's largest |h| just below
// 2^15: 22 bits of every h, and none lost to the range of f16.
#include <cmath>

#include "device_common.hpp"
#include "internal.hpp"

namespace tlhip {

namespace {

constexpr int kWaves = 4;                  // of a workgroup of the products
constexpr int kStageBytes = 32 << 10;      // columns staged in LDS at a time
constexpr int kTokens = 256;               // tokens of one round of launches (moe.cpp)

// ---------------------------------------------------------------------------
// router
// ---------------------------------------------------------------------------
// A workgroup of 16 waves per token: (expert, part of K) tasks over the
// waves, then one wave ranks.  Bound by latency.
__global__ __launch_bounds__(1024) void moe_router_kernel(MoeArgs a) {
    __shared__ float lg[kMoeMaxExperts];
    __shared__ float part[16];
    const int m = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // waves per expert: all 16 waves have work when there are fewer experts
    const int P = a.E <= 2 ? 8 : a.E <= 4 ? 4 : a.E <= 8 ? 2 : 1;
    const uint16_t* x = a.x + (size_t)m * a.K;
    const int pieces = a.K / 8, share = (pieces + P - 1) / P;
    for (int task = wave; task < a.E * P; task += 16) {
        const int e = task / P, k0 = (task % P) * share, k1 = k0 + share < pieces ? k0 + share : pieces;
        const uint16_t* r = a.router + (size_t)e * a.K;
        float s = 0.0f;
#pragma unroll 4
        for (int k = k0 + lane; k < k1; k += 64) {
            const u4 xv = *(const u4*)(x + 8 * k), rv = *(const u4*)(r + 8 * k);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const h2 p = as_h2(xv[i]), q = as_h2(rv[i]);
                s = fmaf((float)p[0], (float)q[0], s);
                s = fmaf((float)p[1], (float)q[1], s);
            }
        }
        s = wave_sum<64>(s);
        if (lane == 0) (P == 1 ? lg : part)[task] = s;
    }
    __syncthreads();
    if (P > 1 && (int)threadIdx.x < a.E) {
        float s = 0.0f;
        for (int i = 0; i < P; i++) s += part[threadIdx.x * P + i];
        lg[threadIdx.x] = s;
    }
    __syncthreads();
    if (wave) return;
    constexpr int NJ = kMoeMaxExperts / 64;
    float v[NJ], big = -INFINITY, z = 0.0f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int e = lane + 64 * j;
        v[j] = e < a.E ? lg[e] : -INFINITY;
        nan |= v[j] != v[j];
        big = fmaxf(big, v[j]);
    }
    nan = __any(nan);   // (then any experts will do: their weights are NaN)
    big = wave_max(big);
#pragma unroll
    for (int j = 0; j < NJ; j++) z += lane + 64 * j < a.E ? __builtin_amdgcn_exp2f((v[j] - big) * 1.44269504f) : 0.0f;
    z = wave_sum<64>(z);
    // rounds of the largest value, at its lowest index; a chosen one leaves
    float chosen = 0.0f, mine = 0.0f;
    uint32_t gone = 0;   // bit j: expert lane + 64 j is chosen, or none
    int id = lane;
#pragma unroll
    for (int j = 0; j < NJ; j++) gone |= (lane + 64 * j >= a.E ? 1u : 0u) << j;
    for (int t = 0; t < a.top && !nan; t++) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NJ; j++) top = fmaxf(top, gone >> j & 1 ? -INFINITY : v[j]);
        top = wave_max(top);
        int e = 0;
#pragma unroll
        for (int j = NJ - 1; j >= 0; j--) {
            const uint64_t who = __ballot(!(gone >> j & 1) && v[j] == top);
            if (who) e = 64 * j + __builtin_ctzll(who);
        }
        if ((e & 63) == lane) gone |= 1u << (e >> 6);
        const float p = __builtin_amdgcn_exp2f((top - big) * 1.44269504f);
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

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
// One lane's weights of one step: a block of 32 (Q types), or 8 values of each
// of four blocks (f16).  sub(j) is its part of A in the j-th of the step's
// four matrix instructions.
template <int WT>
struct Weights;
template <>
struct Weights<TLHIP_Q4_0> {
    u4 q;
    uint32_t d;
    __device__ __forceinline__ void load(const void* w, const uint16_t* wd, size_t row, int nb, int step, int g) {
        const int b = 4 * step + g;
        q = u4{0, 0, 0, 0};
        d = 0;
        if (b < nb) {
            q = __builtin_nontemporal_load((const u4*)((const uint8_t*)w + (row * nb + b) * 16));
            d = wd[row * nb + b];
        }
    }
    __device__ __forceinline__ h8 sub(int j) const {
        h2 o[4];
        q4_unpack(q[j], as_h2(d | d << 16), o);
        return h8{o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1]};
    }
};
template <>
struct Weights<TLHIP_Q8_0> {
    u4 q[2];
    uint32_t d;
    __device__ __forceinline__ void load(const void* w, const uint16_t* wd, size_t row, int nb, int step, int g) {
        const int b = 4 * step + g;
        q[0] = q[1] = u4{0, 0, 0, 0};
        d = 0;
        if (b < nb) {
            const u4* p = (const u4*)((const uint8_t*)w + (row * nb + b) * 32);
            q[0] = __builtin_nontemporal_load(p);
            q[1] = __builtin_nontemporal_load(p + 1);
            d = wd[row * nb + b];
        }
    }
    __device__ __forceinline__ h8 sub(int j) const {
        h2 lo[2], hi[2];
        const h2 dd = as_h2(d | d << 16);
        q8_unpack(q[j >> 1][2 * (j & 1)], dd, lo);
        q8_unpack(q[j >> 1][2 * (j & 1) + 1], dd, hi);
        return h8{lo[0][0], lo[0][1], lo[1][0], lo[1][1], hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
    }
};
template <>
struct Weights<TLHIP_F16> {
    u4 q[4];
    __device__ __forceinline__ void load(const void* w, const uint16_t*, size_t row, int nb, int step, int g) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            q[j] = u4{0, 0, 0, 0};
            if (4 * step + j < nb) q[j] = __builtin_nontemporal_load((const u4*)((const uint16_t*)w + (row * nb + 4 * step + j) * 32 + 8 * g));
        }
    }
    __device__ __forceinline__ h8 sub(int j) const { return __builtin_bit_cast(h8, q[j]); }
};

// Where the 8 elements of piece s (0..3) of a block lie, in the order of A's
// pieces: two runs of four, at r0 and r1, each in the order 0 2 1 3 (Q types,
// as they unpack) or 0 1 2 3 (f16).
template <int WT>
__device__ __forceinline__ int run0(int s) { return WT == TLHIP_Q4_0 ? 4 * s : 8 * s; }
template <int WT>
__device__ __forceinline__ int run1(int s) { return WT == TLHIP_Q4_0 ? 16 + 4 * s : 8 * s + 4; }
template <int WT, typename T>
__device__ __forceinline__ h8 piece(const T& a, const T& b) {   // f16 or f32 runs
    if constexpr (WT == TLHIP_F16) return h8{(h16)a[0], (h16)a[1], (h16)a[2], (h16)a[3], (h16)b[0], (h16)b[1], (h16)b[2], (h16)b[3]};
    else return h8{(h16)a[0], (h16)a[2], (h16)a[1], (h16)a[3], (h16)b[0], (h16)b[2], (h16)b[1], (h16)b[3]};
}
// Which piece of which block of a step lane group g needs in instruction j.
template <int WT>
__device__ __forceinline__ int piece_block(int j, int g) { return WT == TLHIP_F16 ? j : g; }
template <int WT>
__device__ __forceinline__ int piece_sub(int j, int g) { return WT == TLHIP_F16 ? g : j; }

typedef h16 h4 __attribute__((ext_vector_type(4)));

struct MoeShared {
    union {
        h8 stage[kStageBytes / 16];
        float red[kWaves * 4 * 256];
    };
    int list[kTokens];      // the expert's (token, choice) pairs
    float scale[kTokens];   // down: 2^-e of each
    int count;
};

// Fills sh.list with the pairs that chose expert e, in order.  One wave.
__device__ __forceinline__ void find_tokens(const MoeArgs& a, int e, MoeShared& sh) {
    const int n = a.M * a.top, lane = threadIdx.x & 63;
    int have = 0;
    for (int p = 0; p < n; p += 64) {
        const bool is = p + lane < n && a.ids[p + lane] == e;
        const uint64_t who = __ballot(is);
        if (is) sh.list[have + __builtin_popcountll(who & ((1ull << lane) - 1))] = p + lane;
        have += __builtin_popcountll(who);
    }
    if (lane == 0) sh.count = have;
}

// The expert of a workgroup's slot, with sh.list and sh.count filled; -1:
// nothing to do.  With fewer (token, choice) pairs than experts a slot is a
// pair, and only the first pair of an expert works on it; else an expert.
__device__ __forceinline__ int slot_expert(const MoeArgs& a, int slot, MoeShared& sh) {
    if (a.M == 1 && a.top < a.E) {
        if (threadIdx.x == 0) {
            sh.list[0] = slot;
            sh.count = 1;
        }
        __syncthreads();
        return a.ids[slot];
    }
    const bool by_pair = a.M * a.top < a.E;
    const int e = by_pair ? a.ids[slot] : slot;
    if (threadIdx.x < 64) find_tokens(a, e, sh);
    __syncthreads();
    return by_pair && sh.list[0] != slot ? -1 : e;
}

// acc[r][c] += W_r (16 rows from row[r], nb blocks) times the CT * 16 columns
// of `cols` that stage() lays out chunk by chunk.
template <int WT, int NR, int CT, typename STAGE>
__device__ __forceinline__ void multiply(const void* const (&w)[NR], const uint16_t* const (&wd)[NR], size_t row, int nb, int ncol,
                                         const STAGE& stage, MoeShared& sh, f4 (&acc)[NR][CT]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
    // blocks of a chunk: a multiple of what the waves take in one step
    int chunk = kStageBytes / (64 * ncol) / (4 * kWaves) * (4 * kWaves);
    const int all = (nb + 4 * kWaves - 1) / (4 * kWaves) * (4 * kWaves);
    if (chunk > all) chunk = all;
    int col[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) col[c] = 16 * c + c16 < ncol ? 16 * c + c16 : ncol - 1;
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int c = 0; c < CT; c++) acc[r][c] = f4{0, 0, 0, 0};
    constexpr int PD = WT == TLHIP_Q4_0 ? 5 - NR : WT == TLHIP_Q8_0 ? 4 - NR : 3 - NR;   // steps loaded ahead
    Weights<WT> ring[PD][NR];
#pragma unroll
    for (int k = 0; k < PD; k++)
#pragma unroll
        for (int r = 0; r < NR; r++) ring[k][r].load(w[r], wd[r], row + c16, nb, wave + k * kWaves, g);
    for (int c0 = 0; c0 < nb; c0 += chunk) {
        const int blocks = nb - c0 < chunk ? nb - c0 : chunk;
        lds_barrier();
        stage(c0, blocks);
        lds_barrier();
        for (int s = wave; 4 * s < blocks; s += kWaves) {
            Weights<WT> cur[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                cur[r] = ring[0][r];
#pragma unroll
                for (int k = 1; k < PD; k++) ring[k - 1][r] = ring[k][r];
                // (chunks are whole rounds of steps, so the wave's later steps
                // are kWaves apart in this chunk and the next)
                ring[PD - 1][r].load(w[r], wd[r], row + c16, nb, c0 / 4 + s + PD * kWaves, g);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int b = 4 * s + piece_block<WT>(j, g);
                b = b < blocks ? b : blocks - 1;   // (A is zero there)
                const h8* p = sh.stage + (size_t)(b * 4 + piece_sub<WT>(j, g)) * ncol;
                h8 x[CT];
#pragma unroll
                for (int c = 0; c < CT; c++) x[c] = p[col[c]];
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const h8 wv = cur[r].sub(j);
#pragma unroll
                    for (int c = 0; c < CT; c++) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv, x[c], acc[r][c], 0, 0, 0);
                }
            }
        }
    }
    // the waves' sums: red[wave][r * CT + c][col][row]
    lds_barrier();
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int c = 0; c < CT; c++) *(f4*)(sh.red + (((wave * NR + r) * CT + c) * 16 + c16) * 16 + 4 * g) = acc[r][c];
    lds_barrier();
}
template <int NR, int CT>
__device__ __forceinline__ float summed(const MoeShared& sh, int r, int col, int row) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) s += sh.red[(((w * NR + r) * CT + (col >> 4)) * 16 + (col & 15)) * 16 + row];
    return s;
}

// Gate and up of 16 rows of one expert, for tokens list[t0 .. t0 + nt).
template <int WT, int CT>
__device__ __forceinline__ void gate_up_tile(const MoeArgs& a, int e, int i0, int t0, int nt, MoeShared& sh) {
    const void* const w[2] = {a.gate, a.up};
    const uint16_t* const wd[2] = {a.gate_d, a.up_d};
    f4 acc[2][CT];
    auto stage = [&](int c0, int blocks) {
        for (int i = threadIdx.x; i < blocks * 4 * nt; i += kWaves * 64) {
            const int s = i & 3, b = (i >> 2) % blocks, t = (i >> 2) / blocks;
            const uint16_t* x = a.x + (size_t)(sh.list[t0 + t] / a.top) * a.K + (c0 + b) * 32;
            sh.stage[(b * 4 + s) * nt + t] = piece<WT>(*(const h4*)(x + run0<WT>(s)), *(const h4*)(x + run1<WT>(s)));
        }
    };
    multiply<WT, 2, CT>(w, wd, (size_t)e * a.I + i0, a.K / 32, nt, stage, sh, acc);
    for (int i = threadIdx.x; i < 16 * nt; i += kWaves * 64) {
        const int row = i & 15, t = i >> 4, pair = sh.list[t0 + t];
        const float gt = summed<2, CT>(sh, 0, t, row), up = summed<2, CT>(sh, 1, t, row);
        const float h = a.g[pair] * (gt / (1.0f + __expf(-gt)) * up);
        a.h[(size_t)pair * a.I + i0 + row] = h;
        // the tile's largest |h| (a NaN counts as an infinity)
        float m = fabsf(h) <= 3.4028235e38f ? fabsf(h) : INFINITY;
        m = fmaxf(m, dpp_f<0xB1>(m));
        m = fmaxf(m, dpp_f<0x4E>(m));
        m = fmaxf(m, dpp_f<0x141>(m));
        m = fmaxf(m, dpp_f<0x140>(m));
        if (row == 0) a.hmax[(size_t)pair * (a.I / 16) + i0 / 16] = m;
    }
}

template <int WT>
__global__ __launch_bounds__(kWaves * 64) void moe_gate_up_kernel(MoeArgs a) {
    __shared__ MoeShared sh;
    const int tiles = a.I / 16, i0 = (int)(blockIdx.x % tiles) * 16;
    const int e = slot_expert(a, blockIdx.x / tiles, sh);
    if (e < 0) return;
    const int count = sh.count;
    for (int t0 = 0; t0 < count; t0 += 32) {
        const int nt = count - t0 < 32 ? count - t0 : 32;
        if (nt <= 16) gate_up_tile<WT, 1>(a, e, i0, t0, nt, sh);
        else gate_up_tile<WT, 2>(a, e, i0, t0, nt, sh);
        __syncthreads();
    }
}

// Down: 16 rows of one expert; the columns are the hi and lo parts of each
// token's h, one after the other.
template <int WT, int CT>
__device__ __forceinline__ void down_tile(const MoeArgs& a, int e, int n0, int t0, int nt, MoeShared& sh) {
    const void* const w[1] = {a.down};
    const uint16_t* const wd[1] = {a.down_d};
    f4 acc[1][CT];
    auto stage = [&](int c0, int blocks) {
        for (int i = threadIdx.x; i < blocks * 4 * nt; i += kWaves * 64) {
            const int s = i & 3, b = (i >> 2) % blocks, t = (i >> 2) / blocks;
            const float* h = a.h + (size_t)sh.list[t0 + t] * a.I + (c0 + b) * 32;
            const float f = sh.scale[t0 + t];
            const f4 p = *(const f4*)(h + run0<WT>(s)) * f, q = *(const f4*)(h + run1<WT>(s)) * f;
            f4 pl, ql;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                pl[k] = p[k] - (float)(h16)p[k];
                ql[k] = q[k] - (float)(h16)q[k];
            }
            h8* dst = sh.stage + (size_t)(b * 4 + s) * (2 * nt) + 2 * t;
            dst[0] = piece<WT>(p, q);
            dst[1] = piece<WT>(pl, ql);
        }
    };
    multiply<WT, 1, CT>(w, wd, (size_t)e * a.K + n0, a.I / 32, 2 * nt, stage, sh, acc);
    for (int i = threadIdx.x; i < 16 * nt; i += kWaves * 64) {
        const int row = i & 15, t = i >> 4;
        const float v = (summed<1, CT>(sh, 0, 2 * t, row) + summed<1, CT>(sh, 0, 2 * t + 1, row)) / sh.scale[t0 + t];
        a.part[(size_t)sh.list[t0 + t] * a.K + n0 + row] = v;
    }
}

template <int WT>
__global__ __launch_bounds__(kWaves * 64) void moe_down_kernel(MoeArgs a) {
    __shared__ MoeShared sh;
    const int tiles = a.K / 16, n0 = (int)(blockIdx.x % tiles) * 16;
    const int e = slot_expert(a, blockIdx.x / tiles, sh);
    if (e < 0) return;
    const int count = sh.count, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int t = wave; t < count; t += kWaves) {
        const float* hm = a.hmax + (size_t)sh.list[t] * (a.I / 16);
        float m = 0.0f;
        for (int i = lane; i < a.I / 16; i += 64) m = fmaxf(m, hm[i]);
        m = wave_max(m);
        // 2^-e with m 2^-e in [2^14, 2^15); 1 for zeros and the non-finite
        if (lane == 0) sh.scale[t] = m > 0.0f && m < INFINITY ? ldexpf(1.0f, min(14 - ilogbf(m), 126)) : 1.0f;
    }
    __syncthreads();
    for (int t0 = 0; t0 < count; t0 += 16) {
        const int nt = count - t0 < 16 ? count - t0 : 16;
        if (nt <= 8) down_tile<WT, 1>(a, e, n0, t0, nt, sh);
        else down_tile<WT, 2>(a, e, n0, t0, nt, sh);
        __syncthreads();
    }
}

// Down for a single token: all its experts in one workgroup per 16 rows, so
// that no sum is left over.  Sixteen waves share out the (expert, step) pairs;
// the columns are hi and lo of h under one power of two.
constexpr int kOneSteps = 64;   // steps of 4 blocks staged at a time (32 KB)
template <int WT>
__global__ __launch_bounds__(1024) void moe_down_one_kernel(MoeArgs a) {
    __shared__ h8 stage[kOneSteps * 32];
    __shared__ float red[16][2][16], most[16];
    constexpr int PD = WT == TLHIP_F16 ? 1 : 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, nb = a.I / 32, per = (nb + 3) / 4, steps = a.top * per;
    const int ids = a.ids[lane < a.top ? lane : 0];
    auto load = [&](Weights<WT>& w, int n) {
        const int t = n < steps ? n / per : 0, e = __builtin_amdgcn_readlane(ids, t);
        // (past the last step: a step past the row's end, which loads nothing)
        w.load(a.down, a.down_d, (size_t)e * a.K + n0 + c16, nb, n < steps ? n - t * per : per, g);
    };
    Weights<WT> ring[PD];
#pragma unroll
    for (int k = 0; k < PD; k++) load(ring[k], wave + 16 * k);
    float m = 0.0f;
    for (int i = threadIdx.x; i < a.top * (a.I / 16); i += 1024) m = fmaxf(m, a.hmax[i]);
    m = block_max1<16>(m, most);
    const float scale = m > 0.0f && m < INFINITY ? ldexpf(1.0f, min(14 - ilogbf(m), 126)) : 1.0f;
    f4 acc = {0, 0, 0, 0};
    for (int s0 = 0; s0 < steps; s0 += kOneSteps) {
        const int n1 = steps - s0 < kOneSteps ? steps - s0 : kOneSteps;
        lds_barrier();
        for (int i = threadIdx.x; i < n1 * 16; i += 1024) {
            const int s = i & 3, b = i >> 2, n = s0 + (b >> 2), t = n / per, block = 4 * (n - t * per) + (b & 3);
            f4 p = {0, 0, 0, 0}, q = p, pl, ql;
            if (block < nb) {
                const float* h = a.h + (size_t)t * a.I + block * 32;
                p = *(const f4*)(h + run0<WT>(s)) * scale;
                q = *(const f4*)(h + run1<WT>(s)) * scale;
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                pl[k] = p[k] - (float)(h16)p[k];
                ql[k] = q[k] - (float)(h16)q[k];
            }
            stage[2 * i] = piece<WT>(p, q);
            stage[2 * i + 1] = piece<WT>(pl, ql);
        }
        lds_barrier();
        for (int n = wave; n < n1; n += 16) {
            const Weights<WT> cur = ring[0];
#pragma unroll
            for (int k = 1; k < PD; k++) ring[k - 1] = ring[k];
            load(ring[PD - 1], s0 + n + 16 * PD);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const h8 x = stage[((4 * n + piece_block<WT>(j, g)) * 4 + piece_sub<WT>(j, g)) * 2 + (c16 & 1)];
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(cur.sub(j), x, acc, 0, 0, 0);
            }
        }
    }
    if (c16 < 2) *(f4*)&red[wave][c16][4 * g] = acc;
    __syncthreads();
    if (threadIdx.x < 16) {
        float s = 0.0f;
        for (int w = 0; w < 16; w++) s += red[w][0][threadIdx.x] + red[w][1][threadIdx.x];
        a.y[n0 + threadIdx.x] = f2h(s / scale);
    }
}

// y = the sum of a token's experts.
__global__ __launch_bounds__(256) void moe_sum_kernel(MoeArgs a) {
    const int at = blockIdx.x * 256 + threadIdx.x;
    if (at >= a.M * (a.K / 4)) return;
    const int m = at / (a.K / 4), n = at % (a.K / 4) * 4;
    f4 s = {0, 0, 0, 0};
    for (int t = 0; t < a.top; t++) s += *(const f4*)(a.part + ((size_t)m * a.top + t) * a.K + n);
    uint16_t* y = a.y + (size_t)m * a.K + n;
    *(uint64_t*)y = (uint64_t)f2h(s[0]) | (uint64_t)f2h(s[1]) << 16 | (uint64_t)f2h(s[2]) << 32 | (uint64_t)f2h(s[3]) << 48;
}

}  // namespace

template <int WT>
static void launch_gate_up(hipStream_t s, const MoeArgs& a, unsigned slots) {
    moe_gate_up_kernel<WT><<<slots * (a.I / 16), kWaves * 64, 0, s>>>(a);
}
template <int WT>
static void launch_down(hipStream_t s, const MoeArgs& a, unsigned slots) {
    if (a.M == 1) {
        moe_down_one_kernel<WT><<<a.K / 16, 1024, 0, s>>>(a);
        return;
    }
    moe_down_kernel<WT><<<slots * (a.K / 16), kWaves * 64, 0, s>>>(a);
    moe_sum_kernel<<<(a.M * (a.K / 4) + 255) / 256, 256, 0, s>>>(a);
}

tlhip_status launch_moe(hipStream_t s, const MoeArgs& a) {
    moe_router_kernel<<<a.M, 1024, 0, s>>>(a);
    const unsigned slots = a.M * a.top < a.E ? a.M * a.top : a.E;
    if (a.wt_gu == TLHIP_F16) launch_gate_up<TLHIP_F16>(s, a, slots);
    else if (a.wt_gu == TLHIP_Q4_0) launch_gate_up<TLHIP_Q4_0>(s, a, slots);
    else launch_gate_up<TLHIP_Q8_0>(s, a, slots);
    if (a.wt_down == TLHIP_F16) launch_down<TLHIP_F16>(s, a, slots);
    else if (a.wt_down == TLHIP_Q4_0) launch_down<TLHIP_Q4_0>(s, a, slots);
    else launch_down<TLHIP_Q8_0>(s, a, slots);
    return TLHIP_OK;
}

}  // namespace tlhip
