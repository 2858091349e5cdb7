// kernels_logprobs.hip -- token_logprobs: of each row of logits the log
// probability of a given token, the entropy, and the n most likely tokens.
//
// With m = max x, z = sum e^(x - m) and t = sum (x - m) e^(x - m):
//   log p_i = (x_i - m) - log z,   H = log z - t / z.
// One pass over the row keeps m, z and t up to date: when m rises by -d, z
// becomes z e^d and t becomes (t + d z) e^d.  All in f32, in powers of two
// (t in units of ln 2).
//
// The n largest come out of the same pass.  They are the n largest keys
// (value up, index down), all different.  A workgroup's threads are 64 groups
// of four; the n-th largest of the groups' largest keys so far is a bound tau
// that n keys of the row are known to reach, so only keys from tau up are
// kept: a thread compares its batch's maximum, which the softmax needs
// anyway, and looks at single values only if that reaches tau.  tau is found
// after the batches 1, 2, 4, 8, ...; on random rows a doubling adds about n
// to 5 n keys to the list.  Rows made to defeat the bound (rising ones of
// great length) overflow the list and are ranked by n rounds over the row.
//
// Few rows are cut into chunks, a workgroup each, joined by a second kernel.
//
// Bound by memory without alternatives (2048 f16 rows of 32000: 28.6 us, 4.6
// TB/s), with them by the exps and the list beside the loads (333 f32 rows of
// 51200, 20 alternatives: 21 us and 4 for the join, 2.7 TB/s), for one row by
// the two launches (32000 f16: 7 and 3 us).
#include <cmath>

#include "device_common.hpp"
#include "internal.hpp"

namespace tlhip {

namespace {

constexpr float kLog2e = 1.44269504088896f, kLn2 = 0.693147180559945f;
// Elements of a thread's batch, for rows that need more than 256 * kShort
// threads' and for the others (2000 f16 rows of 501, 5 alternatives: 11.4 us
// against 22 with the long batch).
constexpr int kLong = 32, kShort = 8;
constexpr int kBatch = 256 * kLong;     // elements of a workgroup's
constexpr int kList = 2048, kRanked = 512;
constexpr int kMaxChunks = 32;

// The sums in reference to r: e = 2^d2(x).  f32: r = m and d2 = (x - m)
// log2(e), which reaches the type's lowest value; f16: r = m log2(e) and d2 =
// x log2(e) - r in one fused operation.  (Any r near the maximum will do, so
// r's own rounding costs nothing.)
template <bool F32>
struct Stat {
    float m, r, z, t;
    static __device__ __forceinline__ Stat none() {
        Stat s;
        s.m = F32 ? -3.4028234663852886e38f : -65536.0f;   // below every finite logit, or the lowest
        s.r = F32 ? s.m : s.m * kLog2e;
        s.z = s.t = 0.0f;
        return s;
    }
    __device__ __forceinline__ float d2(float x) const { return F32 ? (x - r) * kLog2e : __builtin_fmaf(x, kLog2e, -r); }
    __device__ __forceinline__ void rise(float mn, float rn) {
        const float d = F32 ? (r - rn) * kLog2e : r - rn, f = __builtin_amdgcn_exp2f(d);
        t = f > 0.0f ? fmaf(d, z, t) * f : 0.0f;   // (d may be infinite where f is 0)
        z *= f;
        m = mn;
        r = rn;
    }
    __device__ __forceinline__ void rise(float mn) { rise(mn, F32 ? mn : mn * kLog2e); }
    __device__ __forceinline__ void add(float x) {
        const float d = d2(x), e = __builtin_amdgcn_exp2f(d);
        z += e;                                    // (a NaN or +inf shows in z)
        t = fmaf(fmaxf(d, -300.0f), e, t);         // (-inf: -300 * 0)
    }
    __device__ __forceinline__ void join(Stat o) {
        if (o.m > m) rise(o.m, o.r);
        else o.rise(m, r);
        z += o.z;
        t += o.t;
    }
    // a NaN or +inf among the logits, or nothing but -inf: no distribution
    __device__ __forceinline__ bool ok() const { return z > 0.0f && z < INFINITY; }
    __device__ __forceinline__ float logprob(float x, float lz2) const {
        return F32 ? x - r - lz2 * kLn2 : (d2(x) - lz2) * kLn2;
    }
    __device__ __forceinline__ Stat from_lane(int mask) const {
        Stat o;
        o.m = __shfl_xor(m, mask, 64);
        o.r = __shfl_xor(r, mask, 64);
        o.z = __shfl_xor(z, mask, 64);
        o.t = __shfl_xor(t, mask, 64);
        return o;
    }
};

// Keys ordered as the pairs (value up, index down); -0 is 0.  0: no key.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ int32_t key_index(uint64_t k) { return (int32_t)(0xFFFFFFFFu - (uint32_t)k); }
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <bool F32>
__device__ __forceinline__ float at(const LogprobArgs& a, size_t i) {
    return F32 ? ((const float*)a.x)[i] : h2f(((const uint16_t*)a.x)[i]);
}

// E elements of a thread, in vectors of 16 bytes a workgroup's width apart, of
// a batch that ends at element hi: the vectors past it are moved back to end
// there, and what they repeat counts for none.
struct __attribute__((packed, aligned(4))) f4_any {
    float f[4];
};
template <bool F32, int E>
struct Batch {
    static constexpr int W = F32 ? 4 : 8, NV = E / W, SIZE = 256 * E;
    float f[F32 ? E : 1];
    h8 h[F32 ? 1 : NV];
    int lo, hi, last;   // elements lo .. hi - 1 are new; the last vector's place
    __device__ __forceinline__ float operator[](int j) const {
        if constexpr (F32) return f[j];
        else return (float)h[j / 8][j % 8];
    }
    static __device__ __forceinline__ int place(int v) { return (v * 256 + (int)threadIdx.x) * W; }
    __device__ __forceinline__ int index(int j) const { return min(place(j / W), last) + j % W; }
    __device__ __forceinline__ bool mine(int j) const {
        const int i = index(j);
        return i >= lo && i >= place(j / W) && i < hi;
    }
    // A set of elements, the first at the highest of E bits.
    static constexpr uint32_t ALL = 0xFFFFFFFFu >> (32 - E);
    static __device__ __forceinline__ uint32_t bit(int j) { return 1u << (E - 1 - j); }
    static __device__ __forceinline__ int first(uint32_t set) { return __builtin_clz(set & ALL) - (32 - E); }
    // The elements less than y (above: greater): the differences' signs, shifted
    // in.  (A comparison's mask would take a move and two waits each.)  NaN: any.
    __device__ __forceinline__ uint32_t below(float y, bool above) const {
        if (y == 0.0f) y = above ? 0.0f : -0.0f;   // (either zero minus it is +0)
        uint32_t set = 0;
#pragma unroll
        for (int j = 0; j < E; j++) set = __builtin_amdgcn_alignbit(set, __float_as_uint(above ? y - (*this)[j] : (*this)[j] - y), 31);
        return set;
    }
    __device__ __forceinline__ void set(int j, float x) {
        if constexpr (F32) f[j] = x;
        else h[j / 8][j % 8] = (h16)x;
    }
    // Elements base + index(j); -inf in place of those that are not new.  (No
    // branch among the loads: each would wait for those before it.)
    __device__ __forceinline__ void load(const LogprobArgs& a, size_t base, int lo_, int hi_) {
        lo = lo_;
        hi = hi_;
        last = hi > W ? hi - W : 0;
        if (hi < W) {   // a row shorter than a vector
#pragma unroll
            for (int j = 0; j < E; j++) set(j, j < W && threadIdx.x == 0 && j < hi ? at<F32>(a, base + j) : -INFINITY);
            return;
        }
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const size_t i = base + min(place(v), last);
            if constexpr (F32) {
                const f4_any w = *(const f4_any*)((const float*)a.x + i);
#pragma unroll
                for (int e = 0; e < 4; e++) f[4 * v + e] = w.f[e];
            } else {
                const h8_any w = *(const h8_any*)((const uint16_t*)a.x + i);
                h[v] = __builtin_bit_cast(h8, u4{w.w[0], w.w[1], w.w[2], w.w[3]});
            }
        }
        if (lo || hi < SIZE)
#pragma unroll
            for (int j = 0; j < E; j++)
                if (!mine(j)) set(j, -INFINITY);
    }
};

struct TopShared {
    uint64_t group[64];
    uint64_t ranked[kRanked];
    int list[kList];   // elements of the row
    uint64_t best[4];
    int above[4][64], rank[kRanked];
    int count, kept;
};

// The n-th largest of the 64 groups' keys (0 if there are fewer), the same in
// every thread: a lane stands for a group, and each wave counts the keys above
// it among a quarter of them.
__device__ __forceinline__ uint64_t bound(uint64_t mine, int n, TopShared& sh) {
    for (int k = 1; k < 4; k <<= 1) mine = max64(mine, __shfl_xor((unsigned long long)mine, k, 64));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if ((lane & 3) == 0) sh.group[threadIdx.x >> 2] = mine;
    __syncthreads();
    const uint64_t g = sh.group[lane];
    int above = 0;
#pragma unroll
    for (int k = 0; k < 16; k++) above += sh.group[16 * wave + k] > g;
    sh.above[wave][lane] = above;
    __syncthreads();
    above = sh.above[0][lane] + sh.above[1][lane] + sh.above[2][lane] + sh.above[3][lane];
    const uint64_t who = __ballot(above == n - 1 && g != 0);
    if (!who) return 0;
    const int src = __builtin_ctzll(who);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)g, src), hi = __builtin_amdgcn_readlane((int)(g >> 32), src);
    return (uint64_t)hi << 32 | lo;
}

// Writes the n largest of `count` keys in LDS (0: none) to out in falling
// order, by counting for each the keys above it: a wave per quarter of them.
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int count, int n, uint64_t* out, int* rank) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < count; i += 256) rank[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < count; i0 += 64) {
        const uint64_t k = i0 + lane < count ? keys[i0 + lane] : 0;
        int above = 0;
        for (int j0 = 4 * wave; j0 < count; j0 += 16) {
            uint64_t o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = j0 + j < count ? keys[j0 + j] : 0;
#pragma unroll
            for (int j = 0; j < 4; j++) above += o[j] > k;
        }
        if (i0 + lane < count && above) atomicAdd(&rank[i0 + lane], above);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += 256)
        if (keys[i] && rank[i] < n) out[rank[i]] = keys[i];
}

// The same by n rounds of the largest key below the last one; key(i), i <
// count, may be read n times.
template <typename KEY>
__device__ __forceinline__ void rounds(const KEY& key, int count, int n, uint64_t* out, TopShared& sh) {
    uint64_t below = ~0ull;
    for (int r = 0; r < n; r++) {
        uint64_t b = 0;
        for (int i = threadIdx.x; i < count; i += 256) {
            const uint64_t k = key(i);
            if (k < below && k > b) b = k;
        }
        for (int k = 32; k; k >>= 1) b = max64(b, __shfl_xor((unsigned long long)b, k, 64));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = b;
        __syncthreads();
        for (int k = 0; k < 4; k++) b = max64(b, sh.best[k]);
        if (threadIdx.x == 0) out[r] = b;
        below = b;
    }
}

template <bool F32>
__device__ __forceinline__ void finish(const LogprobArgs& a, int row, const Stat<F32>& s, const uint64_t* top) {
    const bool ok = s.ok();
    const float lz2 = __builtin_amdgcn_logf(s.z);
    const int tid = threadIdx.x;
    if (tid == 0) {
        if (a.logprob) {
            const int id = a.ids[row];
            a.logprob[row] = ok && id >= 0 && id < a.V ? s.logprob(at<F32>(a, (size_t)row * a.V + id), lz2) : NAN;
        }
        if (a.entropy) a.entropy[row] = ok ? (lz2 - s.t / s.z) * kLn2 : NAN;
    }
    if (tid < a.n_top) {
        const uint64_t k = top[tid];
        a.top_logprob[(size_t)row * a.n_top + tid] = ok ? s.logprob(key_value(k), lz2) : NAN;
        a.top_ids[(size_t)row * a.n_top + tid] = ok ? key_index(k) : -1;
    }
}

template <bool F32, bool TOP, int E>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
    __shared__ Stat<F32> st[4];
    __shared__ __align__(16) uint8_t top_raw[TOP ? sizeof(TopShared) : 16];
    __shared__ uint64_t top[TOP ? kMaxTop : 1];
    TopShared& sh = *(TopShared*)top_raw;
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
    const int begin = chunk * a.chunk, count = a.V - begin < a.chunk ? a.V - begin : a.chunk;
    const size_t base = (size_t)row * a.V + begin;
    Stat<F32> s = Stat<F32>::none();
    uint64_t best = 0, tau = 0;
    if (TOP) {
        if (tid < kMaxTop) top[tid] = 0;
        if (tid == 0) sh.count = sh.kept = 0;
    }
    for (int b = 0, nb = 0; b < count; b += Batch<F32, E>::SIZE, nb++) {
        // the last batch of several is moved back to be whole
        const int at0 = count - b < Batch<F32, E>::SIZE && nb ? count - Batch<F32, E>::SIZE : b;
        Batch<F32, E> x;
        x.load(a, base + at0, b - at0, count - at0 < Batch<F32, E>::SIZE ? count - at0 : Batch<F32, E>::SIZE);
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < E; j++) m = fmaxf(m, x[j]);
        if (m > s.m) s.rise(m);
#pragma unroll
        for (int j = 0; j < E; j++) s.add(x[j]);
        if constexpr (TOP) {
            if (!best || m > key_value(best)) {
                // the first element that is m (an -inf in place of another is none)
                int first = -1;
                if (m > -INFINITY) {
                    const uint32_t less = x.below(m, false);
                    first = less != Batch<F32, E>::ALL ? Batch<F32, E>::first(~less) : -1;
                } else {
                    for (int j = E - 1; j >= 0; j--) first = x[j] == m && x.mine(j) ? j : first;
                }
                if (first >= 0) best = key_of(m, begin + at0 + x.index(first));
            }
            if (nb == 0) tau = bound(best, a.n_top, sh);
            const float least = tau ? key_value(tau) : -INFINITY;
            if (m >= least) {
                // the places of the batch's keys from tau up go to the list
                // (-inf has no differences: the lowest finite value stands in)
                const bool any = least == -INFINITY;
                const float l = any ? -3.4028234663852886e38f : least;
                const uint32_t less = x.below(l, false), more = x.below(l, true), same = Batch<F32, E>::ALL & ~(less | more);
                uint32_t hit = any ? more | same : more, even = any ? less : same;
                const int last = tau ? key_index(tau) - begin - at0 : Batch<F32, E>::SIZE;
                for (; even; even ^= Batch<F32, E>::bit(Batch<F32, E>::first(even))) {
                    const int j = Batch<F32, E>::first(even);
                    if (x.mine(j) && x.index(j) <= last) hit |= Batch<F32, E>::bit(j);
                }
                if (hit) {
                    int slot = atomicAdd(&sh.count, __builtin_popcount(hit));
                    for (; hit; hit ^= Batch<F32, E>::bit(Batch<F32, E>::first(hit)), slot++)
                        if (slot < kList) sh.list[slot] = at0 + x.index(Batch<F32, E>::first(hit));
                }
            }
            if (nb && !(nb & (nb + 1)) && b + Batch<F32, E>::SIZE < count) tau = bound(best, a.n_top, sh);
        }
    }
    for (int k = 32; k; k >>= 1) s.join(s.from_lane(k));
    if ((tid & 63) == 0) st[tid >> 6] = s;
    __syncthreads();
    s = st[0];
    for (int k = 1; k < 4; k++) s.join(st[k]);
    if constexpr (TOP) {
        if (count > Batch<F32, E>::SIZE) tau = bound(best, a.n_top, sh);   // (else it stands)
        const int listed = sh.count;
        auto listed_key = [&](int i) { return key_of(at<F32>(a, base + sh.list[i]), begin + sh.list[i]); };
        if (listed <= kList) {
            for (int i = tid; i < listed; i += 256) {
                const uint64_t k = listed_key(i);
                if (k >= tau) {
                    const int slot = atomicAdd(&sh.kept, 1);
                    if (slot < kRanked) sh.ranked[slot] = k;
                }
            }
            __syncthreads();
            const int kept = sh.kept;
            if (kept <= kRanked) rank_keys(sh.ranked, kept, a.n_top, top, sh.rank);
            else rounds(listed_key, listed, a.n_top, top, sh);
        } else {
            rounds([&](int i) { return key_of(at<F32>(a, base + i), begin + i); }, count, a.n_top, top, sh);
        }
        __syncthreads();
    }
    if (a.chunks == 1) {
        finish<F32>(a, row, s, top);
        return;
    }
    // the chunk's sums and keys, for logprobs_join_kernel
    if (tid == 0) *(f4*)(a.part + 4 * (size_t)blockIdx.x) = f4{s.m, s.r, s.z, s.t};
    if (TOP && tid < a.n_top) a.part_keys[(size_t)blockIdx.x * a.n_top + tid] = top[tid];
}

template <bool F32>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    __shared__ uint64_t keys[kMaxChunks * kMaxTop], top[kMaxTop];
    __shared__ int rank[kMaxChunks * kMaxTop];
    const int row = blockIdx.x, n = a.chunks * a.n_top;
    for (int i = threadIdx.x; i < n; i += 256) keys[i] = a.part_keys[(size_t)row * n + i];
    Stat<F32> s = Stat<F32>::none();
    for (int c = 0; c < a.chunks; c++) {
        const f4 p = *(const f4*)(a.part + 4 * ((size_t)row * a.chunks + c));
        Stat<F32> o;
        o.m = p[0];
        o.r = p[1];
        o.z = p[2];
        o.t = p[3];
        s.join(o);
    }
    __syncthreads();
    rank_keys(keys, n, a.n_top, top, rank);
    __syncthreads();
    finish<F32>(a, row, s, top);
}

}  // namespace

// Chunks of a row: enough workgroups for two to a CU, and no more than one for
// each batch of a row.  (333 f32 rows of 51200 with 20 alternatives: 26.3 us,
// with one to a CU 27.2, three 28.8, four 30.9; 700 f16 rows of 128000, 5:
// 56.5, from three on 64.)
constexpr int kWorkgroups = 512;
LogprobPlan logprobs_plan(int rows, int V, int n_top) {
    LogprobPlan p;
    const int64_t batches = ((int64_t)V + kBatch - 1) / kBatch;
    int64_t chunks = rows >= kWorkgroups ? 1 : (kWorkgroups + rows - 1) / rows;
    if (chunks > batches) chunks = batches;
    if (chunks > kMaxChunks) chunks = kMaxChunks;
    const int64_t per = (batches + chunks - 1) / chunks;
    p.chunks = (int)((batches + per - 1) / per);
    p.chunk = per * kBatch < V ? (int)(per * kBatch) : V;
    if (p.chunks > 1) {
        p.part_bytes = align256((size_t)rows * p.chunks * 4 * sizeof(float));
        p.ws_bytes = p.part_bytes + (size_t)rows * p.chunks * n_top * sizeof(uint64_t);
    }
    return p;
}

template <bool F32, int E>
void launch(hipStream_t s, const LogprobArgs& a) {
    const unsigned wg = (unsigned)a.rows * a.chunks;
    if (a.n_top) logprobs_kernel<F32, true, E><<<wg, 256, 0, s>>>(a);
    else logprobs_kernel<F32, false, E><<<wg, 256, 0, s>>>(a);
    if (a.chunks > 1) logprobs_join_kernel<F32><<<a.rows, 256, 0, s>>>(a);
}

tlhip_status launch_logprobs(hipStream_t s, const LogprobArgs& a) {
    if (a.V <= 256 * kShort) a.f32 ? launch<true, kShort>(s, a) : launch<false, kShort>(s, a);
    else a.f32 ? launch<true, kLong>(s, a) : launch<false, kLong>(s, a);
    return TLHIP_OK;
}

}  // namespace tlhip
