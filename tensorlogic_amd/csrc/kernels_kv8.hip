// kernels_kv8.hip -- the 8-bit KV cache: quantising writes, read-back and
// attention.
//
// Blocks of 32 consecutive positions of one KV head, K and V apart, share
// one f32 scale: a = max |x| over the block, scale = a / 127, and each value
// is kept as q = rint(x * (127 / a)), |q| <= 127, stored as the byte q + 128.
// The positions past the last whole block (the tail, at most 31) are kept as
// the f16 values they came as and are quantised once, when their block is
// whole: what the cache holds depends on the rows alone, not on how many
// calls brought them, and no value is rounded twice.
//
// A block or tail of one head is a tile in the order in which the attention
// kernel's lanes read it, so that every load is 16 bytes per lane
// and contiguous over the wave, and neither keys nor probabilities are
// shuffled between lanes:
//   K tile  [D/8][32 keys][8]: 8 dims of a key together
//   V tile  [D/2][4][2][8]: for a pair of dims, four groups of 8 keys; group
//           g holds keys 8g..8g+7 in the order 0 2 4 6 1 3 5 7, the order in
//           which a lane of the score product holds them
//
// Non-finite values: a block of K or V that holds an infinity or NaN gets the
// scale NaN and zeros, a tail row of V the flag NaN (added to the logarithm
// of its scale, which is otherwise 0) and zeros, so a position that a query
// does not see adds exactly nothing to it, and one that it sees shows.
#include <cmath>
#include <type_traits>

#include "device_common.hpp"
#include "internal.hpp"

namespace tlhip {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

// Element offsets inside a tile.
__device__ __forceinline__ int k_at(int key, int d) { return ((d >> 3) * 32 + key) * 8 + (d & 7); }
__device__ __forceinline__ int v_slot(int key) { return ((key & 1) << 2) | ((key & 7) >> 1); }
__device__ __forceinline__ int v_at(int key, int d) {
    return (((d >> 1) * 4 + (key >> 3)) * 2 + (d & 1)) * 8 + v_slot(key);
}

__device__ __forceinline__ float abs_max8(const h8& v, float m) {
    // (a comparison that a NaN fails would drop it: any non-finite value
    // makes the maximum an infinity)
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float a = fabsf((float)v[i]);
        m = fmaxf(m, a <= 65504.0f ? a : INFINITY);
    }
    return m;
}

// A workgroup per (unit, KV head, K or V).  Units 0 .. n_full - 1 are the
// blocks that this call completes: their positions come from the old tail
// (before len0) and the new rows.  The last unit, when rows are left over,
// writes them to the new tail.  Old and new tail are the same buffer only if
// no block is completed, so nothing is written that another workgroup reads.
// Bound by launch and latency below about 1000 rows (46 rows of 4 heads of 64:
// 3.6 us a call), then by memory (2048 rows of 32 heads of 80, 31 MB: 9.6 us,
// 3.3 TB/s; with 256 threads 10.0).
constexpr int kWriteThreads = 128;
template <int D>
__global__ __launch_bounds__(kWriteThreads) void kv8_write_kernel(Kv8Write p) {
    constexpr int PIECES = 4 * D;            // 8 values each
    constexpr int PT = (PIECES + kWriteThreads - 1) / kWriteThreads; // pieces of a thread
    __shared__ float red[kWriteThreads / 64];
    __shared__ int bad_row[32];
    __shared__ __align__(16) uint8_t tile[34 * D];
    // the tile in LDS, 16 bytes between every 256: neighbouring lanes' pieces
    // lie 256 bytes apart in it and would share their banks
    auto lds = [](int at) { return at + (at >> 8) * 16; };
    // Workgroups go round the eight XCDs; the heads of a unit, whose rows share
    // cache lines, stay on one of them when there are enough units.
    const int items = 2 * p.n_kv, units = p.n_full + ((p.len0 + p.S) & 31 ? 1 : 0);
    const int j = units >= 8 ? blockIdx.x >> 3 : blockIdx.x, item = j % items;
    const int unit = units >= 8 ? j / items * 8 + (blockIdx.x & 7) : j / items;
    if (unit >= units) return;
    const int is_v = item >= p.n_kv, head = is_v ? item - p.n_kv : item;
    const int tid = threadIdx.x;
    const size_t row = (size_t)p.n_kv * D;
    const uint16_t* src = (is_v ? p.v : p.k) + (size_t)head * D;
    const int block = (p.len0 >> 5) + unit, old = p.len0 - block * 32;   // keys below old are in the tail

    // The block's new rows, 8 values a piece (no branch among the loads: each
    // would wait for those before it); past the last row, or before the first,
    // that one again.
    h8 x[PT];
#pragma unroll
    for (int j = 0; j < PT; j++) {
        const int i = min(tid + kWriteThreads * j, PIECES - 1), key = i / (D / 8), u = i % (D / 8);
        x[j] = *(const h8*)(src + (size_t)min(max(key - old, 0), p.S - 1) * row + 8 * u);
    }

    if (unit == p.n_full) {   // the rows left over
        // a fresh tail is cleared past its rows: attention reads whole tiles
        const int end = p.len0 + p.S - block * 32, r0 = max(old, 0), r1 = r0 == 0 ? 32 : end;
        const size_t th = (size_t)p.tail_dst * p.n_kv + head;
        uint16_t* t = (is_v ? p.tail_v : p.tail_k) + th * 32 * D;
        if (is_v) {
            if (tid < 32) bad_row[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PT; j++) {
                const int key = min(tid + kWriteThreads * j, PIECES - 1) / (D / 8);
                if (key >= r0 && key < end && abs_max8(x[j], 0.0f) == INFINITY) bad_row[key] = 1;
            }
            __syncthreads();
            if (tid >= r0 && tid < r1) p.tail_flag[th * 32 + tid] = bad_row[tid] ? NAN : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < PT; j++) {
            const int i = tid + kWriteThreads * j, key = i / (D / 8), u = i % (D / 8);
            if (key < r0 || key >= r1) continue;
            if (key >= end || (is_v && bad_row[key])) x[j] = h8{};
            if (is_v) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const h16 v = x[j][e];   // (a bit cast of the vector's element itself takes element 0)
                    t[v_at(key, 8 * u + e)] = __builtin_bit_cast(uint16_t, v);
                }
            } else {
                *(h8*)(t + k_at(key, 8 * u)) = x[j];
            }
        }
        return;
    }

    float m = 0.0f;
    if (old > 0) {   // its first rows are in the tail
        const size_t th = (size_t)p.tail_src * p.n_kv + head;
        const uint16_t* t = (is_v ? p.tail_v : p.tail_k) + th * 32 * D;
        if (is_v && tid < old && p.tail_flag[th * 32 + tid] != 0.0f) m = INFINITY;
#pragma unroll
        for (int j = 0; j < PT; j++) {
            const int i = min(tid + kWriteThreads * j, PIECES - 1), key = i / (D / 8), u = i % (D / 8);
            h8 y;
            if (is_v) {
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = __builtin_bit_cast(h16, t[v_at(key, 8 * u + e)]);
            } else {
                y = *(const h8*)(t + k_at(key, 8 * u));
            }
            x[j] = key < old ? y : x[j];
        }
    }
#pragma unroll
    for (int j = 0; j < PT; j++) m = abs_max8(x[j], m);
    m = block_max1<kWriteThreads / 64>(m, red);
    const bool bad = m == INFINITY;
    const float inv = m > 0.0f && !bad ? 127.0f / m : 0.0f;
    const float scale = bad ? NAN : m / 127.0f;
#pragma unroll
    for (int j = 0; j < PT; j++) {
        const int i = tid + kWriteThreads * j, key = i / (D / 8), u = i % (D / 8);
        if (i >= PIECES) continue;
        uint8_t q[8];
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = bad ? 128 : (uint8_t)((int)rintf((float)x[j][e] * inv) + 128);
        if (is_v) {
#pragma unroll
            for (int e = 0; e < 8; e++) tile[lds(v_at(key, 8 * u + e))] = q[e];
        } else {
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo |= (uint32_t)q[e] << (8 * e);
                hi |= (uint32_t)q[4 + e] << (8 * e);
            }
            *(u2v*)(tile + lds(k_at(key, 8 * u))) = u2v{lo, hi};
        }
    }
    __syncthreads();
    const size_t bt = (size_t)head * p.n_blocks + block;
    uint8_t* dst = (is_v ? p.vq : p.kq) + bt * 32 * D;
    for (int i = tid; i < 2 * D; i += kWriteThreads) *(u4*)(dst + 16 * i) = *(const u4*)(tile + lds(16 * i));
    if (tid == 0) (is_v ? p.vs : p.ks)[bt] = scale;
}

// Read-back of one of K and V as f16 rows [len, n_kv, D]: f16(q * scale), the
// tail as it came (a flagged row of V: NaN).  A thread per 8 dims of a row.
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8Read p) {
    const uint32_t n = (uint32_t)p.len * p.n_kv * (D / 8);   // at most 2^16 * 2^10 * 2^5
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
        const int u = (int)(i % (D / 8));
        const int head = (int)(i / (D / 8) % p.n_kv);
        const int pos = (int)(i / (D / 8) / p.n_kv), key = pos & 31, block = pos >> 5;
        h8 y;
        if (block < p.len >> 5) {
            const size_t bt = (size_t)head * p.n_blocks + block;
            const uint8_t* t = p.q + bt * 32 * D;
            const float s = p.s[bt];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int at = p.is_v ? v_at(key, 8 * u + e) : k_at(key, 8 * u + e);
                y[e] = (h16)((float)((int)t[at] - 128) * s);
            }
        } else {
            const size_t th = (size_t)p.tail_cur * p.n_kv + head;
            const uint16_t* t = p.tail + th * 32 * D;
            const bool nan = p.is_v && p.tail_flag[th * 32 + key] != 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int at = p.is_v ? v_at(key, 8 * u + e) : k_at(key, 8 * u + e);
                y[e] = nan ? (h16)NAN : __builtin_bit_cast(h16, t[at]);
            }
        }
        *(h8*)(p.out + (size_t)8 * i) = y;
    }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// The rows of one KV head are (query, head of its group) pairs, row r = s * G
// + g, which see positions up to q_pos0 + s.  A wave takes NQ * 16 rows and
// walks tiles of 32 keys with v_mfma_f32_16x16x32_f16:
//   S^T[key, row] = K Q^T      A = K (16 keys x 32 dims), B = Q^T
//   O^T[d, row]  += V^T P^T    A = V^T (16 dims x 32 keys), B = P^T
// In the first product's result a lane holds, of its row, 8 of the 32 keys;
// these are the 8 keys that it supplies to the second product as B, so the
// probabilities never leave the lane (the V tile's key order sees to it).
//
// Scales: with x_j = scale * log2(e) * ks_b * (q . kq_j), M a running bound of
// x and C a power of two near the blocks' scales of V, the weights
//   w_j = 2^(x_j - M) vs_b / C
// carry V's scale already:  o = C sum_j w_j vq_j / sum_j (w_j C / vs_b).
// M is raised when a row's largest x passes it by more than 8, C moved (and O
// with it, exactly) when a block's scale is not within C / 2 .. 64 C: so the
// f16 operand P = w stays below 2^14, most tiles rescale nothing, and a weight
// loses bits to f16's range only below 2^-13 of the row's largest.  Scores,
// weights, sums and O are f32; P's rounding to f16 (2^-11 relative, for the
// matrix cores) is the only one before the result's.
//
// Bound: a step of one row by reading K and V (65000 keys of 32 heads of 80,
// 333 MB, 62 us: 5.3 TB/s); prompts by the vector work of a score and of the
// unpacking (2048 rows of 32 / 4 heads of 64 31.3 us, 550 TFLOP/s; 700 after
// 5300 of 32 / 8 of 128 91.5 us, 708 TFLOP/s).
constexpr float kLog2e = 1.44269504088896f;
constexpr float kNone = -3.0e38f;   // M before any key

__device__ __forceinline__ float rows4_max(float v) {   // over the lanes l, l ^ 16, l ^ 32, l ^ 48
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// Four bytes q + 128 -> f16 q: the byte under 0x64 is 1024 + q + 128.
__device__ __forceinline__ void bytes_h4(uint32_t w, h2& a, h2& b) {
    const h2 bias = {(h16)-1152.0f, (h16)-1152.0f};
    a = as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + bias;
    b = as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + bias;
}
__device__ __forceinline__ h8 bytes_h8(uint32_t lo, uint32_t hi) {
    h2 a, b, c, d;
    bytes_h4(lo, a, b);
    bytes_h4(hi, c, d);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int D, int NQ>
struct Kv8Wave {
    static constexpr int NC = (D + 31) / 32;   // 32-dim chunks, the last one maybe half
    h8 q[NQ][NC];
    f32x4 o[NQ][2 * NC];
    float M[NQ], l[NQ];   // the same in a row's four lanes
    int pos[NQ];
    int c16, g;
    float sl;             // |scale| * log2(e) (the queries carry its sign)
    uint32_t C;           // the unit of o, a power of two, as the bits of an f32

    static __device__ __forceinline__ bool chunk_ok(int c, int g) { return D % 32 == 0 || c < NC - 1 || g < 2; }
    static __device__ __forceinline__ bool dim_ok(int p, int c16) { return D % 32 == 0 || p < NC - 1 || c16 < 8; }

    __device__ __forceinline__ void init(const Kv8Attn& p, int head, int row0, int rows) {
        const int lane = threadIdx.x & 63;
        c16 = lane & 15;
        g = lane >> 4;
        sl = fabsf(p.scale) * kLog2e;
        C = 0x3F800000u;
        const uint32_t sign = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int r = row0 + 16 * n + c16, rr = r < rows ? r : rows - 1;
            const int s = rr / p.group, hg = rr - s * p.group;
            pos[n] = p.q_pos0 + s;
            const uint16_t* src = p.q + ((size_t)s * p.H + (size_t)head * p.group + hg) * D;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                u4 v = {0, 0, 0, 0};
                if (chunk_ok(c, g)) v = *(const u4*)(src + 32 * c + 8 * g) ^ sign;
                q[n][c] = __builtin_bit_cast(h8, v);
            }
#pragma unroll
            for (int t = 0; t < 2 * NC; t++) o[n][t] = f32x4{0, 0, 0, 0};
            M[n] = kNone;
            l[n] = 0.0f;
        }
    }

    // One tile: kx(c, t) the lane's keys (8 dims of chunk c of key 2 c16 + t),
    // vx(t) its V^T rows; f: the factor of the score; scale: of V.  TAIL: scale
    // 1 = C, and flag(i) of the lane's key i (8g + 2 (i & 3) + (i >> 2)).
    // Per score a maximum (two to an instruction), one fused operation, one
    // exp and half a conversion; the weights' sum comes from the matrix cores
    // (a row of ones), so that it is the sum of the weights as rounded.
    template <bool MASK, bool TAIL, typename KX, typename VX, typename FLAG>
    __device__ __forceinline__ void tile(const KX& kx, const VX& vx, float f, float scale, const FLAG& flag, int key0) {
        f32x4 sc[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; n++) sc[n][0] = sc[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const h8 a = kx(c, t);
#pragma unroll
                for (int n = 0; n < NQ; n++)
                    sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[n][c], sc[n][t], 0, 0, 0);
            }
        auto seen = [&](int n, int i) { return !MASK || key0 + 8 * g + 2 * (i & 3) + (i >> 2) <= pos[n]; };
        float top[NQ];   // the lane's largest exponent
        bool higher = false;
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float m = kNone;
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, seen(n, i) ? sc[n][i >> 2][i & 3] : kNone);
            top[n] = m * f;
            higher |= top[n] > M[n] + 8.0f;
        }
        float ratio = scale * __uint_as_float(0x7F000000u - C), lv = __builtin_amdgcn_logf(ratio), iv = __builtin_amdgcn_rcpf(ratio);
        if constexpr (!TAIL) higher |= !fits(__float_as_uint(scale) >> 23, C);
        if (__any(higher)) {
            if constexpr (!TAIL) {
                const uint32_t e = __builtin_amdgcn_readfirstlane(__float_as_uint(scale)) >> 23;
                if (!fits(e, C)) {
                    // (a block of zeros: any scale; a NaN: for the keys that are seen)
                    if (e - 1 < 254) unit(e << 23);
                    ratio = e - 1 < 254 ? scale * __uint_as_float(0x7F000000u - C) : 1.0f;
                    lv = e == 255 ? NAN : __builtin_amdgcn_logf(ratio);
                    iv = __builtin_amdgcn_rcpf(ratio);
                }
            }
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                const float m = rows4_max(top[n]), mn = m > M[n] + 8.0f ? m : M[n], r = __builtin_amdgcn_exp2f(M[n] - mn);
                M[n] = mn;
                l[n] *= r;
#pragma unroll
                for (int t = 0; t < 2 * NC; t++) o[n][t] *= r;
            }
        }
        h8 pr[NQ];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const float c = TAIL ? -M[n] : lv - M[n];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x = fmaf(sc[n][i >> 2][i & 3], f, TAIL ? flag(i) + c : c);
                pr[n][i] = (h16)__builtin_amdgcn_exp2f(seen(n, i) ? x : -INFINITY);
            }
        }
        const h8 ones = {(h16)1.0f, (h16)1.0f, (h16)1.0f, (h16)1.0f, (h16)1.0f, (h16)1.0f, (h16)1.0f, (h16)1.0f};
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const f32x4 s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pr[n], f32x4{0, 0, 0, 0}, 0, 0, 0);
            l[n] = TAIL ? l[n] + s[0] : fmaf(s[0], iv, l[n]);
        }
#pragma unroll
        for (int t = 0; t < 2 * NC; t++) {
            const h8 a = vx(t);
#pragma unroll
            for (int n = 0; n < NQ; n++) o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pr[n], o[n][t], 0, 0, 0);
        }
    }

    // Whether a scale of exponent bits e lies within C / 2 .. 64 C.
    static __device__ __forceinline__ bool fits(uint32_t e, uint32_t C) { return e - (C >> 23) + 1 <= 6u; }
    // Moves C to another power of two, and o with it.
    __device__ __forceinline__ void unit(uint32_t to) {
        const float r = __uint_as_float(C) * __uint_as_float(0x7F000000u - to);
        C = to;
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int t = 0; t < 2 * NC; t++) o[n][t] *= r;
    }

    // Tiles t0, t0 + step, ... below t1 (tile nfull, if among them, is the
    // tail).  pos0: the first row's position, which sees whole tiles below it.
    __device__ __forceinline__ void walk(const Kv8Attn& p, int head, int t0, int t1, int step, int pos0) {
        const uint8_t* kq = p.kq + (size_t)head * p.n_blocks * 32 * D + (g * 32 + 2 * c16) * 8;
        const uint8_t* vq = p.vq + (size_t)head * p.n_blocks * 32 * D + (c16 * 4 + g) * 16;
        const float* ks = p.ks + (size_t)head * p.n_blocks;
        const float* vs = p.vs + (size_t)head * p.n_blocks;
        const int tq = t1 < p.n_full ? t1 : p.n_full;
        int t = t0;
        u4 kr[NC], vr[NC];
        float fk = 0.0f, fv = 1.0f;
        auto load = [&](int b) {
            const uint8_t* kb = kq + (size_t)b * 32 * D;
            const uint8_t* vb = vq + (size_t)b * 32 * D;
            fk = ks[b];
            fv = vs[b];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                kr[c] = u4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
                vr[c] = kr[c];
                if (chunk_ok(c, g)) kr[c] = *(const u4*)(kb + c * 4 * 32 * 8);
                if (dim_ok(c, c16)) vr[c] = *(const u4*)(vb + c * 16 * 4 * 16);
            }
        };
        auto step_over = [&](auto mask, int b, int next) {
            u4 kc[NC], vc[NC];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                kc[c] = kr[c];
                vc[c] = vr[c];
            }
            const float f = sl * fk;
            const float scale = fv;
            if (next < tq) load(next);
            tile<decltype(mask)::value, false>([&](int c, int h) { return bytes_h8(kc[c][2 * h], kc[c][2 * h + 1]); },
                                               [&](int h) { return bytes_h8(vc[h >> 1][2 * (h & 1)], vc[h >> 1][2 * (h & 1) + 1]); }, f,
                                               scale, [](int) { return 0.0f; }, 32 * b);
        };
        if (t < tq) load(t);
        const int whole = (pos0 + 1) >> 5;   // tiles below it are seen by every row
        for (; t < tq && t < whole; t += step) step_over(std::false_type{}, t, t + step);
        for (; t < tq; t += step) step_over(std::true_type{}, t, t + step);
        unit(0x3F800000u);
        if (t < t1) {   // the tail: f16 values
            const size_t th = (size_t)p.tail_cur * p.n_kv + head;
            const uint16_t* kt = p.tail_k + th * 32 * D;
            const uint16_t* vt = p.tail_v + th * 32 * D;
            const float* fl = p.tail_flag + th * 32 + 8 * g;
            float flag[8];
#pragma unroll
            for (int i = 0; i < 8; i++) flag[i] = fl[2 * (i & 3) + (i >> 2)];
            tile<true, true>(
                [&](int c, int h) {
                    h8 a = {};
                    if (chunk_ok(c, g)) a = *(const h8*)(kt + ((4 * c + g) * 32 + 2 * c16 + h) * 8);
                    return a;
                },
                [&](int h) {
                    h8 a = {};
                    if (dim_ok(h >> 1, c16)) a = *(const h8*)(vt + ((((h >> 1) * 16 + c16) * 4 + g) * 2 + (h & 1)) * 8);
                    return a;
                },
                sl, 1.0f, [&](int i) { return flag[i]; }, 32 * t);
        }
    }

    // dims of o[n][t][i]: 32 (t / 2) + 8 g + 2 i + (t & 1)
    __device__ __forceinline__ void store(const Kv8Attn& p, int head, int row0, int rows) {
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int r = row0 + 16 * n + c16;
            const float inv = 1.0f / l[n];
            if (r >= rows) continue;
            const int s = r / p.group, hg = r - s * p.group;
            uint16_t* dst = p.out + ((size_t)s * p.H + (size_t)head * p.group + hg) * D;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                if (!chunk_ok(c, g)) continue;
                h8 y;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    y[2 * i] = (h16)(o[n][2 * c][i] * inv);
                    y[2 * i + 1] = (h16)(o[n][2 * c + 1][i] * inv);
                }
                *(h8*)(dst + 32 * c + 8 * g) = y;
            }
        }
    }
};

// Many rows: a wave per NQ * 16 rows, four to a workgroup, each over all its
// keys.  Later rows see more keys: the workgroups of a round (those that start
// together, one to a CU) go down from the longest, those of the next round up,
// so that a CU's share is about the same everywhere.
template <int D, int NQ>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv8_attn_rows_kernel(Kv8Attn p) {
    constexpr int ROUND = 256;
    const int rows = p.S * p.group, wgs = gridDim.x;
    int at = blockIdx.x;   // the place in falling order
    if (at / ROUND & 1) {
        const int first = at / ROUND * ROUND, last = (first + ROUND < wgs ? first + ROUND : wgs) - 1;
        at = first + last - at;
    }
    const int head = at % p.n_kv, tile = wgs / p.n_kv - 1 - at / p.n_kv;
    const int row0 = (tile * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * (16 * NQ);
    if (row0 >= rows) return;
    const int row1 = row0 + 16 * NQ < rows ? row0 + 16 * NQ : rows;
    Kv8Wave<D, NQ> w;
    w.init(p, head, row0, rows);
    w.walk(p, head, 0, ((p.q_pos0 + (row1 - 1) / p.group) >> 5) + 1, 1, p.q_pos0 + row0 / p.group);
    w.store(p, head, row0, rows);
}

// The keys of NQ * 16 rows shared by a workgroup's four waves, which join
// through LDS, and with few rows by gridDim's splits, whose sums go to scratch
// for kv8_join_kernel.  Later rows see more keys: they start first.
template <int D, int NQ>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv8_attn_keys_kernel(Kv8Attn p) {
    constexpr int NC = (D + 31) / 32;
    __shared__ float so[4][16 * NQ][NC * 32 + 4];
    __shared__ float sm[4][16 * NQ], sl[4][16 * NQ];
    const int rows = p.S * p.group;
    const int split = blockIdx.x % p.splits, head = blockIdx.x / p.splits % p.n_kv;
    const int row0 = ((rows - 1) / (16 * NQ) - (int)(blockIdx.x / p.splits / p.n_kv)) * (16 * NQ);
    const int row1 = row0 + 16 * NQ < rows ? row0 + 16 * NQ : rows;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Kv8Wave<D, NQ> w;
    w.init(p, head, row0, rows);
    const int tiles = ((p.q_pos0 + (row1 - 1) / p.group) >> 5) + 1;
    w.walk(p, head, split * 4 + wave, tiles, 4 * p.splits, p.q_pos0 + row0 / p.group);
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r = 16 * n + w.c16;
        if (w.g == 0) {
            sm[wave][r] = w.M[n];
            sl[wave][r] = w.l[n];
        }
        if (row0 + r >= rows) continue;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                so[wave][r][32 * c + 8 * w.g + 2 * i] = w.o[n][2 * c][i];
                so[wave][r][32 * c + 8 * w.g + 2 * i + 1] = w.o[n][2 * c + 1][i];
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NQ * (D / 4); i += 256) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        if (row0 + r >= rows) continue;
        float M = sm[0][r];
#pragma unroll
        for (int k = 1; k < 4; k++) M = fmaxf(M, sm[k][r]);
        float l = 0.0f;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = __builtin_amdgcn_exp2f(sm[k][r] - M);
            l = fmaf(sl[k][r], f, l);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(so[k][r][d + j], f, o[j]);
        }
        const int row = row0 + r;
        if (p.splits == 1) {
            const int s = row / p.group, hg = row - s * p.group;
            uint16_t* dst = p.out + ((size_t)s * p.H + (size_t)head * p.group + hg) * D + d;
            const float inv = 1.0f / l;
#pragma unroll
            for (int j = 0; j < 4; j++) dst[j] = f2h(o[j] * inv);
        } else {   // [head][row][split]: D sums, then M and l
            float* dst = p.scratch + (((size_t)head * rows + row) * p.splits + split) * (D + 4);
            *(f32x4*)(dst + d) = o;
            if (d == 0) {
                dst[D] = M;
                dst[D + 1] = l;
            }
        }
    }
}

// The splits of one (head, row) joined by a workgroup: a thread loads 4 dims of
// one split at a time, all splits' loads in flight together, and the threads
// of the same dims add up in a fixed order through LDS.
template <int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8Attn p) {
    constexpr int Q = D / 4, PER = 256 / Q;   // threads of a split, splits at a time
    __shared__ f32x4 so[256];
    __shared__ float sl[PER];
    const int rows = p.S * p.group;
    const int row = blockIdx.x % rows, head = blockIdx.x / rows;
    const float* src = p.scratch + ((size_t)head * rows + row) * p.splits * (D + 4);
    float M = kNone;
    for (int k = threadIdx.x & 63; k < p.splits; k += 64) M = fmaxf(M, src[(size_t)k * (D + 4) + D]);
    const int part = threadIdx.x / Q, d = threadIdx.x % Q;
    f32x4 o = {0, 0, 0, 0};
    float l = 0.0f;
    constexpr int AHEAD = 4;
    for (int k0 = 0; k0 < p.splits; k0 += AHEAD * PER) {
        f32x4 x[AHEAD], ml[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int k = k0 + a * PER + part;
            const float* at = src + (size_t)(k < p.splits ? k : 0) * (D + 4);
            x[a] = *(const f32x4*)(at + 4 * d);
            ml[a] = *(const f32x4*)(at + D);
        }
        if (k0 == 0) M = wave_max(M);
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            if (part >= PER || k0 + a * PER + part >= p.splits) continue;
            const float f = __builtin_amdgcn_exp2f(ml[a][0] - M);
            l = fmaf(ml[a][1], f, l);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(x[a][j], f, o[j]);
        }
    }
    so[threadIdx.x] = o;
    if (d == 0 && part < PER) sl[part] = l;
    __syncthreads();
    if (threadIdx.x >= Q) return;
    for (int k = 1; k < PER; k++) {
        o += so[k * Q + threadIdx.x];
        l += sl[k];
    }
    const int s = row / p.group, hg = row - s * p.group;
    uint16_t* dst = p.out + ((size_t)s * p.H + (size_t)head * p.group + hg) * D + 4 * threadIdx.x;
    const float inv = 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; j++) dst[j] = f2h(o[j] * inv);
}

template <int D>
tlhip_status attn_d(hipStream_t s, Kv8Attn p, const Kv8Plan& pl) {
    const int rows = p.S * p.group;
    if constexpr (D > 64)
        if (pl.splits == 0) {
            constexpr int NQ = D == 256 ? 1 : 2;
            kv8_attn_rows_kernel<D, NQ><<<(rows + 64 * NQ - 1) / (64 * NQ) * p.n_kv, 256, 0, s>>>(p);
            return TLHIP_OK;
        }
    p.splits = pl.splits;
    const int wg = (rows + 16 * pl.nq - 1) / (16 * pl.nq) * p.n_kv * pl.splits;
    if constexpr (D <= 128)
        if (pl.nq == 2) kv8_attn_keys_kernel<D, 2><<<wg, 256, 0, s>>>(p);
    if constexpr (D <= 64)
        if (pl.nq == 4) kv8_attn_keys_kernel<D, 4><<<wg, 256, 0, s>>>(p);
    if (pl.nq == 1) kv8_attn_keys_kernel<D, 1><<<wg, 256, 0, s>>>(p);
    if (pl.splits > 1) kv8_join_kernel<D><<<rows * p.n_kv, 256, 0, s>>>(p);
    return TLHIP_OK;
}

}  // namespace

bool kv8_head_dim_ok(int D) { return D == 32 || D == 64 || D == 80 || D == 96 || D == 128 || D == 256; }

#define KV8_DISPATCH(D, CALL)                                        \
    switch (D) {                                                     \
        case 32: CALL(32); break;                                    \
        case 64: CALL(64); break;                                    \
        case 80: CALL(80); break;                                    \
        case 96: CALL(96); break;                                    \
        case 128: CALL(128); break;                                  \
        case 256: CALL(256); break;                                  \
        default: return fail(TLHIP_ERR_INVALID_DIMENSION, "8-bit cache: head_dim %d", D); \
    }

tlhip_status launch_kv8_write(hipStream_t s, const Kv8Write& p) {
    const int end = p.len0 + p.S;
    const int units = p.n_full + ((end & 31) ? 1 : 0);
    if (units == 0 || p.S == 0) return TLHIP_OK;
    const dim3 grid((unsigned)(units >= 8 ? (units + 7) / 8 * 8 : units) * p.n_kv * 2);
#define CALL(D) kv8_write_kernel<D><<<grid, kWriteThreads, 0, s>>>(p)
    KV8_DISPATCH(p.D, CALL)
#undef CALL
    return TLHIP_OK;
}

tlhip_status launch_kv8_read(hipStream_t s, const Kv8Read& p) {
    const int64_t n = (int64_t)p.len * p.n_kv * (p.D / 8);
    const int64_t wg = (n + 255) / 256;
    const dim3 grid((unsigned)(wg < 65536 ? wg : 65536));
#define CALL(D) kv8_read_kernel<D><<<grid, 256, 0, s>>>(p)
    KV8_DISPATCH(p.D, CALL)
#undef CALL
    return TLHIP_OK;
}

// How a call is spread over the device (figures: calls on three caches in
// turn, from Python).  A wave takes two columns of 16 rows
// when there are more rows than one has (a tile is unpacked once for both: 700
// rows after 5300, 32 / 8 heads of 128, 104 us against 167 with one), four up
// to head dim 64 if they still make 1024 workgroups (2048 rows of 32 / 4 heads
// of 64 36.5 us against 41.3 with two, after 4000 116 against 137; 1024 rows,
// 512 workgroups, 16.1 against 14.6), one at head dim 256, whose sums fill the
// registers.  From 2048 workgroups of shared keys on, past head dim 64, a wave
// walks all keys of its own instead, and the waves of a workgroup meet in its
// CU's cache (splits = 0: 2048 rows of 32 / 8 heads of 128 62 us against 72);
// else the four waves share them (1024 rows of 32 heads of 80: 20 us against
// 28; up to head dim 64 the two measure the same, 41 us); and below
// 512 workgroups the keys are cut into splits, up to two workgroups a CU, four
// tiles each at least.  (Up to four a CU: 300 rows after 3000, 32 / 4 heads of
// 64, 35 us against 25, one row after 20000, 32 / 8 of 128, 17.4 against 13.9;
// up to one: 12.2 there, but 65000 keys of 32 heads of 80 67.7 against 64.5.)
// Up to 1024 keys (512 for two columns or head dim 256) are not split: a step
// at 400 keys, 32 / 4 heads of 64, 5.7 us against 8.7 with the join's launch, at
// 900 6.4 against 10.1; 1900 of 32 heads of 80 would take 11.6 against 8.7.
Kv8Plan kv8_plan(int S, int group, int n_kv, int D, int len) {
    Kv8Plan pl;
    const int64_t rows = (int64_t)S * group;
    const int tiles = (len + 31) / 32;
    pl.nq = rows <= 16 || D > 128 ? 1 : D <= 64 && rows * n_kv >= 1024 * 64 ? 4 : 2;
    const int64_t wg = (rows + 16 * pl.nq - 1) / (16 * pl.nq) * n_kv;
    if (D > 64 && wg >= 2048) return pl;
    int64_t splits = tiles * pl.nq * (D > 128 ? 2 : 1) <= 32 ? 1 : 512 / wg;
    if (splits < 1) splits = 1;
    if (splits > (tiles + 3) / 4) splits = (tiles + 3) / 4;
    pl.splits = (int)splits;
    pl.scratch_bytes = splits > 1 ? (size_t)n_kv * rows * splits * (D + 4) * sizeof(float) : 0;
    return pl;
}

tlhip_status launch_kv8_attention(hipStream_t s, const Kv8Attn& p, const Kv8Plan& pl) {
#define CALL(D) return attn_d<D>(s, p, pl)
    KV8_DISPATCH(p.D, CALL)
#undef CALL
    return TLHIP_OK;
}

}  // namespace tlhip
