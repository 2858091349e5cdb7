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
// One token of 8 Q4_0 experts 2048 x 5632, two chosen: 20.5 us a call (router
// 3.6, gate and up 8 to 10, down 7 to 8); 13 tokens, Q8_0: 74 us (gate and up
// 41, 4.7 TB/s; down 26; router and sum 4 each).
//
// Four launches: the router (a workgroup per token); gate and up; down; the
// sum over a token's experts (three for one token and for a few, whose down
// sums them itself).  What bounds the middle two is reading the weights of the
// experts that some token chose, so each is read once: a wave takes 16 rows of one
// expert (of gate and of up both) and multiplies by all of that expert's
// tokens on the matrix cores (v_mfma_f32_16x16x32_f16, A = 16 weight rows x 32
// k, B = 32 k x 16 columns; unused columns cost nothing that is scarce).
//
// The weights go through LDS, copied there directly (no registers) in slots
// of 16 rows x 128 bytes (f16: 256): whole cache lines, where A's own layout
// asks for 64 bytes of each of 16 rows at a time.  Through registers in that
// layout, and with the 2-byte scales gathered one by one, 13 Q8_0 tokens' gate
// and up of 5632 x 2048 took 55 us (3.5 TB/s) without any arithmetic.  A tile's
// scales lie together and are copied whole.  Each wave has its own ring of
// slots, so its stream of loads waits for no other.
//
// The product after the activation takes h, f32, as two f16 columns, h 2^-e =
// hi + lo, with the power of two that puts the token's largest |h| just below
// 2^15: 22 bits of every h, and none lost to the range of f16.
#include <cmath>
#include <type_traits>

#include "device_common.hpp"
#include "internal.hpp"

namespace tlhip {

namespace {

constexpr int kTokens = 256;               // tokens of one round of launches (moe.cpp)
// Waves of a workgroup of the products, slots of weights that a wave has in
// flight, and the columns staged in LDS at a time (or one round of slots, if
// that is more): two workgroups fit on a CU with rows of 5632.  (Deeper rings
// and, for gate and up, more columns or waves measured the same or less.)
// Down's columns are f32, to be split in two, so with several tokens to an
// expert eight waves share them: 13 tokens of 8 Q8_0 experts 2048 x 5632, two
// each, 27 us against 33, 30 tokens of 4096 x 5632 12 us less; five tokens of
// 64 experts, six each, are 5 us faster with four.
constexpr int kRing = 2;
constexpr int kWaves = 4, kColumnBytes = 24 << 10;
constexpr int kDownWaves = 8, kDownColumnBytes = 48 << 10;

// ---------------------------------------------------------------------------
// router
// ---------------------------------------------------------------------------
// The wave's maximum without the LDS round trips of a shuffle.
__device__ __forceinline__ float wave_max_u(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    v = fmaxf(v, dpp_f<0x140>(v));
    const int b = __float_as_int(v);
    return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(b, 0)), __int_as_float(__builtin_amdgcn_readlane(b, 16))),
                 fmaxf(__int_as_float(__builtin_amdgcn_readlane(b, 32)), __int_as_float(__builtin_amdgcn_readlane(b, 48))));
}

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
    // U tasks t0, t0 + 16, ... at once, their loads in flight together (E = 32,
    // K = 1024: 4.0 us with two, 5.0 with one after the other)
    auto tasks = [&](auto at_once, int t0) {
        constexpr int U = decltype(at_once)::value;
        const int k0 = t0 % P * share, have = share < pieces - k0 ? share : pieces - k0;   // (U > 1: P = 1)
        const uint16_t* r[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            r[u] = a.router + (size_t)((t0 + 16 * u) / P) * a.K + 8 * k0;
            s[u] = 0.0f;
        }
#pragma unroll 4 / U
        for (int k = lane; k < have; k += 64) {
            const u4 xv = *(const u4*)(x + 8 * (k0 + k));
            u4 rv[U];
#pragma unroll
            for (int u = 0; u < U; u++) rv[u] = *(const u4*)(r[u] + 8 * k);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const h2 p = as_h2(xv[i]), q = as_h2(rv[u][i]);
                    s[u] = fmaf((float)p[0], (float)q[0], s[u]);
                    s[u] = fmaf((float)p[1], (float)q[1], s[u]);
                }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            s[u] = wave_sum<64>(s[u]);
            if (lane == 0) (P == 1 ? lg : part)[t0 + 16 * u] = s[u];
        }
    };
    int t0 = wave;
    if (P == 1) {
        for (; t0 + 48 < a.E; t0 += 64) tasks(std::integral_constant<int, 4>{}, t0);
        for (; t0 + 16 < a.E; t0 += 32) tasks(std::integral_constant<int, 2>{}, t0);
    }
    for (; t0 < a.E * P; t0 += 16) tasks(std::integral_constant<int, 1>{}, t0);
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
    big = wave_max_u(big);
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
        top = wave_max_u(top);
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
// A slot: RB bytes of each of 16 rows, STEPS steps of four blocks of 32.  The
// 16-byte piece at place q of a row is the row's piece q ^ swizzle(row): the 16
// rows' reads of one piece then take 16 different places of the 256 bytes that
// LDS gives in a cycle.
template <int WT>
struct Slot {
    static constexpr int RB = WT == TLHIP_F16 ? 256 : 128, NP = RB / 16, BYTES = 16 * RB, COPIES = BYTES / 1024;
    static constexpr int STEPS = WT == TLHIP_Q4_0 ? 2 : 1, BLOCKS = 4 * STEPS;
    static constexpr int BLOCK_BYTES = WT == TLHIP_Q4_0 ? 16 : WT == TLHIP_Q8_0 ? 32 : 64;
    static __device__ __forceinline__ int swizzle(int row) { return NP == 8 ? row >> 1 & 7 : row; }
};

// One lane's weights of one step: a block (Q4_0), half of each of two (Q8_0) or
// a quarter of each of four (f16).  sub(j) is its part of A in the j-th of the
// step's four matrix instructions.
template <int WT>
struct Weights;
template <>
struct Weights<TLHIP_Q4_0> {
    u4 q;
    uint32_t d;
    __device__ __forceinline__ void read(const uint8_t* slot, const uint16_t* d16, int row, int nb, int block0, int u, int g) {
        q = *(const u4*)(slot + row * 128 + ((4 * u + g) ^ Slot<TLHIP_Q4_0>::swizzle(row)) * 16);
        const int b = block0 + 4 * u + g;
        d = d16[row * nb + (b < nb ? b : nb - 1)];
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
    uint32_t d[2];
    __device__ __forceinline__ void read(const uint8_t* slot, const uint16_t* d16, int row, int nb, int block0, int, int g) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            q[i] = *(const u4*)(slot + row * 128 + ((4 * i + g) ^ Slot<TLHIP_Q8_0>::swizzle(row)) * 16);
            const int b = block0 + 2 * i + (g >> 1);
            d[i] = d16[row * nb + (b < nb ? b : nb - 1)];
        }
    }
    __device__ __forceinline__ h8 sub(int j) const {
        h2 lo[2], hi[2];
        const h2 dd = as_h2(d[j >> 1] | d[j >> 1] << 16);
        q8_unpack(q[j >> 1][2 * (j & 1)], dd, lo);
        q8_unpack(q[j >> 1][2 * (j & 1) + 1], dd, hi);
        return h8{lo[0][0], lo[0][1], lo[1][0], lo[1][1], hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
    }
};
template <>
struct Weights<TLHIP_F16> {
    u4 q[4];
    __device__ __forceinline__ void read(const uint8_t* slot, const uint16_t*, int row, int, int, int, int g) {
#pragma unroll
        for (int j = 0; j < 4; j++) q[j] = *(const u4*)(slot + row * 256 + ((4 * j + g) ^ row) * 16);
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
__device__ __forceinline__ int piece_block(int j, int g) {
    return WT == TLHIP_F16 ? j : WT == TLHIP_Q8_0 ? 2 * (j >> 1) + (g >> 1) : g;
}
template <int WT>
__device__ __forceinline__ int piece_sub(int j, int g) {
    return WT == TLHIP_F16 ? g : WT == TLHIP_Q8_0 ? 2 * (g & 1) + (j & 1) : j;
}

typedef h16 h4 __attribute__((ext_vector_type(4)));

// 16 weight rows whose slots a wave copies to LDS.
template <int WT>
struct Rows {
    using S = Slot<WT>;
    __amdgpu_buffer_rsrc_t q;
    int row_bytes;
    __device__ __forceinline__ Rows(const void* w, size_t row, int nb)
        : q(sk_rsrc((const uint8_t*)w + row * nb * S::BLOCK_BYTES, 16u * nb * S::BLOCK_BYTES)), row_bytes(nb * S::BLOCK_BYTES) {}
    // Slot n to LDS address `lds`.  Pieces past the row's end repeat its last
    // one: their columns are zero.
    __device__ __forceinline__ void copy(int n, uint32_t lds) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < S::COPIES; i++) {
            const int at = i * 64 + lane, row = at / S::NP, byte = n * S::RB + ((at % S::NP) ^ S::swizzle(row)) * 16;
            sk_dma<16>(q, lds + i * 1024, row * row_bytes + (byte < row_bytes ? byte : row_bytes - 16));
        }
    }
};

__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(gl_lds_t)p; }
// This wave's LDS reads are done (their memory may be copied over).
__device__ __forceinline__ void lds_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The scales of 16 rows (nb of each row, which lie together: 2 nb pieces of 16
// bytes) to LDS, copies part, part + parts, ... of 1 KB.  The last copy repeats
// the last piece: room in LDS is in whole KB.
__host__ __device__ constexpr int scale_bytes(int nb) { return (32 * nb + 1023) / 1024 * 1024; }
__device__ __forceinline__ void copy_scales(uint32_t lds, const uint16_t* d, size_t row, int nb, int part, int parts) {
    const __amdgpu_buffer_rsrc_t r = sk_rsrc(d + row * nb, 32u * nb);
    for (int i = part; i * 64 < 2 * nb; i += parts) {
        const int at = i * 64 + (int)(threadIdx.x & 63);
        sk_dma<16>(r, lds + i * 1024, (at < 2 * nb ? at : 2 * nb - 1) * 16);
    }
}

// What a workgroup holds in LDS before its dynamic part, which is: columns,
// rings, scales.
struct MoeShared {
    int list[kTokens];      // the expert's (token, choice) pairs
    float g[kTokens];       // their weights
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
        if (is) {
            const int at = have + __builtin_popcountll(who & ((1ull << lane) - 1));
            sh.list[at] = p + lane;
            sh.g[at] = a.g[p + lane];
        }
        have += __builtin_popcountll(who);
    }
    if (lane == 0) sh.count = have;
}

// The expert of a workgroup's slot, with sh.list and sh.count filled; -1:
// nothing to do.  With fewer (token, choice) pairs than experts a slot is a
// pair, and only the first pair of an expert works on it; else an expert.
__device__ __forceinline__ int slot_expert(const MoeArgs& a, int slot, MoeShared& sh) {
    const bool by_pair = a.M * a.top < a.E;
    const int e = by_pair ? a.ids[slot] : slot;
    if (threadIdx.x < 64) find_tokens(a, e, sh);
    __syncthreads();
    return by_pair && sh.list[0] != slot ? -1 : e;
}

// The columns of a product.  Column c of piece s of block b is 16 bytes at
// (4 b + s) * ncol + c; past the row's nb blocks they are zeros.  A thread
// asks for the first kPieces of a chunk's pieces (fetch) while the chunk
// before is multiplied, and stores them and the rest (put) after it.
constexpr int kPieces = 4;
__device__ __forceinline__ f4 low_part(const f4& p) {
    f4 r;
#pragma unroll
    for (int k = 0; k < 4; k++) r[k] = p[k] - (float)(h16)p[k];
    return r;
}
template <typename LOADER, int NW>
struct Stage : LOADER {
    struct Ahead {
        typename LOADER::Run p[kPieces], q[kPieces];
    };
    // pieces i0 + k * (threads of the workgroup)
    __device__ __forceinline__ void load(Ahead& v, int i0, int c0, int blocks, int nb) const {
        const uint32_t by_nt = 0xFFFFFFFFu / this->nt + 1;   // i / nt = umulhi(i, by_nt): i nt < 2^32
#pragma unroll
        for (int k = 0; k < kPieces; k++) {
            const int i = i0 + k * NW * 64, bs = this->nt == 1 ? i : (int)__umulhi(i, by_nt), t = i - bs * this->nt, b = c0 + (bs >> 2);
            v.p[k] = v.q[k] = typename LOADER::Run{};
            if (i < blocks * 4 * this->nt && b < nb) this->get(v.p[k], v.q[k], t, b, bs & 3);
        }
    }
    __device__ __forceinline__ void store(const Ahead& v, int i0, h8* cols, int blocks) const {
#pragma unroll
        for (int k = 0; k < kPieces; k++)
            if (i0 + k * NW * 64 < blocks * 4 * this->nt) this->set(v.p[k], v.q[k], cols, i0 + k * NW * 64);
    }
    __device__ __forceinline__ void fetch(Ahead& v, int c0, int blocks, int nb) const { load(v, threadIdx.x, c0, blocks, nb); }
    __device__ __forceinline__ void put(Ahead& v, h8* cols, int c0, int blocks, int nb) const {
        store(v, threadIdx.x, cols, blocks);
        for (int i0 = threadIdx.x + kPieces * NW * 64; i0 < blocks * 4 * this->nt; i0 += kPieces * NW * 64) {
            load(v, i0, c0, blocks, nb);
            store(v, i0, cols, blocks);
        }
    }
};
// Gate and up: x of the tokens list[0 .. nt), or of the only token.
template <int WT, bool ONE>
struct LoadX {
    typedef h4 Run;
    const MoeArgs& a;
    const int* list;
    int nt;
    __device__ __forceinline__ int ncol() const { return nt; }
    __device__ __forceinline__ void get(h4& p, h4& q, int t, int b, int s) const {
        const uint16_t* x = a.x + (ONE ? 0 : (size_t)(list[t] / a.top) * a.K) + b * 32;
        p = *(const h4*)(x + run0<WT>(s));
        q = *(const h4*)(x + run1<WT>(s));
    }
    __device__ __forceinline__ void set(const h4& p, const h4& q, h8* cols, int i) const { cols[i] = piece<WT>(p, q); }
};
// Down: hi and lo of each token's h 2^-e, one after the other.
template <int WT>
struct LoadH {
    typedef f4 Run;
    const MoeArgs& a;
    const int* list;
    int nt;
    const float* scale;
    __device__ __forceinline__ int ncol() const { return 2 * nt; }
    __device__ __forceinline__ void get(f4& p, f4& q, int t, int b, int s) const {
        const float* h = a.h + (size_t)list[t] * a.I + b * 32;
        p = *(const f4*)(h + run0<WT>(s)) * scale[t];
        q = *(const f4*)(h + run1<WT>(s)) * scale[t];
    }
    __device__ __forceinline__ void set(const f4& p, const f4& q, h8* cols, int i) const {
        cols[2 * i] = piece<WT>(p, q);
        cols[2 * i + 1] = piece<WT>(low_part(p), low_part(q));
    }
};

// Where the dynamic part of LDS holds what, for a product of nb blocks with
// NR matrices, tiles_wg tiles in a workgroup.
struct Layout {
    int column_bytes, ring_at, scales_at, bytes;
};
template <int WT, int NR, int KS, int NW>
__host__ __device__ inline Layout layout(int nb, int max_cols) {
    constexpr int round = Slot<WT>::BLOCKS * KS;
    Layout l;
    const int whole = (nb + round - 1) / round * round * 64 * max_cols, least = round * 64 * max_cols;
    constexpr int want = NW == kWaves ? kColumnBytes : kDownColumnBytes;
    l.column_bytes = whole < want ? whole : want > least ? want : least;
    l.ring_at = l.column_bytes;
    l.scales_at = l.ring_at + NW * NR * kRing * Slot<WT>::BYTES;
    l.bytes = l.scales_at + (WT == TLHIP_F16 ? 0 : NW / KS * NR * scale_bytes(nb));
    constexpr int red = NW * 4 * 64 * 16;   // the waves' sums, in place of columns and ring at the end
    if (KS > 1 && l.bytes < red) l.bytes = red;
    return l;
}

// acc[r][c] = W_r (16 rows, nb blocks) times the CT * 16 columns that stage()
// lays out chunk by chunk, k shared out over KS waves.  Complete in the first
// of them: lane (c16, g) has rows 4g .. 4g + 3 of column c16.
template <int WT, int NR, int CT, int KS, bool ONE, typename STAGE>
__device__ __forceinline__ void multiply(const Rows<WT> (&w)[NR], const uint16_t* const (&wd)[NR], size_t row, int nb, const STAGE& stage,
                                         const Layout& at, uint8_t* lds, MoeShared& sh, f4 (&acc)[NR][CT]) {
    using S = Slot<WT>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % KS;
    const int c16 = lane & 15, g = lane >> 4, ncol = stage.ncol();
    constexpr int ROUND = S::BLOCKS * KS;
    int chunk = at.column_bytes / (64 * ncol) / ROUND * ROUND;   // blocks of a chunk: whole rounds of the KS waves' slots
    const int all = (nb + ROUND - 1) / ROUND * ROUND;
    if (chunk > all) chunk = all;
    h8* cols = (h8*)lds;
    const uint8_t* ring = lds + at.ring_at + wave * (NR * kRing * S::BYTES);
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_address(ring));
    const uint8_t* scales = lds + at.scales_at + wave / KS * (NR * scale_bytes(nb));
    int col[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) col[c] = 16 * c + c16 < ncol ? 16 * c + c16 : ncol - 1;
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int c = 0; c < CT; c++) acc[r][c] = f4{0, 0, 0, 0};
    const int slots = (nb + S::BLOCKS - 1) / S::BLOCKS;
    auto copy = [&](int n, int k) {   // slot n to ring place k
#pragma unroll
        for (int r = 0; r < NR; r++) w[r].copy(n, ring_lds + (k * NR + r) * S::BYTES);
    };
    // Loads return in order: the columns are asked for before the copies.  One
    // token's do not even wait for the router's choice, which the copies do.
    typename STAGE::Ahead ahead;
    stage.fetch(ahead, 0, chunk, nb);
    if constexpr (ONE) stage.put(ahead, cols, 0, chunk, nb);
    if constexpr (WT != TLHIP_F16) {
        const uint32_t scales_lds = __builtin_amdgcn_readfirstlane(lds_address(scales));
#pragma unroll
        for (int r = 0; r < NR; r++) copy_scales(scales_lds + r * scale_bytes(nb), wd[r], row, nb, part, KS);
    }
    int next = part, place = 0;   // the next slot to copy
#pragma unroll
    for (int k = 0; k < kRing; k++, next += KS)
        if (next < slots) copy(next, k);
    auto scales_landed = [&]() {   // (their copies are older than the slots')
        if (next <= slots - 1 + KS) sk_wait_vm<kRing * NR * S::COPIES>();
        else sk_wait_vm<0>();
    };
    if constexpr (ONE) scales_landed();
    for (int c0 = 0; c0 < all; c0 += chunk) {
        const int blocks = all - c0 < chunk ? all - c0 : chunk;
        if (!ONE || c0) {
            lds_barrier();
            stage.put(ahead, cols, c0, blocks, nb);
            if (c0 == 0) scales_landed();
        }
        lds_barrier();
        if (c0 + chunk < all) stage.fetch(ahead, c0 + chunk, min(all - c0 - chunk, chunk), nb);
        const int end = min((c0 + blocks) / S::BLOCKS, slots);
        for (int n = c0 / S::BLOCKS + part; n < end; n += KS) {
            // the slot has landed when no more copies are in flight than the
            // kRing - 1 later slots'
            if (next > n + (kRing - 1) * KS) sk_wait_vm<(kRing - 1) * NR * S::COPIES>();
            else sk_wait_vm<0>();
            Weights<WT> a[NR][S::STEPS];
            const uint8_t* slot = ring + place * (NR * S::BYTES);
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int u = 0; u < S::STEPS; u++) a[r][u].read(slot + r * S::BYTES, (const uint16_t*)(scales + r * scale_bytes(nb)), c16, nb, n * S::BLOCKS, u, g);
            if (next < slots) {
                lds_reads_done();
                copy(next, place);
                next += KS;
            }
            place = place + 1 == kRing ? 0 : place + 1;
#pragma unroll
            for (int u = 0; u < S::STEPS; u++) {
                h8 x[4][CT];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int b = n * S::BLOCKS - c0 + 4 * u + piece_block<WT>(j, g);
#pragma unroll
                    for (int c = 0; c < CT; c++) x[j][c] = cols[(b * 4 + piece_sub<WT>(j, g)) * ncol + col[c]];
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        const h8 wv = a[r][u].sub(j);
#pragma unroll
                        for (int c = 0; c < CT; c++) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv, x[j][c], acc[r][c], 0, 0, 0);
                    }
            }
        }
    }
    if constexpr (KS > 1) {
        f4* red = (f4*)lds;
        lds_barrier();
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int c = 0; c < CT; c++) red[((wave * NR + r) * CT + c) * 64 + lane] = acc[r][c];
        lds_barrier();
        if (part == 0)
#pragma unroll
            for (int k = 1; k < KS; k++)
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int c = 0; c < CT; c++) acc[r][c] += red[(((wave + k) * NR + r) * CT + c) * 64 + lane];
    }
}

// Gate and up of 16 rows of one expert, for tokens list[t0 .. t0 + nt).
template <int WT, int CT, int KS, bool ONE>
__device__ __forceinline__ void gate_up_tile(const MoeArgs& a, int e, int tile, int t0, int nt, const Layout& at, uint8_t* lds,
                                             MoeShared& sh, int one_pair = 0) {
    f4 acc[2][CT];
    const Stage<LoadX<WT, ONE>, kWaves> stage{{a, sh.list + t0, nt}};
    const int tiles = a.I / 16, nb = a.K / 32;
    // (a wave past the last tile computes that one and stores nothing)
    const size_t row = (size_t)e * a.I + 16 * (tile < tiles ? tile : tiles - 1);
    const Rows<WT> w[2] = {Rows<WT>(a.gate, row, nb), Rows<WT>(a.up, row, nb)};
    const uint16_t* const wd[2] = {a.gate_d, a.up_d};
    multiply<WT, 2, CT, KS, ONE>(w, wd, row, nb, stage, at, lds, sh, acc);
    const int lane = threadIdx.x & 63, c16 = lane & 15, g = lane >> 4;
    if ((threadIdx.x >> 6) % KS || tile >= tiles) return;
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int t = 16 * c + c16 < nt ? 16 * c + c16 : nt - 1, pair = ONE ? one_pair : sh.list[t0 + t];
        const float gw = ONE ? a.g[one_pair] : sh.g[t0 + t];
        f4 h;
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float gt = acc[0][c][i];
            h[i] = gw * (gt / (1.0f + __expf(-gt)) * acc[1][c][i]);
            m = fmaxf(m, fabsf(h[i]) <= 3.4028235e38f ? fabsf(h[i]) : INFINITY);   // (a NaN counts as an infinity)
        }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (16 * c + c16 >= nt) continue;
        *(f4*)(a.h + (size_t)pair * a.I + 16 * tile + 4 * g) = h;
        if (g == 0) a.hmax[(size_t)pair * tiles + tile] = m;   // the tile's largest |h|
    }
}

template <int WT, int KS, int CT, bool ONE>
__global__ __launch_bounds__(kWaves * 64) void moe_gate_up_kernel(MoeArgs a, Layout at) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ MoeShared sh;
    constexpr int TW = kWaves / KS;   // tiles of a workgroup
    const int groups = (a.I / 16 + TW - 1) / TW;
    const int tile = (int)(blockIdx.x % groups) * TW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / KS;
    const int slot = blockIdx.x / groups;
    if constexpr (ONE) {   // a slot is one of the token's choices, each of another expert
        gate_up_tile<WT, 1, KS, true>(a, a.ids[slot], tile, 0, 1, at, lds, sh, slot);
        return;
    }
    const int e = __builtin_amdgcn_readfirstlane(slot_expert(a, slot, sh));
    if (e < 0) return;
    const int count = sh.count;
    for (int t0 = 0; t0 < count; t0 += 16 * CT) {
        const int nt = count - t0 < 16 * CT ? count - t0 : 16 * CT;
        if (CT == 1 || nt <= 16) gate_up_tile<WT, 1, KS, ONE>(a, e, tile, t0, nt, at, lds, sh);
        else gate_up_tile<WT, CT, KS, ONE>(a, e, tile, t0, nt, at, lds, sh);
        __syncthreads();
    }
}

// 2^-e with m 2^-e in [2^14, 2^15); 1 for zeros and the non-finite.
__device__ __forceinline__ float scale_for(float m) {
    return m > 0.0f && m < INFINITY ? ldexpf(1.0f, min(14 - ilogbf(m), 126)) : 1.0f;
}

// Down: 16 rows of one expert; the columns are the hi and lo parts of each
// token's h, one after the other.
template <int WT, int CT, int KS, int NW>
__device__ __forceinline__ void down_tile(const MoeArgs& a, int e, int tile, int t0, int nt, const Layout& at, uint8_t* lds, MoeShared& sh) {
    f4 acc[1][CT];
    const Stage<LoadH<WT>, NW> stage{{a, sh.list + t0, nt, sh.scale + t0}};
    const int tiles = a.K / 16, nb = a.I / 32;
    const size_t row = (size_t)e * a.K + 16 * (tile < tiles ? tile : tiles - 1);
    const Rows<WT> w[1] = {Rows<WT>(a.down, row, nb)};
    const uint16_t* const wd[1] = {a.down_d};
    multiply<WT, 1, CT, KS, false>(w, wd, row, nb, stage, at, lds, sh, acc);
    const int lane = threadIdx.x & 63, c16 = lane & 15, g = lane >> 4;
    if ((threadIdx.x >> 6) % KS || tile >= tiles) return;
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int t = 8 * c + (c16 >> 1);
        f4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = acc[0][c][i] + dpp_f<0xB1>(acc[0][c][i]);   // hi + lo
        if (t >= nt || (c16 & 1)) continue;
        const float f = 1.0f / sh.scale[t0 + t];
        *(f4*)(a.part + (size_t)sh.list[t0 + t] * a.K + 16 * tile + 4 * g) = v * f;
    }
}

template <int WT, int KS, int CT, int NW>
__global__ __launch_bounds__(NW * 64) void moe_down_kernel(MoeArgs a, Layout at) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ MoeShared sh;
    constexpr int TW = NW / KS;
    const int groups = (a.K / 16 + TW - 1) / TW;
    const int tile = (int)(blockIdx.x % groups) * TW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / KS;
    const int e = __builtin_amdgcn_readfirstlane(slot_expert(a, blockIdx.x / groups, sh));
    if (e < 0) return;
    const int count = sh.count, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int t = wave; t < count; t += NW) {
        const float* hm = a.hmax + (size_t)sh.list[t] * (a.I / 16);
        float m = 0.0f;
        for (int i = lane; i < a.I / 16; i += 64) m = fmaxf(m, hm[i]);
        m = wave_max(m);
        if (lane == 0) sh.scale[t] = scale_for(m);
    }
    __syncthreads();
    for (int t0 = 0; t0 < count; t0 += 8 * CT) {
        const int nt = count - t0 < 8 * CT ? count - t0 : 8 * CT;
        if (CT == 1 || nt <= 8) down_tile<WT, 1, KS, NW>(a, e, tile, t0, nt, at, lds, sh);
        else down_tile<WT, CT, KS, NW>(a, e, tile, t0, nt, at, lds, sh);
        __syncthreads();
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

// Down token by token: all its experts in one workgroup per 16 rows, so that
// no sum is left over.  Sixteen waves share out the (expert, slot) pairs;
// the columns are hi and lo of h under one power of two, all of them in LDS at
// once: blocks of expert t from t * per slots on.
constexpr int kOneWaves = 16, kOneRing = 2, kOnePieces = 2;
constexpr int kOneStatic = kOneWaves * 33 * 4;   // its LDS beside the dynamic part
template <int WT>
__host__ __device__ inline Layout layout_one(int nb, int top) {
    const int per = (nb + Slot<WT>::BLOCKS - 1) / Slot<WT>::BLOCKS;
    Layout l;
    l.column_bytes = top * per * Slot<WT>::BLOCKS * 128;
    l.ring_at = l.column_bytes;
    l.scales_at = l.ring_at + kOneWaves * kOneRing * Slot<WT>::BYTES;
    l.bytes = l.scales_at + (WT == TLHIP_F16 ? 0 : top * scale_bytes(nb));
    return l;
}
template <int WT>
__global__ __launch_bounds__(kOneWaves * 64) void moe_down_one_kernel(MoeArgs a, Layout at) {
    using S = Slot<WT>;
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ float red[kOneWaves][2][16], most[kOneWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, nb = a.I / 32, per = (nb + S::BLOCKS - 1) / S::BLOCKS, slots = a.top * per;
    h8* cols = (h8*)lds;
    const uint8_t* ring = lds + at.ring_at + wave * (kOneRing * S::BYTES);
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_address(ring));
    const uint8_t* scales = lds + at.scales_at;
    const size_t pair0 = (size_t)blockIdx.y * a.top;   // of the token
    const int ids = a.ids[pair0 + (lane < a.top ? lane : 0)];
    auto copy = [&](int n, int k) {
        const int t = n / per, e = __builtin_amdgcn_readlane(ids, t);
        Rows<WT>(a.down, (size_t)e * a.K + n0, nb).copy(n - t * per, ring_lds + k * S::BYTES);
    };
    // h and its largest value do not wait for the experts' numbers, which the
    // copies do: they go first, and loads return in order
    f4 p[kOnePieces], q[kOnePieces];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kOnePieces; k++) {
            const int i = i0 + k * kOneWaves * 64, s = i & 3, t = (i >> 2) / (per * S::BLOCKS), b = (i >> 2) - t * (per * S::BLOCKS);
            p[k] = q[k] = f4{0, 0, 0, 0};
            if (i < slots * S::BLOCKS * 4 && b < nb) {
                const float* h = a.h + (pair0 + t) * a.I + b * 32;
                p[k] = *(const f4*)(h + run0<WT>(s));
                q[k] = *(const f4*)(h + run1<WT>(s));
            }
        }
    };
    fetch(threadIdx.x);
    float m = 0.0f;
    for (int i = threadIdx.x; i < a.top * (a.I / 16); i += kOneWaves * 64) m = fmaxf(m, a.hmax[pair0 * (a.I / 16) + i]);
    m = wave_max(m);
    if (lane == 0) most[wave] = m;
    if constexpr (WT != TLHIP_F16) {
        const uint32_t scales_lds = __builtin_amdgcn_readfirstlane(lds_address(scales));
        for (int t = 0; t < a.top; t++)
            copy_scales(scales_lds + t * scale_bytes(nb), a.down_d, (size_t)__builtin_amdgcn_readlane(ids, t) * a.K + n0, nb, wave, kOneWaves);
    }
    int next = wave, place = 0;
#pragma unroll
    for (int k = 0; k < kOneRing; k++, next += kOneWaves)
        if (next < slots) copy(next, k);
    lds_barrier();
    m = most[0];
#pragma unroll
    for (int k = 1; k < kOneWaves; k++) m = fmaxf(m, most[k]);
    const float scale = scale_for(m);
    for (int i0 = threadIdx.x; i0 < slots * S::BLOCKS * 4; i0 += kOnePieces * kOneWaves * 64) {
        if (i0 != (int)threadIdx.x) fetch(i0);
#pragma unroll
        for (int k = 0; k < kOnePieces; k++) {
            const int i = i0 + k * kOneWaves * 64;
            if (i >= slots * S::BLOCKS * 4) continue;
            p[k] *= scale;
            q[k] *= scale;
            cols[2 * i] = piece<WT>(p[k], q[k]);
            cols[2 * i + 1] = piece<WT>(low_part(p[k]), low_part(q[k]));
        }
    }
    // the scales have landed (as many copies as the wave's slots came after them)
    if (next <= slots - 1 + kOneWaves) sk_wait_vm<kOneRing * S::COPIES>();
    else sk_wait_vm<0>();
    lds_barrier();
    f4 acc = {0, 0, 0, 0};
    for (int n = wave; n < slots; n += kOneWaves) {
        if (next > n + (kOneRing - 1) * kOneWaves) sk_wait_vm<(kOneRing - 1) * S::COPIES>();
        else sk_wait_vm<0>();
        const int t = n / per;
        Weights<WT> w[S::STEPS];
#pragma unroll
        for (int u = 0; u < S::STEPS; u++)
            w[u].read(ring + place * S::BYTES, (const uint16_t*)(scales + t * scale_bytes(nb)), c16, nb, (n - t * per) * S::BLOCKS, u, g);
        if (next < slots) {
            lds_reads_done();
            copy(next, place);
            next += kOneWaves;
        }
        place = place + 1 == kOneRing ? 0 : place + 1;
#pragma unroll
        for (int u = 0; u < S::STEPS; u++) {
            h8 x[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] = cols[((n * S::BLOCKS + 4 * u + piece_block<WT>(j, g)) * 4 + piece_sub<WT>(j, g)) * 2 + (c16 & 1)];
#pragma unroll
            for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[u].sub(j), x[j], acc, 0, 0, 0);
        }
    }
    if (c16 < 2) *(f4*)&red[wave][c16][4 * g] = acc;
    __syncthreads();
    if (threadIdx.x < 16) {
        float s = 0.0f;
        for (int w = 0; w < kOneWaves; w++) s += red[w][0][threadIdx.x] + red[w][1][threadIdx.x];
        a.y[(size_t)blockIdx.y * a.K + n0 + threadIdx.x] = f2h(s / scale);
    }
}

// Dynamic LDS beside MoeShared, of 160 KB.  Rows of kMoeMaxRow fit with four
// waves to a tile: at most 64 KB of columns, 64 KB of rings and 64 bytes of
// scales per block (f16: none).
constexpr int kLdsDynamic = 156 << 10;
static_assert(kLdsDynamic + sizeof(MoeShared) <= 160 << 10, "LDS of a CU");
static_assert((64 << 10) + (32 << 10) + 64 * (kMoeMaxRow / 32) <= kLdsDynamic, "rows of a Q type fit");
static_assert(kDownColumnBytes + (64 << 10) <= kLdsDynamic && (32 << 10) + (64 << 10) <= kLdsDynamic, "f16 rows fit");

// Up to 16 (down: 8) tokens, no expert has more columns than one B operand holds.
int gate_up_columns(const MoeArgs& a) { return a.M < 32 ? a.M : 32; }
int down_columns(const MoeArgs& a) { return a.M < 16 ? 2 * a.M : 32; }
template <int WT, int KS>
void gate_up(hipStream_t s, const MoeArgs& a, unsigned slots) {
    const unsigned grid = slots * ((a.I / 16 + kWaves / KS - 1) / (kWaves / KS));
    const Layout at = layout<WT, 2, KS, kWaves>(a.K / 32, gate_up_columns(a));
    if (a.M == 1) moe_gate_up_kernel<WT, KS, 1, true><<<grid, kWaves * 64, at.bytes, s>>>(a, at);
    else if (a.M <= 16) moe_gate_up_kernel<WT, KS, 1, false><<<grid, kWaves * 64, at.bytes, s>>>(a, at);
    else moe_gate_up_kernel<WT, KS, 2, false><<<grid, kWaves * 64, at.bytes, s>>>(a, at);
}
template <int WT, int KS, int NW>
void down(hipStream_t s, const MoeArgs& a, unsigned slots) {
    const unsigned grid = slots * ((a.K / 16 + NW / KS - 1) / (NW / KS));
    const Layout at = layout<WT, 1, KS, NW>(a.I / 32, down_columns(a));
    if (a.M <= 8) moe_down_kernel<WT, KS, 1, NW><<<grid, NW * 64, at.bytes, s>>>(a, at);
    else moe_down_kernel<WT, KS, 2, NW><<<grid, NW * 64, at.bytes, s>>>(a, at);
    moe_sum_kernel<<<(a.M * (a.K / 4) + 255) / 256, 256, 0, s>>>(a);
}
// How often a CU fills up with workgroups until all have run.
template <int WT, int NR, int KS, int NW>
int64_t turns(int64_t tiles, int nb, int columns) {
    const int fit = (160 << 10) / (layout<WT, NR, KS, NW>(nb, columns).bytes + (int)sizeof(MoeShared));
    return (tiles * KS / NW + 256 * fit - 1) / (256 * fit);
}
// Waves that share out the k of a tile of 16 rows: as few as leave two
// workgroups of four waves for every CU (the more tiles a workgroup has, the
// fewer times the columns are staged), and no fewer than LDS has room for; for
// few tiles two, if a CU then fills up with workgroups less often (28 tokens of
// four Q4_0 experts 2656 x 1056, all chosen: 49 us against 75; 12 of six f16
// ones 2048 x 1024, two each: 26 against 33).
template <int WT, int NR, int NW>
int waves_of_tile(int64_t tiles, int nb, int columns) {
    if (tiles >= 2048 && layout<WT, NR, 1, NW>(nb, columns).bytes <= kLdsDynamic) return 1;
    const bool two = layout<WT, NR, 2, NW>(nb, columns).bytes <= kLdsDynamic;
    if (two && (tiles >= 1024 || turns<WT, NR, 2, NW>(tiles, nb, columns) < turns<WT, NR, 4, NW>(tiles, nb, columns))) return 2;
    return 4;
}
template <int WT>
void gate_up(hipStream_t s, const MoeArgs& a, unsigned slots) {
    switch (waves_of_tile<WT, 2, kWaves>((int64_t)slots * (a.I / 16), a.K / 32, gate_up_columns(a))) {
        case 1: return gate_up<WT, 1>(s, a, slots);
        case 2: return gate_up<WT, 2>(s, a, slots);
        default: return gate_up<WT, 4>(s, a, slots);
    }
}
template <int WT, int NW>
void down_waves(hipStream_t s, const MoeArgs& a, unsigned slots) {
    switch (waves_of_tile<WT, 1, NW>((int64_t)slots * (a.K / 16), a.I / 32, down_columns(a))) {
        case 1: return down<WT, 1, NW>(s, a, slots);
        case 2: return down<WT, 2, NW>(s, a, slots);
        default: return down<WT, 4, NW>(s, a, slots);
    }
}
template <int WT>
void down(hipStream_t s, const MoeArgs& a, unsigned slots) {
    // A token's workgroups read its experts' weights whether or not another's
    // do, but no sum is left to launch: taken for one token, and for a few whose
    // workgroups all run at once (two to eight: 4 us less; four of K = 4096,
    // 1024 workgroups of which 256 fit, would take 40 us against 37).
    const Layout at = layout_one<WT>(a.I / 32, a.top);
    const int fit = at.bytes + kOneStatic <= 80 << 10 ? 2 : 1;
    if (at.bytes + kOneStatic <= 160 << 10 && (a.M == 1 || a.M * (a.K / 16) <= 256 * fit)) {
        moe_down_one_kernel<WT><<<dim3(a.K / 16, a.M), kOneWaves * 64, at.bytes, s>>>(a, at);
        return;
    }
    if (a.M * a.top >= 2 * a.E) down_waves<WT, kDownWaves>(s, a, slots);
    else down_waves<WT, kWaves>(s, a, slots);
}

}  // namespace

tlhip_status launch_moe(hipStream_t s, const MoeArgs& a) {
    moe_router_kernel<<<a.M, 1024, 0, s>>>(a);
    const unsigned slots = a.M * a.top < a.E ? a.M * a.top : a.E;
    if (a.wt_gu == TLHIP_F16) gate_up<TLHIP_F16>(s, a, slots);
    else if (a.wt_gu == TLHIP_Q4_0) gate_up<TLHIP_Q4_0>(s, a, slots);
    else gate_up<TLHIP_Q8_0>(s, a, slots);
    if (a.wt_down == TLHIP_F16) down<TLHIP_F16>(s, a, slots);
    else if (a.wt_down == TLHIP_Q4_0) down<TLHIP_Q4_0>(s, a, slots);
    else down<TLHIP_Q8_0>(s, a, slots);
    return TLHIP_OK;
}

}  // namespace tlhip
