// moe.cpp -- tlhip_moe: checks, workspace and launches.
#include "internal.hpp"

using namespace tlhip;

namespace {

// The experts' matrices one after another: [E * n, k], or [E, n, k] for f16.
tlhip_status expert_matrix(tlhip_ctx ctx, tlhip_tensor w, int64_t E, int64_t k, const char* what, int64_t* n) {
    TLHIP_TRY(check_t(w, what));
    TLHIP_TRY(check_here(ctx, w, "moe"));
    if (w->dtype != TLHIP_F16 && w->dtype != TLHIP_Q4_0 && w->dtype != TLHIP_Q8_0)
        return fail(TLHIP_ERR_DTYPE, "moe: %s must be F16, Q4_0 or Q8_0 (dtype %d)", what, (int)w->dtype);
    const bool three = w->ndim == 3;
    const int64_t rows = three ? w->shape[0] * w->shape[1] : w->shape[0];
    if ((w->ndim != 2 && !three) || last_dim(w) != k || rows % E || (three && w->shape[0] != E))
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "moe: %s %s for %lld experts and rows of %lld", what, shape_str(w).c_str(),
                    (long long)E, (long long)k);
    *n = rows / E;
    return TLHIP_OK;
}

constexpr int64_t kSlab = 256;   // tokens of one round of launches

}  // namespace

extern "C" tlhip_status tlhip_moe(tlhip_ctx ctx, tlhip_tensor x, tlhip_tensor router, tlhip_tensor gate, tlhip_tensor up,
                                  tlhip_tensor down, int top_k, int normalize, tlhip_tensor y) try {
    TLHIP_TRY(check_ctx(ctx));
    for (tlhip_tensor t : {x, router, y}) {
        TLHIP_TRY(check_t(t, "moe"));
        TLHIP_TRY(check_dtype(t, TLHIP_F16, "moe"));
        TLHIP_TRY(check_here(ctx, t, "moe"));
    }
    if (x->ndim != 2 || router->ndim != 2 || y->ndim != 2)
        return fail(TLHIP_ERR_INVALID_OPERATION, "moe: x, router and y must be 2-D");
    const int64_t M = x->shape[0], K = x->shape[1], E = router->shape[0];
    if (router->shape[1] != K)
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "moe: router %s for rows of %lld", shape_str(router).c_str(), (long long)K);
    if (y->shape[0] != M || y->shape[1] != K)
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "moe: output %s for x %s", shape_str(y).c_str(), shape_str(x).c_str());
    if (E < 1 || E > kMoeMaxExperts)
        return fail(TLHIP_ERR_INVALID_DIMENSION, "moe: %lld experts not in 1..%d", (long long)E, kMoeMaxExperts);
    if (top_k < 1 || top_k > E || top_k > kMoeMaxTop)
        return fail(TLHIP_ERR_INVALID_DIMENSION, "moe: top_k %d not in 1..min(%lld, %d)", top_k, (long long)E, kMoeMaxTop);
    int64_t I = 0, Iu = 0, Kd = 0;
    TLHIP_TRY(expert_matrix(ctx, gate, E, K, "gate", &I));
    TLHIP_TRY(expert_matrix(ctx, up, E, K, "up", &Iu));
    TLHIP_TRY(expert_matrix(ctx, down, E, I, "down", &Kd));
    if (Iu != I || Kd != K || gate->dtype != up->dtype)
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "moe: gate %s, up %s and down %s (gate and up of one dtype)",
                    shape_str(gate).c_str(), shape_str(up).c_str(), shape_str(down).c_str());
    if (K < 32 || I < 32 || K % 32 || I % 32 || K > kMoeMaxRow || I > kMoeMaxRow)
        return fail(TLHIP_ERR_INVALID_DIMENSION, "moe: rows of %lld and %lld (multiples of 32 up to %d)", (long long)K, (long long)I,
                    kMoeMaxRow);
    if (M == 0) return TLHIP_OK;
    const int64_t slab = M < kSlab ? M : kSlab;
    // ids, g, h, hmax, part: one after another
    const size_t pairs = (size_t)slab * top_k;
    const size_t at_g = align256(pairs * sizeof(int32_t)), at_h = at_g + align256(pairs * sizeof(float));
    const size_t at_max = at_h + align256(pairs * I * sizeof(float)), at_part = at_max + align256(pairs * (I / 16) * sizeof(float));
    const size_t need = at_part + pairs * K * sizeof(float);
    DeviceScope scope(ctx->device);
    OtherStreams others(ctx);
    TLHIP_TRY(others.wait({x, router, gate, up, down, y}));
    uint8_t* ws = (uint8_t*)ctx_workspace(ctx, need);
    if (!ws) return fail(TLHIP_ERR_ALLOCATION, "moe: no workspace of %zu bytes", need);
    MoeArgs a;
    a.router = (const uint16_t*)router->data;
    a.gate = gate->data;
    a.up = up->data;
    a.down = down->data;
    a.gate_d = gate->scales;
    a.up_d = up->scales;
    a.down_d = down->scales;
    a.ids = (int32_t*)ws;
    a.g = (float*)(ws + at_g);
    a.h = (float*)(ws + at_h);
    a.hmax = (float*)(ws + at_max);
    a.part = (float*)(ws + at_part);
    a.K = (int)K;
    a.I = (int)I;
    a.E = (int)E;
    a.top = top_k;
    a.normalize = normalize != 0;
    a.wt_gu = gate->dtype;
    a.wt_down = down->dtype;
    for (int64_t m = 0; m < M; m += kSlab) {
        a.x = (const uint16_t*)x->data + m * K;
        a.y = (uint16_t*)y->data + m * K;
        a.M = (int)(M - m < kSlab ? M - m : kSlab);
        TLHIP_TRY(launch_moe(ctx->stream, a));
    }
    TLHIP_TRY(after_launch(ctx, "moe"));
    return others.done();
} TLHIP_CATCH_STATUS
