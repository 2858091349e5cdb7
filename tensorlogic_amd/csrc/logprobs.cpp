// logprobs.cpp -- tlhip_token_logprobs: checks and launch.
#include "internal.hpp"

using namespace tlhip;

extern "C" tlhip_status tlhip_token_logprobs(tlhip_ctx ctx, tlhip_tensor logits, tlhip_tensor ids, int n_top,
                                             tlhip_tensor logprob, tlhip_tensor entropy, tlhip_tensor top_logprob,
                                             tlhip_tensor top_ids) try {
    const char* op = "token_logprobs";
    TLHIP_TRY(check_ctx(ctx));
    TLHIP_TRY(check_t(logits, op));
    if (logits->dtype != TLHIP_F16 && logits->dtype != TLHIP_F32)
        return fail(TLHIP_ERR_DTYPE, "%s: logits must be f16 or f32 (dtype %d)", op, (int)logits->dtype);
    if (logits->ndim != 1 && logits->ndim != 2)
        return fail(TLHIP_ERR_INVALID_DIMENSION, "%s: expects [V] or [rows, V] logits, got %s", op, shape_str(logits).c_str());
    const int64_t V = last_dim(logits), rows = logits->ndim == 2 ? logits->shape[0] : 1;
    // (a launch holds fewer than 2^32 threads, and a row takes 256 at least)
    if (V < 1 || V > (1 << 30) || rows >= (1 << 24))
        return fail(TLHIP_ERR_INVALID_DIMENSION, "%s: logits %s", op, shape_str(logits).c_str());
    if (n_top < 0 || n_top > kMaxTop || n_top > V)
        return fail(TLHIP_ERR_INVALID_DIMENSION, "%s: n_top %d not in 0..min(%d, %lld)", op, n_top, kMaxTop, (long long)V);
    if ((ids != nullptr) != (logprob != nullptr))
        return fail(TLHIP_ERR_INVALID_ARGUMENT, "%s: ids and logprob go together", op);
    if ((n_top > 0) != (top_logprob != nullptr) || (n_top > 0) != (top_ids != nullptr))
        return fail(TLHIP_ERR_INVALID_ARGUMENT, "%s: top_logprob and top_ids go with n_top > 0", op);
    auto out = [&](tlhip_tensor t, tlhip_dtype dt, int64_t cols, const char* what) -> tlhip_status {
        if (!t) return TLHIP_OK;
        TLHIP_TRY(check_t(t, op));
        TLHIP_TRY(check_dtype(t, dt, op));
        TLHIP_TRY(check_here(ctx, t, op));
        const bool shape_ok = cols ? t->ndim == 2 && t->shape[0] == rows && t->shape[1] == cols
                                   : t->ndim == 1 && t->shape[0] == rows;
        if (!shape_ok)
            return fail(TLHIP_ERR_SHAPE_MISMATCH, "%s: %s %s for %lld rows", op, what, shape_str(t).c_str(), (long long)rows);
        return TLHIP_OK;
    };
    TLHIP_TRY(check_here(ctx, logits, op));
    TLHIP_TRY(out(ids, TLHIP_I32, 0, "ids"));
    TLHIP_TRY(out(logprob, TLHIP_F32, 0, "logprob"));
    TLHIP_TRY(out(entropy, TLHIP_F32, 0, "entropy"));
    TLHIP_TRY(out(top_logprob, TLHIP_F32, n_top, "top_logprob"));
    TLHIP_TRY(out(top_ids, TLHIP_I32, n_top, "top_ids"));
    if (rows == 0) return TLHIP_OK;
    LogprobArgs a;
    a.x = logits->data;
    a.ids = ids ? (const int32_t*)ids->data : nullptr;
    a.logprob = logprob ? (float*)logprob->data : nullptr;
    a.entropy = entropy ? (float*)entropy->data : nullptr;
    a.top_logprob = n_top ? (float*)top_logprob->data : nullptr;
    a.top_ids = n_top ? (int32_t*)top_ids->data : nullptr;
    a.rows = (int)rows;
    a.V = (int)V;
    a.n_top = n_top;
    a.f32 = logits->dtype == TLHIP_F32;
    DeviceScope scope(ctx->device);
    OtherStreams others(ctx);
    TLHIP_TRY(others.wait({logits, ids, logprob, entropy, top_logprob, top_ids}));
    const LogprobPlan pl = logprobs_plan(a.rows, a.V, n_top);
    a.chunks = pl.chunks;
    a.chunk = pl.chunk;
    if (pl.ws_bytes) {
        uint8_t* ws = (uint8_t*)ctx_workspace(ctx, pl.ws_bytes);
        if (!ws) return fail(TLHIP_ERR_ALLOCATION, "%s: no workspace of %zu bytes", op, pl.ws_bytes);
        a.part = (float*)ws;
        a.part_keys = (uint64_t*)(ws + pl.part_bytes);
    }
    TLHIP_TRY(launch_logprobs(ctx->stream, a));
    TLHIP_TRY(after_launch(ctx, op));
    return others.done();
} TLHIP_CATCH_STATUS
