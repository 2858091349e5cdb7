// kv8.cpp -- host side of the 8-bit KV cache (layout and kernels:
// kernels_kv8.hip): its memory, and what tlhip_kvcache_set / append / get and
// the attention entry points do with a cache of dtype Q8_0.
#include "internal.hpp"

namespace tlhip {

namespace {

constexpr int kBlock = 32;   // positions that share a scale

int n_blocks(const tlhip_kvcache_s* c) { return (c->max_ctx + kBlock - 1) / kBlock; }

// The cache's memory and its bookkeeping of the tails belong to its context's
// stream, so every call on it has to come on that context.
tlhip_status own_ctx(tlhip_ctx ctx, const tlhip_kvcache_s* c, const char* op) {
    if (ctx != c->ctx)
        return fail(TLHIP_ERR_INVALID_ARGUMENT, "%s: an 8-bit cache is used on the context it was created on", op);
    return TLHIP_OK;
}

}  // namespace

tlhip_status kv8_alloc(tlhip_kvcache c) {
    if (!kv8_head_dim_ok(c->head_dim))
        return fail(TLHIP_ERR_INVALID_DIMENSION, "8-bit kvcache: head_dim %d is not 32, 64, 80, 96, 128 or 256",
                    c->head_dim);
    if (c->n_kv > 1024) return fail(TLHIP_ERR_INVALID_DIMENSION, "8-bit kvcache: %d KV heads > 1024", c->n_kv);
    const size_t nb = n_blocks(c), hk = c->n_kv, D = c->head_dim;
    const size_t tiles = align256(hk * nb * kBlock * D), scales = align256(hk * nb * sizeof(float));
    const size_t tail = align256(2 * hk * kBlock * D * sizeof(uint16_t)), flags = align256(2 * hk * kBlock * sizeof(float));
    int64_t words = (int64_t)((2 * tiles + 2 * scales + 2 * tail + flags) / sizeof(int32_t));
    c->q8.reserve(c->n_layers);
    for (int i = 0; i < c->n_layers; i++) {
        Kv8Layer l;
        TLHIP_TRY(alloc_tensor(c->ctx, TLHIP_I32, 1, &words, &l.buf));
        uint8_t* at = (uint8_t*)l.buf->data;
        auto cut = [&](size_t bytes) {
            uint8_t* p = at;
            at += bytes;
            return p;
        };
        l.kq = cut(tiles);
        l.vq = cut(tiles);
        l.ks = (float*)cut(scales);
        l.vs = (float*)cut(scales);
        l.tail_k = (uint16_t*)cut(tail);
        l.tail_v = (uint16_t*)cut(tail);
        l.tail_flag = (float*)cut(flags);
        c->q8.push_back(l);
    }
    return TLHIP_OK;
}

tlhip_status kv8_write(tlhip_ctx ctx, tlhip_kvcache c, int layer, tlhip_tensor k, tlhip_tensor v, int start, int S) {
    TLHIP_TRY(own_ctx(ctx, c, "kvcache"));
    TLHIP_TRY(check_here(ctx, k, "kvcache K"));
    TLHIP_TRY(check_here(ctx, v, "kvcache V"));
    DeviceScope scope(ctx->device);
    OtherStreams others(ctx);
    TLHIP_TRY(others.wait({k, v}));
    Kv8Layer& l = c->q8[layer];
    Kv8Write p;
    p.k = (const uint16_t*)k->data;
    p.v = (const uint16_t*)v->data;
    p.kq = l.kq;
    p.vq = l.vq;
    p.ks = l.ks;
    p.vs = l.vs;
    p.tail_k = l.tail_k;
    p.tail_v = l.tail_v;
    p.tail_flag = l.tail_flag;
    p.len0 = start;
    p.S = S;
    p.n_full = (start + S) / kBlock - start / kBlock;
    // a call that completes a block reads the old tail, so the rows it leaves
    // over go to the other one
    p.tail_src = l.tail_cur;
    p.tail_dst = p.n_full ? 1 - l.tail_cur : l.tail_cur;
    p.n_kv = c->n_kv;
    p.D = c->head_dim;
    p.n_blocks = n_blocks(c);
    TLHIP_TRY(launch_kv8_write(ctx->stream, p));
    TLHIP_TRY(after_launch(ctx, "kvcache write"));
    TLHIP_TRY(others.done());
    l.tail_cur = p.tail_dst;
    return TLHIP_OK;
}

tlhip_status kv8_get(tlhip_kvcache c, int layer, int which_v, tlhip_tensor* out) {
    DeviceScope scope(c->ctx->device);
    const Kv8Layer& l = c->q8[layer];
    int64_t shp[3] = {c->len[layer], c->n_kv, c->head_dim};
    tlhip_tensor t = nullptr;
    TLHIP_TRY(alloc_tensor(c->ctx, TLHIP_F16, 3, shp, &t));
    Kv8Read p;
    p.q = which_v ? l.vq : l.kq;
    p.s = which_v ? l.vs : l.ks;
    p.tail = which_v ? l.tail_v : l.tail_k;
    p.tail_flag = l.tail_flag;
    p.out = (uint16_t*)t->data;
    p.tail_cur = l.tail_cur;
    p.len = c->len[layer];
    p.n_kv = c->n_kv;
    p.D = c->head_dim;
    p.n_blocks = n_blocks(c);
    p.is_v = which_v != 0;
    tlhip_status st = launch_kv8_read(c->ctx->stream, p);
    if (st == TLHIP_OK) st = after_launch(c->ctx, "kvcache_get");
    if (st != TLHIP_OK) {
        tlhip_tensor_free(t);
        return st;
    }
    *out = t;
    return TLHIP_OK;
}

tlhip_status kv8_attention(tlhip_ctx ctx, tlhip_tensor q, tlhip_kvcache c, int layer, float scale, tlhip_tensor out) {
    TLHIP_TRY(check_ctx(ctx));
    TLHIP_TRY(own_ctx(ctx, c, "attention"));
    TLHIP_TRY(check_t(out, "attention"));
    TLHIP_TRY(check_dtype(q, TLHIP_F16, "attention"));
    TLHIP_TRY(check_dtype(out, TLHIP_F16, "attention"));
    TLHIP_TRY(check_here(ctx, q, "attention q"));
    TLHIP_TRY(check_here(ctx, out, "attention out"));
    // (q is [S, H, D] with 1 <= S <= len: tlhip_attention_prefill)
    const int64_t S = q->shape[0], H = q->shape[1];
    if (q->shape[2] != c->head_dim)
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "attention: q %s for a cache of head_dim %d", shape_str(q).c_str(), c->head_dim);
    if (H < 1 || H % c->n_kv)
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "attention: %lld heads vs %d KV heads", (long long)H, c->n_kv);
    if (out->ndim != 3 || out->shape[0] != S || out->shape[1] != H || out->shape[2] != q->shape[2])
        return fail(TLHIP_ERR_SHAPE_MISMATCH, "attention q/out: shape %s vs %s", shape_str(q).c_str(), shape_str(out).c_str());
    if (S * H > INT32_MAX / 4) return fail(TLHIP_ERR_INVALID_DIMENSION, "attention: q %s is too large", shape_str(q).c_str());
    DeviceScope scope(ctx->device);
    OtherStreams others(ctx);
    TLHIP_TRY(others.wait({q, out}));
    const Kv8Layer& l = c->q8[layer];
    const int len = c->len[layer];
    Kv8Attn p;
    p.q = (const uint16_t*)q->data;
    p.out = (uint16_t*)out->data;
    p.kq = l.kq;
    p.vq = l.vq;
    p.ks = l.ks;
    p.vs = l.vs;
    p.tail_k = l.tail_k;
    p.tail_v = l.tail_v;
    p.tail_flag = l.tail_flag;
    p.scale = scale;
    p.tail_cur = l.tail_cur;
    p.n_full = len / kBlock;
    p.S = (int)S;
    p.H = (int)H;
    p.n_kv = c->n_kv;
    p.group = (int)(H / c->n_kv);
    p.D = c->head_dim;
    p.n_blocks = n_blocks(c);
    p.q_pos0 = len - (int)S;
    const Kv8Plan pl = kv8_plan(p.S, p.group, p.n_kv, p.D, len);
    if (pl.scratch_bytes) {
        p.scratch = ctx_workspace(ctx, pl.scratch_bytes);
        if (!p.scratch) return fail(TLHIP_ERR_ALLOCATION, "attention: no workspace of %zu bytes", pl.scratch_bytes);
    }
    TLHIP_TRY(launch_kv8_attention(ctx->stream, p, pl));
    TLHIP_TRY(after_launch(ctx, "attention"));
    return others.done();
}

}  // namespace tlhip
