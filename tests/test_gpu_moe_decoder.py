"""A decoder block of experts as a user writes it: projections and RoPE, the
8-bit cache and the attention over it, moe, an output projection and
token_logprobs, a prompt and then tokens one by one; each operator's result
against 64-bit arithmetic on the values that it was given."""
import numpy as np
import pytest

from tensorlogic_amd import F16, F32, I32, Q4_0, Q8_0, Device, KVCache, embedding, moe, token_logprobs
from tensorlogic_amd._lib import call
from test_gpu_kv8 import as_f16, check, held
from test_gpu_logprobs import close
from test_gpu_logprobs import reference as logprobs_reference
from test_gpu_moe import case, upload
from test_gpu_moe import reference as moe_reference

pytestmark = pytest.mark.gpu

K, I, E, TOP, V = 256, 352, 8, 2, 1000


class Block:
    def __init__(self, dev, H, kv, D, gu, dn, max_ctx):
        r = np.random.default_rng([H, kv, D])
        f = lambda n, k: dev.tensor((r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16))  # noqa: E731
        self.dev, self.H, self.kv, self.D, self.gu, self.dn = dev, H, kv, D, gu, dn
        self.table, self.q, self.k, self.v = f(V, K) * 16.0, f(H * D, K), f(kv * D, K), f(kv * D, K)
        self.o, self.head, self.norm = f(K, H * D), f(V, K), dev.tensor(np.ones(K, np.float16))
        self.router, self.mats = case(5, E, K, I, gu, dn)
        self.experts = [upload(dev, raw, s, t) for (raw, _), s, t in
                        zip(self.mats, ((E * I, K), (E * I, K), (E * K, I)), (gu, gu, dn))]
        self.dev_router = dev.tensor(self.router)
        self.cache = KVCache(dev, 1, max_ctx, kv, D, Q8_0)

    def step(self, ids, past):
        """Every value of one pass over the tokens ids, on the host."""
        s, D = len(ids), self.D
        x = embedding(self.table, np.asarray(ids, np.int32))
        n = x.rms_norm([K], self.norm)
        q = n.linear(self.q).reshape((s, self.H, D)).rope(past)
        k = n.linear(self.k).reshape((s, self.kv, D)).rope(past)
        v = n.linear(self.v).reshape((s, self.kv, D))
        (self.cache.append if past else self.cache.set)(0, k, v)
        a = self.cache.attention(q, 0, D ** -0.5)
        x = x.add(a.reshape((s, self.H * D)).linear(self.o))
        n = x.rms_norm([K], self.norm)
        y = moe(n, self.dev_router, *self.experts, TOP)
        logits = x.add(y).rms_norm([K], self.norm).linear(self.head)
        target = (np.asarray(ids) * 7 + 3) % V
        said = token_logprobs(logits, self.dev.tensor(target, I32), 5)
        return [t.numpy() for t in (q, k, v, a, n, y, logits, *said)], target


@pytest.mark.parametrize("H,kv,D,gu,dn", [(8, 2, 64, Q4_0, Q8_0), (4, 4, 80, F16, F16), (8, 2, 128, Q8_0, Q4_0)])
def test_prompt_and_tokens(dev, H, kv, D, gu, dn):
    ids = np.random.default_rng(D).integers(0, V, 70)
    parts = [45] + [1] * 20 + [5]   # a prompt, tokens one by one over a block's end, a few at once
    b = Block(dev, H, kv, D, gu, dn, 80)
    keys, values, past = np.zeros((0, kv, D), np.float16), np.zeros((0, kv, D), np.float16), 0
    for s in parts:
        (q, k, v, a, n, y, logits, *said), target = b.step(ids[past:past + s], past)
        keys, values, past = np.concatenate([keys, k]), np.concatenate([values, v]), past + s
        check(a, q, keys, values, D ** -0.5, f"attention at {past}")
        ref, tol = moe_reference(n, b.router, b.mats, E, TOP, True)
        assert (np.abs(y - ref) <= tol).all(), f"moe at {past}"
        lp, h, top, at, tlp, th, tt = logprobs_reference(logits, target, 5)
        close(said[0], lp, tlp, f"logprob at {past}")
        close(said[1], h, th, f"entropy at {past}")
        close(said[2], top, tt, f"top logprob at {past}")
        assert np.array_equal(said[3], at), f"top ids at {past}"
    assert b.cache.len(0) == 70
    for got, x in ((b.cache.get_k(0), keys), (b.cache.get_v(0), values)):
        assert np.array_equal(got.numpy().view(np.uint16), as_f16(held(x)).view(np.uint16))
    # the same again on the same buffers gives the same bits
    past = 0
    again = []
    for s in parts:
        again.append(b.step(ids[past:past + s], past)[0])
        past += s
    assert np.array_equal(again[-1][6], logits) and all(np.array_equal(x, z) for x, z in zip(again[-1][7:], said))


def test_tensors_of_another_context(dev):
    """Inputs still being computed on another context's stream, results read and inputs overwritten on it."""
    r = np.random.default_rng(3)
    M, E, K, I, top, V = 12, 4, 256, 96, 2, 3001
    w = dev.tensor((r.standard_normal((K, K)) / 16).astype(np.float16))
    wide = dev.tensor((r.standard_normal((4096, K)) / 16).astype(np.float16))
    back = dev.tensor((r.standard_normal((K, 4096)) / 64).astype(np.float16))
    x0 = dev.tensor(r.standard_normal((M, K)).astype(np.float16))
    router, mats = case(6, E, K, I, F16, F16)
    experts = [dev.tensor(m[0]) for m in mats]
    head = dev.tensor((r.standard_normal((V, K)) / 16).astype(np.float16))
    ids = r.integers(0, V, M).astype(np.int32)

    def chain():   # some hundred launches
        x = x0
        for _ in range(60):
            x = x.linear(w).linear(wide).linear(back)
            x = x.rms_norm([K], dev.tensor(np.ones(K, np.float16)))
        return x

    x = chain()
    keys = x.linear(w).reshape((M, 4, 64))
    c = KVCache(dev, 1, 64, 4, 64, Q8_0)
    c.set(0, keys, keys)
    want = [moe(x, dev.tensor(router), *experts, top).numpy(), c.attention(keys, 0, 0.125).numpy(),
            *(t.numpy() for t in token_logprobs(x.linear(head), dev.tensor(ids, I32), 3))]
    other = Device(0)
    try:
        o_router, o_ids = other.tensor(router), other.tensor(ids, I32)
        y, att = other.empty((M, K)), other.empty((M, 4, 64))
        lp, h, tl, ti = other.empty((M,), F32), other.empty((M,), F32), other.empty((M, 3), F32), other.empty((M, 3), I32)
        oc = KVCache(other, 1, 64, 4, 64, Q8_0)
        x = chain()
        keys = x.linear(w).reshape((M, 4, 64))
        logits = x.linear(head)
        call("tlhip_kvcache_set", other.h, oc.h, 0, keys.h, keys.h)
        call("tlhip_attention_prefill", other.h, keys.h, oc.h, 0, 0.125, att.h)
        call("tlhip_moe", other.h, x.h, o_router.h, *(e.h for e in experts), top, 1, y.h)
        call("tlhip_token_logprobs", other.h, logits.h, o_ids.h, 3, lp.h, h.h, tl.h, ti.h)
        del x, keys, logits   # their blocks go to dev's next tensors
        junk = [dev.tensor(np.full((M, n), 7.0, np.float16)).mul_scalar(3.0) for n in (K, K, V, V)]
        got = [t.numpy() for t in (y, att, lp, h, tl, ti)]
        assert all(np.array_equal(a, b) for a, b in zip(want, got))
        del junk, o_router, o_ids, y, att, lp, h, tl, ti, oc
    finally:
        other.close()
