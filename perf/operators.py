"""Operators of one request's step at a long context, as measurable cases.

A case is a dict of plain values.  `kind` says which operator one pass is:

  kv_write   KVCache.set of an 8-bit cache: the K and V rows of a prompt,
             quantised block by block (32 positions of one head, one scale);
             the rows past the last whole block stay f16.
  attention  KVCache.attention over an 8-bit cache: s query rows (the cache's
             last s positions) over past + s cached positions; s = 1 is a
             decode step.
  moe        moe: router, the chosen experts' gate, up and down products and
             their weighted sum, for a few tokens.
  logprobs   token_logprobs: what the vocabulary's softmax says of given
             tokens, its entropy, and the likeliest alternatives.

With `own` false a pass is the operator's plain form: products, sums, exp,
comparisons and indexing of torch in 32 bits, rounded once at the end.  With
`own` true it is the call a user makes of this package, on the package's own
tensors; outputs stay on the device, as a program that goes on computing
leaves them, and are read back when they are looked at.
"""
from __future__ import annotations

import math
import zlib

import numpy as np
import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"   # where inputs are drawn
BLOCK = 32                                              # positions that share a scale of the cache
BYTES = {"f16": 2.0, "q4_0": 18 / 32, "q8_0": 34 / 32}  # per weight


def listed():
    return [
        # the prompt pass of the 46-token chat prompt: one layer's rows, one whole block and a rest
        dict(name="kv_write_46", kind="kv_write", s=46, kv=4, d=64),
        # a prompt that fills a 2048-token context, heads of 80 without sharing
        dict(name="kv_write_2048", kind="kv_write", s=2048, kv=32, d=80),
        # a decode step late in a long conversation, GQA heads of the llama configuration
        dict(name="attn_decode_4000", kind="attention", s=1, past=3999, heads=32, kv=4, d=64),
        # a decode step at the longest context a cache holds, one KV head per query head
        dict(name="attn_decode_65000", kind="attention", s=1, past=64999, heads=32, kv=32, d=80),
        # attention of a prompt that fills a 2048-token context
        dict(name="attn_prompt_2048", kind="attention", s=2048, past=0, heads=32, kv=4, d=64),
        # a 700-token document added to a conversation of 5300 tokens
        dict(name="attn_prompt_700_past_5300", kind="attention", s=700, past=5300, heads=32, kv=8, d=128),
        # one decode step of a small model of many experts, unquantised
        dict(name="moe_f16_m1", kind="moe", wt="f16", m=1, k=1024, i=512, experts=32, top=4, norm=False),
        # one decode step, experts as wide as the llama configuration's FFN
        dict(name="moe_q4_m1", kind="moe", wt="q4_0", m=1, k=2048, i=5632, experts=8, top=2, norm=True),
        # a short question of 13 tokens through the same experts in 8 bits
        dict(name="moe_q8_m13", kind="moe", wt="q8_0", m=13, k=2048, i=5632, experts=8, top=2, norm=True),
        # one decode step: the drawn token's probability and five alternatives
        dict(name="logprobs_1", kind="logprobs", rows=1, v=32000, dtype="f16", top=5, masked=False),
        # scoring a document: what the model gives each of its 2048 tokens
        dict(name="logprobs_2048", kind="logprobs", rows=2048, v=32000, dtype="f16", top=0, masked=False),
        # a prompt's tokens with twenty alternatives each, part of the vocabulary masked out
        dict(name="logprobs_333_top20", kind="logprobs", rows=333, v=51200, dtype="f32", top=20, masked=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 4, 64), (32, 32, 80), (32, 8, 128), (16, 16, 64), (12, 4, 96), (8, 2, 256), (16, 4, 32), (20, 4, 80)]


def draw(rng):
    kind = rng.choice(["kv_write", "attention", "attention", "moe", "moe", "logprobs"])
    if kind == "kv_write":
        _, kv, d = rng.choice(HEADS)
        return dict(kind=kind, s=_log_int(rng, 1, 2048), kv=kv, d=d)
    if kind == "attention":
        while True:
            heads, kv, d = rng.choice(HEADS)
            s = 1 if rng.random() < 0.4 else _log_int(rng, 2, 2048)
            past = _log_int(rng, 1, 65000) if s == 1 else rng.choice([0, _log_int(rng, 1, 8000)])
            if (past + s) * kv * d <= 65000 * 32 * 80 and s * (past + s / 2) * heads * d <= 700 * 5650 * 32 * 128:
                return dict(kind=kind, s=s, past=past, heads=heads, kv=kv, d=d)
    if kind == "moe":
        while True:
            k, i = 32 * _log_int(rng, 4, 128), 32 * _log_int(rng, 2, 176)
            experts = _log_int(rng, 2, 64)
            if experts * i * k <= 8 * 5632 * 2048:
                return dict(kind=kind, wt=rng.choice(["q4_0", "q4_0", "q8_0", "f16"]), m=_log_int(rng, 1, 32), k=k, i=i,
                            experts=experts, top=rng.randrange(1, min(experts, 8) + 1), norm=rng.random() < 0.5)
    while True:
        rows, v, dtype = _log_int(rng, 1, 2048), _log_int(rng, 500, 160000), rng.choice(["f16", "f16", "f32"])
        if rows * v * (2 if dtype == "f16" else 4) <= 2048 * 32000 * 2:
            return dict(kind=kind, rows=rows, v=v, dtype=dtype, top=rng.choice([0, 1, 5, rng.randrange(1, 33)]),
                        masked=rng.random() < 0.3)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, name):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + zlib.crc32(name.encode())) % (1 << 62))


def _normal(seed, name, shape, std=1.0):
    return torch.randn(shape, generator=_gen(seed, name), device=DEV, dtype=torch.float32) * std


def _kv_rows(seed, rows, kv, d):
    """K and V rows [rows, kv, d]; keys have a few channels of large values, as rotated keys do."""
    chan = 1 + 3 * (torch.rand((kv, d), generator=_gen(seed, "chan"), device=DEV) > 0.94).float()
    return (_normal(seed, "k", (rows, kv, d)) * chan).half(), _normal(seed, "v", (rows, kv, d)).half()


def _queries(case, seed):
    # scores of a spread of about 1.5, as attention has where it looks at many positions
    return _normal(seed, "q", (case["s"], case["heads"], case["d"])).half()


def _blocks(w, wt):
    """GGUF bytes (uint8, one row per block of 32) of the f32 matrix w."""
    if wt == "f16":
        return w.half().view(torch.uint8)
    b = w.reshape(-1, 32)
    if wt == "q4_0":   # d = the largest magnitude, signed, over -8
        d = (b.gather(1, b.abs().argmax(1, keepdim=True)) / -8).half()
        q = torch.clamp(torch.round(b / d.float()) + 8, 0, 15).to(torch.uint8)
        return torch.cat([d.view(torch.uint8), q[:, :16] | (q[:, 16:] << 4)], 1)
    d = (b.abs().amax(1, keepdim=True) / 127).half()
    q = torch.clamp(torch.round(b / d.float()), -127, 127).to(torch.int8)
    return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], 1)


def _weights(blk, wt, n, k):
    """The f16 weights [n, k] the GGUF bytes stand for."""
    if wt == "f16":
        return blk.reshape(n, -1).view(torch.float16)
    d = blk[:, :2].contiguous().view(torch.float16).float()
    if wt == "q4_0":
        q = torch.cat([blk[:, 2:] & 15, blk[:, 2:] >> 4], 1).float() - 8
    else:
        q = blk[:, 2:].contiguous().view(torch.int8).float()
    return (q * d).half().reshape(n, k)


def _moe_inputs(case, seed):
    """x, router, and (rows, columns, GGUF bytes) of gate, up and down, the experts' rows one after another."""
    m, k, i, e, wt = case["m"], case["k"], case["i"], case["experts"], case["wt"]
    mats = [(e * n, c, _blocks(_normal(seed, name, (e * n, c), 1 / math.sqrt(c)), wt))
            for name, n, c in (("gate", i, k), ("up", i, k), ("down", k, i))]
    return _normal(seed, "x", (m, k)).half(), _normal(seed, "router", (e, k), 1.5 / math.sqrt(k)).half(), mats


def _logits(case, seed):
    """Logits [rows, v] with a few likely tokens each, and the tokens asked about: mostly likely ones."""
    r, v = case["rows"], case["v"]
    x = _normal(seed, "logits", (r, v), 2.5)
    top = torch.randint(0, v, (r, 6), generator=_gen(seed, "top"), device=DEV)
    x.scatter_add_(1, top, 4 + 2 * _normal(seed, "lift", (r, 6)).abs())
    ids = torch.where(_normal(seed, "pick", (r,)) > -1, top[:, 0], top.flip(0)[:, 1])
    if case["masked"]:   # a grammar's mask: some of the vocabulary cannot follow
        x[torch.rand((r, v), generator=_gen(seed, "mask"), device=DEV) < 0.3] = -math.inf
    return (x.half() if case["dtype"] == "f16" else x), ids.to(torch.int32)


def _host(t):
    return t.cpu().numpy()


_device = None


def _dev():
    """One device context for the process, as a program has."""
    import tensorlogic_amd as tl
    global _device
    if _device is None:
        _device = tl.Device(0)
    return _device


def prepare(case, seed):
    st = {"case": case}
    if case["kind"] == "kv_write":
        k, v = _kv_rows(seed, case["s"], case["kv"], case["d"])
        if own:
            import tensorlogic_amd as tl
            st["k"], st["v"] = _dev().tensor(_host(k)), _dev().tensor(_host(v))
            st["cache"] = tl.KVCache(_dev(), 1, case["s"], case["kv"], case["d"], tl.Q8_0)
        else:
            st["k"], st["v"] = k, v
    elif case["kind"] == "attention":
        k, v = _kv_rows(seed, case["past"] + case["s"], case["kv"], case["d"])
        q = _queries(case, seed)
        if own:   # the cache that the program has filled
            import tensorlogic_amd as tl
            st["q"] = _dev().tensor(_host(q))
            st["cache"] = tl.KVCache(_dev(), 1, k.shape[0], case["kv"], case["d"], tl.Q8_0)
            st["cache"].set(0, _dev().tensor(_host(k)), _dev().tensor(_host(v)))
        else:
            st["q"], st["k"], st["v"] = q, _quantise(k), _quantise(v)
    elif case["kind"] == "moe":
        x, router, mats = _moe_inputs(case, seed)
        if own:
            import tensorlogic_amd as tl
            dev, types = _dev(), {"q4_0": tl.Q4_0, "q8_0": tl.Q8_0}
            st["x"], st["router"] = dev.tensor(_host(x)), dev.tensor(_host(router))
            st["mats"] = [dev.tensor(_host(b.reshape(n, -1).view(torch.float16))) if case["wt"] == "f16"
                          else dev.quantized(_host(b), (n, c), types[case["wt"]]) for n, c, b in mats]
        else:
            st["x"], st["router"], st["mats"] = x, router, mats
    else:
        x, ids = _logits(case, seed)
        if own:
            import tensorlogic_amd as tl
            st["x"] = _dev().tensor(_host(x), tl.F16 if case["dtype"] == "f16" else tl.F32)
            st["ids"] = _dev().tensor(_host(ids), tl.I32)
        else:
            st["x"], st["ids"] = x, ids
    if own:
        _dev().sync()
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
class OnDevice(dict):
    """Outputs left on the device: an entry is read back when it is looked at."""

    def __getitem__(self, key):
        v = super().__getitem__(key)
        return (v() if callable(v) else v).numpy()


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        import tensorlogic_amd as tl
        if kind == "kv_write":
            cache = state["cache"]
            cache.set(0, state["k"], state["v"])
            return OnDevice(k=lambda: cache.get_k(0), v=lambda: cache.get_v(0))   # the cache is the output
        if kind == "attention":
            return OnDevice(out=state["cache"].attention(state["q"], 0, 1.0 / math.sqrt(case["d"])))
        if kind == "moe":
            gate, up, down = state["mats"]
            return OnDevice(y=tl.moe(state["x"], state["router"], gate, up, down, case["top"], case["norm"]))
        logprob, entropy, top_logprob, top_ids = tl.token_logprobs(state["x"], state["ids"], case["top"])
        if case["top"]:
            return OnDevice(logprob=logprob, entropy=entropy, top_logprob=top_logprob, top_ids=top_ids)
        return OnDevice(logprob=logprob, entropy=entropy)
    if kind == "kv_write":
        return {n: _values(*_quantise(state[n])).half() for n in ("k", "v")}
    if kind == "attention":
        return {"out": _attend(state["q"], _values(*state["k"]), _values(*state["v"]), case["past"])}
    if kind == "moe":
        return {"y": _moe(case, state["x"], state["router"], state["mats"])}
    return _logprobs(state["x"].float(), state["ids"], case["top"])


def _quantise(x):
    """Rows [n, kv, d] as the cache keeps them: whole blocks in 8 bits [b, 32, kv, d] with a scale for each
    head, amax / 127, and the rows past them as they are."""
    n = x.shape[0] // BLOCK * BLOCK
    b = x[:n].float().reshape(-1, BLOCK, *x.shape[1:])
    amax = b.abs().amax((1, 3), keepdim=True)
    full = torch.full_like(amax, 127.0)
    scale = torch.where(amax > 0, amax / full, 1.0)
    inv = torch.where(amax > 0, full / amax, 0.0)
    return torch.round(b * inv).to(torch.int8), scale, x[n:]


def _values(q, scale, rest):
    """The rows that _quantise's answer stands for, in 32 bits."""
    return torch.cat([(q.float() * scale).reshape(-1, *rest.shape[1:]), rest.float()])


def _attend(q, k, v, past):
    s, h, d = q.shape
    j, kv = k.shape[0], k.shape[1]
    g = h // kv
    qg = q.float().reshape(s, kv, g, d).permute(1, 2, 0, 3).reshape(kv, g * s, d)
    sc = torch.matmul(qg, k.permute(1, 2, 0).contiguous()) * (1.0 / math.sqrt(d))
    sc = sc.reshape(kv, g, s, j)
    later = torch.arange(j, device=q.device)[None, :] > torch.arange(s, device=q.device)[:, None] + past
    sc = sc.masked_fill(later, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(kv, g * s, j)
    out = torch.matmul(p, v.permute(1, 0, 2).contiguous()).reshape(kv, g, s, d)
    return out.permute(2, 0, 1, 3).reshape(s, h, d).half()


def _gates(x, router, top, norm):
    """What each expert counts for each token [m, experts]: zero for those not among the top (ties: the first)."""
    logits = x @ router.T
    _, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    mask = torch.zeros_like(logits).scatter_(1, order[:, :top], 1.0)
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e * mask / ((e * mask) if norm else e).sum(-1, keepdim=True)


def _moe(case, x, router, mats):
    m, e, i, k, wt = case["m"], case["experts"], case["i"], case["k"], case["wt"]
    gate, up, down = (_weights(b, wt, n, c).float() for n, c, b in mats)
    x = x.float()
    g = _gates(x, router.float(), case["top"], case["norm"])
    a = x @ gate.T
    h = (a / (1 + torch.exp(-a)) * (x @ up.T)).reshape(m, e, i) * g[:, :, None]
    return (h.reshape(m, e * i) @ down.reshape(e, k, i).permute(0, 2, 1).reshape(e * i, k)).half()


def _top(x, n):
    """The n largest of each row and where they are, ties to the lowest index: 64-bit keys without a tie."""
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    at = (torch.topk(key - torch.arange(x.shape[1], device=x.device), n).indices).long()
    return x.gather(1, at), at.to(torch.int32)


def _logprobs(x, ids, n):
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    norm = (m + torch.log(z)).reshape(-1)
    mean = (torch.where(e > 0, e * (x - m), 0.0).sum(-1, keepdim=True) / z).reshape(-1)   # of x - m
    out = {"logprob": x.gather(1, ids.long()[:, None])[:, 0] - norm, "entropy": torch.log(z).reshape(-1) - mean}
    if n:
        val, at = _top(x, n)
        out.update(top_logprob=val - norm[:, None], top_ids=at)
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "kv_write":
        s, row = case["s"], case["kv"] * case["d"]
        whole = s // BLOCK * BLOCK
        return {"bytes": 2.0 * (2 * s * row + whole * row + whole / BLOCK * 4 * case["kv"] + 2 * (s - whole) * row),
                "flops": 4.0 * whole * row}
    if case["kind"] == "attention":
        s, past, h, kv, d = case["s"], case["past"], case["heads"], case["kv"], case["d"]
        j = past + s
        whole = j // BLOCK * BLOCK
        return {"bytes": 2.0 * kv * (whole * d + whole / BLOCK * 4 + 2 * (j - whole) * d) + 4.0 * s * h * d,
                "flops": 4.0 * h * d * (s * past + s * (s + 1) / 2)}
    if case["kind"] == "moe":
        m, k, i, e, t = case["m"], case["k"], case["i"], case["experts"], case["top"]
        used = e * (1 - (1 - t / e) ** m)   # experts that some token chooses
        return {"bytes": used * 3 * i * k * BYTES[case["wt"]] + 2.0 * e * k + 4.0 * m * k,
                "flops": 6.0 * m * t * i * k + 2.0 * m * e * k}
    r, v, n = case["rows"], case["v"], case["top"]
    return {"bytes": r * (v * (2.0 if case["dtype"] == "f16" else 4.0) + 12 + 8 * n), "flops": 5.0 * r * v}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "kv_write":
        return dict(zip("kv", (_stored64(t) for t in _kv_rows(seed, case["s"], case["kv"], case["d"]))))
    if case["kind"] == "attention":
        k, v = (_stored64(t) for t in _kv_rows(seed, case["past"] + case["s"], case["kv"], case["d"]))
        q = _queries(case, seed).double()
        out = torch.empty_like(q)
        share = case["heads"] // case["kv"]
        seen = torch.arange(k.shape[0], device=q.device)[None, :] <= case["past"] + torch.arange(q.shape[0], device=q.device)[:, None]
        for h in range(case["heads"]):
            sc = q[:, h] @ k[:, h // share].T.contiguous() / math.sqrt(case["d"])
            out[:, h] = torch.softmax(torch.where(seen, sc, -math.inf), -1) @ v[:, h // share].contiguous()
        return {"out": out}
    if case["kind"] == "moe":
        return _moe64(case, seed)
    x, ids = _logits(case, seed)
    x = x.double()
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    p = lp.exp()
    out = {"logprob": torch.stack([row[t] for row, t in zip(lp, ids.tolist())]),
           "entropy": -(torch.where(p > 0, p * lp, 0.0)).sum(-1)}
    if case["top"]:
        val, at = torch.sort(lp, dim=-1, descending=True, stable=True)
        out.update(top_logprob=val[:, :case["top"]], top_ids=at[:, :case["top"]].to(torch.int32))
    return out


def _stored64(x):
    """What the cache holds of the rows x, block by block, in 64 bits."""
    out = x.double()
    for b in range(x.shape[0] // BLOCK):
        rows = out[b * BLOCK:(b + 1) * BLOCK]
        step = (rows.abs().amax((0, 2)) / 127)[None, :, None]
        out[b * BLOCK:(b + 1) * BLOCK] = torch.where(step > 0, torch.round(rows / step) * step, 0.0)
    return out


def _moe64(case, seed):
    x, router, mats = _moe_inputs(case, seed)
    x, i, k = x.double(), case["i"], case["k"]
    p = torch.softmax(x @ router.double().T, -1)
    gate, up, down = (_weights(b, case["wt"], n, c) for n, c, b in mats)
    y = torch.zeros_like(x)
    for t in range(case["m"]):
        chosen = sorted(range(case["experts"]), key=lambda e: -p[t, e].item())[:case["top"]]
        total = sum(p[t, e] for e in chosen) if case["norm"] else 1.0
        for e in chosen:
            a = gate[e * i:(e + 1) * i].double() @ x[t]
            h = a * torch.sigmoid(a) * (up[e * i:(e + 1) * i].double() @ x[t])
            y[t] += p[t, e] / total * (down[e * k:(e + 1) * k].double() @ h)
    return {"y": y}
