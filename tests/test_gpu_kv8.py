"""The 8-bit KV cache (csrc/kernels_kv8.hip): what it holds, bit for bit, and
the attention that reads it against 64-bit arithmetic on what it holds."""
import numpy as np
import pytest

from tensorlogic_amd import F32, Q8_0, Device, KVCache, TLHipError

pytestmark = pytest.mark.gpu

HEADS = [(1, 1, 32), (8, 2, 64), (4, 4, 80), (6, 3, 96), (8, 1, 128), (2, 2, 256)]


def rows(seed, n, kv, d):
    """K and V rows; heads of different size, so a block's scale cannot be its neighbour's."""
    r = np.random.default_rng([seed, n, kv, d])
    size = 0.05 * 4.0 ** np.arange(kv)[None, :, None]
    return tuple((r.standard_normal((n, kv, d)) * np.minimum(size, 100)).astype(np.float16) for _ in range(2))


def held(x):
    """The cache's values of rows x, in f32 with the kernel's operations (all exactly rounded): f64 products."""
    out = x.astype(np.float64)
    f = np.float32
    for b in range(x.shape[0] // 32):
        for h in range(x.shape[1]):
            blk = x[32 * b:32 * b + 32, h].astype(f)
            if not np.isfinite(blk).all():
                out[32 * b:32 * b + 32, h] = np.nan
                continue
            a = np.abs(blk).max()
            if a > 0:
                q = np.rint(blk * (f(127) / a)) + f(0)   # (an int8 has no -0)
                out[32 * b:32 * b + 32, h] = q.astype(np.float64) * float(a / f(127))
    return out


def as_f16(v):
    """f16 of the f32 products q * scale, as the read-back rounds them."""
    with np.errstate(over="ignore"):
        return v.astype(np.float32).astype(np.float16)


def attend(q, k, v, scale):
    """Causal attention of the last S positions in 64 bits, and how far the kernel may be from it."""
    S, H, D = q.shape
    J, kv, _ = k.shape
    q, u = q.astype(np.float64), 2.0 ** -24
    out, tol = np.empty_like(q), np.empty_like(q)
    for h in range(H):
        kk, vv = k[:, h // (H // kv)], v[:, h // (H // kv)]
        sc = (q[:, h] @ kk.T) * scale
        dsc = (D + 6) * u * (np.abs(q[:, h]) @ np.abs(kk).T) * abs(scale) + 4 * u * (np.abs(sc) + 40)
        seen = np.arange(J)[None, :] <= np.arange(S)[:, None] + J - S
        p = np.where(seen, np.exp(np.where(seen, sc, -np.inf) - np.where(seen, sc, -np.inf).max(1, keepdims=True)), 0)
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ vv
        absum = p @ np.abs(vv)
        worst = np.where(seen, dsc, 0).max(1, keepdims=True)
        # the result's and the weights' rounding to f16 (2^-11 each; a weight
        # below 2^-14 of the largest: 2^-25 of it), the scores' error on each
        # weight and on their sum, and n f32 sums
        tol[:, h] = (2.0 ** -11 * (np.abs(out[:, h]) + absum) + 2 * worst * absum + J * u * absum
                     + J * 2.0 ** -25 * np.abs(vv).max() + 2.0 ** -25)
    return out, tol


def check(got, q, k, v, scale, what):
    ref, tol = attend(q, held(k), held(v), scale)
    bad = ~(np.abs(got.astype(np.float64) - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                           float(np.nanmax(np.abs(got.astype(np.float64) - ref) / tol)))


@pytest.mark.parametrize("H,kv,D", HEADS)
@pytest.mark.parametrize("n", [1, 31, 32, 33, 95, 200])
def test_holds_what_it_says(dev, H, kv, D, n):
    k, v = rows(1, n, kv, D)
    k[min(n - 1, 5)] = 0
    if n >= 64:
        v[32:64] = 0          # a block of zeros
        k[0, 0, 0] = 65504.0
        k[1, 0, 1] = 6e-8     # the largest and the smallest f16
    c = KVCache(dev, 1, 256, kv, D, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    assert c.len(0) == n
    for got, x in ((c.get_k(0), k), (c.get_v(0), v)):
        assert got.shape == (n, kv, D)
        assert np.array_equal(got.numpy().view(np.uint16), as_f16(held(x)).view(np.uint16))


@pytest.mark.parametrize("kv,D", [(2, 64), (3, 80), (1, 256)])
def test_depends_on_the_rows_not_on_the_calls(dev, kv, D):
    n = 150
    k, v = rows(2, n, kv, D)
    whole = KVCache(dev, 2, 160, kv, D, Q8_0)
    whole.set(1, dev.tensor(k), dev.tensor(v))
    ref = whole.get_k(1).numpy(), whole.get_v(1).numpy()
    for parts in ([1] * n, [33, 1, 30, 64, 22], [31, 2, 95, 22], [32, 32, 86], [5, 0, 145]):
        c = KVCache(dev, 2, 160, kv, D, Q8_0)
        c.set(1, dev.tensor(v[:40]), dev.tensor(k[:40]))   # other contents first
        at = 0
        for i, m in enumerate(parts):
            a = dev.tensor(k[at:at + m]), dev.tensor(v[at:at + m])
            if m:
                (c.append if i else c.set)(1, *a)
            at += m
            if at:
                assert c.len(1) == at and c.len(0) == 0
        got = c.get_k(1).numpy(), c.get_v(1).numpy()
        assert all(np.array_equal(g.view(np.uint16), r.view(np.uint16)) for g, r in zip(got, ref)), parts


def test_read_back_is_a_copy(dev):
    k, v = rows(3, 40, 2, 64)
    c = KVCache(dev, 1, 100, 2, 64, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    a = c.get_k(0)
    c.append(0, dev.tensor(v), dev.tensor(k))
    c.set(0, dev.tensor(v), dev.tensor(k))
    assert np.array_equal(a.numpy().view(np.uint16), as_f16(held(k)).view(np.uint16))


# one row, rows that share waves, whole tiles and rests; more rows than a wave takes
@pytest.mark.parametrize("H,kv,D", HEADS)
@pytest.mark.parametrize("S,past", [(1, 0), (1, 30), (1, 31), (1, 32), (1, 700), (2, 31), (5, 60), (33, 0), (64, 1), (70, 200), (150, 7)])
def test_attention(dev, H, kv, D, S, past):
    n = past + S
    k, v = rows(4, n, kv, D)
    k = (k / np.abs(k).max() * 3).astype(np.float16)
    q = np.random.default_rng([S, past]).standard_normal((S, H, D)).astype(np.float16)
    c = KVCache(dev, 1, n + 40, kv, D, Q8_0)
    if past:
        c.set(0, dev.tensor(k[:past]), dev.tensor(v[:past]))
        c.append(0, dev.tensor(k[past:]), dev.tensor(v[past:]))
    else:
        c.set(0, dev.tensor(k), dev.tensor(v))
    got = c.attention(dev.tensor(q), 0, D ** -0.5).numpy()
    check(got, q, k, v, D ** -0.5, f"S{S} past{past} {H}/{kv} D{D}")


@pytest.mark.parametrize("H,kv,D,S,past", [(32, 4, 64, 300, 0), (32, 32, 80, 40, 100), (16, 1, 64, 1, 5000), (8, 8, 128, 1, 4111),
                                           (40, 1, 64, 1, 500), (128, 2, 32, 3, 100), (4, 1, 64, 700, 1300), (64, 64, 64, 17, 333),
                                           # enough rows for a wave to take all keys of its own
                                           (256, 8, 32, 260, 37), (256, 8, 64, 260, 300), (512, 4, 80, 135, 1), (256, 16, 128, 260, 0), (256, 1, 256, 131, 20),
                                           # few rows of many heads: as many workgroups
                                           (1024, 1024, 32, 40, 5), (1024, 1024, 64, 33, 0), (1024, 1024, 64, 17, 50), (1024, 1024, 80, 33, 2),
                                           (2048, 1024, 96, 20, 0), (1024, 1024, 128, 33, 40), (1024, 512, 256, 40, 3), (1024, 1024, 64, 1, 300)])
def test_attention_larger(dev, H, kv, D, S, past):
    test_attention(dev, H, kv, D, S, past)


@pytest.mark.parametrize("S,past", [(1, 40), (1, 100), (70, 30)])
def test_scores_far_apart(dev, S, past):
    """Keys and values of very different size, a head of zeros, scores past 2^10 and a negative scale."""
    H, kv, D, n = 8, 4, 64, S + past
    r = np.random.default_rng(n)
    k = r.standard_normal((n, kv, D)) * 2.0 ** r.integers(-8, 5, (n, kv, 1))
    v = r.standard_normal((n, kv, D)) * 2.0 ** r.integers(-14, 12, (n // 32 + 1, kv, 1)).repeat(32, 0)[:n]
    k[:, 2], v[:, 3] = 0, 0
    k, v = k.astype(np.float16), v.astype(np.float16)
    q = (r.standard_normal((S, H, D)) * 16).astype(np.float16)
    c = KVCache(dev, 1, n, kv, D, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    for scale in (0.125, -1.0, 0.0):
        check(c.attention(dev.tensor(q), 0, scale).numpy(), q, k, v, scale, f"scale {scale}")


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_non_finite_values_stay_where_they_are_seen(dev, bad):
    """A key and a value in a whole block, a value past the last whole block:
    queries before the block (the row) and other heads are untouched."""
    H, kv, D, n = 4, 4, 64, 90
    k, v = rows(6, n, kv, D)
    k = (k / np.abs(k).max(axis=(0, 2), keepdims=True)).astype(np.float16)
    k[40, 0, 3], v[50, 1, 5], v[80, 2, 7] = bad, bad, bad
    q = np.random.default_rng(6).standard_normal((n, H, D)).astype(np.float16)
    c = KVCache(dev, 1, 96, kv, D, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    assert np.isnan(c.get_k(0).numpy()[32:64, 0]).all() and np.isnan(c.get_v(0).numpy()[80, 2]).all()
    got = c.attention(dev.tensor(q), 0, 0.125).numpy()
    nan = np.isnan(got).all(-1)
    want = np.zeros((n, H), bool)
    want[32:, 0] = want[32:, 1] = want[80:, 2] = True
    assert np.array_equal(nan, want) and np.isfinite(got[~want]).all()
    clean = KVCache(dev, 1, 96, kv, D, Q8_0)
    k2, v2 = np.where(np.isfinite(k), k, 0).astype(np.float16), np.where(np.isfinite(v), v, 0).astype(np.float16)
    clean.set(0, dev.tensor(k2), dev.tensor(v2))
    ref = clean.attention(dev.tensor(q), 0, 0.125).numpy()
    # (the first block and heads without such a value hold the same in both)
    assert np.array_equal(got[:32], ref[:32]) and np.array_equal(got[:, 3], ref[:, 3]) and np.array_equal(got[:80, 2], ref[:80, 2])
    # the row past the last whole block is quantised with its block: NaN there too
    c.append(0, dev.tensor(k2[:6]), dev.tensor(v2[:6]))
    assert np.isnan(c.get_v(0).numpy()[64:96, 2]).all() and np.isfinite(c.get_v(0).numpy()[:, 3]).all()


@pytest.mark.parametrize("S,past", [(70, 30), (9, 25)])
def test_rows_before_a_bad_block_in_one_tile_of_rows(dev, S, past):
    """Queries on both sides of a block's start: those before it see nothing of its NaN."""
    n = S + past
    for which in (0, 1):
        kv = list(rows(11, n, 1, 64))
        kv[which][33, 0, 5] = np.nan if n < 64 else np.inf   # (in f16 still, an infinite key's score is what it is)
        kv[0][:32] = kv[0][:32] / 8
        q = np.random.default_rng(11).standard_normal((S, 2, 64)).astype(np.float16)
        c = KVCache(dev, 1, 128, 1, 64, Q8_0)
        c.set(0, dev.tensor(kv[0]), dev.tensor(kv[1]))
        got = c.attention(dev.tensor(q), 0, 0.125).numpy()
        first = max(32, 33 if n < 64 else 32) - past   # (a bad row past the last whole block is one row)
        assert np.isfinite(got[:first]).all() and np.isnan(got[first:]).all()
        check(got[:first], q[:first], kv[0][:32], kv[1][:32], 0.125, "before") if first == 32 - past else None


@pytest.mark.parametrize("S,past,H,D", [(1, 0, 4, 64), (1, 190, 4, 64), (60, 140, 4, 64), (100, 140, 256, 64), (140, 100, 512, 64), (140, 100, 512, 80)])
@pytest.mark.parametrize("power", [20, 27, 40])
def test_values_of_blocks_far_apart(dev, S, past, H, D, power):
    """Blocks of V whose sizes lie up to 2^40 apart (zeros among them), seen with weights alike: each
    weight counts with its full precision in the sum, and the large values with theirs in the result."""
    n = S + past
    k, v = rows(12, n, 2, D)
    size = np.array([8, 8 - power, 8 - power, 8 - power, None, 8 - power // 2, -14], dtype=object)
    for b in range((n + 31) // 32):
        e = size[b % 7]
        blk = v[32 * b:32 * b + 32].astype(np.float64)
        blk = blk / np.abs(blk).max(axis=(0, 2), keepdims=True)
        v[32 * b:32 * b + 32] = 0 if e is None else np.maximum(np.abs(blk) * 2.0 ** max(e, -24), 2.0 ** -24) * np.sign(blk)
    q = (np.random.default_rng(n).standard_normal((S, H, D)) / 4).astype(np.float16)
    c = KVCache(dev, 1, n, 2, D, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    got = c.attention(dev.tensor(q), 0, 0.125).numpy()
    kk, vv = held(k), held(v)
    ref, tol = attend(q, kk, vv, 0.125)
    for h in range(H):
        sc = np.where(np.arange(n)[None, :] <= np.arange(S)[:, None] + past, (q[:, h].astype(np.float64) @ kk[:, h // (H // 2)].T) * 0.125, -np.inf)
        p = np.exp(sc - sc.max(1, keepdims=True))
        assert p[p > 0].min() > 2.0 ** -12   # all weights are of normal size: attend()'s term for the smaller ones falls away
        p /= p.sum(1, keepdims=True)
        absum = p @ np.abs(vv[:, h // (H // 2)])
        dsc = (D + 6) * 2.0 ** -24 * (np.abs(q[:, h].astype(np.float64)) @ np.abs(kk[:, h // (H // 2)]).T) * 0.125 + 2.0 ** -22 * (np.abs(np.where(sc > -np.inf, sc, 0)) + 40)
        t = 2.0 ** -11 * (np.abs(ref[:, h]) + 2 * absum) + (2 * dsc.max(1, keepdims=True) + n * 2.0 ** -24) * absum + 2.0 ** -25
        assert (np.abs(got[:, h] - ref[:, h]) <= t).all(), float((np.abs(got[:, h] - ref[:, h]) / t).max())


def test_an_infinite_query_spoils_its_row_only(dev):
    k, v = rows(7, 60, 2, 64)
    q = np.random.default_rng(7).standard_normal((20, 4, 64)).astype(np.float16)
    c = KVCache(dev, 1, 64, 2, 64, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    ref = c.attention(dev.tensor(q), 0, 0.125).numpy()
    q[7, 2, 0] = np.inf
    got = c.attention(dev.tensor(q), 0, 0.125).numpy()
    mask = np.ones((20, 4), bool)
    mask[7, 2] = False
    assert np.array_equal(got[mask], ref[mask]) and not np.isfinite(got[7, 2]).all()


def test_same_bits_each_time_and_in_place(dev):
    k, v = rows(8, 3000, 2, 64)
    c = KVCache(dev, 1, 3000, 2, 64, Q8_0)
    c.set(0, dev.tensor(k), dev.tensor(v))
    for S in (1, 9, 130):
        q = dev.tensor(np.random.default_rng(S).standard_normal((S, 16, 64)).astype(np.float16))
        a = [c.attention(q, 0, 0.125).numpy().view(np.uint16) for _ in range(3)]
        assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])
        from tensorlogic_amd._lib import call
        call("tlhip_attention_decode" if S == 1 else "tlhip_attention_prefill", dev.h, q.h, c.h, 0, 0.125, q.h)
        assert np.array_equal(q.numpy().view(np.uint16), a[0])


def test_the_longest_cache(dev):
    """65536 positions; blocks past 2^31 bytes from the layer's start would need more memory than a test takes."""
    n, kv, D = 65536, 1, 64
    k, v = rows(9, n, kv, D)
    c = KVCache(dev, 1, n, kv, D, Q8_0)
    c.set(0, dev.tensor(k[:-1]), dev.tensor(v[:-1]))
    c.append(0, dev.tensor(k[-1:]), dev.tensor(v[-1:]))
    q = np.random.default_rng(9).standard_normal((1, 8, D)).astype(np.float16)
    check(c.attention(dev.tensor(q), 0, 0.125).numpy(), q, k, v, 0.125, "65536 keys")
    with pytest.raises(TLHipError) as e:
        c.append(0, dev.tensor(k[:1]), dev.tensor(v[:1]))
    assert e.value.kind == "IndexOutOfBounds" and c.len(0) == n


def test_refusals(dev):
    def kind(f):
        with pytest.raises(TLHipError) as e:
            f()
        return e.value.kind
    for d in (8, 40, 63, 72, 160, 512):
        assert kind(lambda: KVCache(dev, 1, 64, 1, d, Q8_0)) == "InvalidDimension"
    assert kind(lambda: KVCache(dev, 1, 65537, 1, 64, Q8_0)) == "InvalidDimension"
    assert kind(lambda: KVCache(dev, 1, 64, 1025, 64, Q8_0)) == "InvalidDimension"
    c = KVCache(dev, 2, 64, 2, 64, Q8_0)
    t = dev.empty((3, 2, 64))
    assert kind(lambda: c.get_k(0)) == "InvalidOperation"                       # empty
    assert kind(lambda: c.attention(dev.empty((1, 2, 64)), 0, 1.0)) == "InvalidDimension"
    assert kind(lambda: c.set(2, t, t)) == "IndexOutOfBounds"
    assert kind(lambda: c.set(0, dev.empty((3, 2, 64), F32), dev.empty((3, 2, 64), F32))) == "DtypeError"
    assert kind(lambda: c.set(0, t, dev.empty((2, 2, 64)))) == "ShapeMismatch"
    assert kind(lambda: c.set(0, dev.empty((65, 2, 64)), dev.empty((65, 2, 64)))) == "IndexOutOfBounds"
    c.set(0, t, t)
    assert kind(lambda: c.attention(dev.empty((4, 2, 64)), 0, 1.0)) == "InvalidDimension"   # more rows than positions
    assert kind(lambda: c.attention(dev.empty((1, 3, 64)), 0, 1.0)) == "ShapeMismatch"
    assert kind(lambda: c.attention(dev.empty((1, 2, 32)), 0, 1.0)) == "ShapeMismatch"
    assert kind(lambda: c.attention(dev.empty((1, 2, 64), F32), 0, 1.0)) == "DtypeError"
    other = Device(0)
    try:
        u = other.empty((1, 2, 64))
        other.sync()
        from tensorlogic_amd._lib import call
        assert kind(lambda: call("tlhip_kvcache_append", other.h, c.h, 0, u.h, u.h)) == "InvalidArgument"
        assert kind(lambda: call("tlhip_attention_decode", other.h, u.h, c.h, 0, 1.0, u.h)) == "InvalidArgument"
        del u
    finally:
        other.close()
    assert c.len(0) == 3
