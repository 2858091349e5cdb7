"""moe (csrc/kernels_moe.hip) against 64-bit arithmetic on the f16 weights
that the packed types stand for."""
import numpy as np
import pytest

from tensorlogic_amd import F16, F32, Q4_0, Q6_K, Q8_0, TLHipError, moe

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
MAX_U = 2.0 ** -11


def pack(w, qt):
    """GGUF bytes of w and the f16 values they stand for."""
    if qt == F16:
        h = w.astype(np.float16)
        return h, h.astype(np.float64)
    b = w.astype(np.float32).reshape(-1, 32)
    if qt == Q8_0:
        d = (np.abs(b).max(1) / 127).astype(np.float16)
        q = np.clip(np.rint(b / np.maximum(d.astype(np.float32), 1e-7)[:, None]), -127, 127)
        raw = np.concatenate([d[:, None].view(np.uint8), q.astype(np.int8).view(np.uint8)], 1)
    else:
        d = (np.take_along_axis(b, np.abs(b).argmax(1)[:, None], 1)[:, 0] / -8).astype(np.float16)
        q = np.clip(np.rint(b / np.where(d == 0, 1, d).astype(np.float32)[:, None]) + 8, 0, 15)
        qq = q.astype(np.uint8)
        raw = np.concatenate([d[:, None].view(np.uint8), qq[:, :16] | (qq[:, 16:] << 4)], 1)
        q = q - 8
    val = (q.astype(np.float32) * d.astype(np.float32)[:, None]).astype(np.float16)
    return raw, val.astype(np.float64).reshape(w.shape)


def case(seed, E, K, I, gu, dn):
    r = np.random.default_rng([seed, E, K, I])
    router = (r.standard_normal((E, K)) * 1.5 / np.sqrt(K)).astype(np.float16)
    mats = [pack(r.standard_normal(s) * g / np.sqrt(s[1]), t) for s, g, t in
            (((E * I, K), 2.0, gu), ((E * I, K), 1.0, gu), ((E * K, I), 1.0, dn))]
    return router, mats


def upload(dev, raw, shape, qt):
    return dev.tensor(raw) if qt == F16 else dev.quantized(raw, shape, qt)


def reference(x, router, mats, E, top, norm):
    """y in 64 bits and how far the kernel may be from it."""
    (_, gate), (_, up), (_, down) = mats
    M, K = x.shape
    I = gate.shape[0] // E
    x = x.astype(np.float64)
    l = x @ router.astype(np.float64).T
    # (the router sums in 64 lanes: no term goes through more than K / 64 + 6 sums, less than this)
    dl = (K / 32 + 16) * U * (np.abs(x) @ np.abs(router.astype(np.float64)).T)
    y, tol = np.zeros((M, K)), np.zeros((M, K))
    for m in range(M):
        chosen = np.argsort(-l[m], kind="stable")[:top]
        rest = np.setdiff1d(np.arange(E), chosen)
        if len(rest):   # the inputs leave no doubt about who is chosen
            assert l[m, chosen].min() - l[m, rest].max() > 4 * dl[m].max() or l[m, chosen].min() == l[m, rest].max()
        p = np.exp(l[m] - l[m].max())
        g = p[chosen] / (p[chosen].sum() if norm else p.sum())
        for e, ge in zip(chosen, g):
            wg, wu, wd = gate[e * I:(e + 1) * I], up[e * I:(e + 1) * I], down[e * K:(e + 1) * K]
            a, u = wg @ x[m], wu @ x[m]
            da, du = (K + 2) * U * (np.abs(wg) @ np.abs(x[m])), (K + 2) * U * (np.abs(wu) @ np.abs(x[m]))
            s = 1 / (1 + np.exp(-a))
            h = ge * a * s * u
            # |d silu| <= 1.1; exp and reciprocal within a few ulps of an
            # exponent rounded to f32; the gate's own error; and h as what
            # the second product takes of it, no less than 2^-21 of it
            dh = ge * (1.1 * da * np.abs(u) + np.abs(a * s) * du) + np.abs(h) * ((8 + 2 * np.abs(a)) * U + 4 * dl[m].max() + 8 * U + 2.0 ** -21)
            y[m] += wd @ h
            tol[m] += np.abs(wd) @ dh + (I * top + 4) * U * (np.abs(wd) @ np.abs(h))
    return y, tol + MAX_U * np.abs(y) + 2.0 ** -25


def run(dev, seed, M, E, K, I, top, norm, gu, dn, x=None):
    router, mats = case(seed, E, K, I, gu, dn)
    if x is None:
        x = np.random.default_rng([seed, M]).standard_normal((M, K)).astype(np.float16)
    w = [upload(dev, raw, s, t) for (raw, _), s, t in zip(mats, ((E * I, K), (E * I, K), (E * K, I)), (gu, gu, dn))]
    got = moe(dev.tensor(x), dev.tensor(router), *w, top, norm).numpy()
    ref, tol = reference(x, router, mats, E, top, norm)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), float((np.abs(got - ref) / tol).max()))


@pytest.mark.parametrize("gu,dn", [(F16, F16), (Q4_0, Q4_0), (Q8_0, Q8_0), (Q4_0, Q8_0), (Q8_0, F16), (F16, Q4_0)])
@pytest.mark.parametrize("M,E,K,I,top", [(1, 8, 256, 512, 2), (1, 1, 32, 32, 1), (3, 5, 96, 160, 3), (7, 64, 128, 64, 6), (16, 4, 288, 96, 4),
                                         (17, 3, 64, 1056, 1), (33, 8, 160, 224, 2)])
def test_against_64_bits(dev, gu, dn, M, E, K, I, top):
    run(dev, 1, M, E, K, I, top, (M + E) % 2 == 0, gu, dn)


@pytest.mark.parametrize("gu,dn", [(F16, F16), (Q4_0, Q8_0), (Q8_0, Q4_0)])
@pytest.mark.parametrize("M,E,K,I,top", [(7, 4, 2048, 96, 2), (8, 3, 1088, 224, 3), (9, 4, 2048, 64, 3), (17, 3, 1024, 160, 1),
                                         (24, 64, 512, 64, 6), (33, 8, 352, 224, 2), (40, 5, 416, 96, 2), (130, 2, 160, 96, 1)])
def test_more_workgroups_than_run_at_once(dev, gu, dn, M, E, K, I, top):
    run(dev, 6, M, E, K, I, top, M % 2 == 0, gu, dn)


@pytest.mark.parametrize("M,E,K,I,top,gu", [(1, 8, 2048, 5632, 2, Q4_0), (13, 8, 1024, 1408, 2, Q8_0), (70, 16, 512, 320, 4, Q4_0), (2, 256, 64, 64, 32, F16),
                                            (5, 2, 4096, 32, 2, Q8_0), (4, 2, 32, 4128, 1, Q4_0), (300, 4, 96, 64, 2, Q8_0), (600, 2, 32, 32, 1, F16)])
def test_larger(dev, M, E, K, I, top, gu):
    run(dev, 2, M, E, K, I, top, True, gu, gu)


@pytest.mark.parametrize("t", [F16, Q4_0, Q8_0])
@pytest.mark.parametrize("M", [1, 2, 9, 16, 17, 40])
@pytest.mark.parametrize("K,I", [(16384, 32), (32, 16384), (16384, 64), (96, 16352)])
def test_longest_rows(dev, t, M, K, I):
    """What a workgroup keeps in LDS is largest here.  (All experts where K is long: the bound of a sum
    of 16384 products leaves doubt about which two of three are chosen.)"""
    run(dev, 4, M, 3, K, I, 3 if K == 16384 else 2, False, t, t)


def test_all_tokens_choose_one_expert_and_the_same_row_twice(dev):
    r = np.random.default_rng(5)
    x = np.repeat(r.standard_normal((1, 128)), 40, 0).astype(np.float16)
    run(dev, 3, 40, 6, 128, 96, 2, True, Q4_0, Q4_0, x)


def test_ties_take_the_first_experts(dev):
    """All logits equal (x = 0 is no input here: y would be 0): equal router rows."""
    E, K, I = 70, 64, 32
    router, mats = case(7, E, K, I, F16, F16)
    router[:] = router[:1]
    x = np.random.default_rng(7).standard_normal((5, K)).astype(np.float16)
    w = [dev.tensor(m[0]) for m in mats]
    got = moe(dev.tensor(x), dev.tensor(router), *w, 3, True).numpy()
    ref, tol = reference(x, router, mats, E, 3, True)
    assert (np.abs(got - ref) <= tol).all()


def test_three_dims_in_place_and_same_bits(dev):
    E, K, I, M = 4, 64, 96, 9
    router, mats = case(8, E, K, I, F16, F16)
    x = np.random.default_rng(8).standard_normal((M, K)).astype(np.float16)
    flat = [dev.tensor(m[0]) for m in mats]
    deep = [dev.tensor(m[0].reshape(E, -1, m[0].shape[1])) for m in mats]
    t, rt = dev.tensor(x), dev.tensor(router)
    a = moe(t, rt, *flat, 2).numpy().view(np.uint16)
    assert np.array_equal(a, moe(t, rt, *deep, 2).numpy().view(np.uint16))
    from tensorlogic_amd._lib import call
    call("tlhip_moe", dev.h, t.h, rt.h, *[w.h for w in flat], 2, 1, t.h)
    assert np.array_equal(a, t.numpy().view(np.uint16))


def test_non_finite_rows_stay_alone(dev):
    E, K, I, M = 8, 64, 96, 20
    router, mats = case(9, E, K, I, Q8_0, Q8_0)
    x = np.random.default_rng(9).standard_normal((M, K)).astype(np.float16)
    w = [upload(dev, m[0], s, Q8_0) for m, s in zip(mats, ((E * I, K), (E * I, K), (E * K, I)))]
    ref = moe(dev.tensor(x), dev.tensor(router), *w, 2).numpy()
    x[3, 5], x[11, 0], x[12] = np.nan, np.inf, -np.inf
    got = moe(dev.tensor(x), dev.tensor(router), *w, 2).numpy()
    keep = np.ones(M, bool)
    keep[[3, 11, 12]] = False
    assert np.array_equal(got[keep].view(np.uint16), ref[keep].view(np.uint16))
    assert np.isnan(got[~keep]).all()


def test_no_tokens(dev):
    E, K, I = 2, 32, 32
    router, mats = case(10, E, K, I, F16, F16)
    assert moe(dev.empty((0, K)), dev.tensor(router), *[dev.tensor(m[0]) for m in mats], 1).shape == (0, K)


def test_refusals(dev):
    def kind(x=(3, 64), router=(4, 64), gate=(4 * 96, 64), up=(4 * 96, 64), down=(4 * 64, 96), top=2, types=(F16,) * 5):
        t = [dev.empty(s, d) for s, d in zip((x, router, gate, up, down), types)]
        with pytest.raises(TLHipError) as e:
            moe(*t, top)
        return e.value.kind
    assert kind(router=(4, 32)) == "ShapeMismatch"
    assert kind(gate=(4 * 96, 32)) == "ShapeMismatch"
    assert kind(gate=(4 * 64, 64)) == "ShapeMismatch"
    assert kind(gate=(4 * 96 + 1, 64), up=(4 * 96 + 1, 64)) == "ShapeMismatch"
    assert kind(down=(4 * 64, 64)) == "ShapeMismatch"
    assert kind(down=(4 * 32, 96)) == "ShapeMismatch"
    assert kind(gate=(2, 192, 64), up=(2, 192, 64)) == "ShapeMismatch"
    assert kind(x=(3, 40), router=(4, 40), gate=(4 * 96, 40), up=(4 * 96, 40), down=(4 * 40, 96)) == "InvalidDimension"
    assert kind(gate=(4 * 40, 64), up=(4 * 40, 64), down=(4 * 64, 40)) == "InvalidDimension"
    assert kind(gate=(0, 64), up=(0, 64), down=(4 * 64, 0)) == "InvalidDimension"
    assert kind(top=0) == "InvalidDimension" and kind(top=5) == "InvalidDimension"
    assert kind(router=(300, 64), gate=(300 * 32, 64), up=(300 * 32, 64), down=(300 * 64, 32)) == "InvalidDimension"
    assert kind(x=(64,)) == "InvalidOperation" and kind(router=(0, 64)) == "InvalidDimension"
    assert kind(types=(F32, F16, F16, F16, F16)) == "DtypeError" and kind(types=(F16, F32, F16, F16, F16)) == "DtypeError"
    assert kind(types=(F16, F16, Q4_0, Q8_0, F16)) == "ShapeMismatch"
    assert kind(x=(1, 256), router=(4, 256), gate=(4 * 32, 256), up=(4 * 32, 256), down=(4 * 256, 32),
                types=(F16, F16, Q6_K, Q6_K, F16)) == "DtypeError"
