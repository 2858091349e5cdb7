"""token_logprobs (csrc/kernels_logprobs.hip) against 64-bit arithmetic."""
import numpy as np
import pytest

from tensorlogic_amd import F16, F32, I32, Q8_0, TLHipError, token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, ids, n):
    """logprob, entropy, top_logprob, top_ids in 64 bits of rows x, and the first two's allowed error."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        z = e.sum(1, keepdims=True)
        lp = x - m - np.log(z)
        p = e / z
        h = -np.where(p > 0, p * lp, 0).sum(1)
        mean = np.where(p > 0, p * (m - x), 0).sum(1)
    none = ~((z[:, 0] > 0) & np.isfinite(z[:, 0]))
    lp[none] = np.nan
    h[none] = np.nan
    order = np.argsort(-x, axis=1, kind="stable")[:, :n]
    V = x.shape[1]
    got = np.full(len(x), np.nan)
    for i, t in enumerate(ids):
        if 0 <= t < V and not none[i]:
            got[i] = lp[i, t]
    top = np.take_along_axis(lp, order, 1)
    order[none] = -1
    # z: sums of at most V / 64 + 64 terms in a row, each from an exponent
    # rounded to 2^-24 of it, which weighs (m - x) p on the mean; then a
    # logarithm and two subtractions of what is left
    dz = U * (V / 64 + 64 + 4 * mean)
    with np.errstate(invalid="ignore"):
        tol = lambda v: dz[:, None] + 4 * U * (np.abs(v) + np.abs(np.log(z)))  # noqa: E731
        return got, h, top, order, tol(got[:, None])[:, 0], dz * (2 + mean) + 4 * U * (np.abs(h) + mean + np.log(z)[:, 0]), tol(top)


def close(got, ref, tol, what):
    # (two f32 logits can be further apart than f32 reaches: -inf is that log probability in f32)
    ref = np.where(np.abs(ref) > np.finfo(np.float32).max, np.copysign(np.inf, ref), ref)
    fine = np.isfinite(ref)
    assert np.array_equal(got[~fine], ref[~fine], equal_nan=True), what
    assert (np.abs(got[fine] - ref[fine]) <= tol[fine]).all(), (what, np.abs(got[fine] - ref[fine]).max())


def run(dev, x, ids, n, what):
    dt = F16 if x.dtype == np.float16 else F32
    outs = token_logprobs(dev.tensor(x, dt), dev.tensor(ids, I32), n)
    lp, h, top, at, tlp, th, tt = reference(np.atleast_2d(x), ids, n)
    close(outs[0].numpy(), lp, tlp, what + " logprob")
    close(outs[1].numpy(), h, th, what + " entropy")
    if n:
        assert np.array_equal(outs[3].numpy(), at), what + " top ids"
        close(outs[2].numpy(), top, tt, what + " top logprob")
    else:
        assert outs[2] is None and outs[3] is None


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,V,n", [(1, 1, 1), (1, 2, 2), (3, 7, 7), (2, 64, 64), (5, 255, 3), (4, 257, 64), (3, 1023, 20), (1, 32000, 5),
                                      (9, 32003, 20), (2, 51200, 0), (2, 51201, 64), (1, 151936, 10), (700, 500, 1), (1, 300001, 33)])
def test_against_64_bits(dev, dtype, rows, V, n):
    r = np.random.default_rng([rows, V])
    x = (r.standard_normal((rows, V)) * 3).astype(dtype)
    x[np.arange(rows), r.integers(0, V, rows)] += 12
    run(dev, x, r.integers(0, V, rows).astype(np.int32), n, f"{rows}x{V}")


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("V", [130, 4096, 33001])
def test_ties_and_orders(dev, dtype, V):
    """Equal logits, few values, sorted rows both ways, all of the largest close together, signed zeros."""
    r = np.random.default_rng(V)
    i = np.arange(V)
    x = np.stack([np.zeros(V), r.integers(-3, 4, V), -i * 0.01, i * 0.01, np.where(i // 64 == 1, 5 + i * 1e-2, 0),
                  np.where(i % 256 == 3, 9.0, -9.0), np.where(i % 2, 0.0, -0.0), np.full(V, -60000.0), np.where(i == V - 1, 3, -20)])
    x = x.astype(dtype)
    for n in (1, 20, 64):
        run(dev, x, r.integers(0, V, len(x)).astype(np.int32), n, f"V{V} n{n}")


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("V", [40, 5000, 60000])
def test_masked_and_non_finite_rows(dev, dtype, V):
    r = np.random.default_rng(V)
    x = (r.standard_normal((10, V)) * 3).astype(dtype)
    x[0, r.random(V) < 0.6] = -np.inf
    x[1] = -np.inf
    x[1, V // 2] = 1.0               # one token left
    x[2] = -np.inf
    x[2, [3, V - 1]] = 2.0           # fewer tokens than alternatives asked for
    x[3] = -np.inf                   # no distribution
    x[4, V - 1] = np.nan
    x[5, 0] = np.inf
    x[6] = np.finfo(dtype).min       # the type's lowest value is a logit
    x[7, :] = np.finfo(dtype).min
    x[7, 9] = np.finfo(dtype).max
    x[8, 1:] = -np.inf
    x[8, 0] = np.finfo(dtype).min
    ids = np.array([0, 0, V - 1, 1, 1, 1, 1, 9, 0, V - 1], np.int32)
    for n in (0, 5):
        run(dev, x, ids, n, f"V{V} n{n}")
    for bad in (-1, V, 2 ** 31 - 1, -2 ** 31):
        ids[:] = bad
        run(dev, x, ids, 3, f"id {bad}")


def test_forms(dev):
    """A single row without a rows axis, no ids, no rows; the same bits each time."""
    x = np.random.default_rng(0).standard_normal(1000).astype(np.float16)
    t = dev.tensor(x)
    run(dev, x, np.array([17], np.int32), 4, "1-D")
    lp, h, top, at = token_logprobs(t, None, 2)
    assert lp is None and h.shape == (1,) and top.shape == (1, 2) and at.dtype == I32
    for o in token_logprobs(dev.empty((0, 50)), dev.empty((0,), I32), 3):
        assert o.numpy().size == 0
    ids = dev.tensor(np.array([5], np.int32), I32)
    a, b = ([o.numpy().tobytes() for o in token_logprobs(t, ids, 9)] for _ in range(2))
    assert a == b


def test_refusals(dev):
    def kind(f):
        with pytest.raises(TLHipError) as e:
            f()
        return e.value.kind
    x, ids = dev.empty((3, 100)), dev.empty((3,), I32)
    assert kind(lambda: token_logprobs(x, ids, 65)) == "InvalidDimension"
    assert kind(lambda: token_logprobs(x, ids, -1)) == "InvalidDimension"
    assert kind(lambda: token_logprobs(dev.empty((3, 4)), ids, 5)) == "InvalidDimension"
    assert kind(lambda: token_logprobs(dev.empty((3, 0)), ids)) == "InvalidDimension"
    assert kind(lambda: token_logprobs(dev.empty((1, 3, 100)), ids)) == "InvalidDimension"
    assert kind(lambda: token_logprobs(x, dev.empty((2,), I32))) == "ShapeMismatch"
    assert kind(lambda: token_logprobs(x, dev.empty((3, 1), I32))) == "ShapeMismatch"
    assert kind(lambda: token_logprobs(x, dev.empty((3,), F32))) == "DtypeError"
    assert kind(lambda: token_logprobs(dev.empty((3, 100), I32), ids)) == "DtypeError"
    assert kind(lambda: token_logprobs(dev.empty((3, 96), Q8_0), ids)) == "DtypeError"
    big = dev.empty((2 ** 24, 1))
    assert kind(lambda: token_logprobs(big)) == "InvalidDimension"


def test_most_rows(dev):
    """The largest launch there is: rows of one token, whose probability is 1."""
    n = 2 ** 24 - 1
    x = dev.tensor(np.tile(np.array([[3.0], [-65504.0], [np.nan]], np.float16), (n // 3, 1)))
    h = token_logprobs(x)[1].numpy()
    # not 0: the sums are in reference to a rounded m log2(e), so z = 2^d and t
    # = d 2^d with a |d| of up to half a step of it, and H = log z - t / z
    # keeps the roundings of 2^d, of the logarithm and of the quotient, each of
    # numbers near 1 or 0: reference()'s bound at V = 1, x = m
    tol = U * (1 / 64 + 64) * 2
    assert (np.abs(h[0::3]) <= tol).all() and (np.abs(h[1::3]) <= tol).all() and np.isnan(h[2::3]).all()
