"""How much of q and of the weights reaches the attention over pages: inputs whose leading bits cancel, so that a term too few
shows.  Without a GPU: a model of the arithmetic stays inside the tolerance with all its terms and leaves it with one less.

K and V are small exact numbers in two dims; what is left of a score or of a sum is made of the operand's last bits alone."""
import numpy as np
import pytest

from conftest import bf16, bf16f, rng
from refp import U

FORMS = [(64, 8, 2, 64), (48, 8, 2, 128), (16, 2, 40, 64), (16, 2, 40, 128)]     # sequences, KV heads, heads of each, dim: few rows, and tiles of many


def split(x, terms):
    """The sum of a value's first `terms` bf16 terms, each the rest's nearest."""
    x = np.asarray(x, np.float32)
    out, rest = np.zeros(x.shape), x
    for _ in range(terms):
        h = bf16f(bf16(rest))
        out += h
        rest = (rest - h).astype(np.float32)
    return out


# ---- q: a pair of dims that differ from the 16th bit on, a scale that makes scores of what is left

SCALE_Q, KEYS = 2.0 ** 16, np.array([1.0, -1.0, 0.5, -0.5, 0.25, 0.0, 1.0, -0.25, 0.5, -1.0, 0.125, 0.25])


def rows_q(r, shape, dims):
    """Values of [1, 2) in steps of 2^-21 (all partial sums of their terms times powers of two are exact in f32), the second
    within 2^-14 of the first: scores of at most 4 x 1."""
    q = np.zeros(shape)
    a = 1.0 + r.integers(1 << 14, (1 << 21) - (1 << 14), shape[:-1]) * 2.0 ** -21
    q[..., dims[0]], q[..., dims[1]] = a, a + r.integers(-(1 << 7), (1 << 7) + 1, shape[:-1]) * 2.0 ** -21
    return q


def out_q(diff, v):
    """From the two dims' difference [..] and the values [positions][dim]."""
    s = SCALE_Q * diff[..., None] * KEYS
    w = np.exp(s - s.max(-1, keepdims=True))
    return (w / w.sum(-1, keepdims=True)) @ v


def tolerance_q(v):
    """Scores of at most 4, 5.8 in base 2: the factor scale x log2 e (two roundings), the maximum's product, the difference
    (11.6 at most): (2 x 5.8 + 5.8 + 11.6) U = 29 U of the exponent, 20 U of a weight; its exponential 2 U, its terms 1; a
    weight stands in both sums; those of 12 positions and three terms: 36 U and 12; the quotient, its product, the result: 4."""
    return (2 * 23 + 48 + 4) * U * np.abs(v).max(0)


# ---- weights: 1 and e^x, one value and its negative

def rows_w(r, shape, is_bf16, dim):
    """x in one dim; of either sign, so that either position can have the maximum.  bf16 rows: small ones, as the result's own
    rounding is relative to what is left."""
    q = np.zeros(shape)
    x = r.uniform(2.0 ** -6, 2.0 ** -4, shape[:-1]) if is_bf16 else r.uniform(0.05, 0.69, shape[:-1])
    q[..., dim] = x * r.choice([-1.0, 1.0], shape[:-1])
    return bf16f(bf16(q)).astype(np.float64) if is_bf16 else q.astype(np.float32).astype(np.float64)


def out_w(x, terms=None):
    """(w0 - w1) / (w0 + w1) of weights e^0 and e^x, the larger 1; `terms`: of the weights in the products."""
    m = np.maximum(x, 0)
    w0, w1 = np.exp(-m).astype(np.float32), np.exp(x - m).astype(np.float32)
    if terms is None:
        return (np.exp(-m) - np.exp(x - m)) / (np.exp(-m) + np.exp(x - m))
    return (split(w0, terms) - split(w1, terms)) / (w0.astype(np.float64) + w1)


def tolerance_w(want, is_bf16):
    """Scores of at most 0.69, 1 in base 2: the factor 2 U, the maximum's product U, the difference U: 4 U of the exponent, 3 U of
    a weight; its exponential 2 U, its terms 1 (bf16 rows: 2^-17); of both weights, their share of the sum (each at most 1 of at
    least 1.5, together 1): 6 U.  The product's three additions of at most 1, over 1.5: 2 U.  Sum, quotient and product: relative
    to what is left, with the result's own rounding."""
    return (8 * U if not is_bf16 else 2.0 ** -17 + 8 * U) + (2.0 ** -8 if is_bf16 else 4 * U) * np.abs(want)


# ---- weights of bf16 rows: 1, e^x, e^y, and values whose sum with them is next to nothing, as the result is rounded to bf16

def rows_v(r, n, dim):
    """x, y [n] and values [n][3][dim] of at most 1 in size: the best of 512 pairs for each dim, the third the bf16 value that
    comes nearest to taking the sum away."""
    x, y = (bf16f(bf16(-r.uniform(0.05, 0.69, n))).astype(np.float64) for _ in range(2))
    v = np.empty((n, 3, dim))
    for i in range(n):
        a, b = (bf16f(bf16(s * r.uniform(0.5, 1.0, (512, dim)))).astype(np.float64) for s in (1, -1))
        c = bf16f(bf16(-(a + b * np.exp(x[i])) / np.exp(y[i]))).astype(np.float64)
        left = np.where(np.abs(c) <= 1, np.abs(a + b * np.exp(x[i]) + c * np.exp(y[i])), np.inf)
        best = left.argmin(0), np.arange(dim)
        v[i] = a[best], b[best], c[best]
    return x, y, v


def out_v(x, y, v, terms=None):
    w = np.stack([np.ones(len(x)), np.exp(x), np.exp(y)], 1)
    p = w if terms is None else split(w.astype(np.float32), terms)
    return (p[:, None] @ v)[:, 0] / w.sum(1)[:, None]


def tolerance_v(want):
    """Scores as above: 6 U of a weight, of values of at most 1 the same of the result.  Sums of at most 3, the last one's
    three additions and the one to the lower terms' of U x 3 each, over weights of 2 and more together (1 + 2 x 0.5): 6 U.
    Quotient, product and result relative to what is left."""
    return 12 * U + (2.0 ** -8 + 4 * U) * np.abs(want)


# ---------------------------------------------------------------------------
# the tolerances themselves
# ---------------------------------------------------------------------------

def test_the_tolerances_tell_a_term():
    r = rng(60)
    q = rows_q(r, (400, 2), (0, 1))
    v = r.normal(0, 0.6, (len(KEYS), 64))
    exact = out_q(q[:, 0] - q[:, 1], v)
    off = lambda n: np.abs(out_q(split(q, n)[:, 0] - split(q, n)[:, 1], v) - exact)  # noqa: E731
    assert (off(3) <= tolerance_q(v)).all() and (off(2) > tolerance_q(v)).any(1).mean() > 0.5
    x = rows_w(r, (2000, 1), False, 0)[:, 0]
    off = lambda n: np.abs(out_w(x, n) - out_w(x)) > tolerance_w(out_w(x), False)  # noqa: E731
    assert not off(3).any() and off(2).mean() > 0.1
    x = rows_w(r, (2000, 1), True, 0)[:, 0]
    off = lambda n: np.abs(bf16f(bf16(out_w(x, n))) - out_w(x)) > tolerance_w(out_w(x), True)  # noqa: E731
    assert not off(2).any() and off(1).mean() > 0.1
    x, y, v = rows_v(r, 100, 64)
    want = out_v(x, y, v)
    off = lambda n: np.abs(bf16f(bf16(out_v(x, y, v, n))) - want) > tolerance_v(want)  # noqa: E731
    assert np.abs(want).max() < 2.0 ** -12 and not off(3).any() and off(2).mean() > 0.1


# ---------------------------------------------------------------------------
# the kernels
# ---------------------------------------------------------------------------

def cache(dev, n_seq, heads, dim, keys, dims, values):
    """A page a sequence: K has `keys` in the first of `dims` and their negatives in the second (if there is one)."""
    from test_gpu_hypotheses import Cache
    n = len(keys)
    c = Cache(dev, rng(1), [n] * n_seq, 16, heads, dim, fill=False, width=2)
    k, v = np.zeros((n_seq, heads, 16, dim)), np.zeros((n_seq, heads, 16, dim))
    k[:, :, :n, dims[0]] = keys
    if len(dims) > 1:
        k[:, :, :n, dims[1]] = -keys
    v[:, :, :n] = values
    for j in range(n_seq):
        c.bits["k"][c.table[j, 0]], c.bits["v"][c.table[j, 0]] = bf16(k[j]), bf16(v[j])
    c.upload()
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [(0, 1), (3, 60), (17, 16)])
@pytest.mark.parametrize("n_seq,heads,g,dim", FORMS)
def test_every_bit_of_q(dev, n_seq, heads, g, dim, apart):
    from test_gpu_hypotheses import attention
    print(f"bits of q {n_seq} heads={heads} x {g} dim={dim} {apart}", flush=True)
    r = rng(61 + dim + g)
    v = bf16f(bf16(r.normal(0, 0.6, (len(KEYS), dim)))).astype(np.float64)
    c = cache(dev, n_seq, heads, dim, KEYS, apart, v)
    q = rows_q(r, (n_seq, heads * g, dim), apart)
    got = attention(dev, c, q, [1] * n_seq, [len(KEYS) - 1] * n_seq, g, scale=SCALE_Q)
    want = out_q(q[..., apart[0]] - q[..., apart[1]], v)
    off = np.abs(got - want)
    assert (off <= tolerance_q(v)).all(), np.max(off / tolerance_q(v))


@pytest.mark.gpu
@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("at", [0, 37])
@pytest.mark.parametrize("n_seq,heads,g,dim", FORMS)
def test_every_bit_of_a_weight(dev, n_seq, heads, g, dim, at, is_bf16):
    from test_gpu_hypotheses import attention
    print(f"bits of weights {n_seq} heads={heads} x {g} dim={dim} {at} bf16={is_bf16}", flush=True)
    r = rng(62 + dim + g)
    c = cache(dev, n_seq, heads, dim, np.array([0.0, 1.0]), (at,), np.array([[1.0], [-1.0]]) * np.where(np.arange(dim) % 3 == 1, -1.0, 1.0))
    q = rows_w(r, (n_seq, heads * g, dim), is_bf16, at)
    got = attention(dev, c, q, [1] * n_seq, [1] * n_seq, g, is_bf16=is_bf16, scale=1.0) * np.where(np.arange(dim) % 3 == 1, -1.0, 1.0)
    want = out_w(q[..., at])[..., None]
    off = np.abs(got - want)
    assert (off <= tolerance_w(want, is_bf16)).all(), np.max(off / tolerance_w(want, is_bf16))


@pytest.mark.gpu
@pytest.mark.parametrize("power", [-100, 60])
@pytest.mark.parametrize("n_seq,heads,g,dim", FORMS[1:3])
def test_every_bit_of_small_and_large_q(dev, n_seq, heads, g, dim, power):
    """From 2^-100 on the last term is a normal number."""
    from test_gpu_hypotheses import attention
    r = rng(63 + dim)
    v = bf16f(bf16(r.normal(0, 0.6, (len(KEYS), dim)))).astype(np.float64)
    c = cache(dev, n_seq, heads, dim, KEYS * 2.0 ** -power, (2, 9), v)
    q = rows_q(r, (n_seq, heads * g, dim), (2, 9))
    got = attention(dev, c, q * 2.0 ** power, [1] * n_seq, [len(KEYS) - 1] * n_seq, g, scale=SCALE_Q)
    assert (np.abs(got - out_q(q[..., 2] - q[..., 9], v)) <= tolerance_q(v)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hints", [dict(max_len=48), dict(max_len=3000), {}])
@pytest.mark.parametrize("n_seq,dim", [(60, 64), (24, 128)])
def test_every_bit_of_a_weight_of_few_bf16_rows(dev, n_seq, dim, hints):
    """Of up to 32 rows x heads; 2^-17 of a weight would show."""
    from test_gpu_hypotheses import Cache, attention
    r, heads = rng(64 + dim), 8
    x, y, v = rows_v(r, n_seq * heads, dim)
    c = Cache(dev, rng(1), [3] * n_seq, 16, heads, dim, fill=False, width=200)
    k, val = np.zeros((n_seq, heads, 16, dim)), np.zeros((n_seq, heads, 16, dim))
    k[:, :, 1, 5] = k[:, :, 2, 6] = 1.0
    val[:, :, :3] = v.reshape(n_seq, heads, 3, dim)
    for j in range(n_seq):
        c.bits["k"][c.table[j, 0]], c.bits["v"][c.table[j, 0]] = bf16(k[j]), bf16(val[j])
    c.upload()
    q = np.zeros((n_seq, heads, dim))
    q[..., 5], q[..., 6] = x.reshape(n_seq, heads), y.reshape(n_seq, heads)
    got = attention(dev, c, q, [1] * n_seq, [2] * n_seq, 1, is_bf16=True, scale=1.0, **hints).reshape(-1, dim)
    want = out_v(x, y, v)
    off = np.abs(got - want)
    assert (off <= tolerance_v(want)).all(), np.max(off / tolerance_v(want))
