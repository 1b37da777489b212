"""Single-row attention over f32 and bf16 caches with many KV heads and all 64 splits: the shapes whose partial results
take most of a handle's scratch area.  Against float64."""
import numpy as np
import pytest

from conftest import bf16, bf16f, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("heads", [126, 127, 200, 256])
def test_many_heads(dev, heads, is_bf16):
    from qwenasr_amd import kernels as K
    dim, n = 128, 64 * 256                                   # 256 positions a split
    r = rng(heads)
    # heads may share memory: head h begins at row h
    k, v = (r.normal(0, 1, (heads + n, dim)).astype(np.float32) for _ in range(2))
    q = r.normal(0, 3, (2 * heads, dim)).astype(np.float32)
    out = dev.zeros((2 * heads, dim), np.float32)
    if is_bf16:
        dk, dv, k, v = dev.upload(bf16(k)), dev.upload(bf16(v)), bf16f(bf16(k)), bf16f(bf16(v))
        K.causal_attention_bf16kv(out, dev.upload(q), dk, dv, dim, n, 2 * heads, heads, dim, dim ** -0.5, n - 1)
    else:
        K.causal_attention(out, dev.upload(q), dev.upload(k), dev.upload(v), dim, 1, n, 2 * heads, heads, dim, dim ** -0.5, n - 1)
    got = out.numpy().astype(np.float64)
    u = 2.0 ** -24
    for h in sorted({0, 1, 63, 64, heads - 2, heads - 1}):
        kk, vv = k[h:h + n].astype(np.float64), v[h:h + n].astype(np.float64)
        for g in (0, 1):
            x = q[2 * h + g].astype(np.float64)
            s = dim ** -0.5 * (kk @ x)
            w = np.exp(s - s.max())
            w /= w.sum()
            # a score: dim products and sums, its scale and the difference; a weight and its product: those twice (the
            # weights' sum has them too), the exponential, and sums of n terms in any order
            e = (dim + 2) * u * dim ** -0.5 * (np.abs(kk) @ np.abs(x)) + 2 * u * np.abs(s)
            err = (w * (2 * e.max() + (2 * n + 8) * u)) @ np.abs(vv)
            assert (np.abs(got[2 * h + g] - w @ vv) <= err).all(), (h, g, np.abs(got[2 * h + g] - w @ vv).max(), err.max())
    assert np.isfinite(got).all() and (np.abs(got).max(1) > 0).all()


def test_more_heads_are_refused(dev):
    from qwenasr_amd import kernels as K
    b = dev.zeros(2 * 257 * 128, np.float32)
    for f in (lambda: K.causal_attention(b, b, b, b, 128, 1, 1, 514, 257, 128, 0.1, 0),
              lambda: K.causal_attention_bf16kv(b, b, b, b, 128, 1, 514, 257, 128, 0.1, 0)):
        with pytest.raises(RuntimeError):
            f()
