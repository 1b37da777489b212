"""The attention over the int8 cache where its numbers leave the ordinary range: very large scores, one position far
above the rest.  Against float64."""
import numpy as np
import pytest

import ref8
from conftest import rng
from test_gpu_layer8 import BF16, F32, DevCache, held, prefix, up, values

pytestmark = pytest.mark.gpu


def attend(dev, ref, q, counts, pos, scale, is_bf16, window=0, sinks=0, max_len=0):
    """The call's result [rows][heads][dim]."""
    from qwenasr_amd import kernels as K
    n, heads, cap, dim = ref.shape
    d, total, hq = DevCache(dev, ref), sum(counts), q.shape[1]
    out = up(dev, np.full((total, hq * dim), 3.0), is_bf16)
    K.attention_kv8(out, up(dev, q.reshape(total, -1), is_bf16), *d.buf, dev.upload(np.array(pos, np.int32)), total, n, max(counts), hq,
                    heads, dim, cap, scale, row_start=dev.upload(prefix(counts)), max_len=max_len, window=window, sinks=sinks,
                    bf16=is_bf16)
    return values(out, is_bf16).reshape(q.shape)


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(dev, rows, sign, is_bf16):
    """Scores of 2^17 ... 2^24 (x log2 e), one position 2^11 or more above all others: the result is that position's row of V."""
    r = rng(31 + rows + sign)
    heads, group, dim, cap, pos, at = 2, 4, 64, 256, 130, 37          # `at` lies in a block that every row sees
    ref = ref8.Cache(1, heads, cap, dim)
    ref.q["v"] = r.integers(-127, 128, ref.shape)
    ref.s["v"][:] = 2.0 ** -6
    ref.s["k"][:] = 1.0
    # dim 0 decides: the score is q x 127 against 0, or q x -63 against -127
    ref.q["k"][0, :, :, 0] = 0 if sign > 0 else -127
    ref.q["k"][0, :, at, 0] = 127 if sign > 0 else -63
    q = np.zeros((rows, heads * group, dim))
    q[:, :, 0] = 2.0 ** r.uniform(17, 24, q.shape[:2]) * np.log(2) / 63
    got = attend(dev, ref, q, [rows], [pos], 1.0, is_bf16)
    want = np.broadcast_to(np.repeat(ref.values("v")[0, :, at], group, 0), got.shape)
    # the only weight is not rounded by more than its terms', the products are exact, their quotient is rounded and the result is
    err = ((2.0 ** -16 if is_bf16 else 4 * F32) + (BF16 if is_bf16 else F32)) * np.abs(want)
    over = np.abs(got - want) > err
    assert not over.any(), (np.argwhere(over)[:3], got[over][:3], want[over][:3])
