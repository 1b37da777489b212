"""The attention over the int8 cache where its numbers leave the ordinary range: very large scores, one position far
above the rest, rows of q with one value far above the rest, more tiles than the card holds at a time.  Against
float64."""
import numpy as np
import pytest

import ref8
from conftest import rng
from test_gpu_layer8 import BF16, F32, DevCache, held, prefix, up, values

pytestmark = pytest.mark.gpu

BLOCK = ref8.BLOCK


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


def weighted(ref, q, pos, scale, is_bf16, window=0, sinks=0):
    """(result, bound) of one sequence's rows: the formula, and what arithmetic in 32 bits may lose of
    sum_i weight_i |v_i|, the sum whose terms the result adds."""
    u, (n, hq, dim) = F32, q.shape
    k, v = ref.values("k")[0], ref.values("v")[0]
    heads, cap, _ = k.shape
    out, bound, p = np.zeros(q.shape), np.zeros(q.shape), np.arange(cap)
    for i in range(n):
        last = pos + i
        seen = (p <= last) & ((p > last - window) | (p < sinks) if window else True)
        if not seen.any():
            continue
        for h in range(hq):
            kk, vv = k[h * heads // hq][seen], v[h * heads // hq][seen]
            s = scale * (kk @ q[i, h])
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv
            # a score's products are exact in up to 3 terms of q; sums of 3 dim of them in any order: 3 dim roundings of
            # what they add up to.  Six more of the score itself (scale x log2 e, the block's scale, the row's factor, the
            # product, the difference from the reference, the exponential's argument)
            e = scale and (3 * dim * u * abs(scale) * (np.abs(kk) @ np.abs(q[i, h])) + 6 * u * np.abs(s - s.max()) + 6 * u * np.abs(s))
            e = np.broadcast_to(e, s.shape)
            # a weight: the exponential's two units; the terms that it goes into the product in (2^-17 of it in two, 2^-24
            # in three); the product's sums, 64 positions in 3 terms in any order; the rescaling and the addition of each
            # block, and the joining of at most 64 + 4 parts.  And the weights' sum, whose relative error is the largest one's
            blocks = seen.sum() // BLOCK + 2
            each = np.expm1(e) + (2.0 ** -17 if is_bf16 else u) + (2 + 192 + 2 * blocks + 72) * u
            # and what f32 does not hold: a weight, the largest of which is 1 or more, and each of its three terms may lose
            # what lies below 2^-126, and so may the result
            bound[i, h] = (w * each) @ np.abs(vv) + (w @ each) * np.abs(out[i, h]) + 2.0 ** -126 * (4 * np.abs(vv).sum(0) + 1)
    t = BF16 if is_bf16 else F32
    return out, bound + t * (np.abs(out) + bound)


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


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("positions", [64, 384, 2048])
@pytest.mark.parametrize("gap", [8, 10, 12, 20, 40])
def test_dominant_position(dev, gap, positions, rows, is_bf16):
    """One position `gap` above all others whose row of V is zero (a sink): the others alone make the result, and it is
    as near as if their weights stood alone."""
    r = rng(int(gap) + positions + rows)
    heads, group, dim, cap = 2, 2, 64, 2176
    ref = ref8.Cache(1, heads, cap, dim)
    # the others' scores are all 0, so that what their weights lose does not average out
    ref.q["k"][:, :, 5, 0] = 127
    ref.q["v"] = r.integers(20, 128, ref.shape)
    ref.q["v"][:, :, 5] = 0
    ref.s["k"][:] = 2.0 ** -5
    ref.s["v"][:] = r.uniform(0.01, 0.04, ref.s["v"].shape).astype(np.float32)
    q = np.zeros((rows, heads * group, dim))
    q[:, :, 0] = held(np.array(gap * 32 / 127), is_bf16)
    pos = positions - 1
    got = attend(dev, ref, q, [rows], [pos], 1.0, is_bf16)
    want, err = weighted(ref, q, pos, 1.0, is_bf16)
    over = np.abs(got - want) > err
    assert not over.any(), (np.abs(got / want - 1).max(), (err / np.abs(want)).max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("big", [1e3, 1e6, 1e12, 1e30])
def test_row_with_one_large_value(dev, big, rows, is_bf16):
    """A value of q far above its row's others where K has zeros: the others decide the scores as if they stood alone."""
    r = rng(int(np.log10(big)) + rows)
    heads, group, dim, cap, pos = 2, 2, 128, 256, 190
    ref = ref8.Cache(1, heads, cap, dim).fill(r)
    ref.q["k"][..., 77] = 0
    q = held(r.normal(0, 1, (rows, heads * group, dim)), is_bf16)
    scale = dim ** -0.5
    want, err = weighted(ref, q, pos, float(np.float32(scale)), is_bf16)
    q[..., 77] = held(np.array(big), is_bf16)
    got = attend(dev, ref, q, [rows], [pos], scale, is_bf16)
    over = np.abs(got - want) > err
    assert not over.any(), (np.argwhere(over)[:3], np.abs(got - want).max(), err.max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,spread", [(1, 1), (1, 4), (1, 12), (40, 1), (40, 4), (40, 12)])
def test_peaked_rows(dev, rows, spread, is_bf16):
    """Random rows whose scores spread over `spread`, K and V of outlying positions: what is lost, against the sum of weight x |v|."""
    r = rng(rows + spread)
    heads, group, dim, cap, pos = 2, 2, 128, 1024, 960
    ref = ref8.Cache(1, heads, cap, dim).fill(r)
    ref.q["v"][:, :, ::97] //= 32                            # some positions with next to nothing in V
    q = held(r.normal(0, spread, (rows, heads * group, dim)), is_bf16)
    scale = dim ** -0.5
    got = attend(dev, ref, q, [rows], [pos], scale, is_bf16)
    want, err = weighted(ref, q, pos, float(np.float32(scale)), is_bf16)
    over = np.abs(got - want) > err
    assert not over.any(), (np.argwhere(over)[:3], np.abs(got - want).max(), err.max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
def test_rows_of_any_size(dev, rows, is_bf16):
    """Rows of q from 1e-30 to 1e30 with a block scale that brings their scores back: no product of the two is out of range."""
    r = rng(rows)
    heads, group, dim, cap, pos = 2, 2, 64, 256, 150
    for size in (1e-30, 1e-10, 1e10, 1e30):
        ref = ref8.Cache(1, heads, cap, dim).fill(r)
        ref.s["k"] = (ref.s["k"] / np.float32(size)).astype(np.float32)
        q = held(r.normal(0, size, (rows, heads * group, dim)), is_bf16)
        got = attend(dev, ref, q, [rows], [pos], 0.125, is_bf16)
        want, err = weighted(ref, q, pos, 0.125, is_bf16)
        over = np.abs(got - want) > err
        assert not over.any(), (size, np.argwhere(over)[:3], np.abs(got - want).max(), err.max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
def test_negative_block_scales(dev, rows, is_bf16):
    """A value is int8 x scale, whatever the scale's sign."""
    r = rng(rows)
    heads, group, dim, cap, pos = 2, 2, 128, 512, 400
    ref = ref8.Cache(1, heads, cap, dim).fill(r)
    for n in "kv":
        ref.s[n] *= r.choice([-1, 1], ref.s[n].shape).astype(np.float32)
    q = held(r.normal(0, 8, (rows, heads * group, dim)), is_bf16)
    got = attend(dev, ref, q, [rows], [pos], 0.125, is_bf16)
    want, err = weighted(ref, q, pos, 0.125, is_bf16)
    over = np.abs(got - want) > err
    assert not over.any(), (np.argwhere(over)[:3], np.abs(got - want).max(), err.max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
def test_scores_out_of_range(dev, rows, is_bf16):
    """A block whose largest score f32 does not hold makes the rows that see it NaN, an infinite scale among them; a score
    below f32's range beside others that it holds weighs nothing."""
    r = rng(rows)
    heads, group, dim, cap, pos = 1, 2, 64, 256, 40
    ref = ref8.Cache(1, heads, cap, dim).fill(r)
    ref.q["k"][..., 0] = -np.maximum(np.abs(ref.q["k"][..., 0]), 4)
    q = np.zeros((rows, heads * group, dim))
    q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
    see = np.arange(rows) + pos >= 64
    for scale in (np.inf, np.float32(3e38)):
        ref.s["k"][0, 0, 1] = scale
        got = attend(dev, ref, q, [rows], [pos], 0.5, is_bf16)
        assert np.isfinite(got[~see]).all() and np.isnan(got[see]).all()
    ref.s["k"][0, 0, 1] = 3e38
    ref.q["k"][0, 0, 64, 0] = 0                              # the one score of that block that f32 holds, for head 0 its largest
    got = attend(dev, ref, q, [rows], [pos], 0.5, is_bf16)
    more = np.arange(rows) + pos > 64                        # a row that sees only that position of the block is finite in both heads
    assert np.isnan(got[more][:, 1]).all() and np.isfinite(got[~more]).all() and np.isfinite(got[:, 0]).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("counts,pos,heads", [([1100], [0], 8), ([2100], [0], 8), ([700, 1, 431], [5, 60, 0], 5)])
def test_many_tiles(dev, counts, pos, heads, is_bf16):
    """More blocks than the card holds at a time, in whatever order they come: every row is written, and is right."""
    r = rng(sum(counts) + is_bf16)
    group, dim, cap = 2, 64, 2176
    ref = ref8.Cache(len(counts), heads, cap, dim).fill(r)
    q = held(r.normal(0, 1, (sum(counts), heads * group, dim)), is_bf16)
    got = attend(dev, ref, q, counts, pos, 0.125, is_bf16)
    assert (np.abs(got - 3.0) > 0).any(2).all()              # the output held 3.0 before
    start = prefix(counts)
    for j, n in enumerate(counts):
        one = ref8.Cache(1, heads, cap, dim)
        for name in "kv":
            one.q[name], one.s[name] = ref.q[name][j:j + 1], ref.s[name][j:j + 1]
        for i in sorted({*range(0, n, 97), *range(n - 1, 0, -211)}):
            want, err = weighted(one, q[start[j] + i:start[j] + i + 1], pos[j] + i, 0.125, is_bf16)
            over = np.abs(got[start[j] + i] - want[0]) > err[0]
            assert not over.any(), (j, i, np.abs(got[start[j] + i] - want[0]).max(), err.max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("sinks", [0, 3, 70])
@pytest.mark.parametrize("pos,window", [(2000, 256), (2000, 257), (2000, 1000), (2000, 1900), (2000, 2000), (2000, 2010), (2000, 1 << 40), (250, 257),
                                        (250, 1000), (3, 1 << 62), ((1 << 31) - 1, (1 << 31) - 1), ((1 << 31) - 1, (1 << 31) - 70), (1 << 30, (1 << 30) - 5)])
def test_window_and_capacity(dev, pos, window, sinks, is_bf16):
    """Rows past the capacity, windows around it and far larger: a row at p sees what is stored of (p - window, p] and the
    first sinks.  One sequence of few rows, one of many."""
    r = rng(sinks + window % 1000)
    counts, heads, group, dim, cap = [3, 40], 2, 2, 64, 256
    ref = ref8.Cache(2, heads, cap, dim).fill(r)
    for rows in (counts, [2, 3]):
        q = held(r.normal(0, 1, (sum(rows), heads * group, dim)), is_bf16)
        got = attend(dev, ref, q, rows, [pos, pos], 0.125, is_bf16, window=window, sinks=sinks)
        start = prefix(rows)
        for j in range(2):
            one = ref8.Cache(1, heads, cap, dim)
            for name in "kv":
                one.q[name], one.s[name] = ref.q[name][j:j + 1], ref.s[name][j:j + 1]
            want, err = weighted(one, q[start[j]:start[j + 1]], pos, 0.125, is_bf16, window, sinks)
            over = np.abs(got[start[j]:start[j + 1]] - want) > err
            assert not over.any(), (rows, j, np.argwhere(over)[:3], np.abs(got[start[j]:start[j + 1]] - want).max())


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("scale", [-0.1, 2.0])
def test_very_peaked_rows(dev, scale, rows, is_bf16):
    """Rows a thousand times an ordinary one's size: each result against the bound that its scores' size allows, and where
    that leaves no doubt which position has all the weight, that position's row of V."""
    r = rng(rows)
    heads, group, dim, cap, pos = 2, 2, 128, 256, 120
    ref = ref8.Cache(1, heads, cap, dim).fill(r)
    q = held(r.normal(0, 1000, (rows, heads * group, dim)), is_bf16)
    got = attend(dev, ref, q, [rows], [pos], scale, is_bf16)
    want, err = weighted(ref, q, pos, float(np.float32(scale)), is_bf16)
    over = np.abs(got - want) > err
    assert not over.any(), (np.argwhere(over)[:3], np.abs(got - want).max(), err.max())
    k, v = ref.values("k")[0], ref.values("v")[0]
    sure = 0
    for i in range(rows):
        for h in range(heads * group):
            s = float(np.float32(scale)) * (k[h // group, :pos + i + 1] @ q[i, h])
            first, second = np.sort(s)[::-1][:2]
            off = 3 * dim * F32 * abs(scale) * (np.abs(k[h // group, :pos + i + 1]) @ np.abs(q[i, h])).max()
            if first - second > 2 * off + 40:
                sure += 1
                x = v[h // group, s.argmax()]
                # the others together weigh less than a position's e^-40 each
                rest = (pos + rows) * np.exp(-40) * np.abs(v).max()
                err = ((2.0 ** -16 if is_bf16 else 8 * F32) + (BF16 if is_bf16 else F32)) * np.abs(x) + 1.01 * rest
                assert (np.abs(got[i, h] - x) <= err).all(), (i, h)
    assert sure >= rows                                      # most of them are


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 40])
def test_smallest_weights(dev, rows, is_bf16):
    """Weights 2^-99 of the one in front of them, whose row of V is zero, keep their bits."""
    test_dominant_position(dev, 99 * np.log(2), 384, rows, is_bf16)
