"""Attention over pages where its parts are joined: rows, keys and whole parts that are not finite, against the formula in
float64, with the work split, behind a shared prefix, and in one piece."""
import numpy as np
import pytest

import refp
from conftest import rng
from refp import U
from test_gpu_hypotheses import BF16, Cache, attention, check_attention, held

pytestmark = pytest.mark.gpu

NAN, INF, NEG = 0x7FC0, 0x7F80, 0xFF80


def formula(c, q, counts, pos, is_bf16):
    """softmax(scale q k) v and its bound; NaN where the formula has it, zeros for rows that see nothing."""
    pools, at = c.floats(), 0
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    q, scale = held(q, is_bf16), c.dim ** -0.5
    for j, n in enumerate(counts):
        end = min(max(pos[j] + n, 0), c.width * c.page)
        k, there = refp.gather(pools["k"], c.table[j], end, c.page)
        v, _ = refp.gather(pools["v"], c.table[j], end, c.page)
        for i in range(n):
            see = (np.arange(end) <= pos[j] + i) & there
            for h in range(q.shape[1]):
                with np.errstate(invalid="ignore"):
                    s = scale * (k[see, h // (q.shape[1] // c.heads)] @ q[at + i, h])
                if see.any() and not (np.isfinite(s).any() and (np.isfinite(s) | np.isneginf(s)).all()):
                    want[at + i, h] = np.nan                 # NaN, +infinity, or -infinity alone
                    continue
                use = np.flatnonzero(see)[np.isfinite(s)]    # a score of -infinity: weight 0
                g = h // (q.shape[1] // c.heads)
                o, b = refp.attend(q[at + i:at + i + 1, h:h + 1], k[use, g:g + 1], v[use, g:g + 1], np.ones((1, len(use)), bool), scale,
                                   2.0 ** -17 if is_bf16 else U)
                want[at + i, h], bound[at + i, h] = o[0, 0], b[0, 0]
        at += n
    return want, bound * (1 + BF16) + (BF16 if is_bf16 else U) * np.abs(want)


def check(c, q, counts, pos, g, is_bf16, forms):
    want, bound = formula(c, q, counts, pos, is_bf16)
    for group, shared, more in forms:
        got = attention(c.dev, c, q, counts, pos, g, group, shared, is_bf16, **more)
        assert (np.isnan(got) == np.isnan(want)).all(), (group, shared, more, np.argwhere(np.isnan(got) != np.isnan(want))[:4])
        ok = ~np.isnan(want)
        assert (np.abs(got - want)[ok] <= bound[ok]).all(), (group, shared, more)
    return want


def put(c, x, j, positions, heads, dims, bits):
    for p in positions:
        c.bits[x][c.table[j, p // c.page], heads, p % c.page, dims] = bits


# rows a sequence x heads a KV head: few rows, and tiles of many; capacities of 1024 and more, which are split if no hint says
# that less of them is in use
FORMS = [(1, 2), (3, 5), (40, 2)]
PIECES = [(1, None, {}), (1, None, dict(max_len=64)), (1, None, dict(max_len=300)), (1, None, dict(max_len=1000))]


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,g", FORMS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_a_row_of_nan_is_nan_in_every_part(dev, rows, g, dim, page, is_bf16):
    print(f"row of NaN rows={rows} g={g} dim={dim} page={page} bf16={is_bf16}", flush=True)
    r = rng(50 + dim)
    counts, pos = [rows] * 3, [700, 20, 330]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], page, 2, dim, 3, [20], width=1024 // page)
    q = r.normal(0, 1, (3 * rows, 2 * g, dim))
    q[0, 0, 5] = q[2 * rows, 2 * g - 1, 0] = q[3 * rows - 1, 1, dim - 1] = np.nan
    want = check(c, q, counts, pos, g, is_bf16, PIECES + [(3, [20], {}), (3, [20], dict(max_len=1000, max_own=900)), (2, [3, 20], {})])
    assert np.isnan(want).any(2).sum() == 3


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,g", FORMS)
def test_a_part_of_nan_keys(dev, rows, g, is_bf16):
    """Keys of NaN in one stretch, of which a whole part is made (a table of 1024 positions is split into parts of 288), or the
    last one: the rows that see it are NaN, those before it are not."""
    r = rng(51)
    counts, pos = [rows] * 3, [800, 310, 250]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 16, 2, 128, width=64)
    put(c, "k", 0, range(288, 576), 1, slice(None), NAN)
    put(c, "k", 1, range(300, 310 + rows), 0, 7, NAN)
    put(c, "k", 2, range(max(1, 250 + rows // 2), 250 + rows), slice(None), 3, NAN)
    c.upload()
    q = r.normal(0, 1, (3 * rows, 2 * g, 128))
    want = check(c, q, counts, pos, g, is_bf16, PIECES)
    assert np.isnan(want[:rows, g:]).all() and np.isnan(want[rows:2 * rows, :g]).all() and np.isfinite(want[:rows, :g]).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16)])
def test_nan_in_the_only_position_behind_a_prefix(dev, dim, page, is_bf16):
    """A finite prefix, and one position of its own a member: NaN in that of two members, and in nobody else's."""
    r = rng(52)
    counts, pos = [1] * 6, [96] * 6
    c = Cache(dev, r, [97] * 6, page, 2, dim, 6, [96], width=1024 // page)
    put(c, "k", 2, [96], 1, 3, NAN)
    put(c, "v", 4, [96], 0, 9, NAN)
    c.upload()
    q = r.normal(0, 1, (6, 4, dim))
    want = check_members(c, q, counts, pos, is_bf16, [(6, [96], {}), (6, [96], dict(max_len=97, max_own=1)), (1, None, {}), (1, None, dict(max_len=97))])
    assert np.isnan(want[2, 2:]).all() and np.isnan(want[4, :2, 9]).all() and np.isnan(want).sum() == 2 * dim + 2


def check_members(c, q, counts, pos, is_bf16, forms):
    """As check, where a value of V is NaN: that dim of the rows that see it."""
    bits = c.bits["v"].copy()
    v = c.floats()["v"]
    nan = [np.isnan(refp.gather(v, c.table[j], pos[j] + n, c.page)[0]).any(0) for j, n in enumerate(counts)]
    c.bits["v"] = np.where((bits & 0x7FFF) > 0x7F80, 0, bits).astype(np.uint16)
    want, bound = formula(c, q, counts, pos, is_bf16)
    c.bits["v"] = bits
    g = q.shape[1] // c.heads
    for j in range(len(counts)):
        want[j][np.repeat(nan[j], g, 0)] = np.nan
    for group, shared, more in forms:
        got = attention(c.dev, c, q, counts, pos, g, group, shared, is_bf16, **more)
        assert (np.isnan(got) == np.isnan(want)).all(), (group, shared, more, np.argwhere(np.isnan(got) != np.isnan(want))[:4])
        ok = ~np.isnan(want)
        assert (np.abs(got - want)[ok] <= bound[ok]).all(), (group, shared, more)
    return want


@pytest.mark.parametrize("is_bf16", [False, True])
def test_every_part_of_a_prefix_of_nan_keys(dev, is_bf16):
    """A prefix of NaN keys for one head, and finite positions behind it."""
    r = rng(53)
    counts, pos = [1, 2, 1, 1], [700, 710, 705, 690]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 16, 2, 64, 4, [690], width=80)
    put(c, "k", 0, range(690), 1, 11, NAN)
    for j in (1, 2, 3):                                      # the copies of the part of a page
        put(c, "k", j, range(688, 690), 1, 11, NAN)
    c.upload()
    q = r.normal(0, 1, (5, 6, 64))
    want = check(c, q, counts, pos, 3, is_bf16, [(4, [690], {}), (4, [690], dict(max_len=720, max_own=40)), (1, None, {}), (1, None, dict(max_len=100))])
    assert np.isnan(want[:, 3:]).all() and np.isfinite(want[:, :3]).all()


# a dim of q that is 1 and of K that is -infinity: a score of -infinity
def low(c, j, positions, heads=slice(None)):
    put(c, "k", j, positions, heads, 2, NEG)


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,g", FORMS)
@pytest.mark.parametrize("dim,page", [(64, 64), (128, 16)])
def test_scores_of_minus_infinity_alone(dev, rows, g, dim, page, is_bf16):
    """What a row sees has scores of -infinity: 0 / 0, as the formula has it.  Where one score is finite, the others weigh
    nothing; a row that sees nothing gives zeros."""
    print(f"-infinity rows={rows} g={g} dim={dim} page={page} bf16={is_bf16}", flush=True)
    r = rng(54 + dim)
    counts, pos = [rows] * 6, [800, 0, 700, 30, -5, 40]
    c = Cache(dev, r, [max(a + b, 1) for a, b in zip(counts, pos)], page, 2, dim, width=1024 // page)
    low(c, 0, range(288, 576))                               # a whole part; the others are finite
    low(c, 1, range(0, rows), 0)                             # all there is, of one head
    low(c, 2, range(0, 700 + rows - 1))                      # all but what the last row sees last
    low(c, 3, range(30 + rows // 2, 30 + rows), 1)
    if rows > 5:
        low(c, 4, range(0, rows - 6))                        # rows that see nothing, -infinity alone, and (the last) something
    low(c, 5, range(page, 40 + rows))
    c.table[5, 0] = -1                                       # no page, and -infinity behind it
    c.upload()
    q = r.normal(0, 1, (6 * rows, 2 * g, dim))
    q[:, :, 2] = 1.0
    if rows == 1:
        q[2, 1, 2] = -1.0                                    # +infinity
    want = check(c, q, counts, pos, g, is_bf16, PIECES)
    assert np.isfinite(want[:rows]).all() and np.isnan(want[rows:2 * rows, :g]).all() and np.isnan(want[2 * rows:3 * rows - 1]).all()
    assert (want[4 * rows:4 * rows + min(rows, 5)] == 0).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_minus_infinity_behind_a_prefix(dev, rows, dim, is_bf16):
    """-infinity in the prefix, in what a member has behind it, and in both."""
    r = rng(55 + dim)
    counts, pos = [rows] * 8, [331, 340, 350, 331, 120, 130, 121, 5]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 16, 2, dim, 4, [331, 120], width=64)
    low(c, 0, range(331), 1)                                 # the first group's prefix for one head, with the copies of its last page
    for j in (1, 2, 3):
        low(c, j, range(320, 331), 1)
    low(c, 1, range(331, 340 + rows))                        # with what the second member has behind it
    low(c, 2, range(331, 345))                               # with a part of that
    low(c, 5, range(120, 130 + rows))                        # behind a finite prefix
    low(c, 4, range(0, 6))                                   # what the last member sees of the second prefix
    c.upload()
    q = r.normal(0, 1, (8 * rows, 4, dim))
    q[:, :, 2] = 1.0
    forms = [(4, [331, 120], {}), (4, [331, 120], dict(max_len=360, max_own=30)), (4, [331, 120], dict(max_len=1000, max_own=60)), (1, None, {}),
             (1, None, dict(max_len=200))]
    want = check(c, q, counts, pos, 2, is_bf16, forms)
    assert np.isnan(want[rows:2 * rows, 2:]).all() and np.isfinite(want[:rows]).all() and np.isfinite(want[5 * rows:6 * rows]).all()
    assert np.isnan(want[7 * rows]).all()


# The forms that the work's size picks, reached with small caches: which one runs goes by the hints and the table's width.
# sequences, rows, lengths (of the first ones, and at most of the others), heads, g, dim, page, width, group, shared, hints
PICKED = [
    # eight waves a block, K and V past the caches: in one piece, and split
    (34, 1, [700, 1, 257, 256, 64], 150, 8, 2, 128, 64, 40, 1, None, dict(max_len=2200)),
    (34, 2, [600, 2, 520, 33], 150, 8, 3, 64, 16, 270, 1, None, dict(max_len=4300)),
    (34, 1, [500], 90, 8, 16, 128, 16, 140, 1, None, {}),
    (12, 1, [3000, 2817, 2816, 2815, 1], 300, 8, 2, 128, 64, 90, 1, None, dict(max_len=5600)),
    (16, 3, [4400, 4193, 4191, 3], 200, 8, 2, 64, 256, 33, 1, None, dict(max_len=8300)),
    # four waves, in the caches and past them; two
    (40, 1, [600, 513, 128, 129, 1], 200, 8, 2, 128, 32, 20, 1, None, {}),
    (40, 2, [400, 129, 2], 100, 8, 5, 128, 16, 32, 1, None, dict(max_len=450)),
    (100, 1, [600, 129, 128, 1], 120, 8, 2, 64, 16, 64, 1, None, dict(max_len=1000)),
    (60, 1, [400], 120, 8, 3, 128, 128, 7, 1, None, dict(max_len=880)),
    (140, 1, [300, 65, 64, 63, 1], 80, 8, 2, 64, 16, 20, 1, None, {}),
    (140, 2, [250, 2], 60, 8, 4, 64, 64, 4, 1, None, dict(max_len=200)),
    # a prefix read once: prefixes and what is behind them in one part or several
    (130, 1, [450], 330, 8, 2, 64, 16, 45, 10, [300, 0, 17, 256, 300, 31, 1, 300, 299, 64, 128, 300, 300], {}),
    (40, 1, [700, 650], 500, 8, 16, 64, 16, 48, 10, [290, 300, 0, 100], {}),
    (40, 1, [700, 650], 400, 8, 16, 128, 64, 12, 10, [290, 300, 0, 100], {}),
    (12, 2, [1500, 900], 300, 1, 4, 64, 32, 50, 6, [640, 280], {}),
    # many rows: four groups over the positions, in one piece and split
    (3, 65, [1090, 1000, 641], 0, 16, 1, 128, 64, 18, 1, None, dict(max_len=1100)),
    (3, 65, [1090, 1025, 66], 0, 16, 1, 64, 16, 70, 1, None, dict(max_len=1100)),
    (4, 70, [570, 513, 512, 100], 0, 16, 1, 128, 16, 36, 1, None, {}),
    (4, 70, [570, 513, 512, 100], 0, 16, 1, 64, 32, 18, 1, None, {}),
]


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("n_seq,rows,first,most,heads,g,dim,page,width,group,shared,hints", PICKED)
def test_forms_that_sizes_pick(dev, n_seq, rows, first, most, heads, g, dim, page, width, group, shared, hints, is_bf16):
    print(f"form {n_seq} x {rows} of {first[:3]} {most} heads={heads} x {g} dim={dim} page={page} width={width} group={group} {hints} bf16={is_bf16}", flush=True)
    r = rng(n_seq + rows + dim)
    lengths = (first + [int(x) for x in r.integers(rows, max(most, rows + 1), n_seq)])[:n_seq]
    if shared:                                               # members hold the prefix, but for some that end inside it
        lengths = [m if j % 7 == 5 else max(m, shared[j // group] + rows) for j, m in enumerate(lengths)]
    counts, pos = [rows] * n_seq, [m - rows for m in lengths]
    c = Cache(dev, r, lengths, page, heads, dim, group, shared, width=width)
    q = r.normal(0, 1, (sum(counts), heads * g, dim))
    got = attention(dev, c, q, counts, pos, g, group, shared, is_bf16, **hints)
    check_attention(c, got, q, counts, pos, is_bf16)
    assert (attention(dev, c, q, counts, pos, g, group, shared, is_bf16, **hints) == got).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 64)])
def test_not_finite_in_groups_over_the_positions(dev, dim, page, is_bf16):
    """The same with one, two and four groups of a block over the positions, split and in one piece."""
    r = rng(56 + dim)
    counts, pos = [65] * 3, [1000, 0, 440]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], page, 16, dim, width=1120 // page)
    put(c, "k", 0, range(0, 576), 1, 7, NAN)                 # the first part, and every group's first positions
    put(c, "k", 0, range(1030, 1065), 2, 0, NAN)
    low(c, 0, range(0, 1064), 3)                             # all but the last position
    low(c, 1, range(0, 65), 0)                               # all
    low(c, 1, range(0, 32), 1)                               # what one group has
    low(c, 2, range(32, 500), 5)                             # what the others have, and all of it in the first rows but one group's
    c.upload()
    q = r.normal(0, 1, (195, 16, dim))
    q[:, :, 2] = 1.0
    q[70, 4, 9] = q[194, 15, 0] = q[3, 15, dim - 1] = np.nan
    want = check(c, q, counts, pos, 1, is_bf16, [(1, None, m) for m in ({}, dict(max_len=600), dict(max_len=200), dict(max_len=32))])
    assert np.isnan(want[:65, 1]).all() and np.isnan(want[:64, 3]).all() and np.isfinite(want[64, 3]).all() and np.isnan(want[65:130, 0]).all()
    assert np.isnan(want[65:97, 1]).all() and np.isfinite(want[97:130, 1]).all() and np.isfinite(want[130:, 5]).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,group,shared,hints", [(1, 1, None, dict(max_len=64)), (1, 1, None, {}), (2, 4, [300], {}), (50, 1, None, {}), (50, 1, None, dict(max_len=100)),
                                                      (50, 1, None, dict(max_len=30))])
def test_results_in_the_rows_of_q(dev, rows, group, shared, hints, is_bf16):
    """out may be q: the same bits."""
    from qwenasr_amd import kernels as K
    from test_gpu_hypotheses import ints, prefix, up
    r = rng(57)
    counts, pos = [rows] * 4, [900, 310, 320, 305]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 16, 2, 128, group, shared, width=64)
    q = r.normal(0, 1, (4 * rows, 6, 128))
    a, b = up(dev, q, is_bf16), up(dev, q, is_bf16)
    out = up(dev, np.zeros((4 * rows, 768)), is_bf16)
    more = dict(row_start=ints(dev, prefix(counts)), group=group, shared=None if shared is None else ints(dev, shared), bf16=is_bf16, **hints)
    for o, x in ((out, a), (b, b)):
        K.attention_kvp(o, x, c.k, c.v, c.n_pages, c.t, c.width, ints(dev, pos), 4 * rows, 4, rows, 6, 2, 128, 16, 128 ** -0.5, **more)
    assert (out.numpy().reshape(-1) == b.numpy().reshape(-1)).all() and (a.numpy() == up(dev, q, is_bf16).numpy()).all()
