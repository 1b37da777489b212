"""The operators for several hypotheses of one prompt against lists and float64: pages of a KV cache forked, compacted
and written, the attention over them, log probabilities of tokens."""
import ctypes as C

import numpy as np
import pytest

import refp
from conftest import bf16, bf16f, rng
from refp import U, pages_of

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8                 # half a step of bf16, relative
NAN16 = 0x7FC1                   # what stands where nothing was written


class At:
    """A device array from element `off` on."""

    def __init__(self, d, off):
        self.d, self.dev, self.shape, self.ptr = d, d.dev, d.shape, d.offset(off)


def up(dev, a, is_bf16):
    return dev.upload(bf16(a) if is_bf16 else np.asarray(a, np.float32))


def held(a, is_bf16):
    """What the type keeps of a."""
    return (bf16f(bf16(a)) if is_bf16 else np.asarray(a, np.float32)).astype(np.float64)


def values(d, is_bf16):
    a = d.numpy()
    return (bf16f(a) if is_bf16 else a).astype(np.float64)


def ints(dev, v):
    return dev.upload(np.asarray(v, np.int32).reshape(np.shape(v)))


def prefix(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


# ---------------------------------------------------------------------------
# fork and compact
# ---------------------------------------------------------------------------

class Pools:
    """Pools of random bits on both sides."""

    def __init__(self, dev, r, n_pools, n_pages, heads, page, row_bytes, gap=0):
        self.geo = (n_pools, n_pages, heads, page, row_bytes)
        self.one = n_pages * heads * page * row_bytes
        self.stride = self.one + 16 * gap
        self.host = r.integers(0, 256, n_pools * self.stride, dtype=np.uint8)
        self.dev = dev.upload(self.host)

    def pages(self):
        n_pools, n_pages, heads, page, row = self.geo
        return [self.host[i * self.stride:i * self.stride + self.one].reshape(n_pages, heads, page, row) for i in range(n_pools)]

    def args(self):
        n_pools, n_pages, heads, page, row = self.geo
        return self.dev, n_pools, n_pages, heads, page, row

    def same(self):
        return (self.dev.numpy() == self.host).all()


def run_fork(dev, pools, table, length, parent, rows, max_rows=None, null_parent=False):
    """Both sides; returns the new (table, len), checked."""
    from qwenasr_amd import kernels as K
    n, (n_seq, width), page = len(parent), table.shape, pools.geo[3]
    uniform = max_rows is None and len(set(rows)) <= 1
    most = (rows[0] if n else 1) if uniform else max(rows, default=1) if max_rows is None else max_rows
    t, p, m, s = ints(dev, np.full((n + 1, width), 7)), ints(dev, np.full(n + 1, 7)), ints(dev, np.full(n + 1, 7)), ints(dev, [7, 7, 7])
    K.kvp_fork(t, p, m, s, ints(dev, table) if table.size else dev.zeros(1, np.int32), ints(dev, length) if n_seq else dev.zeros(1, np.int32), n, n_seq,
               width, *pools.args(), parent=None if null_parent else ints(dev, parent) if n else dev.zeros(1, np.int32),
               row_start=None if uniform else ints(dev, prefix(rows)), max_rows=most, pool_stride=pools.stride)
    want = refp.fork(table, length, parent, [min(x, most) for x in rows], pools.geo[1], page)
    for src, dst, part in want[4]:
        for pool in pools.pages():
            pool[dst, :, :part] = pool[src, :, :part]
    got = t.numpy(), p.numpy(), m.numpy(), s.numpy()
    assert tuple(got[3]) == (*want[3], 7)
    assert (got[0][:n] == want[0]).all() and (got[1][:n] == want[1]).all() and (got[2][:n] == want[2]).all()
    assert (got[0][n:] == 7).all() and got[1][n] == 7 and got[2][n] == 7
    assert pools.same()
    return got[0][:n], got[2][:n], want[3][0]


def run_compact(dev, pools, table, length, in_place=False):
    from qwenasr_amd import kernels as K
    n, width = table.shape
    t, s = ints(dev, np.vstack([table, np.full((1, width), 7)])), ints(dev, [7, 7, 7])
    o = t if in_place else ints(dev, np.full((n + 1, width), 7))
    K.kvp_compact(o, s, t, ints(dev, length), n, width, *pools.args(), pool_stride=pools.stride)
    want, status, moved = refp.compact(table, length, pools.geo[1], pools.geo[3])
    for pool in pools.pages():
        for a, b in moved.items():
            pool[b] = pool[a]
    got = o.numpy()
    assert tuple(s.numpy()) == (*status, 7) and (got[:n] == want).all() and (got[n] == 7).all() and pools.same()
    return got[:n]


@pytest.mark.parametrize("page,n_pages,heads,row,n_pools,gap,seed", [(16, 60, 2, 16, 3, 0, 0), (16, 333, 1, 256, 2, 5, 1), (64, 40, 3, 128, 4, 1, 2),
                                                                      (256, 33, 2, 48, 1, 0, 3), (32, 2100, 1, 16, 2, 3, 4)])
def test_forks_in_a_row(dev, page, n_pages, heads, row, n_pools, gap, seed):
    """Random forks and compactions one after another: every table, every byte of every pool."""
    r = rng(seed)
    pools = Pools(dev, r, n_pools, n_pages, heads, page, row, gap)
    width = max(4, n_pages // 6)
    table, length = np.full((1, width), -1, np.int32), np.zeros(1, np.int32)
    for step in range(12):
        n = int(r.integers(1, 9)) if step % 4 else int(r.integers(1, 70))
        parent = r.integers(-1, len(length) + 1, n)
        rows = [int(x) for x in r.choice([0, 1, 1, 2, page - 1, page, 2 * page + 3], n)] if step % 3 else [int(r.integers(0, page + 2))] * n
        print(f"fork page={page} step={step} {len(length)} -> {n}", flush=True)
        t, m, missing = run_fork(dev, pools, table, length, parent, rows)
        if missing:                                  # the old ones still hold: keep a few and go on
            table, length = table[:2], length[:2] // 2
            continue
        table, length = t, m
        if step % 5 == 4:
            table = run_compact(dev, pools, table, length, in_place=step % 2 == 0)


def test_fork_who_keeps_the_last_page(dev):
    """The sequence with the most positions of a common last page goes on in it if it gets rows, the first of equals; a
    page that one holds full is gone on in by nobody."""
    pools = Pools(dev, rng(9), 2, 24, 2, 16, 32)
    table = np.array([[3, 5, -1, -1]] * 6, np.int32)
    for length, rows in [([20] * 6, [1] * 6), ([20] * 6, [0, 0, 1, 1, 0, 1]), ([20, 25, 20, 25, 18, 17], [1] * 6), ([20, 25, 20, 25, 18, 17], [1, 0, 1, 1, 1, 0]),
                         ([20, 25, 20, 24, 18, 17], [1, 0, 1, 1, 1, 0]), ([20, 32, 20, 24, 18, 17], [1, 0, 1, 1, 1, 0]), ([20, 40, 20, 16, 0, 31], [1] * 6)]:
        print("who keeps", length, rows, flush=True)
        run_fork(dev, pools, table, length, list(range(6)), rows, max_rows=1, null_parent=True)


def test_fork_with_odd_tables(dev):
    """Entries that name no page, lengths out of range, the same page twice in one table, no sequences, empty parents."""
    pools = Pools(dev, rng(10), 1, 20, 1, 16, 16)
    table = np.array([[2, -5, 20, 4], [1 << 30, 3, -1, -1], [6, 6, 6, 6], [-1, 9, 9, 1]], np.int32)
    run_fork(dev, pools, table, [40, 17, 50, 70], [0, 1, 2, 3, 0, 2], [3, 1, 1, 0, 1, 1])
    run_fork(dev, pools, table, [-7, 1 << 30, 16, 2 ** 31 - 1], [0, 2, 2, -1, 4, 1 << 30, -(1 << 31), 1], [1, 1, 1, 1, 1, 1, 0, 0])
    run_fork(dev, pools, table, [20, 3, 0, 0], [], [])
    run_fork(dev, pools, np.zeros((0, 3), np.int32), [], [0, -1], [5, 2])
    run_compact(dev, pools, table, [40, 17, 50, 70])
    run_compact(dev, pools, table, [64, 64, 64, 64], in_place=True)
    run_compact(dev, pools, table, [-1, 0, 0, 0])


def test_fork_that_does_not_fit(dev):
    """Too few pages, or too long a table: nothing but empty sequences and the number that is missing."""
    pools = Pools(dev, rng(11), 2, 10, 1, 16, 16)
    table = np.array([[0, 1, 2, 3], [4, 5, 6, -1]], np.int32)
    assert run_fork(dev, pools, table, [50, 33], [0, 1, 0, 0, 1], [1] * 5)[2] == 0          # three copies: the last three pages
    assert run_fork(dev, pools, table, [50, 33], [0, 1, 0, 0, 0, 1], [1] * 6)[2] == 1       # four
    assert run_fork(dev, pools, table, [50, 33], [0, 1], [15, 60], max_rows=60)[2] == -2
    assert run_fork(dev, pools, table, [50, 33], [0, 1], [14, 31], max_rows=60)[2] == 0
    # rows past max_rows do not count
    assert run_fork(dev, pools, table, [50, 33], [0, 1], [14, 1 << 20], max_rows=3)[2] == 0
    big = Pools(dev, rng(12), 1, 16, 1, 16, 16)
    wide = np.full((40, 1 << 16), -1, np.int32)
    assert run_fork(dev, big, wide, [0] * 40, list(range(40)), [(1 << 20) - 5] * 40, null_parent=True)[2] == 40 * (1 << 16) - 16


def test_fork_of_many(dev):
    """The most sequences and pages there may be."""
    r = rng(13)
    n, n_pages, width, page = 2048, 1 << 18, 130, 16
    pools = Pools(dev, r, 1, n_pages, 1, page, 16)
    table = r.permutation(n_pages)[:n * 120].reshape(n, 120).astype(np.int32)
    table = np.hstack([table, np.full((n, 10), -1, np.int32)])
    length = r.integers(1, 1920, n)
    table[1::2, :60] = table[0::2, :60]                              # pairs share what both have of their first half
    parent = r.integers(0, n, n)
    print("fork 2048 of 2048", flush=True)
    t, m, missing = run_fork(dev, pools, table, length, parent, [1] * n)
    assert not missing
    run_compact(dev, pools, t, m)


def test_copies_past_32_bits(dev):
    """Pages more than 2^32 bytes into a pool are copied and moved to their place."""
    from qwenasr_amd import kernels as K
    n_pages, heads, page, row = 5000, 8, 256, 512                    # 1 MiB pages
    one = heads * page * row
    pool = dev.empty(n_pages * one, np.uint8)
    table = ints(dev, [[4990, 4995], [4990, 4995], [1, 4999]])
    marks = {p: rng(p).integers(0, 256, one, dtype=np.uint8) for p in (4990, 4995, 4999, 1)}
    raw = lambda p: C.c_void_p(pool.offset(p * one).value)  # noqa: E731
    from qwenasr_amd._lib import check, lib
    for p, v in marks.items():
        check(lib().qasr_hip_upload(dev.h, raw(p), v.ctypes.data_as(C.c_void_p), one))

    def read(p):
        v = np.empty(one, np.uint8)
        check(lib().qasr_hip_download(dev.h, v.ctypes.data_as(C.c_void_p), raw(p), one))
        return v

    t, p_, m, s = ints(dev, np.zeros((3, 2))), ints(dev, [0] * 3), ints(dev, [0] * 3), ints(dev, [0, 0])
    K.kvp_fork(t, p_, m, s, table, ints(dev, [300, 300, 512]), 3, 3, 2, pool, 1, n_pages, heads, page, row, max_rows=1)
    assert tuple(s.numpy()) == (-1, 4)                               # the third is full
    K.kvp_fork(t, p_, m, s, table, ints(dev, [300, 300, 511]), 3, 3, 2, pool, 1, n_pages, heads, page, row, max_rows=1)
    assert (t.numpy() == [[4990, 4995], [4990, 0], [1, 4999]]).all() and tuple(s.numpy()) == (0, 5)
    got, want = read(0).reshape(heads, page, row), marks[4995].reshape(heads, page, row)
    assert (got[:, :44] == want[:, :44]).all()
    K.kvp_compact(t, s, t, m, 3, 2, pool, 1, n_pages, heads, page, row)
    assert (t.numpy() == [[2, 3], [2, 0], [1, 4]]).all() and tuple(s.numpy()) == (3, 5)
    assert (read(2) == marks[4990]).all() and (read(3) == marks[4995]).all() and (read(4) == marks[4999]).all()


# ---------------------------------------------------------------------------
# the paged cache
# ---------------------------------------------------------------------------

class Cache:
    """K and V pools whose unwritten places hold NaN, and random tables; members of a group name the same pages for the
    whole pages of their first `shared` positions and hold copies of the rest of those."""

    def __init__(self, dev, r, lengths, page, heads, dim, group=1, shared=None, spare=3, width=None, fill=True):
        self.dev, self.page, self.heads, self.dim = dev, page, heads, dim
        n = len(lengths)
        shared = [0] * pages_of(n, group) if shared is None else shared
        # a group's first sequence names its whole prefix, also where it does not see all of it
        lengths = [m if j % group else max(m, shared[j // group]) for j, m in enumerate(lengths)]
        need = [pages_of(max(m, 0), page) for m in lengths]
        self.width = width or max(max(need), 1) + 1
        table = np.full((n, self.width), -1, np.int64)
        count = 0
        for j in range(n):
            f = j // group * group
            common = min(shared[j // group] // page, need[j], need[f]) if j != f else 0
            table[j, :common] = table[f, :common]
            table[j, common:need[j]] = np.arange(count, count + need[j] - common)
            count += need[j] - common
        self.n_pages = count + spare
        order = r.permutation(self.n_pages)
        table[table >= 0] = order[table[table >= 0]]
        self.table = table.astype(np.int32)
        shape = (self.n_pages, heads, page, dim)
        self.bits = {x: np.full(shape, NAN16, np.uint16) for x in "kv"}
        if fill:
            for j in range(n):
                f = j // group * group
                for s in range(need[j]):
                    m = min(page, lengths[j] - s * page)
                    for x in "kv":
                        to = self.bits[x][self.table[j, s]]
                        fresh = to[0, :m, 0] == NAN16
                        val = bf16(r.normal(0, 1 if x == "k" else 0.6, (heads, m, dim)))
                        both = max(0, min(m, shared[j // group] - s * page)) if j != f else 0
                        val[:, :both] = self.bits[x][self.table[f, s], :, :both]
                        to[:, :m][:, fresh] = val[:, fresh]
        self.upload()

    def upload(self):
        self.k, self.v = self.dev.upload(self.bits["k"]), self.dev.upload(self.bits["v"])
        self.t = ints(self.dev, self.table)

    def floats(self):
        return {x: bf16f(b).astype(np.float64) for x, b in self.bits.items()}


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("counts,pos,heads,dim,page,pad,off", [
    ([1], [0], 1, 64, 16, 0, 0), ([1] * 32, list(range(0, 640, 20)), 8, 128, 64, 0, 0), ([5, 0, 17, 1], [3, 9, 15, 40], 2, 128, 16, 3, 1),
    ([100, 33], [0, 250], 3, 64, 256, 8, 2), ([7, 7], [-3, 44], 2, 64, 16, 64, 0), ([300], [17], 8, 128, 32, 1024, 0), ([9, 2], [1000, -9], 1, 128, 16, 1, 3)])
def test_write(dev, counts, pos, heads, dim, page, pad, off, is_bf16):
    from qwenasr_amd import kernels as K
    print(f"write {counts} at {pos} heads={heads} dim={dim} page={page} bf16={is_bf16}", flush=True)
    r = rng(sum(counts) + 7 * dim + page)
    cap = max(64, max(a + b for a, b in zip(counts, pos) if b < 900))
    c = Cache(dev, r, [cap] * len(counts), page, heads, dim, fill=False, width=pages_of(cap, page))
    c.table[-1, 0], c.table[0, -1] = (c.n_pages, -1) if len(counts) > 1 else (c.table[-1, 0], c.table[0, -1])
    c.upload()
    hd, total = heads * dim, sum(counts)
    ld = hd + pad
    k, v = r.normal(0, 1, total * ld + 8), r.normal(0, 1e3, total * ld + 8)
    k[off], v[off + 1] = np.inf, -np.inf
    if not is_bf16:
        v[off + 2] = 3.4e38                                          # past bf16's largest
    K.kvp_write(c.k, c.v, c.n_pages, At(up(dev, k, is_bf16), off), At(up(dev, v, is_bf16), off), c.t, c.width, ints(dev, pos), total + 1, len(counts),
                max(counts), heads, dim, page, row_start=ints(dev, prefix(counts)), ld=ld, bf16=is_bf16)
    for x, d, rows in (("k", c.k, k), ("v", c.v, v)):
        want, bits = c.bits[x], bf16(rows)
        for j, n in enumerate(counts):
            for i in range(n):
                p, at = pos[j] + i, off + (prefix(counts)[j] + i) * ld
                if 0 <= p < c.width * page and 0 <= c.table[j, p // page] < c.n_pages:
                    want[c.table[j, p // page], :, p % page] = bits[at:at + hd].reshape(heads, dim)
        assert (d.numpy() == want).all(), x


def test_write_nan_and_rows_past_max_rows(dev):
    from qwenasr_amd import kernels as K
    c = Cache(dev, rng(1), [40, 40], 16, 2, 64, fill=False)
    x = rng(2).normal(0, 1, (20, 128)).astype(np.float32)
    x[0, 0], x[1, 3] = np.nan, -np.nan
    d = dev.upload(x)
    K.kvp_write(c.k, c.v, c.n_pages, d, d, c.t, c.width, ints(dev, [0, 4]), 20, 2, 3, 2, 64, 16, row_start=ints(dev, [0, 5, 20]))
    got = bf16f(c.k.numpy())
    assert np.isnan(got[c.table[0, 0], 0, 0, 0]) and np.isnan(got[c.table[0, 0], 0, 1, 3])
    written = ~np.isnan(got[:, :, :, 5]).all(1)
    assert written.sum() == 6 and written[c.table[0, 0], :3].all() and written[c.table[1, 0], 4:7].all()
    # max_rows each, without row starts; row starts outside the buffer are held to it
    K.kvp_write(c.k, c.v, c.n_pages, d, d, c.t, c.width, ints(dev, [20, 20]), 20, 2, 2, 2, 64, 16)
    assert (c.k.numpy()[c.table[1, 1], :, 4] == bf16(x[2]).reshape(2, 64)).all()
    K.kvp_write(c.k, c.v, c.n_pages, d, d, c.t, c.width, ints(dev, [30, 30]), 20, 2, 50, 2, 64, 16, row_start=ints(dev, [-5, 1, 1 << 30]))
    assert (c.k.numpy()[c.table[1, 1], :, 14] == bf16(x[1]).reshape(2, 64)).all()


def attention(dev, c, q, counts, pos, g, group=1, shared=None, is_bf16=False, pad=0, off=0, behind=2, scale=None, max_rows=None, **more):
    """[rows][heads][dim] float64; rows behind the last one and columns between rows are checked to be left alone."""
    from qwenasr_amd import kernels as K
    hq, total = c.heads * g, int(sum(counts))
    width = hq * c.dim
    ld = width + pad
    rows = np.full((total + behind) * ld + 8, 3.0)
    rows[off:off + (total + behind) * ld].reshape(-1, ld)[:total, :width] = q.reshape(total, width)
    out = up(dev, np.full((total + behind, width), 7.0), is_bf16)
    K.attention_kvp(out, At(up(dev, rows, is_bf16), off), c.k, c.v, c.n_pages, c.t, c.width, ints(dev, pos), total + behind, len(counts),
                    max(counts) if max_rows is None else max_rows, hq, c.heads, c.dim, c.page, c.dim ** -0.5 if scale is None else scale,
                    row_start=ints(dev, prefix(counts)), ldq=ld, group=group, shared=None if shared is None else ints(dev, shared), bf16=is_bf16, **more)
    got = values(out, is_bf16)
    assert (got[total:] == 7.0).all()
    return got[:total].reshape(total, hq, c.dim)


def check_attention(c, got, q, counts, pos, is_bf16=False, scale=None):
    pools, at = {x: np.nan_to_num(v) for x, v in c.floats().items()}, 0
    for j, n in enumerate(counts):
        end = min(max(pos[j] + n, 0), c.width * c.page)
        k, there = refp.gather(pools["k"], c.table[j], end, c.page)
        v, _ = refp.gather(pools["v"], c.table[j], end, c.page)
        seen = (np.arange(end)[None] <= pos[j] + np.arange(n)[:, None]) & there
        want, bound = refp.attend(held(q[at:at + n], is_bf16), k, v, seen, c.dim ** -0.5 if scale is None else scale, 2.0 ** -17 if is_bf16 else U)
        # and the result's own rounding
        bound = bound * (1 + BF16) + (BF16 if is_bf16 else U) * np.abs(want)
        off = np.abs(got[at:at + n] - want)
        assert (off <= bound).all(), (j, np.nanmax(off / np.maximum(bound, 1e-300)))
        assert (got[at:at + n][~seen.any(1)] == 0).all()
        at += n


ATTN = [
    # counts, pos, group, shared, heads, g, dim, page
    ([1], [0], 1, None, 1, 1, 64, 16),
    ([1], [403], 1, None, 8, 2, 128, 64),
    ([1] * 8, [404 + 5 * j for j in range(8)], 8, [384], 8, 2, 128, 64),
    ([1] * 8, [404 + 5 * j for j in range(8)], 8, [397], 2, 2, 128, 16),                  # ends inside a page and a tile
    ([1] * 12, [50, 90, 3, 70, 75, 80, 100, 33, 64, 65, 63, 40], 4, [31, 0, 33], 2, 3, 64, 32),
    ([1] * 7, [200, 210, 220, 230, 240, 250, 260], 3, [200, 100, 260], 4, 1, 128, 128),   # a last group of one
    ([2, 0, 5, 1, 3, 1], [300, 300, 310, 320, 290, 301], 6, [290], 2, 4, 128, 256),       # members without rows
    ([0, 3, 1], [100, 70, 99], 3, [70], 1, 5, 64, 16),                                    # the first among them
    ([1, 1, 1, 1], [-5, 0, 10, 40], 2, [30, 41], 2, 2, 128, 16),                          # positions before the prefix' end
    ([3, 2], [-2, -1], 1, None, 2, 2, 64, 16),
    ([1] * 3, [2000, 1999, 37], 1, None, 1, 16, 128, 16),
    ([1] * 40, [300 + 3 * j for j in range(40)], 40, [300], 1, 7, 64, 32),
    ([16, 5], [100, 0], 2, [90], 2, 2, 64, 64),                                           # 32 queries a sequence
    ([17, 5, 40], [100, 0, 3], 3, [2], 2, 2, 128, 32),                                    # 80
    ([130, 1, 77], [0, 500, 31], 1, None, 2, 2, 128, 16),
    ([67, 200], [700, 0], 2, [64], 1, 3, 64, 256),
    ([333], [0], 1, None, 1, 1, 128, 64),
    ([1] * 2, [5000, 7000], 2, [4999], 1, 2, 128, 64),
    ([1] * 34, [4100 + 3 * (j % 17) for j in range(34)], 17, [4090, 4100], 2, 2, 128, 16),    # read once by the hints, too
    ([300, 1, 131], [10, 600, 0], 3, [0], 2, 3, 128, 64),
    ([45], [2500], 1, None, 1, 1, 64, 32),                                                # splits of one tile
    ([129, 128], [-20, 333], 1, None, 1, 1, 128, 128),
    ([30, 17] * 10, [3 * j for j in range(20)], 1, None, 8, 2, 64, 16),                   # a tile for each of 160 CUs
    ([33, 50, 20, 41] * 4, [9 * j for j in range(16)], 4, [0] * 4, 8, 1, 128, 32),
    ([17 + j % 23 for j in range(140)], [j % 50 for j in range(140)], 1, None, 1, 2, 64, 16),    # more sequences than lanes
]


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("counts,pos,group,shared,heads,g,dim,page", ATTN)
def test_attention(dev, counts, pos, group, shared, heads, g, dim, page, is_bf16):
    print(f"attention {counts[:8]} at {pos[:8]} group={group} shared={shared} heads={heads} x {g} dim={dim} page={page} bf16={is_bf16}", flush=True)
    r = rng(sum(counts) + heads + page)
    # tables of 700 positions and more: without hints prefixes are read once (shorter ones are not worth a merge)
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], page, heads, dim, group, shared,
              width=pages_of(max(700, *(a + b for a, b in zip(counts, pos))), page) + 1)
    q = r.normal(0, 1, (sum(counts), heads * g, dim))
    pad, off = ((0, 0), (8, 0), (3, 1))[(sum(counts) + page // 16) % 3]
    got = attention(dev, c, q, counts, pos, g, group, shared, is_bf16, pad, off)
    check_attention(c, got, q, counts, pos, is_bf16)
    # the hints change the split, the prefix' rows may be read from every sequence's own table: rounding
    longest = max(max(a + b for a, b in zip(counts, pos)), 1)
    for more in (dict(max_len=longest, max_own=max(1, longest - min(shared or [0]))), dict(max_len=1), dict(max_len=64, max_own=32), dict(max_own=100)):
        again = attention(dev, c, q, counts, pos, g, group, shared, is_bf16, pad, off, **more)
        check_attention(c, again, q, counts, pos, is_bf16)
    alone = attention(dev, c, q, counts, pos, g, 1, None, is_bf16, pad, off)
    check_attention(c, alone, q, counts, pos, is_bf16)
    # the same call gives the same bits
    assert (attention(dev, c, q, counts, pos, g, group, shared, is_bf16, pad, off) == got).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("scale,rows", [(0.0, 1), (-0.3, 1), (-0.3, 40), (0.0, 40), (40.0, 3), (40.0, 60), (1e-6, 2)])
def test_attention_scale(dev, scale, rows, is_bf16):
    r = rng(17)
    counts, pos = [rows, max(1, rows - 1)], [70, 3]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 16, 2, 64)
    q = r.normal(0, 1, (sum(counts), 4, 64))
    check_attention(c, attention(dev, c, q, counts, pos, 2, is_bf16=is_bf16, scale=scale), q, counts, pos, is_bf16, scale)


@pytest.mark.parametrize("rows", [1, 6, 50])
def test_attention_pages_that_are_none(dev, rows):
    """Positions of entries that name no page do not exist; a sequence of none gives zeros; positions past the table too."""
    r = rng(18)
    counts, pos = [rows] * 4, [90, 90, 40, 200]
    c = Cache(dev, r, [90 + rows] * 3 + [176], 16, 2, 128, width=11)        # the last: all that its table names
    c.table[0, 1] = -1
    c.table[0, 4] = c.n_pages
    c.table[1, :] = -(1 << 31)
    c.table[2, 2] = 1 << 30
    c.upload()
    q = r.normal(0, 1, (4 * rows, 4, 128))
    for group, shared in ((1, None), (4, [0]), (2, [0, 0])):
        got = attention(dev, c, q, counts, pos, 2, group, shared)
        check_attention(c, got, q, counts, pos)
        assert (got[rows:2 * rows] == 0).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [4, 40])
def test_attention_not_finite(dev, rows, is_bf16):
    """What a row does not see does not reach it; what it sees counts as in the formula."""
    r = rng(19)
    counts, pos = [rows, rows], [50, 20]
    c = Cache(dev, r, [50 + rows, 20 + rows], 16, 2, 64)
    q = r.normal(0, 1, (2 * rows, 4, 64))
    clean = attention(dev, c, q, counts, pos, 2, is_bf16=is_bf16)

    def put(x, j, p, h, d, bits):
        c.bits[x][c.table[j, p // 16], h, p % 16, d] = bits
        c.upload()

    # the position of the last row but one: seen by two rows
    put("v", 0, 50 + rows - 2, 0, 5, 0x7F80)
    got = attention(dev, c, q, counts, pos, 2, is_bf16=is_bf16)
    see = got[rows - 2:rows, :2, 5]
    assert np.isposinf(see).all()
    rest = got.copy()
    rest[rows - 2:rows, :2, 5] = clean[rows - 2:rows, :2, 5]
    assert np.isfinite(rest).all() and np.allclose(rest, clean, rtol=1e-2 if is_bf16 else 1e-4, atol=1e-2 if is_bf16 else 1e-5)
    # NaN in K of the same position, and -infinity against a K of the other sequence
    put("k", 0, 50 + rows - 2, 1, 7, 0x7FC0)
    got = attention(dev, c, q, counts, pos, 2, is_bf16=is_bf16)
    assert np.isnan(got[rows - 2:rows, 2:]).all() and np.isfinite(got[:rows - 2]).all() and np.isfinite(got[rows:]).all()
    # an infinite K: its score is an infinity: weight 0, or NaN for the row
    c.bits["k"][c.table[1, 0], 0, 3, 0] = 0x7F80
    c.upload()
    got = attention(dev, c, q, counts, pos, 2, is_bf16=is_bf16)
    positive = held(q, is_bf16)[rows:, :2, 0] > 0
    assert (np.isnan(got[rows:, :2]).all(2) == positive).all() and np.isfinite(got[rows:, :2][~positive]).all()
    assert np.isfinite(got[rows:, 2:]).all() and np.isfinite(got[:rows - 2]).all()
    # a row of q that holds NaN: that row and head alone
    q[1, 3, 9] = np.nan
    got = attention(dev, c, q, counts, pos, 2, is_bf16=is_bf16)
    assert np.isnan(got[1, 3]).all() and np.isfinite(got[0]).all() and np.isfinite(got[1, :3]).all()


@pytest.mark.parametrize("is_bf16", [False, True])
def test_attention_not_finite_behind_a_shared_prefix(dev, is_bf16):
    """NaN in what one member holds behind the prefix, and in the prefix past what a short member sees."""
    r = rng(20)
    counts, pos = [1] * 6, [100, 101, 102, 103, 60, 105]
    c = Cache(dev, r, [p + 1 for p in pos], 16, 2, 128, 6, [96], width=50)
    q = r.normal(0, 1, (6, 4, 128))
    clean = attention(dev, c, q, counts, pos, 2, 6, [96], is_bf16)
    for x in "kv":
        c.bits[x][c.table[2, 6], :, 2, 3] = 0x7FC0                    # member 2's position 98
        c.bits[x][c.table[0, 5], :, 1, 3] = 0x7FC0                    # the prefix' position 81: member 4 does not see it
    c.upload()
    got = attention(dev, c, q, counts, pos, 2, 6, [96], is_bf16)
    assert np.isnan(got[[0, 1, 2, 3, 5]]).any(2).all()
    assert np.allclose(got[4], clean[4], rtol=1e-2 if is_bf16 else 1e-4, atol=1e-2 if is_bf16 else 1e-5)


def test_attention_bound_of_rows(dev):
    """max_rows may be far above what there is."""
    r = rng(23)
    counts, pos = [3, 1], [20, 900]
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 32, 2, 64)
    q = r.normal(0, 1, (4, 4, 64))
    check_attention(c, attention(dev, c, q, counts, pos, 2, max_rows=1 << 24), q, counts, pos)


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("n_seq,rows,heads,g,dim,width", [(2048, 1, 1, 32, 64, 60), (2048, 1, 2, 16, 128, 60), (300, 20, 1, 32, 64, 60), (2048, 1, 1, 32, 128, 20),
                                                          (2048, 1, 2, 16, 64, 20), (700, 1, 2, 2, 128, 10), (400, 1, 1, 3, 64, 150), (700, 2, 2, 8, 128, 24)])
def test_attention_of_many_sequences(dev, n_seq, rows, heads, g, dim, width, is_bf16):
    """Up to the most sequences, and so many rows x heads that the scratch area holds one part of each or none: no prefix and
    no split, whatever the hints."""
    r = rng(29)
    counts, pos = [rows] * n_seq, [int(x) for x in r.integers(30, 70, n_seq)]
    groups = pages_of(n_seq, 16)
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 16, heads, dim, 16, [30] * groups, width=width)
    q = r.normal(0, 1, (sum(counts), heads * g, dim))
    check_attention(c, attention(dev, c, q, counts, pos, g, 16, [30] * groups, is_bf16), q, counts, pos, is_bf16)
    check_attention(c, attention(dev, c, q, counts, pos, g, is_bf16=is_bf16), q, counts, pos, is_bf16)


def test_attention_rows_past_max_rows(dev):
    """Rows past max_rows are left as they were, also inside a group."""
    from qwenasr_amd import kernels as K
    r = rng(21)
    counts, pos, most = [5, 2, 7, 1], [60, 61, 62, 63], 3
    c = Cache(dev, r, [a + b for a, b in zip(counts, pos)], 32, 2, 64, 4, [60], width=25)
    q = r.normal(0, 1, (15, 4, 64))
    for group, shared in ((1, None), (4, [60]), (2, [60, 32])):
        got = attention(dev, c, q, counts, pos, 2, group, shared, max_rows=most)
        at = 0
        for j, n in enumerate(counts):
            m = min(n, most)
            assert (got[at + m:at + n] == 7.0).all()
            pools = c.floats()
            k, _ = refp.gather(np.nan_to_num(pools["k"]), c.table[j], pos[j] + m, 32)
            v, _ = refp.gather(np.nan_to_num(pools["v"]), c.table[j], pos[j] + m, 32)
            seen = np.arange(pos[j] + m)[None] <= pos[j] + np.arange(m)[:, None]
            want, bound = refp.attend(held(q[at:at + m], False), k, v, seen, 0.125, U)
            assert (np.abs(got[at:at + m] - want) <= bound + U * np.abs(want)).all()
            at += n
    # max_rows each, without row starts; row starts outside the buffers are held to them
    out = dev.upload(np.full((15, 256), 7.0, np.float32))
    K.attention_kvp(out, dev.upload(q.astype(np.float32)), c.k, c.v, c.n_pages, c.t, c.width, ints(dev, pos), 15, 4, 3, 4, 2, 64, 32, 0.125)
    assert (out.numpy()[12:] == 7.0).all() and (out.numpy()[:12] != 7.0).all()
    out = dev.upload(np.full((15, 256), 7.0, np.float32))
    K.attention_kvp(out, dev.upload(q.astype(np.float32)), c.k, c.v, c.n_pages, c.t, c.width, ints(dev, pos), 15, 4, 3, 4, 2, 64, 32, 0.125,
                    row_start=ints(dev, [-9, 4, 2, 1 << 30, 1 << 30]))
    assert (out.numpy()[6:] == 7.0).all()


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_past_32_bits(dev, rows):
    """Pages more than 2^32 bytes into a pool: written, and read by the attention."""
    from qwenasr_amd import kernels as K
    r = rng(22)
    n_pages, heads, page, dim = 40000, 8, 64, 128                    # 128 KiB pages, 5.2 GB a pool
    kp, vp = dev.empty((n_pages, heads, page, dim), np.uint16), dev.empty((n_pages, heads, page, dim), np.uint16)
    ids = np.array([[39999, 39000, 35001, 39998], [3, 37777, 36666, 12]], np.int32)
    lengths = [200 + rows, 180 + rows] if rows == 1 else [rows + 130, rows + 100]
    pos = [m - rows for m in lengths]
    k, v = r.normal(0, 1, (sum(lengths), heads * dim)), r.normal(0, 0.6, (sum(lengths), heads * dim))
    t = ints(dev, ids)
    K.kvp_write(kp, vp, n_pages, dev.upload(k.astype(np.float32)), dev.upload(v.astype(np.float32)), t, 4, ints(dev, [0, 0]), sum(lengths), 2,
                max(lengths), heads, dim, page, row_start=ints(dev, prefix(lengths)))
    q = r.normal(0, 1, (2 * rows, heads * 2, dim))
    out = dev.zeros((2 * rows, heads * 2 * dim), np.float32)
    K.attention_kvp(out, dev.upload(q.astype(np.float32)), kp, vp, n_pages, t, 4, ints(dev, pos), 2 * rows, 2, rows, 16, heads, dim, page, dim ** -0.5)
    got, at = out.numpy().astype(np.float64).reshape(2 * rows, 16, dim), 0
    for j, m in enumerate(lengths):
        kk, vv = (bf16f(bf16(x[at:at + m])).astype(np.float64).reshape(m, heads, dim) for x in (k, v))
        pick = [0, rows - 1]
        seen = np.arange(m)[None] <= pos[j] + np.array(pick)[:, None]
        want, bound = refp.attend(held(q, False)[j * rows:][pick], kk, vv, seen, dim ** -0.5, U)
        assert (np.abs(got[j * rows:][pick] - want) <= bound + U * np.abs(want)).all()
        at += m


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------

def check_logp(x, targets, k, got, sign=1):
    logp, entropy, ids, top = got
    lp, ent, want_ids, want_top, m, first = refp.logprobs(x, targets, k)
    x = x.astype(np.float64)
    cols = x.shape[1]
    # a term of the sums: the difference and its product with log2 e, the exponential's unit, the additions (at most one a
    # value in a thread, then a few levels); log1p and the two differences
    d = np.where(np.isfinite(x), x - m[:, None], 0.0)
    p = np.exp(np.where(np.isfinite(x), x - m[:, None], -np.inf))
    rest = p.copy()
    rest[np.arange(len(x)), first] = 0
    s = rest.sum(1)
    es = ((3 * np.abs(d) + 90) * U * rest).sum(1)
    tail = es / (1 + s) + 3 * U * np.log1p(s)
    at = np.arange(len(x)), targets
    dt = np.abs(x[at] - m)
    ok = np.isfinite(lp)
    assert (np.abs(np.where(ok, logp, 0) - np.where(ok, lp, 0))[ok] <= (tail + 1.01 * U * (dt + np.abs(lp)))[ok]).all()
    assert (np.isneginf(logp) == np.isneginf(lp)).all()
    eh = ((6 * np.abs(d) + 96) * U * np.abs(d) * rest).sum(1)
    hs = np.abs(np.where(rest > 0, d, 0) * rest).sum(1)
    assert (np.abs(entropy - ent) <= tail + eh / (1 + s) + hs * (es / (1 + s) + 4 * U) / (1 + s) + 2 * U * np.abs(ent)).all()
    assert (ids == want_ids).all()
    ok = np.isfinite(want_top)
    dt = np.abs(np.take_along_axis(x, want_ids, 1) - m[:, None])
    assert (np.abs(np.where(ok, top, 0) - np.where(ok, want_top, 0))[ok] <= (tail[:, None] + 1.01 * U * (dt + np.abs(want_top)))[ok]).all()
    assert (np.isneginf(top) == np.isneginf(want_top)).all()


def logprobs(dev, x, targets, k, is_bf16, pad=0, off=0):
    from qwenasr_amd import kernels as K
    rows, cols = x.shape
    ld = cols + pad
    flat = np.full(rows * ld + off, 50.0)                            # between the rows: larger than any of theirs
    flat[off:].reshape(rows, ld)[:, :cols] = x
    out = [dev.upload(np.full(n, 7, t)) for n, t in ((rows + 1, np.float32), (rows + 1, np.float32), ((rows + 1, k), np.int32), ((rows + 1, k), np.float32))]
    K.token_logprobs(At(up(dev, flat, is_bf16), off), rows, cols, ld=ld, targets=ints(dev, targets), logp=out[0], entropy=out[1], top_ids=out[2],
                     top_logp=out[3], k=k, bf16=is_bf16)
    got = [o.numpy() for o in out]
    assert all((g[rows:] == 7).all() for g in got)
    return [g[:rows].astype(np.float64) if g.dtype == np.float32 else g[:rows] for g in got]


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,cols,k,pad,off", [(1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (5, 31, 31, 1, 1), (2, 63, 32, 0, 3), (9, 64, 5, 8, 0), (4, 1000, 32, 0, 0),
                                                 (3, 2041, 8, 0, 1), (3, 2048, 8, 0, 0), (2, 2049, 9, 0, 0), (4, 4999, 1, 0, 0), (3, 8185, 32, 2, 1),
                                                 (2, 8192, 32, 0, 0), (2, 8192, 3, 0, 5), (2, 8193, 16, 3, 0), (2, 20011, 32, 1, 2), (3, 151936, 16, 0, 0),
                                                 (400, 700, 4, 0, 0), (1, 1 << 20, 32, 0, 1), (3, 16383, 8, 0, 3), (2, 16384, 5, 0, 0), (3, 24001, 32, 1, 1),
                                                 (2, 32761, 9, 7, 2), (2, 32768, 4, 0, 0), (2, 32768, 32, 0, 1), (3, 40003, 12, 2, 0), (600, 20001, 3, 0, 0),
                                                 (2100, 8500, 2, 0, 1)])
def test_logprobs(dev, rows, cols, k, pad, off, is_bf16):
    print(f"logprobs {rows} x {cols} k={k} pad={pad} off={off} bf16={is_bf16}", flush=True)
    r = rng(cols + rows)
    x = r.normal(0, 3, (rows, cols))
    x[:, 0] += np.linspace(0, 40, rows)                              # from flat rows to sure ones
    if cols > 3 and rows > 1:
        x[1, 1:cols // 2] = -np.inf
        x[1, 2] = 0.0
    x = held(x, is_bf16).astype(np.float32)
    targets = np.where(np.arange(rows) % 2, r.integers(0, cols, rows), 0)
    check_logp(x, targets, k, logprobs(dev, x, targets, k, is_bf16, pad, off))


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("cols", [40, 2000, 9000, 30000, 40000])
def test_logprobs_ties_go_to_the_lowest_index(dev, cols, is_bf16):
    r = rng(cols)
    x = np.stack([np.zeros(cols), np.full(cols, -3.5), np.repeat(np.arange(cols // 40 + 1), 40)[:cols] % 2.0, -np.repeat(np.arange(cols // 40 + 1.0), 40)[:cols],
                  np.arange(cols) // 8.0 % 50, np.where(np.arange(cols) % 3 == 0, -0.0, 0.0), r.integers(-2, 3, cols) * 1.0,
                  np.where(np.arange(cols) >= cols - 5, 1.0, -np.inf), np.where(np.arange(cols) == 17, 1.0, -np.inf)])
    x = np.concatenate([x, np.sort(held(r.normal(0, 4, (2, cols)), is_bf16))[:, ::1], np.sort(held(r.normal(0, 4, (1, cols)), is_bf16))[:, ::-1]])
    x = held(x, is_bf16).astype(np.float32)
    targets = np.full(len(x), 17)
    check_logp(x, targets, 32, logprobs(dev, x, targets, 32, is_bf16))


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(12, 3000), (12, 9000), (60, 30000), (5, 151936), (60, 50000)])
def test_logprobs_masked_vocabularies(dev, rows, cols, is_bf16):
    """Few values left, the others -infinity or the type's lowest; and places of a few lanes that hold all the large ones."""
    r = rng(rows + cols)
    x = r.normal(0, 2, (rows, cols))
    low = -3.3895314e38
    for i in range(rows):
        left = r.permutation(cols)[:(1, 3, 31, 32, 33, 200)[i % 6]]
        masked = np.full(cols, (-np.inf, low, -1e4)[i // 6 % 3])
        masked[left] = x[i, left]
        if i % 7 != 6:
            x[i] = masked
        else:
            at = np.arange(cols)
            x[i, at % (512 if is_bf16 else 256) // (8 if is_bf16 else 4) < 8] += 60
    x[1] = low
    x[1, cols // 2:] = -np.inf
    x = held(x, is_bf16).astype(np.float32)
    targets = x.argmax(1)
    check_logp(x, targets, 32, logprobs(dev, x, targets, 32, is_bf16))


@pytest.mark.parametrize("cols", [50, 9000, 40000])
def test_logprobs_next_to_one(dev, cols):
    """A probability of 1 - 1e-9 has a logarithm of -1e-9, not 0; its entropy likewise."""
    x = np.full((3, cols), -60.0, np.float32)
    x[0, 7], x[1, 7], x[2, 7] = 0.0, -35.0, 40.0
    x[0, 30] = -20.0
    got = logprobs(dev, x, [7, 7, 30], 2, False)
    lp, ent, _, top, _, _ = refp.logprobs(x, [7, 7, 30], 2)
    assert -3e-9 < lp[0] < -1e-9
    # e^-20: twice 20 half steps, the exponential's and log1p's units.  The last row's entropy is 50 terms of e^-100 = 3.7e-44
    # times 100, 2e-40 at most together with 9000 of them 3e-38: its terms are below 2^-126 = 1.2e-38, f32's smallest normal
    # number, under which the exponential gives 0 (40000 of them: 1.5e-37)
    tiny = max(1e-37, 4e-42 * cols) if cols > 50 else 2.0 ** -126
    assert np.allclose(got[0], lp, rtol=60 * 3 * U, atol=0) and np.allclose(got[1], ent, rtol=60 * 8 * U, atol=tiny)
    assert np.allclose(got[3], top, rtol=60 * 3 * U, atol=2.0 ** -126)       # the last row's: 9000 e^-100 = 3e-40


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("cols", [60, 9000, 40000])
def test_logprobs_not_finite(dev, cols, is_bf16):
    """NaN or +infinity: NaN values, ids by value with NaN last; -infinity alone: log 0; targets outside: NaN."""
    x = held(rng(cols).normal(0, 1, (7, cols)), is_bf16).astype(np.float32)
    x[0, 5] = np.nan
    x[1, 9] = np.inf
    x[2, :] = -np.inf
    x[3, :] = np.nan
    x[4, :-2] = -np.inf
    x[4, -1] = np.nan
    logp, entropy, ids, top = logprobs(dev, x, [0, 0, 3, 0, 0, -1, cols], 4, is_bf16)
    assert np.isnan(logp[[0, 1, 3, 4, 5, 6]]).all() and np.isneginf(logp[2])
    assert np.isnan(entropy[[0, 1, 3, 4]]).all() and entropy[2] == 0 and np.isfinite(entropy[5:]).all()
    assert np.isnan(top[[0, 1, 3, 4]]).all() and np.isneginf(top[2]).all() and np.isfinite(top[5:]).all()
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x).astype(np.float64), axis=1, kind="stable")[:, :4]
    assert (ids == order).all()


def test_logprobs_parts(dev):
    """Any of the results alone: the same bits as all of them."""
    from qwenasr_amd import kernels as K
    for cols in (500, 20000, 40000):
        x = rng(3).normal(0, 2, (5, cols)).astype(np.float32)
        d, g = dev.upload(x), ints(dev, [1, 2, 3, 4, 5])
        want = [a.astype(np.float32) if a.dtype == np.float64 else a for a in logprobs(dev, x, [1, 2, 3, 4, 5], 6, False)]
        for which in range(4):
            o = dev.zeros(want[which].shape, want[which].dtype)
            K.token_logprobs(d, 5, cols, targets=g if which == 0 else None, k=6, **{["logp", "entropy", "top_ids", "top_logp"][which]: o})
            assert (o.numpy() == want[which]).all(), which
        K.token_logprobs(d, 5, cols)
        K.token_logprobs(d, 0, cols, entropy=d)
    assert (d.numpy() == x).all()


def test_logprobs_many_rows(dev):
    """More rows than one launch and the scratch area take."""
    from qwenasr_amd import kernels as K
    r = rng(5)
    for rows, cols, k in ((70001, 33, 2), (13000, 8200, 32)):
        x = r.normal(0, 1, (rows, cols)).astype(np.float32)
        ids, ent = dev.zeros((rows, k), np.int32), dev.zeros(rows, np.float32)
        K.token_logprobs(dev.upload(x), rows, cols, entropy=ent, top_ids=ids, k=k)
        got, e = ids.numpy(), ent.numpy()
        for i in (0, 1, rows // 2, 65534, 65535, rows - 1):
            if i < rows:
                assert (got[i] == np.argsort(-x[i], kind="stable")[:k]).all() and e[i] > 0
        assert (got[:, 0] == x.argmax(1)).all()


def test_nothing_to_do(dev):
    from qwenasr_amd import kernels as K
    z = dev.zeros(4096, np.int32)
    K.kvp_write(z, z, 1, z, z, z, 1, z, 0, 0, 0, 1, 64, 16)
    K.kvp_write(z, z, 1, z, z, z, 1, z, 0, 1, 0, 1, 64, 16)
    K.attention_kvp(z, z, z, z, 1, z, 1, z, 0, 0, 0, 1, 1, 64, 16, 1.0)
    K.attention_kvp(z, z, z, z, 1, z, 1, z, 4, 0, 4, 1, 1, 64, 16, 1.0, row_start=z)
    K.kvp_compact(z, At(z, 100), z, z, 0, 1, z, 1, 1, 1, 16, 16)
    assert (z.numpy() == 0).all()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

class Step:
    """One step of n-best decoding over a toy model: fork, per layer write and attention, the head, log probabilities.  The
    model: a token's rows of q, k, v per layer, and a head over the sum of the layers' attention."""
    PAGE, HEADS, G, DIM, LAYERS, VOCAB, PAGES, WIDTH = 16, 2, 2, 64, 2, 300, 120, 48

    def __init__(self, dev, r, n, group):
        self.dev, self.n, self.group = dev, n, group
        hd, hq = self.HEADS * self.DIM, self.HEADS * self.G * self.DIM
        self.rows = {x: r.normal(0, 1 if x != "v" else 0.6, (self.LAYERS, self.VOCAB, hq if x == "q" else hd)).astype(np.float32) for x in "qkv"}
        self.head = bf16(r.normal(0, 0.5, (self.VOCAB, hq)))
        self.head_dev = dev.upload(self.head)
        self.pools = dev.upload(np.full((2 * self.LAYERS, self.PAGES, self.HEADS, self.PAGE, self.DIM), NAN16, np.uint16))
        self.one = self.PAGES * self.HEADS * self.PAGE * self.DIM
        z = lambda *s: ints(dev, np.zeros(s))  # noqa: E731
        self.tables = [(z(n, self.WIDTH), z(n)), (z(n, self.WIDTH), z(n))]
        self.pos, self.status, self.parent = z(n), z(2), z(n)
        self.shared = z(n // group)
        self.q = [dev.zeros((n, hq), np.float32) for _ in range(self.LAYERS)]
        self.k = [dev.zeros((n, hd), np.float32) for _ in range(self.LAYERS)]
        self.v = [dev.zeros((n, hd), np.float32) for _ in range(self.LAYERS)]
        self.o, self.sum, self.logits = dev.zeros((n, hq), np.float32), dev.zeros((n, hq), np.float32), dev.zeros((n, self.VOCAB), np.float32)
        self.targets, self.lp, self.ent = z(n), dev.zeros(n, np.float32), dev.zeros(n, np.float32)
        self.ids, self.top = z(n, 6), dev.zeros((n, 6), np.float32)

    def feed(self, tokens, parent, shared, targets):
        self.parent.copy_from(np.asarray(parent, np.int32))
        self.shared.copy_from(np.asarray(shared, np.int32))
        self.targets.copy_from(np.asarray(targets, np.int32))
        for layer in range(self.LAYERS):
            for x, d in (("q", self.q), ("k", self.k), ("v", self.v)):
                d[layer].copy_from(self.rows[x][layer][tokens])

    def launch(self, turn):
        from qwenasr_amd import kernels as K
        (t0, l0), (t1, l1) = self.tables[turn], self.tables[1 - turn]
        n, page = self.n, self.PAGE
        K.kvp_fork(t1, self.pos, l1, self.status, t0, l0, n, n, self.WIDTH, self.pools, 2 * self.LAYERS, self.PAGES, self.HEADS, page, 2 * self.DIM,
                   parent=self.parent, max_rows=1)
        for layer in range(self.LAYERS):
            kp, vp = At(self.pools, 2 * layer * self.one), At(self.pools, (2 * layer + 1) * self.one)
            K.kvp_write(kp, vp, self.PAGES, self.k[layer], self.v[layer], t1, self.WIDTH, self.pos, n, n, 1, self.HEADS, self.DIM, page)
            o = self.sum if layer == 0 else self.o
            K.attention_kvp(o, self.q[layer], kp, vp, self.PAGES, t1, self.WIDTH, self.pos, n, n, 1, self.HEADS * self.G, self.HEADS, self.DIM, page,
                            self.DIM ** -0.5, group=self.group, shared=self.shared)
        K.linear(self.logits, self.sum, self.head_dev, None, n, self.HEADS * self.G * self.DIM, self.VOCAB)
        K.linear(self.logits, self.o, self.head_dev, None, n, self.HEADS * self.G * self.DIM, self.VOCAB, accumulate=True)
        K.token_logprobs(self.logits, n, self.VOCAB, targets=self.targets, logp=self.lp, entropy=self.ent, top_ids=self.ids, top_logp=self.top, k=6)

    def results(self):
        return [d.numpy() for d in (self.lp, self.ent, self.ids, self.top, self.pos, self.status)]

    def expected(self, history):
        """Log probabilities after a hypothesis' tokens, in 64 bits."""
        out = np.zeros(self.VOCAB)
        for layer in range(self.LAYERS):
            k = bf16f(bf16(self.rows["k"][layer][history])).astype(np.float64).reshape(-1, self.HEADS, self.DIM)
            v = bf16f(bf16(self.rows["v"][layer][history])).astype(np.float64).reshape(-1, self.HEADS, self.DIM)
            q = self.rows["q"][layer][history[-1:]].astype(np.float64).reshape(1, -1, self.DIM)
            o, _ = refp.attend(q, k, v, np.ones((1, len(history)), bool), self.DIM ** -0.5, U)
            out += bf16f(self.head).astype(np.float64) @ o.reshape(-1)
        out -= out.max()
        return out - np.log(np.exp(out).sum())


def choose(top_lp, ids, n, group, step):
    """Parents and tokens of the next step: of every group some members twice, some not at all."""
    parent, tokens = [], []
    for j in range(n):
        f, i = j // group * group, j % group
        p = f + (i * 2 + step) % max(1, group - 1 - step % 2)
        parent.append(p)
        tokens.append(int(ids[p][(i + step) % 6]))
    return parent, tokens


def test_decoding_steps(dev):
    """Twenty-five steps of two prompts with four hypotheses each, forked at every step, against 64-bit histories."""
    s = Step(dev, rng(40), 8, 4)
    history = [[1 + j // 4] for j in range(8)]
    parent, tokens, shared = [-1] * 8, [h[0] for h in history], [0, 0]
    for step in range(25):
        targets = [(7 * step + j) % s.VOCAB for j in range(8)]
        s.feed(tokens, parent, shared, targets)
        s.launch(step % 2)
        lp, ent, ids, top, pos, status = s.results()
        assert status[0] == 0 and (pos == step).all()
        want = np.stack([s.expected(h) for h in history])
        # logits of size 30 summed over 256 products in f32: 2e-4 bounds 256 x 30 x U = 4.6e-4 / 2; attention 1e-4
        assert np.abs(lp - want[np.arange(8), targets]).max() < 1e-3
        assert np.abs(top - np.sort(want)[:, ::-1][:, :6]).max() < 1e-3
        assert np.abs(ent + (np.exp(want) * want).sum(1)).max() < 1e-2
        parent, tokens = choose(top, ids, 8, 4, step)
        history = [history[p] + [t] for p, t in zip(parent, tokens)]
        # what the members of a group have in common from the start
        shared = []
        for g in range(2):
            hs = history[4 * g:4 * g + 4]
            shared.append(next((i for i in range(len(hs[0])) if len({tuple(h[:i + 1]) for h in hs}) > 1), len(hs[0])) if step % 3 else 0)


def captured(dev, launch):
    from qwenasr_amd._lib import lib
    hip = C.CDLL("libamdhip64.so.7")     # the HIP runtime the library already loaded
    stream = C.c_void_p(lib().qasr_hip_stream(dev.h))
    graph, exe = C.c_void_p(), C.c_void_p()
    dev.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        launch()
    finally:
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    return hip, stream, graph, exe


def test_captured(dev):
    """Steps captured into two graphs (one for each turn of the tables) and replayed with other inputs, eager work on the
    same handle and synchronisations in between: the bits of the eager steps."""
    eager, s = Step(dev, rng(41), 12, 4), Step(dev, rng(41), 12, 4)
    parent, tokens, shared = [-1] * 12, [1] * 4 + [2] * 4 + [3] * 4, [0, 0, 0]
    graphs = []
    try:
        for turn in range(2):
            graphs.append(captured(dev, lambda: s.launch(turn)))
        for step in range(9):
            for x in (eager, s):
                x.feed(tokens, parent, shared, [(step + j) % 300 for j in range(12)])
            eager.launch(step % 2)
            want = eager.results()
            hip, stream, _, exe = graphs[step % 2]
            assert hip.hipGraphLaunch(exe, stream) == 0
            eager.launch(step % 2)                               # the handle's scratch is used again behind the graph
            got = s.results()
            assert all((a == b).all() for a, b in zip(got, want)), step
            assert (s.tables[1 - step % 2][0].numpy() == eager.tables[1 - step % 2][0].numpy()).all()
            parent, tokens = choose(got[3], got[2], 12, 4, step)
            shared = [1, 0, 1] if step % 2 else [0, 0, 0]       # every member of a group begins with the same token
    finally:
        for hip, _, graph, exe in graphs:
            hip.hipGraphExecDestroy(exe)
            hip.hipGraphDestroy(graph)


def test_two_handles(dev):
    """Steps in turn on two handles, nothing waited for in between: each has its own scratch area."""
    from qwenasr_amd import Device
    other = Device(0)
    try:
        a, b, alone = Step(dev, rng(42), 8, 4), Step(other, rng(42), 8, 4), Step(dev, rng(42), 8, 4)
        parent, tokens = [-1] * 8, list(range(8))
        for step in range(5):
            for x in (a, b, alone):
                x.feed(tokens, parent, [0, 0], tokens)
                x.dev.sync()
            alone.launch(step % 2)
            want = alone.results()
            a.launch(step % 2)
            b.launch(step % 2)
            for got in (a.results(), b.results()):
                assert all((x == y).all() for x, y in zip(got, want)), step
            parent, tokens = choose(want[3], want[2], 8, 4, step)
        del b
    finally:
        other.close()
