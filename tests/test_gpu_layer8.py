"""The 8-bit layer operators over many rows and sequences against float64: int8
activation rows, the int8 x int8 product, the int8 KV cache and its attention."""
import ctypes as C

import numpy as np
import pytest

import ref8
from conftest import bf16, bf16f, rng

pytestmark = pytest.mark.gpu

F32, BF16 = 2.0 ** -24, 2.0 ** -8           # half a step, relative


def up(dev, a, is_bf16):
    return dev.upload(bf16(a) if is_bf16 else np.asarray(a, np.float32))


def held(a, is_bf16):
    """What the type keeps of a."""
    return (bf16f(bf16(a)) if is_bf16 else np.asarray(a, np.float32)).astype(np.float64)


def values(d, is_bf16):
    a = d.numpy()
    return (bf16f(a) if is_bf16 else a).astype(np.float64)


# ---------------------------------------------------------------------------
# int8 rows
# ---------------------------------------------------------------------------

# rows, hidden, padding of the row stride, residual, norm
ROWS = [(1, 1024, 0, True, True), (3, 1, 0, True, True), (5, 7, 2, True, True), (2, 63, 0, False, True), (33, 1000, 24, True, True),
        (4, 2048, 8, False, False), (1, 2049, 0, True, True), (2, 4096, 0, True, True), (3, 8192, 0, True, True), (2, 8200, 1, True, False),
        (2, 16384, 0, True, True), (301, 1024, 0, True, True), (700, 136, 0, True, True),
        (4100, 2048, 0, True, True), (4193, 2001, 0, False, True), (513, 16384, 8, True, False)]        # and from 2^23 values on


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows,hidden,pad,res,norm", ROWS)
def test_rows(dev, rows, hidden, pad, res, norm, is_bf16):
    from qwenasr_amd import kernels as K
    print(f"rows8 {rows} x {hidden} + {pad} res={res} norm={norm} bf16={is_bf16}", flush=True)
    r = rng(rows * 31 + hidden + 7 * is_bf16)
    ld = hidden + pad
    x, d, w = r.normal(0, 1, (rows, ld)), r.normal(0, 0.3, (rows, ld)), (1 + r.normal(0, 0.1, hidden)).astype(np.float32)
    x[0, :] *= 1e-3
    if rows > 2:
        x[2, :hidden] = 0.0
        d[2, :hidden] = 0.0
    dx, dd = up(dev, x, is_bf16), up(dev, d, is_bf16)
    q, s = dev.zeros((rows + 1, hidden), np.int8), dev.zeros(rows + 1, np.float32)
    out = up(dev, np.full((rows, ld), 5.0), is_bf16)
    K.add_rms_norm_int8(q, s, dx, dev.upload(w) if norm else None, rows, hidden, res=dd if res else None, sum_out=out, ld=ld,
                        eps=1e-6, bf16=is_bf16)
    hx, hd = held(x, is_bf16)[:, :hidden], held(d, is_bf16)[:, :hidden]
    want_s, want_q, want_sc = ref8.norm8(hx, hd if res else None, w.astype(np.float64), 1e-6, norm)
    got_q, got_s, got = q.numpy(), s.numpy().astype(np.float64), values(out, is_bf16)
    assert (got_q[:rows] == want_q).all() and (got_q[rows] == 0).all() and got_s[rows] == 0
    # one rounding of a 64-bit value, whose own sums are off by far less
    assert (np.abs(got_s[:rows] - want_sc) <= 1.001 * F32 * want_sc).all()
    assert (np.abs(got[:, :hidden] - want_s) <= (BF16 if is_bf16 else F32) * np.abs(want_s)).all()
    assert (got[:, hidden:] == 5.0).all()                    # nothing behind a row


@pytest.mark.parametrize("is_bf16", [False, True])
def test_rows_in_place(dev, is_bf16):
    """sum may be x or res: the same results and the sum in its place."""
    from qwenasr_amd import kernels as K
    r = rng(5)
    x, d, w = r.normal(0, 1, (9, 1032)), r.normal(0, 1, (9, 1032)), r.uniform(0.5, 1.5, 1032)
    dw = dev.upload(w.astype(np.float32))
    want = None
    for where in ("apart", "x", "res"):
        dx, dd, o = up(dev, x, is_bf16), up(dev, d, is_bf16), up(dev, 0 * x, is_bf16)
        to = {"apart": o, "x": dx, "res": dd}[where]
        q, s = dev.zeros((9, 1032), np.int8), dev.zeros(9, np.float32)
        K.add_rms_norm_int8(q, s, dx, dw, 9, 1032, res=dd, sum_out=to, bf16=is_bf16)
        got = (q.numpy(), s.numpy(), to.numpy())
        want = want or got
        assert all((a == b).all() for a, b in zip(got, want)), where


def test_rows_not_finite(dev):
    """A row with a value that is not finite: q 0, scale NaN; its neighbours as alone."""
    from qwenasr_amd import kernels as K
    x = rng(6).normal(0, 1, (6, 520)).astype(np.float32)
    clean = x.copy()
    x[1, 3], x[2, 519], x[4, 0] = np.nan, np.inf, -np.inf
    w = np.ones(520, np.float32)
    q, s = dev.zeros((6, 520), np.int8), dev.zeros(6, np.float32)
    K.add_rms_norm_int8(q, s, dev.upload(x), dev.upload(w), 6, 520)
    _, want_q, _ = ref8.norm8(clean.astype(np.float64), None, w.astype(np.float64), 1e-6)
    for i in range(6):
        if i in (1, 2, 4):
            assert (q.numpy()[i] == 0).all() and np.isnan(s.numpy()[i])
        else:
            assert (q.numpy()[i] == want_q[i]).all() and np.isfinite(s.numpy()[i])


def test_rows_halves(dev):
    """Values halfway between two int8 values go away from zero, exactly: k + 1/2 steps of a row whose largest value is 127 steps."""
    from qwenasr_amd import kernels as K
    step = np.array([1.0, 0.75, 3.0, 1.625, 2.0 ** -20], np.float64)
    k = np.arange(0, 127) + 0.5
    x = np.concatenate([k, -k, [127.0, -127.0]])[None] * step[:, None]
    q, s = dev.zeros(x.shape, np.int8), dev.zeros(len(step), np.float32)
    K.add_rms_norm_int8(q, s, dev.upload(x.astype(np.float32)), None, *x.shape)
    want = np.concatenate([np.arange(1, 128), -np.arange(1, 128), [127, -127]])
    assert (q.numpy() == want).all() and (s.numpy() == step).all()


# ---------------------------------------------------------------------------
# int8 x int8 products
# ---------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 5, 64), (3, 70, 17), (16, 64, 64), (17, 130, 100), (32, 2048, 1024), (33, 1000, 1040), (64, 256, 2048),
          (65, 66, 63), (130, 514, 192), (257, 4100, 320), (404, 1024, 1024), (100, 1003, 999), (300, 2050, 6144), (1000, 771, 128),
          (2, 3000, 16400), (5, 33, 131071), (31, 20000, 256), (48, 12290, 512)]


def check_gemm(got, acc, as_, ws, bias, y0, mode, is_bf16):
    """f32: the sum's conversion and two products; bias and y0 one rounding of the total each; bf16 one more."""
    sa, sw = as_.astype(np.float64)[:, None], ws.astype(np.float64)
    p = acc * sa * sw
    err = 3.01 * F32 * np.abs(p)
    y = p
    if bias is not None:
        y = y + bias
        err = err + 1.01 * F32 * (np.abs(y) + err)
    if mode == "add":
        b0 = y0 + (0.0 if bias is None else bias)
        y = y + y0
        err = 3.01 * F32 * np.abs(p) + 1.01 * F32 * np.abs(b0) + 1.01 * F32 * np.abs(y)
    if mode == "swiglu":
        g, u, eg, eu = y[:, 0::2], y[:, 1::2], err[:, 0::2], err[:, 1::2]
        with np.errstate(over="ignore"):
            sig = 1 / (1 + np.exp(-g))
        y = g * sig * u
        # d silu <= 1.1 |dg|; the exponential's 2 units (of e^-g / (1 + e^-g) <= 1), the sum, the quotient, the product
        err = 1.1 * eg * np.abs(u) + np.abs(g * sig) * eu + 1.01 * (4 + 3) * F32 * np.abs(y) + np.abs(y) * np.abs(g) * F32 + 1e-37
    if is_bf16:
        err = err + BF16 * (np.abs(y) + err)
    assert got.shape == y.shape
    over = np.abs(got - y) > err
    assert not over.any(), (np.argwhere(over)[:5], np.abs(got - y).max())


@pytest.mark.parametrize("mode,with_bias,is_bf16", [("plain", False, False), ("plain", True, True), ("add", True, False), ("add", False, True),
                                                    ("swiglu", False, False), ("swiglu", True, True)])
@pytest.mark.parametrize("M,N,Kd", SHAPES)
def test_gemm(dev, M, N, Kd, mode, with_bias, is_bf16):
    from qwenasr_amd import kernels as K
    print(f"w8a8 {M} x {N} x {Kd} {mode} bias={with_bias} bf16={is_bf16}", flush=True)
    if mode == "swiglu":
        N += N % 2
    r = rng(M * 1009 + N * 31 + Kd)
    a, w = r.integers(-127, 128, (M, Kd), dtype=np.int8), r.integers(-127, 128, (N, Kd), dtype=np.int8)
    sa, sw = r.uniform(0.01, 0.03, M).astype(np.float32), (r.uniform(0.01, 0.02, N) / np.sqrt(Kd) / 60).astype(np.float32)
    bias = r.normal(0, 0.5, N).astype(np.float32) if with_bias else None
    cols = N // 2 if mode == "swiglu" else N
    y0 = r.normal(0, 1, (M + 1, cols))
    y = up(dev, y0, is_bf16)
    K.gemm_w8a8(y, dev.upload(a), dev.upload(sa), dev.upload(w), dev.upload(sw), M, N, Kd, bias=dev.upload(bias) if with_bias else None,
                accumulate=mode == "add", swiglu=mode == "swiglu", bf16=is_bf16)
    got, was = values(y, is_bf16), held(y0, is_bf16)
    acc, _ = ref8.gemm8(a, sa, w, sw)
    check_gemm(got[:M], acc, sa, sw, None if bias is None else bias.astype(np.float64), was[:M], mode, is_bf16)
    assert (got[M] == was[M]).all()                           # nothing past the last row


# what the larger tiles, and long K-steps in eight groups, are chosen for: edges inside a tile, rows of y of every alignment, K-steps that end inside 128
LARGE = [(1500, 4102, 336), (900, 5004, 2000), (1337, 6001, 80), (641, 12290, 464), (1153, 4100, 1104), (1700, 4999, 1040),
         (2100, 8192, 272), (2100, 4032, 1040), (2000, 6144, 1024), (40, 1003, 6000), (17, 515, 2000),
         (2000, 2501, 1023), (40, 1003, 6001), (33, 6001, 1030), (130, 4099, 519), (400, 20004, 4016)]                            # the last: weights past the caches


@pytest.mark.parametrize("mode,with_bias,is_bf16", [("plain", True, False), ("add", True, True), ("swiglu", True, True)])
@pytest.mark.parametrize("M,N,Kd", LARGE)
def test_gemm_large(dev, M, N, Kd, mode, with_bias, is_bf16):
    test_gemm(dev, M, N, Kd, mode, with_bias, is_bf16)


@pytest.mark.parametrize("off_a,off_w", [(1, 0), (0, 1), (4, 8), (15, 15)])
def test_gemm_alignment(dev, off_a, off_w):
    """Buffers that start at any byte."""
    from qwenasr_amd._lib import check, lib
    M, N, Kd = 70, 200, 256
    r = rng(off_a * 16 + off_w)
    a, w = r.integers(-127, 128, (M, Kd), dtype=np.int8), r.integers(-127, 128, (N, Kd), dtype=np.int8)
    sa, sw = r.uniform(0.5, 1, M).astype(np.float32), r.uniform(0.5, 1, N).astype(np.float32)
    da = dev.upload(np.concatenate([np.zeros(off_a, np.int8), a.reshape(-1)]))
    dw = dev.upload(np.concatenate([np.zeros(off_w, np.int8), w.reshape(-1)]))
    dsa, dsw, y = dev.upload(sa), dev.upload(sw), dev.zeros((M, N), np.float32)
    check(lib().qasr_hip_gemm_w8a8(dev.h, y.ptr, da.offset(off_a), dsa.ptr, dw.offset(off_w), dsw.ptr, None, M, N, Kd, 0, 0))
    check_gemm(y.numpy().astype(np.float64), ref8.gemm8(a, sa, w, sw)[0], sa, sw, None, None, "plain", False)


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("mode", ["plain", "add", "swiglu"])
@pytest.mark.parametrize("M,N,Kd", [(70, 200, 256), (300, 2050, 1040), (1500, 4100, 336), (40, 301, 16), (9, 333, 77)])
def test_gemm_result_anywhere(dev, M, N, Kd, mode, is_bf16):
    """y, bias and scales that start one element off: rows of y at any alignment, nothing written around them."""
    from qwenasr_amd._lib import check, lib
    print(f"w8a8 {M} x {N} x {Kd} {mode} bf16={is_bf16}, one element off", flush=True)
    N += N % 2 if mode == "swiglu" else 0
    r = rng(M + N + Kd + is_bf16)
    a, w = r.integers(-127, 128, (M, Kd), dtype=np.int8), r.integers(-127, 128, (N, Kd), dtype=np.int8)
    sa, sw = r.uniform(0.01, 0.03, M).astype(np.float32), (r.uniform(0.01, 0.02, N) / np.sqrt(Kd) / 60).astype(np.float32)
    bias, cols = r.normal(0, 0.5, N).astype(np.float32), N // 2 if mode == "swiglu" else N
    y0 = np.concatenate([[7.0], r.normal(0, 1, M * cols), [7.0]])
    y, dsa, dsw, db = up(dev, y0, is_bf16), *(dev.upload(np.concatenate([[0.0], v]).astype(np.float32)) for v in (sa, sw, bias))
    da, dw = dev.upload(a), dev.upload(w)
    check(lib().qasr_hip_gemm_w8a8(dev.h, y.offset(1), da.ptr, dsa.offset(1), dw.ptr, dsw.offset(1), db.offset(1), M, N, Kd,
                                   ["plain", "add", "swiglu"].index(mode), 1 if is_bf16 else 0))
    got = values(y, is_bf16)
    assert got[0] == 7.0 and got[-1] == 7.0
    check_gemm(got[1:-1].reshape(M, cols), ref8.gemm8(a, sa, w, sw)[0], sa, sw, bias.astype(np.float64),
               held(y0, is_bf16)[1:-1].reshape(M, cols), mode, is_bf16)


def test_gemm_largest_sums(dev):
    """Every product -128 x -128 at the longest K: the sum is the largest that 32 bits hold."""
    from qwenasr_amd import kernels as K
    Kd = 131071
    a, w = np.full((2, Kd), -128, np.int8), np.full((3, Kd), -128, np.int8)
    one = np.ones(3, np.float32)
    y = dev.zeros((2, 3), np.float32)
    K.gemm_w8a8(y, dev.upload(a), dev.upload(one), dev.upload(w), dev.upload(one), 2, 3, Kd)
    assert (y.numpy() == np.float32(16384 * Kd)).all()


def test_gemm_row_alone(dev):
    """A row's bits do not depend on how many rows share the call, and are those of the int8 matvec on its values."""
    from qwenasr_amd import kernels as K
    M, N, Kd = 77, 1024, 1024
    r = rng(8)
    x = r.normal(0, 1, (M, Kd)).astype(np.float32)
    w, sw = r.integers(-127, 128, (N, Kd), dtype=np.int8), r.uniform(1e-4, 2e-3, N).astype(np.float32)
    dw, dsw = dev.upload(w), dev.upload(sw)
    q, s = dev.zeros((M, Kd), np.int8), dev.zeros(M, np.float32)
    K.add_rms_norm_int8(q, s, dev.upload(x), None, M, Kd)
    y = dev.zeros((M, N), np.float32)
    K.gemm_w8a8(y, q, s, dw, dsw, M, N, Kd)
    for i in (0, 41, 76):
        q1, s1, y1 = dev.upload(q.numpy()[i]), dev.upload(s.numpy()[i:i + 1]), dev.zeros(N, np.float32)
        K.gemm_w8a8(y1, q1, s1, dw, dsw, 1, N, Kd)
        assert (y1.numpy() == y.numpy()[i]).all()
        xq, xs = dev.zeros(Kd, np.int8), dev.zeros(1, np.float32)
        dx = dev.upload(x[i])
        K.quantize_f32_to_int8(dx, xq, xs)
        if (xq.numpy() == q.numpy()[i]).all():               # the two quantizers differ next to halves
            ym = dev.zeros(N, np.float32)
            K.linear_int8(ym, dx, dw, dsw, None, Kd, N)
            assert xs.numpy()[0] == s.numpy()[i] and (ym.numpy() == y.numpy()[i]).all()


# ---------------------------------------------------------------------------
# the int8 KV cache
# ---------------------------------------------------------------------------

class DevCache:
    def __init__(self, dev, ref):
        self.dev, self.ref = dev, ref
        self.n_seq, self.heads, self.cap, self.dim = ref.shape
        self.buf = [dev.upload(np.ascontiguousarray(a)) for a in ref.stored()]

    def geometry(self):
        return self.heads, self.dim, self.cap

    def check(self):
        """The device's bytes are the reference's."""
        for name, d, want in zip(("k8", "v8", "k_scales", "v_scales"), self.buf, self.ref.stored()):
            got = d.numpy()
            assert (got == want).all(), (name, np.argwhere(got != want)[:4])


def prefix(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


# counts of rows per sequence, first positions, heads, dim, capacity
WRITES = [([1], [0], 1, 64, 64), ([1, 1, 1], [63, 64, 10], 8, 128, 128), ([64, 0, 3], [0, 5, 62], 2, 128, 192),
          ([130, 65, 1, 63], [1, 63, 191, 65], 3, 64, 256), ([200, 7], [0, 250], 8, 128, 256), ([5, 5, 5], [-3, -9, 254], 2, 128, 256),
          ([300], [17], 14, 64, 320), ([2, 2], [600, -(1 << 31)], 1, 128, 256)]


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("counts,pos,heads,dim,cap", WRITES)
def test_kv8_write_read(dev, counts, pos, heads, dim, cap, is_bf16):
    """Into caches that hold something already, out of wide rows (an offset and a stride); then back."""
    from qwenasr_amd import kernels as K
    print(f"kv8 {counts} at {pos} heads={heads} dim={dim} cap={cap} bf16={is_bf16}", flush=True)
    r = rng(sum(counts) * 7 + heads + dim + is_bf16)
    n, hd = len(counts), heads * dim
    start = prefix(counts)
    total = int(start[-1]) + 3                               # rows behind the last sequence
    ref = ref8.Cache(n, heads, cap, dim).fill(r)
    d = DevCache(dev, ref)
    ld = 3 * hd + 8
    rows = r.normal(0, 1, (total, ld)) * r.uniform(0.2, 4, (total, 1))
    if sum(counts) > 1:
        rows[1, hd:2 * hd] = 0.0
    dr = up(dev, rows, is_bf16)
    es = 2 if is_bf16 else 4

    class At:                                                # k and v inside the fused projection's rows
        def __init__(self, e):
            self.ptr, self.dev = C.c_void_p(dr.ptr.value + e * es), dev
    dpos, dstart = dev.upload(np.array(pos, np.int32)), dev.upload(start)
    K.kv8_write(*d.buf, At(hd), At(2 * hd), dpos, total, n, max(counts), *d.geometry(), row_start=dstart, ld=ld, bf16=is_bf16)
    h = held(rows, is_bf16)
    for j in range(n):
        x = h[start[j]:start[j + 1]]
        ref.write(j, pos[j], {"k": x[:, hd:2 * hd].reshape(-1, heads, dim), "v": x[:, 2 * hd:3 * hd].reshape(-1, heads, dim)})
    d.check()
    # back: f32 values are the products, bf16 ones rounded once
    back = np.full((total, ld), 9.0)
    for as_bf16 in (False, True):
        o = up(dev, back, as_bf16)
        es = 2 if as_bf16 else 4

        class To:
            def __init__(self, e):
                self.ptr, self.dev = C.c_void_p(o.ptr.value + e * es), dev
        K.kv8_read(To(0), To(hd), *d.buf, dpos, total, n, max(counts), *d.geometry(), row_start=dstart, ld=ld, bf16=as_bf16)
        got = values(o, as_bf16)
        want = back.copy()
        for j in range(n):
            for i in range(counts[j]):
                if 0 <= pos[j] + i < cap:
                    want[start[j] + i, :hd] = ref.values("k")[j, :, pos[j] + i].reshape(-1)
                    want[start[j] + i, hd:2 * hd] = ref.values("v")[j, :, pos[j] + i].reshape(-1)
        assert (np.abs(got - want) <= (BF16 if as_bf16 else F32) * np.abs(want) * (want != 9.0)).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_kv8_grow(dev, dim):
    """Position by position, as decoding writes: the scale rises and what the block holds is rounded again."""
    from qwenasr_amd import kernels as K
    r = rng(dim)
    heads, cap, n = 2, 128, 3
    ref = ref8.Cache(n, heads, cap, dim)
    d = DevCache(dev, ref)
    at = [0, 30, 62]
    for step in range(40):
        rows = r.normal(0, 1, (n, heads * dim)) * (1 + step / 10)
        dr, dp = up(dev, rows, False), dev.upload(np.array(at, np.int32))
        K.kv8_write(*d.buf, dr, dr, dp, n, n, 1, *d.geometry())
        x = held(rows, False).reshape(n, 1, heads, dim)
        for j in range(n):
            ref.write(j, at[j], {"k": x[j], "v": x[j]})
            at[j] += 1
    d.check()


def test_kv8_not_finite(dev):
    """NaN is stored as 0, infinities as +-127; neither moves the scale.  A block of zeros has scale 0."""
    from qwenasr_amd import kernels as K
    heads, dim, cap, n = 2, 64, 128, 70
    rows = rng(3).normal(0, 1, (n, heads * dim)).astype(np.float32)
    rows[0, 0], rows[1, 5], rows[2, 100], rows[63, 64:] = np.nan, np.inf, -np.inf, np.nan
    zero = np.zeros_like(rows)
    zero[3, 7] = np.inf
    ref = ref8.Cache(1, heads, cap, dim)
    d = DevCache(dev, ref)
    dk, dv = dev.upload(rows), dev.upload(zero)
    K.kv8_write(*d.buf, dk, dv, dev.zeros(1, np.int32), n, 1, n, *d.geometry())
    ref.write(0, 0, {"k": rows.astype(np.float64).reshape(n, heads, dim), "v": zero.astype(np.float64).reshape(n, heads, dim)})
    d.check()
    assert (d.buf[3].numpy()[0, 0, 0] == 0) and (d.buf[1].numpy() == 0).all()


# ---------------------------------------------------------------------------
# attention over it
# ---------------------------------------------------------------------------

def attention(dev, d, q, counts, pos, group, window=0, sinks=0, is_bf16=False, pad=0, max_len=0, behind=2):
    """(got, start) of a call on ragged rows; checks that rows behind the last sequence stay."""
    from qwenasr_amd import kernels as K
    start = prefix(counts)
    total, hq = int(start[-1]) + behind, d.heads * group
    wide = np.zeros((total, hq * d.dim + pad))
    wide[:len(q), :hq * d.dim] = q.reshape(len(q), -1)
    out = up(dev, np.full((total, hq * d.dim), 3.0), is_bf16)
    K.attention_kv8(out, up(dev, wide, is_bf16), *d.buf, dev.upload(np.array(pos, np.int32)), total, d.n_seq, max(max(counts), 1),
                    hq, d.heads, d.dim, d.cap, d.dim ** -0.5, row_start=dev.upload(start), ldq=hq * d.dim + pad, max_len=max_len,
                    window=window, sinks=sinks, bf16=is_bf16)
    got = values(out, is_bf16)
    assert (got[start[-1]:] == 3.0).all()
    return got[:start[-1]].reshape(-1, hq, d.dim)


def check_attention(got, ref, q, counts, pos, window=0, sinks=0, is_bf16=False):
    start, dim = prefix(counts), ref.shape[3]
    k, v = ref.values("k"), ref.values("v")
    for j, n in enumerate(counts):
        rows = slice(start[j], start[j] + n)
        want, err = ref8.attend(q[rows], k[j], v[j], pos[j], dim ** -0.5, window, sinks, 32000.0 if is_bf16 else 8.0e6)
        err = err + (BF16 if is_bf16 else F32) * (np.abs(want) + err)
        over = np.abs(got[rows] - want) > err
        assert not over.any(), (j, np.argwhere(over)[:4], np.abs(got[rows] - want).max(), err.max())


# counts, positions of the first rows, heads, group, dim, capacity, window, sinks
ATTN = [([1], [0], 1, 1, 64, 64, 0, 0), ([1], [403], 8, 2, 128, 512, 0, 0), ([1, 1, 1, 1], [0, 63, 64, 700], 8, 2, 128, 768, 0, 0),
        ([0, 3, 1], [5, -1, -4], 2, 3, 128, 128, 0, 0), ([17, 1, 40], [0, 100, 63], 2, 2, 128, 192, 0, 0), ([70], [0], 3, 4, 64, 128, 0, 0),
        ([5, 9], [60, 126], 1, 7, 64, 128, 0, 0), ([133], [0], 2, 1, 128, 192, 0, 0), ([1, 1], [3000, 1500], 2, 2, 128, 3200, 0, 0),
        ([1, 1], [900, 40], 8, 2, 128, 1024, 100, 4), ([30, 66], [700, 0], 2, 2, 64, 1024, 65, 70), ([33], [512], 2, 2, 128, 1024, 1, 0),
        ([1, 20], [1000, 900], 1, 16, 128, 1024, 64, 0), ([3], [2000], 2, 2, 128, 256, 100, 5), ([130], [0], 1, 2, 128, 256, 1000, 3),
        ([1], [5000], 4, 33, 64, 5120, 0, 0), ([260, 259, 100], [0, 1, 60], 16, 1, 64, 320, 0, 0), ([40], [3000], 2, 2, 128, 3136, 1500, 70),
        ([2, 1], [3000, 2999], 1, 4, 128, 3136, 2500, 100), ([9], [4000], 1, 2, 64, 4096, 0, 0)]


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("counts,pos,heads,group,dim,cap,window,sinks", ATTN)
def test_attention(dev, counts, pos, heads, group, dim, cap, window, sinks, is_bf16):
    print(f"attn8 {counts} at {pos} {heads} x {group} x {dim} cap={cap} window={window}+{sinks} bf16={is_bf16}", flush=True)
    r = rng(sum(counts) + cap + heads * 10 + is_bf16)
    ref = ref8.Cache(len(counts), heads, cap, dim).fill(r)
    d = DevCache(dev, ref)
    q = r.normal(0, 1, (sum(counts), heads * group, dim)) * r.uniform(0.1, 3, (sum(counts), heads * group, 1))
    got = attention(dev, d, q, counts, pos, group, window, sinks, is_bf16, pad=0 if sum(counts) % 2 else 8)
    check_attention(got, ref, held(q, is_bf16), counts, pos, window, sinks, is_bf16)


@pytest.mark.parametrize("max_len", [1, 64, 5000])
def test_attention_max_len_is_a_hint(dev, max_len):
    """Whatever max_len says, every position counts."""
    r = rng(12)
    ref = ref8.Cache(2, 2, 1024, 128).fill(r)
    d = DevCache(dev, ref)
    q = r.normal(0, 1, (3, 4, 128))
    got = attention(dev, d, q, [1, 2], [1000, 333], 2, max_len=max_len)
    check_attention(got, ref, held(q, False), [1, 2], [1000, 333])


def test_attention_sink_holds_the_maximum(dev):
    """One position far above a long context of equal ones: each weighs 2^-22 of it, together they count."""
    heads, dim, cap = 1, 128, 8192
    ref = ref8.Cache(1, heads, cap, dim)
    ref.q["k"][:], ref.q["v"][:] = 0, 100
    ref.q["k"][0, 0, 0, 0] = 127
    ref.q["v"][0, 0, 0, :] = -3
    ref.s["k"][:], ref.s["v"][:] = 1.0, 0.01
    q = np.zeros((1, 1, dim))
    q[0, 0, 0] = 22 * np.log(2) * dim ** 0.5 / 127
    d = DevCache(dev, ref)
    got = attention(dev, d, q, [1], [cap - 1], 1)
    check_attention(got, ref, held(q, False), [1], [cap - 1])


def test_attention_not_finite(dev):
    """A row of q that is not finite gives NaN where it sees something; a block's scale that is not finite reaches only rows that see the block."""
    r = rng(13)
    ref = ref8.Cache(1, 2, 256, 64).fill(r)
    clean = DevCache(dev, ref)
    q = r.normal(0, 1, (100, 4, 64))
    want = attention(dev, clean, q, [100], [20], 2)
    ref.s["k"][0, 0, 1], ref.s["v"][0, 1, 1] = np.nan, np.inf
    got = attention(dev, DevCache(dev, ref), q, [100], [20], 2)
    see = np.arange(100) + 20 >= 64
    assert (got[~see] == want[~see]).all()
    assert np.isnan(got[see][:, :2]).all() and not np.isfinite(got[see][:, 2:]).any()
    q[7, 1, 5], q[8, 3, 0] = np.nan, np.inf
    got = attention(dev, clean, q, [100], [20], 2)
    assert np.isnan(got[7, 1]).all() and np.isnan(got[8, 3]).all()
    keep = np.ones((100, 4), bool)
    keep[7, 1] = keep[8, 3] = False
    assert (got[keep] == want[keep]).all()


def test_rows_past_max_rows(dev):
    """A sequence's rows past max_rows are left out: of the cache, of what is read back and of the attention's output."""
    from qwenasr_amd import kernels as K
    r = rng(16)
    heads, dim, cap, counts, most = 2, 64, 128, [5, 2, 40], 3
    start, n, total = prefix(counts), len(counts), sum(counts)
    ref = ref8.Cache(n, heads, cap, dim).fill(r)
    d = DevCache(dev, ref)
    dpos, dstart = dev.upload(np.array([60, 0, 7], np.int32)), dev.upload(start)
    rows, q = r.normal(0, 1, (total, heads * dim)), r.normal(0, 1, (total, 4 * dim))
    dr, back = up(dev, rows, False), up(dev, np.full(rows.shape, 3.0), False)
    out = up(dev, np.full((total, 4 * dim), 3.0), False)
    K.kv8_write(*d.buf, dr, dr, dpos, total, n, most, *d.geometry(), row_start=dstart)
    K.kv8_read(back, dev.zeros(rows.shape, np.float32), *d.buf, dpos, total, n, most, *d.geometry(), row_start=dstart)
    K.attention_kv8(out, up(dev, q, False), *d.buf, dpos, total, n, most, 4, heads, dim, cap, dim ** -0.5, row_start=dstart)
    keep = [min(c, most) for c in counts]
    for j in range(n):
        x = held(rows, False)[start[j]:start[j] + keep[j]].reshape(-1, heads, dim)
        ref.write(j, [60, 0, 7][j], {"k": x, "v": x})
    d.check()
    taken = np.concatenate([np.arange(start[j], start[j] + keep[j]) for j in range(n)])
    left = np.setdiff1d(np.arange(total), taken)
    assert (back.numpy()[left] == 3.0).all() and (out.numpy()[left] == 3.0).all() and (back.numpy()[taken] != 3.0).all()
    check_attention(values(out, False)[taken].reshape(-1, 4, dim), ref, held(q, False)[taken].reshape(-1, 4, dim), keep, [60, 0, 7])


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
def test_long_cache(dev, rows, is_bf16):
    """Positions whose bytes lie past 2^31 in the cache: with a window, the bits of a short cache that holds the same
    positions; without, against the formula (positions never written have scale 0: their scores and values are 0)."""
    from qwenasr_amd import kernels as K
    r = rng(17 + rows)
    n, heads, group, dim, cap, short, pos = 3, 8, 2, 128, 1 << 20, 512, 400
    hq, base, total = heads * group, cap - short, n * rows
    k, v = r.normal(0, 1, (n * (pos + rows), heads * dim)), r.normal(0, 1, (n * (pos + rows), heads * dim))
    q = up(dev, r.normal(0, 1, (total, hq * dim)), is_bf16)
    dk, dv = up(dev, k, False), up(dev, v, False)
    out = {}
    for name, c, b in (("short", short, 0), ("long", cap, base)):
        buf = [dev.zeros((n, heads, c, dim), np.int8), dev.zeros((n, heads, c // 64, dim, 64), np.int8),
               dev.zeros((n, heads, c // 64), np.float32), dev.zeros((n, heads, c // 64), np.float32)]
        K.kv8_write(*buf, dk, dv, dev.upload(np.full(n, b, np.int32)), len(k), n, pos + rows, heads, dim, c)
        back = [dev.zeros((len(k), heads * dim), np.float32) for _ in range(2)]
        K.kv8_read(*back, *buf, dev.upload(np.full(n, b, np.int32)), len(k), n, pos + rows, heads, dim, c)
        o, dp = up(dev, np.zeros((total, hq * dim)), is_bf16), dev.upload(np.full(n, b + pos, np.int32))
        K.attention_kv8(o, q, *buf, dp, total, n, rows, hq, heads, dim, c, dim ** -0.5, window=200, bf16=is_bf16)
        out[name] = [o.numpy()] + [a.numpy() for a in back]
        if name == "long":
            K.attention_kv8(o, q, *buf, dp, total, n, rows, hq, heads, dim, c, dim ** -0.5, bf16=is_bf16)
            full = values(o, is_bf16).reshape(n, rows, hq, dim)
    assert all((a == b).all() for a, b in zip(out["short"], out["long"]))
    back_k, back_v = (a.astype(np.float64).reshape(n, pos + rows, heads, dim) for a in out["long"][1:])
    qh = values(q, is_bf16).reshape(n, rows, hq, dim)
    for j, i, h in ((2, 0, 15), (2, rows - 1, 14), (1, 1, 0)):
        kk, vv = np.zeros((1, cap, dim)), np.zeros((1, cap, dim))
        kk[0, base:base + pos + rows], vv[0, base:base + pos + rows] = back_k[j, :, h // group], back_v[j, :, h // group]
        want, err = ref8.attend(qh[j, i:i + 1, h:h + 1], kk, vv, base + pos + i, dim ** -0.5, 0, 0, 32000.0 if is_bf16 else 8.0e6)
        # back_k and back_v are the cache's values rounded once to f32
        err = err + (BF16 if is_bf16 else F32) * (np.abs(want) + err) + 2 * F32 * np.abs(vv).max()
        assert (np.abs(full[j, i, h] - want[0, 0]) <= err[0, 0]).all()


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("counts,dim,off,pad", [([1, 1], 128, 1, 1), ([2, 19], 128, 3, 5), ([40, 1], 64, 1, 7), ([2, 1], 64, 5, 2)])
def test_rows_anywhere(dev, counts, dim, off, pad, is_bf16):
    """Rows that start at any element and lie any number of elements apart: into the cache, back, and the attention's."""
    from qwenasr_amd import kernels as K
    r = rng(off * 8 + pad + dim + is_bf16)
    heads, group, cap, pos = 2, 2, 256, [70, 3]
    n, hd, hq, es = len(counts), heads * dim, heads * group * dim, 2 if is_bf16 else 4
    start, total, ld = prefix(counts), sum(counts), hd + pad
    ref = ref8.Cache(n, heads, cap, dim).fill(r)
    d = DevCache(dev, ref)
    dpos, dstart = dev.upload(np.array(pos, np.int32)), dev.upload(start)

    class Off:
        def __init__(self, b):
            self.b, self.ptr, self.dev = b, C.c_void_p(b.ptr.value + off * es), dev
    flat = [r.normal(0, 1, off + total * ld) for _ in range(2)]
    k, v = (Off(up(dev, f, is_bf16)) for f in flat)
    K.kv8_write(*d.buf, k, v, dpos, total, n, max(counts), *d.geometry(), row_start=dstart, ld=ld, bf16=is_bf16)
    kh, vh = (held(f, is_bf16)[off:].reshape(total, ld)[:, :hd].reshape(total, heads, dim) for f in flat)
    for j in range(n):
        rows = slice(start[j], start[j + 1])
        ref.write(j, pos[j], {"k": kh[rows], "v": vh[rows]})
    d.check()
    bk, bv = (Off(up(dev, np.full(off + total * ld, 9.0), is_bf16)) for _ in range(2))
    K.kv8_read(bk, bv, *d.buf, dpos, total, n, max(counts), *d.geometry(), row_start=dstart, ld=ld, bf16=is_bf16)
    for o, name in ((bk, "k"), (bv, "v")):
        got = values(o.b, is_bf16)
        assert (got[:off] == 9.0).all() and (got[off:].reshape(total, ld)[:, hd:] == 9.0).all()
        want = np.concatenate([ref.values(name)[j, :, pos[j]:pos[j] + counts[j]].transpose(1, 0, 2) for j in range(n)])
        got = got[off:].reshape(total, ld)[:, :hd].reshape(want.shape)
        assert (np.abs(got - want) <= (BF16 if is_bf16 else F32) * np.abs(want)).all()
    ldq = hq + pad
    qf = r.normal(0, 1, off + total * ldq)
    o = Off(up(dev, np.full(off + total * hq + 1, 9.0), is_bf16))
    K.attention_kv8(o, Off(up(dev, qf, is_bf16)), *d.buf, dpos, total, n, max(counts), heads * group, heads, dim, cap, dim ** -0.5,
                    row_start=dstart, ldq=ldq, bf16=is_bf16)
    got = values(o.b, is_bf16)
    assert (got[:off] == 9.0).all() and got[-1] == 9.0
    q = held(qf, is_bf16)[off:].reshape(total, ldq)[:, :hq].reshape(total, heads * group, dim)
    check_attention(got[off:-1].reshape(q.shape), ref, q, counts, pos, is_bf16=is_bf16)


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0])
def test_attention_scale(dev, scale, rows, is_bf16):
    """Any scale; rows of zeros, and rows of very small and large values."""
    from qwenasr_amd import kernels as K
    r = rng(rows + is_bf16)
    heads, dim, cap, pos = 2, 128, 256, 120
    ref = ref8.Cache(1, heads, cap, dim).fill(r)
    d = DevCache(dev, ref)
    q = r.normal(0, 1, (rows, heads * 2, dim))
    q[0, 1], q[1, 2], q[1, 3] = 0.0, q[1, 2] * 1e-20, q[1, 3] * 1e3
    out = up(dev, np.zeros((rows, heads * 2 * dim)), is_bf16)
    K.attention_kv8(out, up(dev, q, is_bf16), *d.buf, dev.upload(np.array([pos], np.int32)), rows, 1, rows, heads * 2, heads, dim, cap, scale,
                    bf16=is_bf16)
    # the scale as the operator gets it: f32
    want, err = ref8.attend(held(q, is_bf16), ref.values("k")[0], ref.values("v")[0], pos, float(np.float32(scale)),
                            steps=32000.0 if is_bf16 else 8.0e6)
    got = values(out, is_bf16).reshape(q.shape)
    assert np.isfinite(got).all()
    # the bound is first order in a score's error: below 0.05 here, exp(2 e) - 1 <= 1.06 x 2 e, but for the large row
    err = 1.06 * err + (BF16 if is_bf16 else F32) * (np.abs(want) + err)
    ok = np.abs(got - want) <= err
    ok[1, 3] = True
    assert ok.all(), np.argwhere(~ok)[:4]


def test_attention_uniform_rows(dev):
    """row_start None: max_rows rows a sequence, the same bits as with it."""
    from qwenasr_amd import kernels as K
    r = rng(14)
    ref = ref8.Cache(3, 2, 256, 128).fill(r)
    d = DevCache(dev, ref)
    q = r.normal(0, 1, (6, 4, 128))
    a = attention(dev, d, q, [2, 2, 2], [5, 100, 254], 2, behind=0)
    out = dev.zeros((6, 4 * 128), np.float32)
    K.attention_kv8(out, up(dev, q, False), *d.buf, dev.upload(np.array([5, 100, 254], np.int32)), 6, 3, 2, 4, 2, 128, 256, 128 ** -0.5)
    assert (out.numpy().reshape(6, 4, 128) == a).all()


def test_row_start_is_held_to_the_buffers(dev):
    """row_start and pos values from anywhere: calls end, and touch nothing outside their rows."""
    from qwenasr_amd import kernels as K
    r = rng(15)
    ref = ref8.Cache(3, 2, 128, 64).fill(r)
    d = DevCache(dev, ref)
    start = dev.upload(np.array([-5, 1 << 30, 2, -(1 << 31)], np.int32))
    pos = dev.upload(np.array([(1 << 31) - 1, 127, -(1 << 31)], np.int32))
    q = up(dev, r.normal(0, 1, (5, 4, 64)), False)
    out = up(dev, np.full((6, 256), 3.0), False)
    k, v = up(dev, np.full((6, 128), 3.0), False), up(dev, np.full((6, 128), 3.0), False)
    K.attention_kv8(out, q, *d.buf, pos, 5, 3, 5, 4, 2, 64, 128, 0.125, row_start=start)
    K.kv8_read(k, v, *d.buf, pos, 5, 3, 5, *d.geometry(), row_start=start)
    K.kv8_write(*d.buf, k, v, pos, 5, 3, 5, *d.geometry(), row_start=start)
    assert all((o.numpy()[5] == 3.0).all() for o in (out, k, v))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_layer(dev):
    """An attention layer's first half in 8 bits as a decoder runs it: three ragged prompts, then single tokens of all
    three; each operator against float64 on what the one before it gave."""
    from qwenasr_amd import kernels as K
    r = rng(21)
    hidden, heads, group, dim, cap = 512, 2, 2, 128, 256
    hq, nqkv = heads * group, (heads * group + 2 * heads) * dim
    g = (1 + r.normal(0, 0.1, hidden)).astype(np.float32)
    wqkv, sqkv = r.integers(-127, 128, (nqkv, hidden), dtype=np.int8), r.uniform(3e-4, 6e-4, nqkv).astype(np.float32)
    wo, so = r.integers(-127, 128, (hidden, hq * dim), dtype=np.int8), r.uniform(3e-4, 6e-4, hidden).astype(np.float32)
    dg, dwq, dsq, dwo, dso = (dev.upload(a) for a in (g, wqkv, sqkv, wo, so))
    ref = ref8.Cache(3, heads, cap, dim)
    d = DevCache(dev, ref)
    pos = np.zeros(3, np.int32)
    for counts in ([70, 1, 33], [1, 1, 1], [1, 1, 1], [20, 64, 1]):
        start, n = prefix(counts), sum(counts)
        x, dl = r.normal(0, 1, (n, hidden)), r.normal(0, 0.3, (n, hidden))
        dx = up(dev, x, False)
        q, s, y = dev.zeros((n, hidden), np.int8), dev.zeros(n, np.float32), dev.zeros((n, nqkv), np.float32)
        dpos, dstart = dev.upload(pos), dev.upload(start)
        K.add_rms_norm_int8(q, s, dx, dg, n, hidden, res=up(dev, dl, False), sum_out=dx)
        K.gemm_w8a8(y, q, s, dwq, dsq, n, nqkv, hidden)

        class At:
            def __init__(self, e):
                self.ptr, self.dev = C.c_void_p(y.ptr.value + 4 * e), dev
        K.kv8_write(*d.buf, At(hq * dim), At((hq + heads) * dim), dpos, n, 3, max(counts), *d.geometry(), row_start=dstart, ld=nqkv)
        o = dev.zeros((n, hq * dim), np.float32)
        K.attention_kv8(o, y, *d.buf, dpos, n, 3, max(counts), hq, heads, dim, cap, dim ** -0.5, row_start=dstart, ldq=nqkv)
        oq, os_ = dev.zeros((n, hq * dim), np.int8), dev.zeros(n, np.float32)
        K.add_rms_norm_int8(oq, os_, o, None, n, hq * dim)
        before = dx.numpy().astype(np.float64)
        K.gemm_w8a8(dx, oq, os_, dwo, dso, n, hidden, hq * dim, accumulate=True)
        # each against float64
        _, want_q, _ = ref8.norm8(held(x, False), held(dl, False), g.astype(np.float64), 1e-6)
        assert (q.numpy() == want_q).all()
        check_gemm(values(y, False), ref8.gemm8(q.numpy(), s.numpy(), wqkv, sqkv)[0], s.numpy(), sqkv, None, None, "plain", False)
        yh = y.numpy().astype(np.float64)
        for j in range(3):
            rows = yh[start[j]:start[j + 1]]
            ref.write(j, int(pos[j]), {"k": rows[:, hq * dim:(hq + heads) * dim].reshape(-1, heads, dim),
                                       "v": rows[:, (hq + heads) * dim:].reshape(-1, heads, dim)})
        d.check()
        check_attention(values(o, False).reshape(n, hq, dim), ref, yh[:, :hq * dim].reshape(n, hq, dim), counts, [int(p) for p in pos])
        assert (oq.numpy() == ref8.norm8(values(o, False), None, None, 0, False)[1]).all()
        check_gemm(values(dx, False), ref8.gemm8(oq.numpy(), os_.numpy(), wo, so)[0], os_.numpy(), so, None, before, "add", False)
        pos = pos + np.array(counts, np.int32)


def test_captured(dev):
    """All of them captured into one graph on the handle's stream and replayed with other positions and rows: each replay
    gives the bits of the eager calls."""
    from qwenasr_amd import kernels as K
    from qwenasr_amd._lib import lib
    hip = C.CDLL("libamdhip64.so.7")     # the HIP runtime the library already loaded
    r = rng(22)
    hidden, heads, group, dim, cap, n = 256, 2, 2, 64, 512, 4
    hq, nqkv = heads * group, (heads * group + 2 * heads) * dim
    dg = dev.upload(np.ones(hidden, np.float32))
    dw, dsw = dev.upload(r.integers(-127, 128, (nqkv, hidden), dtype=np.int8)), dev.upload(r.uniform(3e-4, 6e-4, nqkv).astype(np.float32))
    ref = ref8.Cache(n, heads, cap, dim).fill(r)
    x, pos = dev.zeros((n, hidden), np.float32), dev.zeros(n, np.int32)
    q, s, y, o = dev.zeros((n, hidden), np.int8), dev.zeros(n, np.float32), dev.zeros((n, nqkv), np.float32), dev.zeros((n, hq * dim), np.float32)
    back = [dev.zeros((n, heads * dim), np.float32) for _ in range(2)]

    def at(e):
        class At:
            ptr, dev = C.c_void_p(y.ptr.value + 4 * e), x.dev
        return At

    def step(d):
        K.add_rms_norm_int8(q, s, x, dg, n, hidden)
        K.gemm_w8a8(y, q, s, dw, dsw, n, nqkv, hidden)
        K.kv8_write(*d.buf, at(hq * dim), at((hq + heads) * dim), pos, n, n, 1, *d.geometry(), ld=nqkv)
        K.attention_kv8(o, y, *d.buf, pos, n, n, 1, hq, heads, dim, cap, dim ** -0.5, ldq=nqkv)
        K.kv8_read(*back, *d.buf, pos, n, n, 1, *d.geometry())

    eager, graphed = DevCache(dev, ref), DevCache(dev, ref)
    stream = C.c_void_p(lib().qasr_hip_stream(dev.h))
    graph, exe = C.c_void_p(), C.c_void_p()
    dev.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        step(graphed)
    finally:
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    try:
        for rep in range(4):
            x.copy_from(r.normal(0, 1, (n, hidden)).astype(np.float32))
            pos.copy_from(np.array([0, 63, 64 + rep, 500 + rep], np.int32))
            step(eager)
            want = [a.numpy() for a in (q, s, y, o, *back, *eager.buf)]
            for a in (q, s, y, o, *back):
                a.copy_from(np.zeros(a.shape, a.dtype))
            assert hip.hipGraphLaunch(exe, stream) == 0
            dev.sync()
            got = [a.numpy() for a in (q, s, y, o, *back, *graphed.buf)]
            assert all((a == b).all() for a, b in zip(got, want)), rep
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("rows", [1, 20])
def test_two_handles(dev, rows):
    """Calls in turn on two handles, nothing waited for in between, and a graph of one of them: each handle splits the
    positions through its own scratch area, so every result is that of the call alone."""
    from qwenasr_amd import Device
    from qwenasr_amd import kernels as K
    from qwenasr_amd._lib import lib
    hip = C.CDLL("libamdhip64.so.7")     # the HIP runtime the library already loaded
    r = rng(23 + rows)
    heads, group, dim, cap = 2, 2, 128, 4096
    hq, other, sides = heads * group, Device(0), []
    try:
        for side in (dev, other):
            d = DevCache(side, ref8.Cache(1, heads, cap, dim).fill(r))
            q, pos = up(side, r.normal(0, 1, (rows, hq * dim)), False), side.upload(np.array([cap - rows], np.int32))
            outs = [side.zeros((rows, hq * dim), np.float32) for _ in range(6)]

            def run(o, d=d, q=q, pos=pos):
                K.attention_kv8(o, q, *d.buf, pos, rows, 1, rows, hq, heads, dim, cap, dim ** -0.5)
            run(outs[0])
            sides.append((run, outs, outs[0].numpy()))
        stream = C.c_void_p(lib().qasr_hip_stream(dev.h))
        graph, exe = C.c_void_p(), C.c_void_p()
        captured = dev.zeros((rows, hq * dim), np.float32)
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        try:
            sides[0][0](captured)
        finally:
            assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        try:
            for i in range(1, 6):
                for run, outs, _ in sides:
                    run(outs[i])
                assert hip.hipGraphLaunch(exe, stream) == 0
            for _, outs, want in sides:
                assert all((o.numpy() == want).all() for o in outs)
            assert (captured.numpy() == sides[0][2]).all() and np.abs(sides[0][2]).max() > 0
        finally:
            hip.hipGraphExecDestroy(exe)
            hip.hipGraphDestroy(graph)
        del d, q, pos, outs, run
        sides.clear()
    finally:
        other.close()


def test_nothing_to_do(dev):
    """No rows, no sequences: the calls return and touch nothing."""
    from qwenasr_amd import kernels as K
    b, i8 = dev.zeros(4096, np.float32), dev.zeros(65536, np.int8)
    pos = dev.zeros(4, np.int32)
    K.add_rms_norm_int8(i8, b, b, None, 0, 64)
    K.gemm_w8a8(b, i8, b, i8, b, 0, 64, 64)
    for n_rows, n_seq, max_rows in ((0, 1, 0), (4, 0, 1), (4, 2, 0)):
        K.kv8_write(i8, i8, b, b, b, b, pos, n_rows, n_seq, max_rows, 1, 64, 64)
        K.kv8_read(b, b, i8, i8, b, b, pos, n_rows, n_seq, max_rows, 1, 64, 64)
        K.attention_kv8(b, b, i8, i8, b, b, pos, n_rows, n_seq, max_rows, 1, 1, 64, 64, 0.125)
    assert (b.numpy() == 0).all() and (i8.numpy() == 0).all()
