"""What the 8-bit layer operators refuse: arguments are checked before the handle
and the device, so these run without a GPU (a null handle comes last)."""
import ctypes as C

import pytest

BUF = C.create_string_buffer(4096)
P = (C.addressof(BUF) + 255) // 256 * 256          # any non-null, aligned address: no call here reaches a device


def call(name, *args):
    from qwenasr_amd import _lib
    L = _lib.lib()
    rc = getattr(L, name)(None, *args)
    return rc, L.qasr_hip_last_error().decode()


def norm(**kw):
    a = dict(q=P, scales=P, sum=P, x=P, res=P, norm_w=P, rows=4, hidden=64, ld=64, eps=1e-6, bf16=0)
    a.update(kw)
    return call("qasr_hip_add_rms_norm_int8", *a.values())


def gemm(**kw):
    a = dict(y=P, a=P, sa=P, w=P, sw=P, bias=P, M=4, N=64, K=64, mode=0, bf16=0)
    a.update(kw)
    return call("qasr_hip_gemm_w8a8", *a.values())


KV = dict(k8=P, v8=P, ks=P, vs=P)
ROWS = dict(row_start=P, pos=P, n_rows=8, n_seq=2, max_rows=4)


def write(**kw):
    a = dict(**KV, k=P, v=P, ld=256, **ROWS, heads=2, dim=128, cap=128, bf16=0)
    a.update(kw)
    return call("qasr_hip_kv8_write", *a.values())


def read(**kw):
    a = dict(k=P, v=P, ld=256, **KV, **ROWS, heads=2, dim=128, cap=128, bf16=0)
    a.update(kw)
    return call("qasr_hip_kv8_read", *a.values())


def attn(**kw):
    a = dict(out=P, q=P, ldq=512, **KV, **ROWS, max_len=0, n_heads=4, heads=2, dim=128, cap=128, scale=0.1, window=0, sinks=0, bf16=0)
    a.update(kw)
    return call("qasr_hip_attention_kv8", *a.values())


CACHE = [dict(k8=None), dict(v8=None), dict(ks=None), dict(vs=None), dict(pos=None), dict(dim=96), dict(dim=0), dict(cap=0), dict(cap=100),
         dict(cap=1 << 31), dict(heads=0), dict(n_seq=-1), dict(n_seq=1 << 20), dict(n_rows=-1), dict(n_rows=1 << 31), dict(max_rows=-1),
         dict(max_rows=1 << 25), dict(row_start=None, n_rows=7), dict(k8=P + 8), dict(v8=P + 1)]
BAD = ([(norm, k) for k in (dict(q=None), dict(scales=None), dict(x=None), dict(rows=-1), dict(rows=1 << 31), dict(hidden=0), dict(hidden=16385, ld=16385),
                            dict(ld=63), dict(eps=-1.0), dict(eps=float("nan")))]
       + [(gemm, k) for k in (dict(y=None), dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(M=-1), dict(M=1 << 23), dict(N=0),
                              dict(N=1 << 29), dict(K=0), dict(K=131072), dict(mode=3), dict(mode=-1), dict(mode=2, N=63))]
       + [(f, k) for f in (write, read, attn) for k in CACHE]
       + [(f, k) for f in (write, read) for k in (dict(k=None), dict(v=None), dict(ld=255), dict(ld=1 << 31))]
       + [(attn, k) for k in (dict(out=None), dict(q=None), dict(ldq=511), dict(n_heads=3), dict(n_heads=0), dict(window=-1), dict(sinks=-1),
                              dict(max_len=-1))])


@pytest.mark.parametrize("f,kw", BAD, ids=lambda v: v.__name__ if callable(v) else "-".join(f"{k}" for k in v))
def test_refused(f, kw):
    from qwenasr_amd import _lib
    rc, msg = f(**kw)
    assert rc == _lib.QASR_ERR_INVALID and "handle" not in msg, (rc, msg)


@pytest.mark.parametrize("f", [norm, gemm, write, read, attn])
def test_what_is_right_reaches_the_handle(f):
    from qwenasr_amd import _lib
    rc, msg = f()
    assert rc == _lib.QASR_ERR_INVALID and msg == "handle is null"


def test_accumulate_and_swiglu_exclude_each_other():
    from qwenasr_amd import kernels as K
    with pytest.raises(ValueError):
        K.gemm_w8a8(None, None, None, None, None, 1, 2, 64, accumulate=True, swiglu=True)
