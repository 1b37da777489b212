"""What the operators for several hypotheses of one prompt refuse: arguments are checked before the handle and the
device, so these run without a GPU (a null handle comes last)."""
import ctypes as C

import pytest

BUF = C.create_string_buffer(1 << 16)
P = (C.addressof(BUF) + 255) // 256 * 256          # any non-null, aligned address: no call here reaches a device
AT = [P + 4096 * i for i in range(12)]             # apart from one another


def call(name, *args):
    from qwenasr_amd import _lib
    L = _lib.lib()
    rc = getattr(L, name)(None, *args)
    return rc, L.qasr_hip_last_error().decode()


POOLS = dict(pools=AT[8], n_pools=2, pool_stride=8 * 2 * 16 * 256, n_pages=8, n_heads=2, page=16, row_bytes=256)


def fork(**kw):
    a = dict(table_out=AT[0], pos_out=AT[1], len_out=AT[2], status=AT[3], table=AT[4], len=AT[5], parent=AT[6], row_start=AT[7], max_rows=1,
             n_out=3, n_seq=2, table_ld=4, **POOLS)
    a.update(kw)
    return call("qasr_hip_kvp_fork", *a.values())


def compact(**kw):
    a = dict(table_out=AT[0], status=AT[3], table=AT[4], len=AT[5], n_seq=2, table_ld=4, **POOLS)
    a.update(kw)
    return call("qasr_hip_kvp_compact", *a.values())


ROWS = dict(row_start=P, pos=P, n_rows=8, n_seq=2, max_rows=4)


def write(**kw):
    a = dict(kp=P, vp=P, n_pages=8, k=P, v=P, ld=256, table=P, table_ld=4, **ROWS, heads=2, dim=128, page=16, bf16=0)
    a.update(kw)
    return call("qasr_hip_kvp_write", *a.values())


def attn(**kw):
    a = dict(out=P, q=P, ldq=512, kp=P, vp=P, n_pages=8, table=P, table_ld=4, **ROWS, max_len=0, group=2, shared=P, max_own=0, n_heads=4,
             heads=2, dim=128, page=16, scale=0.1, bf16=0)
    a.update(kw)
    return call("qasr_hip_attention_kvp", *a.values())


def logp(**kw):
    a = dict(logp=P, entropy=P, top_ids=P, top_logp=P, k=4, logits=P, ld=64, targets=P, rows=4, cols=64, bf16=0)
    a.update(kw)
    return call("qasr_hip_token_logprobs", *a.values())


PAGED = [dict(page=0), dict(page=8), dict(page=48), dict(page=512), dict(n_pages=0), dict(n_pages=(1 << 18) + 1), dict(n_seq=-1), dict(n_seq=2049),
         dict(table_ld=0), dict(table_ld=-1), dict(table_ld=1 << 27), dict(table=None)]
POOL = [dict(pools=None), dict(pools=AT[8] + 8), dict(n_pools=0), dict(n_pools=65536), dict(pool_stride=8 * 2 * 16 * 256 - 16),
        dict(pool_stride=8 * 2 * 16 * 256 + 8), dict(n_heads=0), dict(n_heads=1025), dict(row_bytes=0), dict(row_bytes=24), dict(row_bytes=4112)]
CACHE = [dict(kp=None), dict(vp=None), dict(kp=P + 8), dict(vp=P + 2), dict(pos=None), dict(dim=96), dict(dim=0), dict(heads=0), dict(heads=1025),
         dict(n_rows=-1), dict(n_rows=1 << 31), dict(max_rows=-1), dict(max_rows=1 << 25), dict(row_start=None, n_rows=7)]
BAD = ([(f, k) for f in (fork, compact, write, attn) for k in PAGED] + [(f, k) for f in (fork, compact) for k in POOL]
       + [(f, k) for f in (write, attn) for k in CACHE]
       + [(fork, k) for k in (dict(table_out=None), dict(pos_out=None), dict(len_out=None), dict(status=None), dict(len=None), dict(n_out=-1),
                              dict(n_out=2049), dict(parent=None), dict(max_rows=-1), dict(max_rows=1 << 25), dict(table_out=AT[4]),
                              dict(table_out=AT[4] + 28), dict(pos_out=AT[5]), dict(len_out=AT[6] + 8), dict(status=AT[7] + 12),
                              dict(pos_out=AT[2]), dict(status=AT[0] + 44))]
       + [(compact, k) for k in (dict(table_out=None), dict(status=None), dict(len=None), dict(table_out=AT[4] + 16), dict(status=AT[4]),
                                 dict(status=AT[5] + 4), dict(status=AT[0]), dict(table_out=AT[5] - 4))]
       + [(write, k) for k in (dict(k=None), dict(v=None), dict(ld=255), dict(ld=1 << 31))]
       + [(attn, k) for k in (dict(out=None), dict(q=None), dict(ldq=511), dict(ldq=1 << 31), dict(n_heads=3), dict(n_heads=0), dict(group=0),
                              dict(group=-1), dict(max_len=-1), dict(max_own=-1), dict(scale=float("nan")), dict(scale=float("inf")))]
       + [(logp, k) for k in (dict(logits=None), dict(targets=None), dict(cols=0), dict(cols=(1 << 20) + 1, ld=1 << 21), dict(ld=63), dict(rows=-1),
                              dict(rows=1 << 25), dict(k=-1), dict(k=33), dict(k=5, cols=4), dict(logits=P + 2), dict(logits=P + 1, bf16=1))])


@pytest.mark.parametrize("f,kw", BAD, ids=lambda v: v.__name__ if callable(v) else "-".join(f"{k}" for k in v))
def test_refused(f, kw):
    from qwenasr_amd import _lib
    rc, msg = f(**kw)
    assert rc == _lib.QASR_ERR_INVALID and "handle" not in msg, (rc, msg)


@pytest.mark.parametrize("f,kw", [(fork, {}), (fork, dict(parent=None, n_out=2)), (fork, dict(row_start=None)), (fork, dict(n_out=0)),
                                  (compact, {}), (compact, dict(table_out=AT[4])), (write, {}), (attn, {}), (attn, dict(shared=None)),
                                  (attn, dict(scale=0.0)), (attn, dict(group=1 << 62)), (logp, {}), (logp, dict(logp=None, targets=None)), (logp, dict(k=0)),
                                  (logp, dict(logits=P + 2, bf16=1))])
def test_what_is_right_reaches_the_handle(f, kw):
    from qwenasr_amd import _lib
    rc, msg = f(**kw)
    assert rc == _lib.QASR_ERR_INVALID and msg == "handle is null"
