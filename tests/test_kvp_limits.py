"""Arguments at the ends of their types, refused by the operators for several hypotheses of one prompt before the handle and
the device are looked at (no GPU: a null handle comes last)."""
import pytest

from test_kvp_refusals import P, attn, compact, fork, write

INT64 = (1 << 63) - 1


@pytest.mark.parametrize("f", [fork, compact, write, attn], ids=lambda f: f.__name__)
@pytest.mark.parametrize("page,table_ld", [(16, 1 << 60), (16, 3 << 60), (32, 1 << 59), (256, 1 << 56), (256, (1 << 56) + 1), (64, 1 << 58), (128, 1 << 57),
                                           (16, INT64), (256, INT64), (16, (1 << 26) + 1), (256, (1 << 22) + 1), (16, 1 << 32)])
def test_a_table_longer_than_positions_count(f, page, table_ld):
    """table_ld x page past 2^30, also where the product does not fit its type."""
    from qwenasr_amd import _lib
    rc, msg = f(page=page, table_ld=table_ld)
    assert rc == _lib.QASR_ERR_INVALID and "table_ld" in msg, (rc, msg)


@pytest.mark.parametrize("f,name", [(write, "k"), (write, "v"), (attn, "q"), (attn, "out")], ids=lambda v: getattr(v, "__name__", v))
@pytest.mark.parametrize("bf16,off,taken", [(0, 1, False), (0, 2, False), (0, 3, False), (0, 4, True), (1, 1, False), (1, 2, True), (1, 3, False), (1, 6, True)])
def test_rows_that_are_not_aligned_to_their_type(f, name, bf16, off, taken):
    from qwenasr_amd import _lib
    rc, msg = f(**{name: P + (1 << 15) + off, "bf16": bf16})
    assert rc == _lib.QASR_ERR_INVALID and ("handle is null" == msg if taken else "aligned" in msg), (rc, msg)


@pytest.mark.parametrize("scale,taken", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False), (float("inf"), False)])
def test_a_scale_whose_product_with_log2_e_is_not_finite(scale, taken):
    """Scores are taken in base 2: 2.4e38 x log2 e is no f32, and 0 times it no score of 0."""
    from qwenasr_amd import _lib
    rc, msg = attn(scale=scale)
    assert rc == _lib.QASR_ERR_INVALID and ("handle is null" == msg if taken else "scale" in msg), (rc, msg)


# 8 rows of 4 heads of 128: q's rows 512 elements apart, or 600
@pytest.mark.parametrize("kw,taken", [(dict(), True), (dict(bf16=1), True), (dict(ldq=600), False), (dict(out=P + 16), False), (dict(out=P + 4096 * 4 - 16), False),
                                      (dict(out=P + 4096 * 4), True), (dict(out=P + 4096 * 2, bf16=1), True), (dict(out=P + 4096 * 2 - 2, bf16=1), False),
                                      (dict(q=P + 16), False), (dict(out=P + 2048, ldq=600), False), (dict(out=P + (7 * 600 + 512) * 4, ldq=600), True),
                                      (dict(q=P + 4096 * 4), True)])
def test_results_over_rows_that_are_still_to_be_read(kw, taken):
    """out may be q, row by row; else the two are apart."""
    from qwenasr_amd import _lib
    rc, msg = attn(**kw)
    assert rc == _lib.QASR_ERR_INVALID and ("handle is null" == msg if taken else "overlaps" in msg), (rc, msg)
