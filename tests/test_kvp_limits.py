"""Arguments at the ends of their types, refused by the operators for several hypotheses of one prompt before the handle and
the device are looked at (no GPU: a null handle comes last)."""
import pytest

from test_kvp_refusals import attn, compact, fork, write

INT64 = (1 << 63) - 1


@pytest.mark.parametrize("f", [fork, compact, write, attn], ids=lambda f: f.__name__)
@pytest.mark.parametrize("page,table_ld", [(16, 1 << 60), (16, 3 << 60), (32, 1 << 59), (256, 1 << 56), (256, (1 << 56) + 1), (64, 1 << 58), (128, 1 << 57),
                                           (16, INT64), (256, INT64), (16, (1 << 26) + 1), (256, (1 << 22) + 1), (16, 1 << 32)])
def test_a_table_longer_than_positions_count(f, page, table_ld):
    """table_ld x page past 2^30, also where the product does not fit its type."""
    from qwenasr_amd import _lib
    rc, msg = f(page=page, table_ld=table_ld)
    assert rc == _lib.QASR_ERR_INVALID and "table_ld" in msg, (rc, msg)
