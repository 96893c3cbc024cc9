"""Arrays of the drafted-token operators that may not share memory, without a GPU."""
import pytest

from test_cache_ops import INVALID, Call


@pytest.mark.parametrize("op", ["commit", "evict"])
@pytest.mark.parametrize("off", [-8, 0, 8])
def test_new_len_over_pos(q3, op, off):
    """Other CTAs read pos while one writes new_len."""
    c = Call(q3)
    c.with_(pos=c.p + 1024, new_len=c.p + 1024 + off)
    assert getattr(c, op)() == INVALID
    assert b"new_len" in q3.lib().q3_last_error()
