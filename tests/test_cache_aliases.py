"""Arrays of the drafted-token operators that may not share memory, without a GPU."""
import pytest

from cache_reference import host_buffer
from test_cache_ops import INVALID, Call


@pytest.mark.parametrize("op", ["commit", "evict"])
@pytest.mark.parametrize("off", [-8, 0, 8])
def test_new_len_over_pos(q3, op, off):
    """Other CTAs read pos while one writes new_len."""
    c = Call(q3)
    c.with_(pos=c.p + 1024, new_len=c.p + 1024 + off)
    assert getattr(c, op)() == INVALID
    assert b"new_len" in q3.lib().q3_last_error()


@pytest.mark.parametrize("op", ["tree", "scored"])
@pytest.mark.parametrize("off", [-8, 0, 8, 2 * 4 * 4096 * 2 - 8])
def test_out_over_qkv(q3, op, off):
    """Other CTAs read qkv while one writes its rows of out."""
    c = Call(q3)
    c.with_(new_weight=c.p + 40000)
    n = 2 * (4 if op == "tree" else 1) * 4096 * 2
    c.with_(qkv=c.p + (1 << 14), out=c.p + (1 << 14) + min(off, n - 8))
    assert getattr(c, op)() == INVALID
    assert b"qkv" in q3.lib().q3_last_error()


@pytest.mark.parametrize("which", ["x", "w"])
@pytest.mark.parametrize("off", [-2, 0, 2])
def test_gemv_output_over_an_input(q3, which, off):
    _, p = host_buffer(1 << 16)
    w, x = p, p + 16384
    y = (w if which == "w" else x) + off
    assert q3.lib().q3_gemv_q4(w, x, y, 16, 256, 1, None) == INVALID
    assert b"apart" in q3.lib().q3_last_error()
