"""Sequences that the drafted-token operators leave as they were, on the GPU."""
import numpy as np
import pytest

from cache_reference import Cache, up
from test_gpu_cache_ops import BAD_POS, bits, evict_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pos", [-1, -(1 << 40)])
def test_evict_bad_position(gpu, pos):
    """A negative position would make every slot one of the newest."""
    rng = np.random.default_rng(1)
    c = Cache(rng, 2, 1, 50, 2, 1).upload(gpu)
    w, sp = evict_inputs(rng, c)
    new_w, new_sp = up(gpu, np.full_like(w, -3)), up(gpu, np.full_like(sp, -3))
    lens, new_len, err = np.array([50, 15]), up(gpu, np.full(2, -7, np.int64)), up(gpu, np.zeros(1, np.int32))
    d = [up(gpu, x) for x in (lens, np.array([pos, pos]), w, sp)]
    gpu.call("q3_cache_evict", c.kv, 0, 1, 2, 20, 5, *(x.ptr for x in d), new_len.ptr, new_w.ptr, new_sp.ptr, err.ptr, None)
    assert err.download()[0] == BAD_POS
    assert np.array_equal(new_len.download(), lens)
    assert (new_w.download() == -3).all() and (new_sp.download() == -3).all()
    k, v = c.download()
    assert np.array_equal(bits(k), bits(c.k)) and np.array_equal(bits(v), bits(c.v))
