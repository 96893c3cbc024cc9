"""Sequences that the drafted-token operators leave as they were, on the GPU."""
import numpy as np
import pytest

from cache_reference import Cache, up
from test_gpu_cache_ops import BAD_POS, BAD_TREE, bits, commit, evict_inputs

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


@pytest.mark.parametrize("acc,n,length,pos", [([1, 2, 4], 4, 10, 10), ([1, 2, 4], -1, 10, 10), ([1, 2, 4], 3, -1, 10),
                                              ([1, 2, 4], 3, 88, 99), ([1, 2, 5], 3, 85, 99), ([2, 1, 4], 3, 10, 10),
                                              ([1, 1, 4], 3, 10, 10), ([1, 2, 64], 3, 10, 10), ([-1, 2, 4], 3, 10, 10),
                                              ([1, 2, 4], 3, 10, -1), ([1, 2, 4], 3, 10, 1 << 31)],
                         ids=["count", "negative count", "length", "full", "behind the slots", "descending", "twice",
                              "token 64", "token -1", "position", "large position"])
def test_commit_refuses_the_whole_path(gpu, acc, n, length, pos):
    """One sequence's path is bad: nothing of it moves, its length stays and the code is 6; the other's moves."""
    c = Cache(np.random.default_rng(3), 2, 2, 90).upload(gpu)
    shape = (2, 2, 8, 90)
    w, sp = np.ones(shape, np.float32), np.full(shape, 5, np.int32)
    given = [up(gpu, x) for x in (np.array([pos, 30]), w, sp)]
    new_len, err = commit(gpu, c, 0, 2, np.array([acc, [0, 3, 9]], np.int32), np.array([n, 3], np.int32),
                          np.array([length, 20]), given)
    assert err == BAD_TREE and new_len.tolist() == [length, 23]
    k, v = c.k.copy(), c.v.copy()
    for x in (k, v):
        c.view(x)[1, :, :, 21], c.view(x)[1, :, :, 22] = c.view(x)[1, :, :, 23].copy(), c.view(x)[1, :, :, 29].copy()
    w[1, :, :, 20:23], sp[1, :, :, 20:23] = 0, [30, 31, 32]
    got_k, got_v = c.download()
    assert np.array_equal(bits(got_k), bits(k)) and np.array_equal(bits(got_v), bits(v))
    assert np.array_equal(given[1].download(), w) and np.array_equal(given[2].download(), sp)
