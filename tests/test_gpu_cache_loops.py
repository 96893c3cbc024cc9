"""Drafted-token kernels where their loops run long: rings that are filled many times over, on the GPU,
against the plain 64-bit forms (cache_reference)."""
import numpy as np
import pytest

from test_gpu_cache_ops import Tree, bits

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- tree attention, tcgen05 form
@pytest.mark.parametrize("T", [20, 32, 33, 60])
@pytest.mark.parametrize("length", [9984, 10001, 10049, 31999])
def test_tree_of_many_tiles_a_cta(gpu, T, length):
    """One kv head, so at most 16 CTAs for all of the cache: 9 to 32 tiles each, lengths at and around
    multiples of a tile; every launch gives the same bits."""
    t = Tree(gpu, T + length, T, [length], q_heads=2, kv_heads=1, gap=3).upload()
    first = bits(t.call().check()).copy()
    for _ in range(20):
        t.call()
        assert np.array_equal(bits(t.out.download()), first)


@pytest.mark.parametrize("T", [20, 60])
def test_tree_of_many_sequences(gpu, T):
    """More (sequence, kv head) than SMs: a CTA each, of up to 11 tiles; and some of a tile or two."""
    rng = np.random.default_rng(T)
    lens = [640, 639, 641, 0, 1, 63, 64, 65, 128, 577, *rng.integers(0, 641, 30).tolist()]
    counts = [T] * 10 + rng.integers(1, T + 1, 30).tolist()
    t = Tree(gpu, T, T, lens, counts, S=640 + T + 1).upload()
    first = bits(t.call().check()).copy()
    for _ in range(5):
        t.call()
        assert np.array_equal(bits(t.out.download()), first)
