"""Drafted-token kernels where their loops run long: rings that are filled many times over, on the GPU,
against the plain 64-bit forms (cache_reference)."""
import numpy as np
import pytest

from cache_reference import HD, attend, norm_rope, paths, q4_blocks, q4_dequant
from test_gpu_cache_ops import Scored, Tree, bits, gemv

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


def _attend(t, b=0):
    """Output, its tolerance and the slot weights of sequence b, as cache_reference derives them."""
    n, c = int(t.counts[b]), t.c
    return attend(c, c.view(c.k), c.view(c.v), t.layer, b, int(t.lens[b]), int(t.pos[b]), t.parents[b, :n].tolist(),
                  t.qkv[b, :n], t.gq, t.gk, t.cos, t.sin)


def _queries(t, b=0):
    """Roped queries [n, q_heads, 128] of sequence b."""
    n = int(t.counts[b])
    at = [int(t.pos[b]) + len(p) - 1 for p in paths(t.parents[b, :n].tolist())]
    x = t.qkv[b, :n].reshape(n, -1, HD)[:, :t.c.nq]
    return norm_rope(x, t.gq, t.cos[at][:, None], t.sin[at][:, None]).astype(np.float64)


# ------------------------------------------------------------------ small softmax weights
def _sinks(t, drop):
    """Every sixteenth slot takes nearly the whole weight and has V = 0, as the first slots of a model's
    cache do; all others score `drop` powers of two below, the same in every row, with V in 50..100."""
    c, x = t.c, t.qkv.reshape(t.B, t.T, -1, HD)
    t.gq[:], t.gk[:], t.cos[:], t.sin[:] = 1, 1, 1, 0
    x[:, :, :c.nq] = x[:, :1, :1]                      # one query
    x[:, :, c.nq:c.nq + c.nkv] = 0                     # new keys score 0
    q = norm_rope(x[0, 0, 0], t.gq, t.cos[0], t.sin[0]).astype(np.float64)
    k, v = c.view(c.k), c.view(c.v)
    m = int(t.lens[0])
    k[0, 0, :, :m], k[0, 0, :, :m:16] = 0, q * (drop * np.log(2) * np.sqrt(HD) / (q @ q))
    v[0, 0, :, :m] = t.rng.uniform(50, 100, v[0, 0, :, :m].shape)
    v[0, 0, :, :m:16] = 0
    return t


def _check_small(t, held):
    """`held`: a weight at most this far (in powers of two) below the row's largest is held to half an f16
    step, 2^-11 of itself; a smaller one to half the smallest step, 2^-25 where f16's normal range begins at
    2^-14: so 2^-(held + 11) of the largest weight, which is at most 1.  The largest lies at 2^15 in the
    mma.sync form (held = 15 + 14), at 2^9 at least in the tcgen05 form, which rescales late (9 + 14)."""
    o, tol, _, vn, _, _ = _attend(t)
    m = int(t.lens[0])
    mass = np.abs(t.c.view(t.c.v)[0, 0, :, :m].astype(np.float64)).sum(1) + np.abs(vn.astype(np.float64)).sum(0)
    tol = tol.reshape(len(o), t.c.nkv, -1, HD) + 2.0 ** -(held + 11) * mass[:, None]
    got = t.out.download()[0].reshape(tol.shape).astype(np.float64)
    far = np.abs(got - o.reshape(tol.shape))
    assert (far <= tol).all(), (far / tol).max()
    assert (o > 0).all()


SMALL = [17.3, 20.6, 23.9, 26.4, 29.2]


@pytest.mark.parametrize("drop", SMALL)
@pytest.mark.parametrize("T", [1, 5, 8])
def test_tree_small_weights(gpu, T, drop):
    _check_small(_sinks(Tree(gpu, 70 + T, T, [1500], q_heads=2, kv_heads=1), drop).upload().call(), 29)


@pytest.mark.parametrize("drop", SMALL)
@pytest.mark.parametrize("T", [20, 60])
def test_tree_tc_small_weights(gpu, T, drop):
    _check_small(_sinks(Tree(gpu, 70 + T, T, [1500], q_heads=2, kv_heads=1), drop).upload().call(), 23)


@pytest.mark.parametrize("drop", SMALL)
def test_scored_small_weights(gpu, drop):
    t = _sinks(Scored(gpu, 80, [1500], q_heads=2, kv_heads=1), drop).upload().call()
    _check_small(t, 29)
    *_, w, wt = _attend(t)
    got, want = t.dn.download()[0, 0, :, :1501], w.copy()
    want[:, :1500] += t.weight[0, 0, :, :1500]
    assert (np.abs(got - want) <= wt + 8 * 2.0 ** -24 * want).all()


# ----------------------------------------------------------------------- growing maxima
@pytest.mark.parametrize("T", [5, 8, 20, 33, 60])
def test_tree_maxima_that_grow(gpu, T):
    """Scores that climb by eight (nats) from tile to tile over ten tiles, again and again, each tile for
    one row in particular: the output is rescaled in some rows and tiles and not in others."""
    t = Tree(gpu, 90 + T, T, [10001], q_heads=2, kv_heads=1)
    q = _queries(t).reshape(-1, HD)
    k = t.c.view(t.c.k)[0, 0, 0]
    for j in range(0, 10001, 64):
        r = t.rng.integers(len(q))
        at = slice(j, min(j + 64, 10001))
        k[at] = q[r] * (8 * (j // 64 % 10 + 1) * np.sqrt(HD) / (q[r] @ q[r])) + 0.3 * k[at]
    t.upload().call().check()


@pytest.mark.parametrize("gamma", [1, 24])
@pytest.mark.parametrize("T", [3, 8, 20, 60])
def test_tree_huge_scores(gpu, T, gamma):
    """Scores of thousands up to millions: some rows give one slot the whole weight."""
    t = Tree(gpu, 110 + T, T, [700], q_heads=2, kv_heads=1)
    t.gq[:] = gamma
    t.c.view(t.c.k)[0, 0, :, 40] = 60000
    assert np.isfinite(t.upload().call().check()).all()


# ------------------------------------------------------------------------- 4-bit GEMV
@pytest.mark.parametrize("N,K,R", [(151936, 256, 1), (151936, 256, 16), (151936, 1024, 8), (151936, 1024, 16),
                                   (90001, 1280, 3), (60007, 2048, 8), (151935, 512, 9)])
def test_gemv_q4_of_many_tiles(gpu, N, K, R):
    """Every ring stage of the streaming kernel is filled several times; and the same bits again."""
    rng = np.random.default_rng(N + K + R)
    blocks, x = q4_blocks(rng, N, K), rng.standard_normal((R, K)).astype(np.float16)
    got = gemv(gpu, blocks, x)
    xd = x.astype(np.float64)
    for n in range(0, N, 8192):
        w = q4_dequant(blocks[n:n + 8192])
        y = xd @ w.T
        # 32 exact products of a block summed in f32 by two MMAs, a chain of K / 64 blocks a warp, the
        # two warps' sums: each step off by up to 2^-23 of the sum of magnitudes; one rounding to f16
        tol = (34 + K / 64 + 2) * 2.0 ** -23 * (np.abs(xd) @ np.abs(w).T) + 2.0 ** -11 * np.abs(y) + 2.0 ** -25
        assert (np.abs(got[:, n:n + 8192] - y) <= tol).all(), n
    assert np.array_equal(bits(gemv(gpu, blocks, x)), bits(got))
