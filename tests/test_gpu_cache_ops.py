"""Drafted-token operators on the GPU against plain 64-bit forms (cache_reference)."""
import ctypes

import numpy as np
import pytest
from cache_reference import HD, Cache, attend, evict, q4_blocks, q4_dequant, rope_tables, up

pytestmark = pytest.mark.gpu

BAD_POS, BAD_TREE = 5, 6


def bits(a):
    return np.ascontiguousarray(a).view(np.uint16)


# ------------------------------------------------------------------ 4-bit GEMV
def gemv(gpu, blocks, x, stream=None):
    N, K, R = blocks.shape[0], blocks.shape[1] * 32, x.shape[0]
    w, dx, y = up(gpu, blocks), up(gpu, x), gpu.DeviceArray((R + 1, N), np.float16)
    y.fill_bytes(0x55)
    gpu.call("q3_gemv_q4", w.ptr, dx.ptr, y.ptr, N, K, R, stream)
    out = y.download(stream)
    assert (bits(out[R]) == 0x5555).all()  # nothing behind the last row
    return out[:R]


def gemv_tolerance(blocks, x):
    """A block's two MMAs sum 32 exact products in f32 (each step off by up to 2^-23 of the sum of
    magnitudes: the tensor core may truncate), K / 256 blocks a warp and 8 warps follow; one rounding."""
    w, x = q4_dequant(blocks), x.astype(np.float64)
    y = x @ w.T
    steps = 34 + 2 + w.shape[1] / 256 + 8
    return y, steps * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + 2.0 ** -11 * np.abs(y) + 2.0 ** -25


@pytest.mark.parametrize("N,K,R", [(1, 256, 1), (15, 256, 2), (16, 512, 1), (17, 768, 3), (100, 1024, 7), (2048, 1024, 1),
                                   (1000, 1280, 8), (6007, 1280, 5), (33, 2048, 9), (48, 2304, 16), (20, 16384, 1),
                                   (20, 16384, 16), (4099, 256, 12), (40000, 512, 8), (50021, 1024, 4),
                                   (20000, 768, 16), (12000, 2048, 3), (13001, 1280, 9), (10007, 256, 1),
                                   (9990, 4096, 2)])
def test_gemv_q4(gpu, N, K, R):
    rng = np.random.default_rng(N + K + R)
    blocks, x = q4_blocks(rng, N, K), rng.standard_normal((R, K)).astype(np.float16)
    y, tol = gemv_tolerance(blocks, x)
    assert (np.abs(gemv(gpu, blocks, x) - y) <= tol).all()


def test_gemv_q4_extremes(gpu):
    """Zero, negative, smallest and large scales; nibbles at both ends; a row that overflows f16."""
    rng = np.random.default_rng(3)
    blocks, x = q4_blocks(rng, 32, 512), rng.standard_normal((3, 512)).astype(np.float16)
    d = np.ascontiguousarray(blocks[..., :2]).view(np.float16)
    d[0], d[1], d[2], d[3] = 0, -0.01, 2.0 ** -24, 30000
    blocks[..., :2] = d.view(np.uint8)
    blocks[4, :, 2:], blocks[5, :, 2:] = 0x00, 0xff
    y, tol = gemv_tolerance(blocks, x)
    with np.errstate(over="ignore"):
        want = y.astype(np.float16).astype(np.float64)
    got = gemv(gpu, blocks, x).astype(np.float64)
    over = np.isinf(want)
    assert over[:, 3].any() and np.array_equal(got[over], want[over])
    assert (np.abs(got - y)[~over] <= tol[~over]).all()


def test_gemv_q4_rows_do_not_mix(gpu):
    """An infinite and a NaN row of x change no other row."""
    rng = np.random.default_rng(4)
    blocks, x = q4_blocks(rng, 64, 256), rng.standard_normal((5, 256)).astype(np.float16)
    clean = gemv(gpu, blocks, x)
    x[1, 7], x[3, 200] = np.inf, np.nan
    got = gemv(gpu, blocks, x)
    assert np.array_equal(bits(got[[0, 2, 4]]), bits(clean[[0, 2, 4]]))
    w = q4_dequant(blocks)[:, 7]
    assert np.array_equal(got[1][w != 0], np.sign(w[w != 0]) * np.inf) and np.isnan(got[1][w == 0]).all()
    assert np.isnan(got[3]).all()


# --------------------------------------------------------------- tree attention
def random_tree(rng, n, kind):
    if kind == "chain":
        return np.arange(n) - 1
    if kind == "star":
        return np.full(n, -1)
    return np.array([rng.integers(max(-1, i - 6), i) for i in range(n)])


class Tree:
    """Inputs of a tree (or scored) call and its check."""

    def __init__(self, gpu, seed, T, lens, counts=None, kind="mixed", layers=1, layer=0, S=None, q_heads=16, kv_heads=8,
                 layout="flat", gap=0):
        rng = self.rng = np.random.default_rng(seed)
        self.gpu, self.T, self.layer, self.B = gpu, T, layer, len(lens)
        self.lens = np.array(lens, np.int64)
        self.counts = np.array([T] * self.B if counts is None else counts, np.int32)
        self.given = counts is not None
        S = S or int(max(lens)) + T + 3
        self.c = Cache(rng, self.B, layers, S, q_heads, kv_heads, layout)
        self.pos = self.lens + gap
        # what lies behind the cached slots must not be read
        for x in (self.c.k, self.c.v):
            v = self.c.view(x)
            for b in range(self.B):
                v[b, layer, :, lens[b]:] = np.nan
        self.qkv = rng.standard_normal((self.B, T, (q_heads + 2 * kv_heads) * HD)).astype(np.float16)
        self.gq, self.gk = ((1 + 0.1 * rng.standard_normal(HD)).astype(np.float16) for _ in range(2))
        self.cos, self.sin = rope_tables(gpu, max(S, int(self.pos.max()) + T + 1))
        self.parents = np.zeros((self.B, T), np.int32)
        for b in range(self.B):
            self.parents[b] = random_tree(rng, T, kind)

    def upload(self):
        g = self.gpu
        self.c.upload(g)
        self.d = {n: up(g, getattr(self, n)) for n in ("qkv", "gq", "gk", "cos", "sin", "parents", "counts", "lens", "pos")}
        self.out = g.DeviceArray((self.B, self.T, self.c.nq * HD), np.float16)
        self.out.fill_bytes(0x55)
        self.err = up(g, np.zeros(1, np.int32))
        return self

    def call(self, stream=None):
        d = self.d
        self.gpu.call("q3_tree_attention", d["qkv"].ptr, d["gq"].ptr, d["gk"].ptr, d["cos"].ptr, d["sin"].ptr,
                      self.cos.shape[0], self.c.kv, self.layer, self.B, self.T, d["parents"].ptr,
                      d["counts"].ptr if self.given else None, d["lens"].ptr, d["pos"].ptr, self.out.ptr, self.err.ptr, stream)
        return self

    def check(self, stream=None, skip=()):
        out = self.out.download(stream)
        k, v = self.c.download()
        wk, wv = self.c.k.copy(), self.c.v.copy()
        for b in range(self.B):
            n = int(self.counts[b]) if b not in skip else 0
            assert (bits(out[b, max(n, 0):]) == 0x5555).all()  # rows behind the last token
            if n == 0:
                continue
            m = int(self.lens[b])
            o, tol, kn, vn, _, _ = attend(self.c, self.c.view(self.c.k), self.c.view(self.c.v), self.layer, b, m,
                                          int(self.pos[b]), self.parents[b, :n].tolist(), self.qkv[b, :n], self.gq, self.gk,
                                          self.cos, self.sin)
            far = np.abs(out[b, :n] - o)
            assert (far <= tol).all(), (b, np.nanmax(far / tol), np.isnan(far).sum())
            self.c.view(wk)[b, self.layer, :, m:m + n] = kn.swapaxes(0, 1)
            self.c.view(wv)[b, self.layer, :, m:m + n] = vn.swapaxes(0, 1)
        assert np.array_equal(bits(k), bits(wk)) and np.array_equal(bits(v), bits(wv))  # new rows bit for bit, no others
        return out


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("length", [0, 1, 64, 333])
def test_tree_attention(gpu, T, length):
    Tree(gpu, T * 1000 + length, T, [length]).upload().call().check()


@pytest.mark.parametrize("length", [15, 16, 17, 63, 65, 127, 128, 129, 1023, 1024, 1025, 4097])
def test_tree_attention_lengths(gpu, length):
    Tree(gpu, length, 5, [length], gap=7).upload().call().check()


@pytest.mark.parametrize("layout", ["flat", "head", "padded"])
@pytest.mark.parametrize("kind", ["mixed", "chain", "star"])
def test_tree_attention_batch(gpu, layout, kind):
    t = Tree(gpu, 5, 20, [130, 0, 700, 64, 1, 257], [20, 3, 1, 0, 20, 13], kind, layers=3, layer=1, layout=layout, gap=11)
    t.upload().call().check()


@pytest.mark.parametrize("q_heads,kv_heads,T", [(8, 8, 64), (8, 8, 3), (1, 1, 5), (2, 1, 64), (32, 8, 32), (32, 8, 4),
                                                (64, 8, 16), (64, 8, 2), (6, 3, 10)])
def test_tree_attention_heads(gpu, q_heads, kv_heads, T):
    Tree(gpu, q_heads, T, [200, 77], q_heads=q_heads, kv_heads=kv_heads).upload().call().check()


@pytest.mark.parametrize("B", [3, 20, 40, 100])
def test_tree_attention_cluster_sizes(gpu, B):
    """More sequences, fewer CTAs each."""
    rng = np.random.default_rng(B)
    Tree(gpu, B, 4, rng.integers(0, 500, B).tolist()).upload().call().check()


def test_tree_attention_full_cache(gpu):
    Tree(gpu, 8, 6, [58, 122], S=128, counts=[6, 6]).upload().call().check()


def test_tree_attention_bad_values(gpu):
    """A sequence with a bad count, length, position or tree is left alone; the others are not."""
    t = Tree(gpu, 9, 4, [30, 40, 50, 20, 10, 60, 25, 35], [4, 5, 4, 4, 4, -1, 4, 4], S=70)
    t.lens[2], t.pos[3], t.pos[4] = 67, -1, t.cos.shape[0] - 2
    t.parents[4] = [-1, 0, 1, 2]          # its last tokens run out of the rope table
    t.parents[6] = [-1, 0, 2, 1]          # a token that is its own parent
    t.parents[7] = [-1, -2, 0, 0]
    t.upload().call()
    t.check(skip=(1, 2, 3, 4, 5, 6, 7))
    assert t.err.download()[0] in (BAD_POS, BAD_TREE)
    with pytest.raises(gpu.Q3Error):
        gpu.call("q3_check_error_word", t.err.ptr, None)


@pytest.mark.parametrize("b,code", [(0, BAD_POS), (1, BAD_TREE)])
def test_tree_attention_error_code(gpu, b, code):
    t = Tree(gpu, 9, 4, [30, 40])
    if b == 0:
        t.lens[0] = -2
    else:
        t.parents[1, 2] = 3
    t.upload().call().check(skip=(b,))
    assert t.err.download()[0] == code


def test_tree_attention_huge_scores(gpu):
    """Scores of several thousand, where some rows give one slot the whole weight and some give it none."""
    t = Tree(gpu, 11, 3, [100])
    t.c.view(t.c.k)[0, 0, :, 40] = 60000
    out = t.upload().call().check()
    assert np.isfinite(out).all()


@pytest.mark.parametrize("T", [6, 30, 60])
def test_tree_attention_odd_values_stay_on_their_branch(gpu, T):
    """An infinity and a NaN in a drafted token's V row reach the tokens that see it, in their dims, and
    no other; a token whose Q and K are NaN spoils only its descendants."""
    t = Tree(gpu, 30 + T, T, [130], kind="mixed")
    clean = t.upload().call().check()
    par = t.parents[0]
    sees = lambda i, j: i == j or (par[i] >= 0 and sees(par[i], j))
    bad, lost = T // 3, T - 2
    par[lost] = -1                                        # apart from the first
    par[bad] = -1
    base = t.upload().call().check()
    x = t.qkv[0].reshape(T, 32, HD)
    x[bad, 24:, 3], x[bad, 24:, 90] = -np.inf, np.nan     # V of every kv head
    x[lost, :24] = np.nan                                 # its Q and K
    t.upload().call()
    got, k = t.out.download()[0].reshape(T, 16, HD), t.c.download()[0]
    want = base[0].reshape(T, 16, HD)
    for i in range(T):
        dims = np.ones(HD, bool)
        if sees(i, lost):
            assert np.isnan(got[i]).all()
            continue
        if sees(i, bad):
            dims[[3, 90]] = False
            assert (got[i, :, 3] == -np.inf).all() and np.isnan(got[i, :, 90]).all()
        assert np.array_equal(bits(got[i][:, dims]), bits(want[i][:, dims])), i
    v = t.c.view(t.c.download()[1])[0, 0, :, 130 + bad]
    assert (v[:, 3] == -np.inf).all() and np.isnan(v[:, 90]).all()  # the cache holds them as they are
    assert clean.shape == base.shape


def test_first_calls_inside_a_capture(gpu):
    """A process whose first call of each operator is captured: set-up is legal there, and the replay
    gives what eager calls give."""
    import subprocess
    import sys

    code = """
import sys, ctypes
sys.path[:0] = %r
import numpy as np, q3b200 as q3
from cache_reference import *
q3.set_device(0)
rng = np.random.default_rng(5)
c = Cache(rng, 1, 1, 200).upload(q3)
cos, sin = (up(q3, x) for x in rope_tables(q3, 256))
g = up(q3, np.ones(HD, np.float16))
n, zero = 40, up(q3, np.zeros(1, np.int32))
qkv = up(q3, rng.standard_normal((n, 4096)).astype(np.float16))
par = up(q3, (np.arange(n) - 1).astype(np.int32))
lens, new_len, newer = (up(q3, np.array([x])) for x in (100, 0, 0))
acc = up(q3, np.arange(1, n, 2).astype(np.int32)); nacc = up(q3, np.array([20], np.int32))
w, w2 = (up(q3, np.ones((1, 1, 8, 200), np.float32)) for _ in range(2))
sp, sp2 = (up(q3, np.tile(np.arange(200, dtype=np.int32), (1, 1, 8, 1))) for _ in range(2))
blocks = up(q3, q4_blocks(rng, 4096, 256)); many = up(q3, q4_blocks(rng, 20000, 256))
x = up(q3, rng.standard_normal((2, 256)).astype(np.float16))
ys = [q3.DeviceArray((2, m), np.float16) for m in (4096, 20000)]
outs = [q3.DeviceArray((n, 2048), np.float16, zero=True) for _ in range(3)]
def step(st):
    q3.call("q3_gemv_q4", blocks.ptr, x.ptr, ys[0].ptr, 4096, 256, 2, st)
    q3.call("q3_gemv_q4", many.ptr, x.ptr, ys[1].ptr, 20000, 256, 2, st)
    for T, o in ((n, outs[0]), (8, outs[1])):
        q3.call("q3_tree_attention", qkv.ptr, g.ptr, g.ptr, cos.ptr, sin.ptr, 256, c.kv, 0, 1, T, par.ptr, None, lens.ptr, lens.ptr, o.ptr, zero.ptr, st)
    q3.call("q3_tree_commit", c.kv, 0, 1, 1, 20, acc.ptr, nacc.ptr, lens.ptr, new_len.ptr, lens.ptr, w.ptr, sp.ptr, zero.ptr, st)
    q3.call("q3_decode_attention_scored", qkv.ptr, g.ptr, g.ptr, cos.ptr, sin.ptr, 256, c.kv, 0, 1, new_len.ptr, new_len.ptr, w.ptr, w2.ptr, sp.ptr, outs[2].ptr, zero.ptr, st)
    q3.call("q3_cache_evict", c.kv, 0, 1, 1, 64, 8, new_len.ptr, new_len.ptr, w2.ptr, sp.ptr, newer.ptr, w.ptr, sp2.ptr, zero.ptr, st)
st, ex = ctypes.c_void_p(), ctypes.c_void_p()
q3.call("q3_stream_create", ctypes.byref(st))
q3.call("q3_graph_capture_begin", st); step(st); q3.call("q3_graph_capture_end", st, ctypes.byref(ex))
def run(f):
    c.dk.upload(c.k); c.dv.upload(c.v); w.upload(np.ones((1, 1, 8, 200), np.float32))
    f(); q3.call("q3_stream_synchronize", st)
    return [a.download().tobytes() for a in (*ys, *outs, w2, sp2, newer, c.dk, c.dv, zero)]
a = run(lambda: q3.call("q3_graph_launch", ex, st)); b = run(lambda: step(st))
assert a == b and zero.download()[0] == 0 and newer.download()[0] == 64
q3.call("q3_graph_destroy", ex)
print("same")
""" % [p for p in sys.path if p.endswith(("qwen3-iree_b200", "tests"))]
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_tree_attention_beyond_4_gb(gpu):
    """The second sequence's rows lie more than 2^32 bytes (and 2^31 elements) behind the first's."""
    t = Tree(gpu, 12, 3, [70, 90], S=128)
    far = (1 << 31) + 1024
    bufs = [gpu.DeviceArray((far * 2 + 128 * 8 * HD * 2,), np.uint8) for _ in range(2)]
    t.upload()
    per = 128 * 8 * HD
    for buf, x in zip(bufs, (t.c.k, t.c.v)):
        for b in range(2):
            a = np.ascontiguousarray(x[b])
            gpu.call("q3_memcpy_htod", buf.ptr + 2 * far * b, a.ctypes.data, a.nbytes, None)
    gpu.synchronize()
    dk, dv = t.c.dk, t.c.dv
    t.c.kv = gpu.KVCache(bufs[0].ptr, bufs[1].ptr, far, per, 8 * HD, HD, 128, 1, 16, 8)
    t.call()
    for buf, d in zip(bufs, (dk, dv)):
        for b in range(2):
            gpu.call("q3_memcpy_dtod", d.ptr + 2 * per * b, buf.ptr + 2 * far * b, 2 * per, None)
    gpu.synchronize()
    t.check()


def test_tree_attention_is_deterministic_and_captured(gpu):
    """Replays of a captured call follow the lengths on the device and give the eager call's bits."""
    t = Tree(gpu, 13, 9, [300, 45], S=400).upload()
    t.call()
    first = t.check()
    s = ctypes.c_void_p()
    gpu.call("q3_stream_create", ctypes.byref(s))
    gpu.call("q3_graph_capture_begin", s)
    t.call(s)
    ex = ctypes.c_void_p()
    gpu.call("q3_graph_capture_end", s, ctypes.byref(ex))
    for _ in range(3):
        gpu.call("q3_graph_launch", ex, s)
    assert np.array_equal(bits(t.check(s)), bits(first))
    u = Tree(gpu, 14, 9, [120, 390], S=400)
    for n in ("qkv", "lens", "pos", "parents"):
        t.d[n].upload(getattr(u, n))
    u.gq, u.gk, u.cos, u.sin = t.gq, t.gk, t.cos, t.sin
    t.c.dk.upload(u.c.k)
    t.c.dv.upload(u.c.v)
    gpu.call("q3_graph_launch", ex, s)
    u.c.dk, u.c.dv, u.out = t.c.dk, t.c.dv, t.out
    u.check(s)
    gpu.call("q3_graph_destroy", ex)
    gpu.call("q3_stream_destroy", s)


def test_smallest_cache(gpu):
    """One slot, one head, one sequence: the strides of all dimensions but the row's are unused."""
    t = Scored(gpu, 50, [0], S=1, q_heads=1, kv_heads=1)
    t.upload()
    t.c.kv = gpu.KVCache(t.c.dk.ptr, t.c.dv.ptr, 0, 0, 0, 0, 1, 1, 1, 1)
    t.call().check()
    t = Tree(gpu, 51, 1, [0], S=1, q_heads=1, kv_heads=1)
    t.upload()
    t.c.kv = gpu.KVCache(t.c.dk.ptr, t.c.dv.ptr, 0, 0, 0, 0, 1, 1, 1, 1)
    t.call().check()
    c = Cache(np.random.default_rng(1), 1, 1, 1, 1, 1).upload(gpu)
    c.kv = gpu.KVCache(c.dk.ptr, c.dv.ptr, 0, 0, 0, 0, 1, 1, 1, 1)
    new_len, err = commit(gpu, c, 0, 1, np.zeros((1, 1), np.int32), np.array([1], np.int32), np.array([0]))
    assert err == 0 and new_len[0] == 1
    w = np.ones((1, 1, 1, 1), np.float32)
    assert run_evict(gpu, c, 0, 1, w, w.astype(np.int32), np.array([1]), np.array([1]), 1, 0) == 0


def test_two_streams(gpu):
    """Calls on different buffers at the same time."""
    ts = [Tree(gpu, 20 + i, T, [n], S=3000).upload() for i, (T, n) in enumerate([(3, 2900), (64, 2500), (20, 1000)])]
    ss = []
    for _ in ts:
        s = ctypes.c_void_p()
        gpu.call("q3_stream_create", ctypes.byref(s))
        ss.append(s)
    for _ in range(20):
        for t, s in zip(ts, ss):
            t.call(s)
    for t, s in zip(ts, ss):
        t.check(s)
        gpu.call("q3_stream_destroy", s)


# ------------------------------------------------------------------------ commit
def commit(gpu, c, layer0, n_layers, accepted, n, lens, given=(None, None, None)):
    d = [up(gpu, x) for x in (accepted, n, lens)]
    new_len, err = up(gpu, np.full(c.B, -7, np.int64)), up(gpu, np.zeros(1, np.int32))
    gpu.call("q3_tree_commit", c.kv, layer0, n_layers, c.B, accepted.shape[1], d[0].ptr, d[1].ptr, d[2].ptr, new_len.ptr,
             *(x and x.ptr for x in given), err.ptr, None)
    return new_len.download(), err.download()[0]


@pytest.mark.parametrize("layout", ["flat", "head", "padded"])
def test_tree_commit(gpu, layout):
    rng = np.random.default_rng(1)
    c = Cache(rng, 5, 3, 90, layout=layout).upload(gpu)
    acc = np.zeros((5, 40), np.int32)
    n = np.array([40, 1, 0, 7, 12], np.int32)
    lens = np.array([26, 0, 80, 83, 50], np.int64)
    acc[0] = np.sort(rng.choice(64, 40, replace=False))
    acc[1, 0] = 63
    acc[3, :7] = np.arange(7)                      # nothing moves
    acc[4, :12] = [0, 1, 2, 5, 6, 7, 9, 11, 12, 20, 38, 39]
    shape = (5, 3, 8, 90)
    pos = lens + 9
    w, sp = rng.standard_normal(shape).astype(np.float32), rng.integers(0, 99, shape).astype(np.int32)
    given = [up(gpu, x) for x in (pos, w, sp)]
    new_len, err = commit(gpu, c, 1, 2, acc, n, lens, given)
    for b in range(5):
        w[b, 1:, :, lens[b]:lens[b] + n[b]] = 0
        sp[b, 1:, :, lens[b]:lens[b] + n[b]] = pos[b] + np.arange(n[b])
    assert np.array_equal(given[1].download(), w) and np.array_equal(given[2].download(), sp)
    assert err == 0 and np.array_equal(new_len, lens + n)
    k, v = c.download()
    for x, got in ((c.k, k), (c.v, v)):
        w = x.copy()
        for b in range(5):
            src = lens[b] + acc[b, :n[b]]
            c.view(w)[b, 1:, :, lens[b]:lens[b] + n[b]] = c.view(x)[b, 1:, :, src].transpose(1, 2, 0, 3)
        assert np.array_equal(bits(got), bits(w))


def test_tree_commit_bad_values(gpu):
    rng = np.random.default_rng(2)
    c = Cache(rng, 7, 2, 90).upload(gpu)
    acc = np.tile(np.array([1, 3, 5], np.int32), (7, 1))
    n = np.array([3, 4, -1, 3, 3, 3, 3], np.int32)
    lens = np.array([10, 10, 10, -1, 85, 10, 10], np.int64)
    acc[5], acc[6] = [1, 1, 2], [-1, 3, 5]
    new_len, err = commit(gpu, c, 0, 2, acc, n, lens)
    assert err == BAD_TREE and np.array_equal(new_len, [13, *lens[1:]])
    w = c.k.copy()
    c.view(w)[0, :, :, 10:13] = c.view(c.k)[0, :, :, [11, 13, 15]].transpose(1, 2, 0, 3)
    assert np.array_equal(bits(c.download()[0]), bits(w))


@pytest.mark.parametrize("pos", [-1, 1 << 31])
def test_tree_commit_bad_position(gpu, pos):
    c = Cache(np.random.default_rng(3), 1, 1, 90).upload(gpu)
    w, sp = np.ones((1, 1, 8, 90), np.float32), np.full((1, 1, 8, 90), 5, np.int32)
    given = [up(gpu, x) for x in (np.array([pos]), w, sp)]
    new_len, err = commit(gpu, c, 0, 1, np.array([[1, 2]], np.int32), np.array([2], np.int32), np.array([10]), given)
    assert err == BAD_TREE and new_len[0] == 10
    assert np.array_equal(given[1].download(), w) and np.array_equal(given[2].download(), sp)
    assert np.array_equal(bits(c.download()[0]), bits(c.k))


# ------------------------------------------------------------------------ scored
class Scored(Tree):
    def __init__(self, gpu, seed, lens, **kw):
        super().__init__(gpu, seed, 1, [max(n, 0) for n in lens], **kw)
        self.lens = np.array(lens, np.int64)
        self.parents[:] = -1
        shape = (self.B, self.c.layers, self.c.nkv, self.c.S)
        self.weight = np.exp(self.rng.standard_normal(shape)).astype(np.float32)
        self.slot_pos = self.rng.integers(0, 1000, shape).astype(np.int32)

    def upload(self, in_place=False):
        super().upload()
        g = self.gpu
        self.dw, self.dsp = up(g, self.weight), up(g, self.slot_pos)
        self.dn = self.dw if in_place else up(g, np.full_like(self.weight, -3))
        return self

    def call(self, stream=None):
        d = self.d
        self.gpu.call("q3_decode_attention_scored", d["qkv"].ptr, d["gq"].ptr, d["gk"].ptr, d["cos"].ptr, d["sin"].ptr,
                      self.cos.shape[0], self.c.kv, self.layer, self.B, d["lens"].ptr, d["pos"].ptr, self.dw.ptr, self.dn.ptr,
                      self.dsp.ptr, self.out.ptr, self.err.ptr, stream)
        return self

    def check(self, stream=None, skip=()):
        skip = (*skip, *np.flatnonzero(self.lens == -1))
        super().check(stream, skip)
        got, sp = self.dn.download(stream), self.dsp.download(stream)
        want = self.weight.astype(np.float64) if self.dn is self.dw else np.full(got.shape, -3.0)
        tol, wsp = np.zeros(got.shape), self.slot_pos.copy()
        for b in set(range(self.B)) - set(skip):
            m = int(self.lens[b])
            _, _, _, _, w, wt = attend(self.c, self.c.view(self.c.k), self.c.view(self.c.v), self.layer, b, m,
                                       int(self.pos[b]), [-1], self.qkv[b], self.gq, self.gk, self.cos, self.sin)
            old = self.weight[b, self.layer, :, :m].astype(np.float64)
            want[b, self.layer, :, :m] = old + w[:, :m]
            want[b, self.layer, :, m] = w[:, m]
            # a rounding to f32 after each head of the group
            tol[b, self.layer, :, :m + 1] = wt + 8 * 2.0 ** -24 * np.abs(want[b, self.layer, :, :m + 1])
            wsp[b, self.layer, :, m] = self.pos[b]
        assert (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-30))
        assert np.array_equal(sp, wsp)


@pytest.mark.parametrize("length", [0, 1, 15, 16, 63, 64, 65, 500, 1024, 4095])
@pytest.mark.parametrize("in_place", [False, True])
def test_scored(gpu, length, in_place):
    Scored(gpu, length, [length], gap=5).upload(in_place).call().check()


@pytest.mark.parametrize("layout", ["flat", "head", "padded"])
def test_scored_batch(gpu, layout):
    t = Scored(gpu, 2, [130, -1, 700, 64, 0, 257], layers=3, layer=2, layout=layout, gap=11)
    t.upload().call().check()
    assert t.err.download()[0] == 0


@pytest.mark.parametrize("q_heads,kv_heads", [(8, 8), (1, 1), (32, 8), (64, 8), (6, 3)])
def test_scored_heads(gpu, q_heads, kv_heads):
    Scored(gpu, q_heads, [200, 77], q_heads=q_heads, kv_heads=kv_heads).upload().call().check()


def test_scored_long(gpu):
    """Long enough that a CTA's scores take most of the shared memory."""
    Scored(gpu, 7, [130003], q_heads=2, kv_heads=1, gap=2).upload().call().check()


def test_scored_many_sequences_of_a_long_cache(gpu):
    """Many sequences would take few CTAs each; the scores ask for more."""
    Scored(gpu, 8, [5, 20000, *[40] * 40], q_heads=8, kv_heads=1, S=20100).upload().call().check()


def test_scored_bad_values(gpu):
    t = Scored(gpu, 9, [30, 40, 50, 20], S=51)
    t.lens[1], t.pos[2], t.lens[3] = 51, t.cos.shape[0], -2
    t.upload().call().check(skip=(1, 2, 3))
    assert t.err.download()[0] == BAD_POS


# ---------------------------------------------------------------------- eviction
def run_evict(gpu, c, layer0, n_layers, weight, slot_pos, lens, pos, budget, recent):
    """Calls and checks bit for bit."""
    d = [up(gpu, x) for x in (lens, pos, weight, slot_pos)]
    new_len, err = up(gpu, np.full(c.B, -7, np.int64)), up(gpu, np.zeros(1, np.int32))
    nw, nsp = up(gpu, np.full_like(weight, -3)), up(gpu, np.full_like(slot_pos, -3))
    gpu.call("q3_cache_evict", c.kv, layer0, n_layers, c.B, budget, recent, *(x.ptr for x in d), new_len.ptr, nw.ptr, nsp.ptr,
             err.ptr, None)
    wk, wv, ww, wsp = c.k.copy(), c.v.copy(), np.full_like(weight, -3), np.full_like(slot_pos, -3)
    want_len = lens.copy()
    for b in range(c.B):
        if not 0 <= lens[b] <= c.S:
            continue
        want_len[b] = min(lens[b], budget)
        for l in range(layer0, layer0 + n_layers):
            for h in range(c.nkv):
                w, sp = evict(c.view(wk)[b, l, h], c.view(wv)[b, l, h], weight[b, l, h], slot_pos[b, l, h], int(lens[b]),
                              int(pos[b]), budget, recent)
                ww[b, l, h, :len(w)], wsp[b, l, h, :len(w)] = w, sp
    k, v = c.download()
    assert np.array_equal(new_len.download(), want_len)
    assert np.array_equal(nw.download().view(np.uint32), ww.view(np.uint32)) and np.array_equal(nsp.download(), wsp)
    assert np.array_equal(bits(k), bits(wk)) and np.array_equal(bits(v), bits(wv))
    return err.download()[0]


def evict_inputs(rng, c, kind="plain"):
    shape = (c.B, c.layers, c.nkv, c.S)
    w = np.exp(1.5 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = np.round(w)
    elif kind == "equal":
        w[...] = 0.25
    elif kind == "odd":
        w = rng.choice(np.array([0.0, -0.0, np.nan, np.inf, -np.inf, -1.5, 1e-40, 3.0], np.float32), shape)
    sp = np.argsort(rng.random(shape), -1).astype(np.int32)
    return w, sp


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "odd"])
@pytest.mark.parametrize("S,budget,recent", [(2, 1, 0), (2, 1, 1), (33, 32, 3), (64, 31, 31), (100, 1, 0), (700, 512, 64),
                                             (1024, 1023, 5), (3000, 700, 0), (3000, 2100, 2100)])
def test_evict(gpu, kind, S, budget, recent):
    rng = np.random.default_rng(S + budget)
    c = Cache(rng, 1, 1, S, 4, 2).upload(gpu)
    w, sp = evict_inputs(rng, c, kind)
    assert run_evict(gpu, c, 0, 1, w, sp, np.array([S]), np.array([S]), budget, recent) == 0


@pytest.mark.parametrize("layout", ["flat", "head", "padded"])
def test_evict_batch(gpu, layout):
    rng = np.random.default_rng(3)
    c = Cache(rng, 6, 4, 300, 4, 2, layout=layout).upload(gpu)
    w, sp = evict_inputs(rng, c, "ties")
    lens = np.array([300, 0, 129, 128, 127, 201])
    assert run_evict(gpu, c, 1, 2, w, sp, lens, lens + 4, 128, 16) == 0


def test_evict_more_newest_than_budget(gpu):
    """Repeated positions: more slots count as newest than may stay; the lower slots do."""
    rng = np.random.default_rng(4)
    c = Cache(rng, 2, 1, 200, 2, 1).upload(gpu)
    w, sp = evict_inputs(rng, c)
    sp[:] = 7
    run_evict(gpu, c, 0, 1, w, sp, np.array([200, 150]), np.array([8, 8]), 60, 1)


@pytest.mark.parametrize("S", [32768, 32769, 70001])
def test_evict_long(gpu, S):
    """On both sides of where the keys still fit on chip."""
    rng = np.random.default_rng(S)
    c = Cache(rng, 1, 1, S, 2, 1).upload(gpu)
    w, sp = evict_inputs(rng, c, "ties")
    run_evict(gpu, c, 0, 1, w, sp, np.array([S - 3]), np.array([S]), S // 2, 1000)


def test_evict_all_layers_of_many(gpu):
    """More (sequence, layer, head) than there are CTAs at once."""
    rng = np.random.default_rng(6)
    c = Cache(rng, 20, 28, 40, 16, 8, layout="head").upload(gpu)
    w, sp = evict_inputs(rng, c)
    lens = rng.integers(0, 41, 20)
    run_evict(gpu, c, 0, 28, w, sp, lens, np.full(20, 40), 25, 6)


def test_evict_bad_values(gpu):
    rng = np.random.default_rng(7)
    c = Cache(rng, 3, 1, 50, 2, 1).upload(gpu)
    w, sp = evict_inputs(rng, c)
    assert run_evict(gpu, c, 0, 1, w, sp, np.array([50, 51, -1]), np.array([50, 50, 50]), 20, 5) == BAD_POS


# -------------------------------------------------------------- a run of them all
def test_draft_verify_commit_evict(gpu):
    """Three rounds as a server runs them: the draft's 4-bit projections of a tree, verification, the
    accepted path, one scored step, and an eviction once the cache is over its budget; the whole
    state against the plain forms after every step, captured as one graph the last time."""
    rng = np.random.default_rng(40)
    T, S, B, budget, recent, K = 6, 96, 2, 64, 16, 1024
    c = Cache(rng, B, 1, S)
    c.upload(gpu)
    cos, sin = rope_tables(gpu, 512)
    gq, gk = ((1 + 0.1 * rng.standard_normal(HD)).astype(np.float16) for _ in range(2))
    blocks = q4_blocks(rng, 4096, K)
    lens, pos = np.array([60, 75], np.int64), np.array([60, 90], np.int64)
    weight = np.zeros((B, 1, 8, S), np.float32)
    sp = np.tile(np.arange(S, dtype=np.int32), (B, 1, 8, 1))
    d = {n: up(gpu, a) for n, a in dict(w=blocks, cos=cos, sin=sin, gq=gq, gk=gk, lens=lens, pos=pos, weight=weight, sp=sp).items()}
    x = gpu.DeviceArray((B * T, K), np.float16)
    qkv = gpu.DeviceArray((B, T, 4096), np.float16)
    one = gpu.DeviceArray((B, 1, 4096), np.float16)
    out, out1 = gpu.DeviceArray((B, T, 2048), np.float16), gpu.DeviceArray((B, 1, 2048), np.float16)
    par, acc, nacc = (gpu.DeviceArray(s, np.int32) for s in ((B, T), (B, 3), (B,)))
    len2, len3 = gpu.DeviceArray((B,), np.int64), gpu.DeviceArray((B,), np.int64)
    pos2, pos3 = gpu.DeviceArray((B,), np.int64), gpu.DeviceArray((B,), np.int64)
    nw, nsp = up(gpu, weight), up(gpu, sp)
    err = up(gpu, np.zeros(1, np.int32))
    st = ctypes.c_void_p()
    gpu.call("q3_stream_create", ctypes.byref(st))
    n1 = np.array([3, 2], np.int64)

    def heads(q):
        return (q, d["gq"].ptr, d["gk"].ptr, d["cos"].ptr, d["sin"].ptr, 512, c.kv, 0, B)

    def device_step():
        gpu.call("q3_gemv_q4", d["w"].ptr, x.ptr, qkv.ptr, 4096, K, B * T, st)
        gpu.call("q3_tree_attention", *heads(qkv.ptr), T, par.ptr, None, d["lens"].ptr, d["pos"].ptr, out.ptr, err.ptr, st)
        gpu.call("q3_tree_commit", c.kv, 0, 1, B, 3, acc.ptr, nacc.ptr, d["lens"].ptr, len2.ptr, d["pos"].ptr,
                 d["weight"].ptr, d["sp"].ptr, err.ptr, st)
        gpu.call("q3_decode_attention_scored", *heads(one.ptr), len2.ptr, pos2.ptr, d["weight"].ptr, d["weight"].ptr,
                 d["sp"].ptr, out1.ptr, err.ptr, st)
        gpu.call("q3_cache_evict", c.kv, 0, 1, B, budget, recent, len3.ptr, pos3.ptr, d["weight"].ptr, d["sp"].ptr, d["lens"].ptr,
                 nw.ptr, nsp.ptr, err.ptr, st)
        gpu.call("q3_memcpy_dtod", d["weight"].ptr, nw.ptr, nw.nbytes, st)
        gpu.call("q3_memcpy_dtod", d["sp"].ptr, nsp.ptr, nsp.nbytes, st)

    ex = None
    for step in range(3):
        hx = rng.standard_normal((B * T, K)).astype(np.float16)
        hp = np.stack([random_tree(rng, T, "mixed") for _ in range(B)]).astype(np.int32)
        ha = np.array([[0, 2, 5], [1, 4, 0]], np.int32)
        hone = rng.standard_normal((B, 1, 4096)).astype(np.float16)
        for dev, host in ((x, hx), (par, hp), (acc, ha), (nacc, n1.astype(np.int32)), (one, hone), (pos2, pos + n1),
                          (pos3, pos + n1 + 1), (len3, lens + n1 + 1)):
            dev.upload(host)
        if step == 2:
            gpu.call("q3_graph_capture_begin", st)
            device_step()
            ex = ctypes.c_void_p()
            gpu.call("q3_graph_capture_end", st, ctypes.byref(ex))
            gpu.call("q3_graph_launch", ex, st)
        else:
            device_step()
        gpu.call("q3_stream_synchronize", st)
        assert err.download()[0] == 0
        y, tol = gemv_tolerance(blocks, hx)
        hq = qkv.download()
        assert (np.abs(hq.reshape(B * T, -1) - y) <= tol).all()
        k, v = c.view(c.k), c.view(c.v)
        for b in range(B):
            m, n = int(lens[b]), int(n1[b])
            o, tol, kn, vn, _, _ = attend(c, k, v, 0, b, m, int(pos[b]), hp[b].tolist(), hq[b], gq, gk, cos, sin)
            assert (np.abs(out.download()[b] - o) <= tol).all()
            for dst, rows in ((k, kn), (v, vn)):
                dst[b, 0, :, m:m + T] = rows.swapaxes(0, 1)
                dst[b, 0, :, m:m + n] = rows[ha[b, :n]].swapaxes(0, 1)
            sp[b, 0, :, m:m + n] = pos[b] + np.arange(n)
            weight[b, 0, :, m:m + n] = 0
            m += n
            o, tol, kn, vn, w, wt = attend(c, k, v, 0, b, m, int(pos[b]) + n, [-1], hone[b], gq, gk, cos, sin)
            assert (np.abs(out1.download()[b] - o) <= tol).all()
            k[b, 0, :, m], v[b, 0, :, m] = kn[0], vn[0]
            sp[b, 0, :, m] = pos[b] + n
            weight[b, 0, :, :m] += w[:, :m]
            weight[b, 0, :, m] = w[:, m]
            for h in range(8):
                kept = evict(k[b, 0, h], v[b, 0, h], weight[b, 0, h], sp[b, 0, h], m + 1, int(pos[b]) + n + 1, budget, recent)
                weight[b, 0, h, :len(kept[0])], sp[b, 0, h, :len(kept[1])] = kept
            lens[b], pos[b] = min(m + 1, budget), pos[b] + n + 1
            live = int(lens[b])
            gw = d["weight"].download()
            assert np.allclose(gw[b, 0, :, :live], weight[b, 0, :, :live], rtol=2e-5, atol=1e-7)
            assert np.array_equal(d["sp"].download()[b, 0, :, :live], sp[b, 0, :, :live])
            weight[b] = gw[b]
        gk_, gv_ = (c.view(z) for z in c.download())
        for b in range(B):
            assert np.array_equal(bits(gk_[b, 0, :, :lens[b]]), bits(k[b, 0, :, :lens[b]]))
            assert np.array_equal(bits(gv_[b, 0, :, :lens[b]]), bits(v[b, 0, :, :lens[b]]))
        assert np.array_equal(d["lens"].download(), lens)
        d["pos"].upload(pos)
    gpu.call("q3_graph_destroy", ex)
    gpu.call("q3_stream_destroy", st)


@pytest.mark.parametrize("op", ["q4", "tree", "scored", "evict"])
def test_benchmark_command(gpu, op, capsys):
    from q3b200.benchmark import main

    assert main(["--cache-op", op, "--batch", "2", "--context", "0", "500", "--tokens", "6", "--reps", "2"]) == 0
    assert op in capsys.readouterr().out
