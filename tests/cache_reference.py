"""Plain 64-bit numpy forms of the drafted-token operators, for the tests."""
import ctypes

import numpy as np

HD = 128
EPS = np.float32(9.99999997e-7)


# ------------------------------------------------------------------ Q4_0
def q4_blocks(rng, N, K, d_scale=0.005):
    """Random Q4_0 bytes [N][K/32][18] with every nibble value."""
    q = rng.integers(0, 16, (N, K // 32, 32), dtype=np.uint8)
    d = (d_scale * (1 + 0.3 * rng.standard_normal((N, K // 32, 1)))).astype(np.float16)
    return np.concatenate([d.view(np.uint8), q[..., :16] | (q[..., 16:] << 4)], -1)


def q4_dequant(blocks):
    """[N][K/32][18] -> float64 [N][K]."""
    d = np.ascontiguousarray(blocks[..., :2]).view(np.float16).astype(np.float64)
    q = np.concatenate([blocks[..., 2:] & 15, blocks[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (d * q).reshape(blocks.shape[0], -1)


# ----------------------------------------------------------------- heads
def norm_rope(x, gamma, cos, sin):
    """f16 head vectors [..., 128] -> roped f16, with the operations, order and
    roundings of the one-token engines (f32; lane l holds dims l + 32 i; the
    sum of squares is a chain per lane, then a butterfly over lanes)."""
    x = x.astype(np.float32)
    v = x.reshape(*x.shape[:-1], 4, 32)
    ss = np.zeros(v.shape[:-2] + (32,), np.float32)
    for i in range(4):  # an f32 fma: the square is exact in f64
        ss = (v[..., i, :].astype(np.float64) ** 2 + ss).astype(np.float32)
    lane = np.arange(32)
    for off in (16, 8, 4, 2, 1):
        ss = ss + ss[..., lane ^ off]
    r = np.sqrt(ss[..., :1] / np.float32(128) + EPS)
    n = ((x / r) * gamma.astype(np.float32)).astype(np.float16).astype(np.float32)
    a, b = n[..., :64], n[..., 64:]
    return np.concatenate([a * cos - b * sin, a * sin + b * cos], -1).astype(np.float16)


def paths(parents):
    """Ancestors and self of each token."""
    out = []
    for t, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [t])
    return out


class Cache:
    """A host cache in a flat, head-major or padded layout, with what the library is told of it."""

    def __init__(self, rng, B, layers, S, q_heads=16, kv_heads=8, layout="flat", fill=None):
        self.B, self.layers, self.S, self.nq, self.nkv = B, layers, S, q_heads, kv_heads
        H = kv_heads
        pad = 16 if layout == "padded" else 0
        if layout == "head":
            shape, order = (B, layers, H, S, HD), (0, 1, 3, 2)
        else:
            shape, order = (B, layers, S, H, HD + pad), (0, 1, 2, 3)
        self.k = rng.standard_normal(shape).astype(np.float16)
        self.v = rng.standard_normal(shape).astype(np.float16)
        if fill is not None:
            self.k[...] = fill
            self.v[...] = fill
        el = [s // 2 for s in self.k.strides]
        self.strides = tuple(el[i] for i in (order.index(0), order.index(1), order.index(2), order.index(3)))
        if layout == "head":
            self.strides = (el[0], el[1], el[3], el[2])

    def view(self, x):
        """[B, layers, kv_heads, S, 128] of self.k, self.v or a downloaded copy."""
        if x.shape[2:4] == (self.nkv, self.S) and x.strides[2] > x.strides[3] and self.strides[2] == HD:
            return x[..., :HD]
        return np.swapaxes(x, 2, 3)[..., :HD]

    def upload(self, q3):
        self.dk, self.dv = q3.DeviceArray.from_host(self.k), q3.DeviceArray.from_host(self.v)
        self.kv = q3.KVCache(self.dk.ptr, self.dv.ptr, *self.strides, self.S, self.layers, self.nq, self.nkv)
        return self

    def download(self):
        return self.dk.download(), self.dv.download()


def attend(c, k, v, layer, b, length, pos, parents, qkv, gq, gk, cos, sin):
    """One sequence's drafted tokens (qkv [n, (nq + 2 nkv) * 128] f16) over views
    k, v [B, layers, nkv, S, 128] (f16).  Returns float64 out [n, nq * 128], its
    tolerance, K rows, V rows [n, nkv, 128] f16 and slot weights [nkv, length + n]
    with their tolerance."""
    n, G = len(parents), c.nq // c.nkv
    pth = paths(parents)
    at = [pos + len(p) - 1 for p in pth]
    cs, sn = cos[at][:, None], sin[at][:, None]
    x = qkv.reshape(n, c.nq + 2 * c.nkv, HD)
    q = norm_rope(x[:, :c.nq], gq, cs, sn)
    kn = norm_rope(x[:, c.nq:c.nq + c.nkv], gk, cs, sn)
    vn = x[:, c.nq + c.nkv:]
    see = np.zeros((n, length + n), bool)
    see[:, :length] = True
    for t, p in enumerate(pth):
        see[t, [length + a for a in p]] = True
    out, tol = np.zeros((n, c.nq, HD)), np.zeros((n, c.nq, HD))
    w, wtol = np.zeros((c.nkv, length + n)), np.zeros((c.nkv, length + n))
    for h in range(c.nkv):
        keys = np.concatenate([k[b, layer, h, :length], kn[:, h]]).astype(np.float64)
        vals = np.concatenate([v[b, layer, h, :length], vn[:, h]]).astype(np.float64)
        for j in range(G):
            qq = q[:, h * G + j].astype(np.float64)
            s = np.where(see, qq @ keys.T / np.sqrt(HD), -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            # a score: 128 exact products summed in f32 (each step off by at most 2^-23 of the
            # running sum of magnitudes, the tensor core may truncate), then scaled
            es = 130 * 2.0 ** -23 * np.where(see, np.abs(qq) @ np.abs(keys).T, 0).max(-1, keepdims=True) / np.sqrt(HD)
            # exp2 and the rescalings: 2^-22 each, a handful of them; sums over n keys in f32
            ee = 2 * es + 2.0 ** -18 + (length + n) ** 0.5 * 2.0 ** -23
            out[:, h * G + j] = p @ vals
            # weights go to the MMA as f16 (half a step: 2^-11), the result is rounded to f16
            tol[:, h * G + j] = (2.0 ** -11 + ee) * (p @ np.abs(vals)) + 2.0 ** -11 * np.abs(out[:, h * G + j]) + 2.0 ** -24
            w[h] += p.sum(0)
            wtol[h] += (ee * p).sum(0)
    return out.reshape(n, -1), tol.reshape(n, -1), kn, vn, w, wtol


def evict(k, v, w, sp, length, pos, budget, recent):
    """One head's cache rows [S, 128], weights and positions; in place for k and v.
    Returns (weights, positions) of the slots that stay."""
    w, sp = w[:length].copy(), sp[:length].copy()
    if length <= budget:
        return w, sp
    rank = np.where(np.isnan(w), -np.inf, w.astype(np.float64))
    group = np.where(np.isnan(w), 2, 1)           # a NaN counts least, below -inf
    group[sp.astype(np.int64) >= pos - recent] = 0
    rank[group == 0] = 0
    kept = sorted(range(length), key=lambda i: (group[i], -rank[i], i))[:budget]
    stay = np.zeros(length, bool)
    stay[kept] = True
    dst, src = np.flatnonzero(~stay[:budget]), budget + np.flatnonzero(stay[budget:])
    for x in (k, v, w, sp):
        x[dst] = x[src]
    return w[:budget], sp[:budget]


def rope_tables(q3, rows):
    c, s = np.empty((rows, 64), np.float32), np.empty((rows, 64), np.float32)
    assert q3.lib().q3_rope_table(rows, c.ctypes.data, s.ctypes.data) == 0
    return c, s


def up(q3, a):
    return q3.DeviceArray.from_host(np.ascontiguousarray(a))


def host_buffer(n):
    """A 16-byte aligned host address, to stand in for a device pointer in refusals."""
    buf = ctypes.create_string_buffer(n + 16)
    return buf, (ctypes.addressof(buf) + 15) & ~15
