"""Drafted-token operators without a GPU: the Q4_0 quantizer, and that every
argument the entry points refuse is a status before anything is launched."""
import numpy as np
import pytest
from cache_reference import HD, host_buffer, q4_dequant

INVALID, UNSUPPORTED = 1, 6


def quantize(q3, w):
    w = np.ascontiguousarray(w, np.float32)
    out = np.empty(w.size // 32 * 18, np.uint8)
    assert q3.lib().q3_quantize_q4_0(w.ctypes.data, w.size, out.ctypes.data) == 0
    return out.reshape(w.shape[0], -1, 18)


def test_quantizer_is_within_half_a_step(q3):
    rng = np.random.default_rng(0)
    w = (rng.standard_normal((7, 256)) * 0.02).astype(np.float32)
    blocks = quantize(q3, w)
    d = np.abs(np.ascontiguousarray(blocks[..., :2]).view(np.float16).astype(np.float64))
    err = np.abs(q4_dequant(blocks) - w).reshape(7, -1, 32)
    # half a step inside the range; d is rounded to f16 (8 steps of it, half a unit each), and +8
    # steps are not held: the side opposite to the largest value ends at 7
    top = np.abs(w.reshape(7, -1, 32)).max(-1, keepdims=True)
    assert (err <= d / 2 + 8 * d * 2.0 ** -11 + (np.abs(w.reshape(7, -1, 32)) > 7 * d) * d).all()
    assert (err[np.abs(w.reshape(7, -1, 32)) == top] <= (top * 2.0 ** -11 + 1e-12)[..., 0].ravel()).all()


def test_quantizer_zero_and_signs(q3):
    w = np.zeros((3, 32), np.float32)
    w[1, 5], w[2, 20] = 0.8, -0.8
    y = q4_dequant(quantize(q3, w))
    assert not y[0].any()
    assert np.allclose(y[1:], w[1:], rtol=2.0 ** -11, atol=0)


def test_quantizer_refusals(q3):
    buf, p = host_buffer(64)
    assert q3.lib().q3_quantize_q4_0(p, 33, p) == INVALID
    assert q3.lib().q3_quantize_q4_0(None, 32, p) == INVALID


@pytest.mark.parametrize("change", [{"w": 0}, {"x": 0}, {"y": 0}, {"w": 8}, {"x": 2}, {"y": 1}, {"N": 0}, {"N": -4},
                                    {"K": 0}, {"K": 128}, {"K": 300}, {"K": 16640}, {"R": 0}, {"R": 17}])
def test_gemv_q4_refusals(q3, change):
    buf, p = host_buffer(64)
    a = {"w": 0, "x": 0, "y": 0, "N": 16, "K": 256, "R": 1}
    ptr = {n: p for n in "wxy"}
    for n, v in change.items():
        if n in ptr:
            ptr[n] = p + v if v else None
        else:
            a[n] = v
    assert q3.lib().q3_gemv_q4(ptr["w"], ptr["x"], ptr["y"], a["N"], a["K"], a["R"], None) == INVALID


class Call:
    """A call that would be accepted, on host addresses; `with_` changes one thing."""

    def __init__(self, q3):
        self.q3 = q3
        self.buf, self.p = host_buffer(1 << 16)
        self.kv = dict(k=self.p, v=self.p + 4096, seq_stride=0, layer_stride=64 * 8 * HD, slot_stride=8 * HD,
                       head_stride=HD, slots=64, layers=2, q_heads=16, kv_heads=8)
        self.kv["seq_stride"] = 2 * self.kv["layer_stride"]
        self.a = dict(layer=0, n_layers=2, B=2, T=4, A=4, rope_rows=64, budget=32, recent=4, qkv=self.p, q_norm=self.p,
                      k_norm=self.p, cos=self.p, sin=self.p, parents=self.p, n=self.p, len=self.p, pos=self.p,
                      weight=self.p, new_weight=self.p + 16384, slot_pos=self.p, new_slot_pos=self.p + 16384,
                      out=self.p, accepted=self.p, new_len=self.p + 64, err=None)

    def with_(self, **change):
        for k, v in change.items():
            (self.kv if k in self.kv and k != "layer" else self.a)[k] = v
        return self

    def cache(self):
        return self.q3.KVCache(*(self.kv[n] for n, _ in self.q3.KVCache._fields_))

    def tree(self):
        a = self.a
        return self.q3.lib().q3_tree_attention(a["qkv"], a["q_norm"], a["k_norm"], a["cos"], a["sin"], a["rope_rows"],
                                               self.cache(), a["layer"], a["B"], a["T"], a["parents"], a["n"], a["len"],
                                               a["pos"], a["out"], a["err"], None)

    def scored(self):
        a = self.a
        return self.q3.lib().q3_decode_attention_scored(
            a["qkv"], a["q_norm"], a["k_norm"], a["cos"], a["sin"], a["rope_rows"], self.cache(), a["layer"], a["B"],
            a["len"], a["pos"], a["weight"], a["new_weight"], a["slot_pos"], a["out"], a["err"], None)

    def commit(self):
        a = self.a
        return self.q3.lib().q3_tree_commit(self.cache(), a["layer"], a["n_layers"], a["B"], a["A"], a["accepted"],
                                            a["n"], a["len"], a["new_len"], a["pos"], a["weight"], a["slot_pos"],
                                            a["err"], None)

    def evict(self):
        a = self.a
        return self.q3.lib().q3_cache_evict(self.cache(), a["layer"], a["n_layers"], a["B"], a["budget"], a["recent"],
                                            a["len"], a["pos"], a["weight"], a["slot_pos"], a["new_len"],
                                            a["new_weight"], a["new_slot_pos"], a["err"], None)


OPS = ["tree", "scored", "commit", "evict"]
CACHE = [{"k": None}, {"v": None}, {"slots": 0}, {"slots": 1 << 31}, {"layers": 0}, {"layer": -1}, {"layer": 2},
         {"kv_heads": 0}, {"q_heads": 0}, {"q_heads": 12}, {"q_heads": 24}, {"q_heads": 128}, {"slot_stride": 0},
         {"slot_stride": 8 * HD - 8}, {"head_stride": 64}, {"head_stride": HD + 4}, {"seq_stride": 64 * 8 * HD},
         {"layer_stride": 64 * 8 * HD - 8}, {"seq_stride": 0}, {"seq_stride": -8}, {"seq_stride": 1 << 62}, {"B": 0}, {"B": 65536}]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("change", CACHE, ids=str)
def test_cache_refusals(q3, op, change):
    assert getattr(Call(q3).with_(**change), op)() == INVALID


@pytest.mark.parametrize("op", OPS)
def test_misaligned_cache(q3, op):
    c = Call(q3)
    assert getattr(c.with_(k=c.p + 8), op)() == INVALID


@pytest.mark.parametrize("op,change", [
    *(("tree", {n: None}) for n in ("qkv", "q_norm", "k_norm", "cos", "sin", "parents", "len", "pos", "out")),
    ("tree", {"T": 0}), ("tree", {"T": 65}), ("tree", {"T": 33, "q_heads": 32}), ("tree", {"T": 17, "q_heads": 64}),
    ("tree", {"rope_rows": 0}),
    *(("scored", {n: None}) for n in ("qkv", "q_norm", "k_norm", "cos", "sin", "len", "pos", "weight", "new_weight",
                                      "slot_pos", "out")),
    ("scored", {"rope_rows": 1 << 31}),
    *(("commit", {n: None}) for n in ("accepted", "n", "len", "new_len", "pos", "weight", "slot_pos")),
    ("commit", {"A": 0}), ("commit", {"A": 65}), ("commit", {"n_layers": 0}), ("commit", {"n_layers": 3}),
    *(("evict", {n: None}) for n in ("len", "pos", "weight", "slot_pos", "new_len", "new_weight", "new_slot_pos")),
    ("evict", {"budget": 0}), ("evict", {"budget": 65}), ("evict", {"recent": -1}), ("evict", {"recent": 33}),
    ("evict", {"n_layers": 3}),
], ids=str)
def test_argument_refusals(q3, op, change):
    assert getattr(Call(q3).with_(**change), op)() == INVALID


ALIGNED = {"tree": {2: ("q_norm", "k_norm"), 4: ("cos", "sin", "parents", "n", "err"), 8: ("qkv", "out", "len", "pos")},
           "scored": {2: ("q_norm", "k_norm"), 4: ("cos", "sin", "weight", "new_weight", "slot_pos", "err"),
                      8: ("qkv", "out", "len", "pos")},
           "commit": {4: ("accepted", "n", "weight", "slot_pos", "err"), 8: ("len", "new_len", "pos")},
           "evict": {4: ("weight", "slot_pos", "new_weight", "new_slot_pos", "err"), 8: ("len", "new_len", "pos")}}


@pytest.mark.parametrize("op,name,size", [(op, n, s) for op, a in ALIGNED.items() for s, ns in a.items() for n in ns])
def test_misaligned_arrays(q3, op, name, size):
    c = Call(q3)
    c.a[name] = (c.a[name] or c.p + 32768) + size // 2
    assert getattr(c, op)() == INVALID
    assert b"aligned" in q3.lib().q3_last_error()


def test_overlapping_arrays(q3):
    c = Call(q3)
    assert c.with_(new_len=c.p + 8).commit() == INVALID
    c = Call(q3)
    assert c.with_(new_weight=c.p).evict() == INVALID
    c = Call(q3)
    assert c.with_(new_slot_pos=c.p + 4).evict() == INVALID
    c = Call(q3)
    assert c.with_(new_weight=c.p + 4).scored() == INVALID     # neither the same array nor apart
    c = Call(q3)
    assert c.with_(qkv=c.p + 4).tree() == INVALID
    c = Call(q3)
    assert c.with_(out=c.p + 4).scored() == INVALID


def test_sizes_that_are_not_covered(q3):
    big = dict(slots=1 << 20, slot_stride=HD, head_stride=HD << 20, layer_stride=HD << 23, seq_stride=HD << 24)
    c = Call(q3).with_(**big, new_weight=1 << 40, new_slot_pos=1 << 40)
    assert c.scored() == UNSUPPORTED
    assert c.evict() == UNSUPPORTED


def test_gguf_q4_0_blocks(tmp_path, q3):
    from q3b200 import gguf
    from test_gguf import _write_gguf

    blocks = quantize(q3, np.random.default_rng(1).standard_normal((8, 256)).astype(np.float32))
    path = str(tmp_path / "q4.gguf")
    _write_gguf(path, [("blk.0.attn_q.weight", (8, 256), gguf.GGML_Q4_0, blocks.tobytes()),
                       ("odd", (3, 11), gguf.GGML_F32, b"\0" * 132)])
    _, t = gguf.read_gguf(path)
    assert np.array_equal(gguf.q4_0(t, "blk.0.attn_q.weight", 8, 256), blocks.ravel())
    for name, N, K in (("none", 8, 256), ("odd", 3, 11), ("blk.0.attn_q.weight", 4, 512)):
        with pytest.raises(gguf.GGUFError):
            gguf.q4_0(t, name, N, K)
