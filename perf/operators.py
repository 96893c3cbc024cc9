"""Decoding with drafted tokens over a bounded KV cache: the cases the operators are measured on.

Five entry points of the library, each with its plain form (elementary torch
operations, what a user writes without the library):

  gemv    q3_gemv_q4                 y[R, N] = x[R, K] . W[N, K]^T with 4-bit weights in groups of
                                     32 (18 bytes: an f16 scale d, then 16 bytes of nibbles; byte j
                                     holds element j low and j + 16 high; w = d * (q - 8))
  tree    q3_tree_attention          a tree of drafted tokens attends to the cache and to its own
                                     ancestors; its K/V rows go behind the cached ones
  commit  q3_tree_commit             the accepted path's rows move together, in every layer; their
                                     slots start with weight 0 and hold the path's positions
  scored  q3_decode_attention_scored one token's attention, which adds every slot's attention weight
                                     to an accumulator
  evict   q3_cache_evict             the slots with the largest accumulated weight and the newest
                                     ones stay; kept rows from behind the budget fill the holes

Heads are 16 query and 8 key/value heads of 128, values f16, accumulators f32.
"flat" caches are [B][layers * S][8][128], "head" ones [B][layers][8][S][128].
Nothing here reads the library unless `own` is true.
"""
import os
import sys

import torch

own = False

HD, NQ, NKV, EPS, THETA = 128, 16, 8, 9.99999997e-7, 1.0e6
G = NQ // NKV
SCALE = HD ** -0.5
ROW = (NQ + 2 * NKV) * HD


def listed():
    return [
        # one token through the query projection of a 4-bit copy of the weights: a draft step, all latency
        {"name": "gemv q 1", "op": "gemv", "N": 2048, "K": 1024, "R": 1},
        # a ragged output width and a few beams
        {"name": "gemv ragged 3", "op": "gemv", "N": 6007, "K": 1280, "R": 3},
        # the vocabulary head for eight drafted tokens
        {"name": "gemv vocab 8", "op": "gemv", "N": 151936, "K": 1024, "R": 8},
        # verifying a small tree in a chat-length cache
        {"name": "tree 8 at 500", "op": "tree", "B": 1, "T": 8, "L": 500, "ragged": False, "layout": "flat"},
        # a wide tree over a long document
        {"name": "tree 64 at 32k", "op": "tree", "B": 1, "T": 64, "L": 32749, "ragged": False, "layout": "flat"},
        # a served batch: every sequence has its own length and its own tree, the batched decoder's layout
        {"name": "tree 17 batch 16", "op": "tree", "B": 16, "T": 17, "L": 4001, "ragged": True, "layout": "head"},
        # accepting a path in all 28 layers
        {"name": "commit 1", "op": "commit", "B": 1, "T": 16, "A": 5, "S": 1024, "layers": 28, "layout": "flat"},
        {"name": "commit batch 32", "op": "commit", "B": 32, "T": 64, "A": 9, "S": 300, "layers": 28, "layout": "flat"},
        # one decode step whose weights are kept for a later eviction
        {"name": "scored at 1000", "op": "scored", "B": 1, "L": 1000, "ragged": False, "layout": "flat"},
        {"name": "scored batch 32", "op": "scored", "B": 32, "L": 4095, "ragged": True, "layout": "head"},
        # a full chat cache down to its half, and a batch of longer ones down to three quarters
        {"name": "evict 1", "op": "evict", "B": 1, "S": 1024, "budget": 512, "recent": 64, "layers": 28, "layout": "flat"},
        {"name": "evict batch 4", "op": "evict", "B": 4, "S": 4096, "budget": 3077, "recent": 256, "layers": 28, "layout": "head"},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["gemv", "tree", "commit", "scored", "evict"])
    layout = rng.choice(["flat", "head"])
    if op == "gemv":
        return {"op": op, "N": log(100, 151936), "K": 256 * rng.randint(1, 4), "R": rng.randint(1, 8)}
    if op == "tree":
        T = log(1, 64)
        B = log(1, 16)
        return {"op": op, "B": B, "T": T, "L": log(1, min(32749, 32749 * 64 // (B * max(T, 32)))), "ragged": rng.random() < 0.5,
                "layout": layout}
    if op == "commit":
        A = rng.randint(2, 9)
        return {"op": op, "B": log(1, 32), "T": rng.randint(2 * A, 64), "A": A, "S": rng.randint(100, 300),
                "layers": rng.randint(1, 28), "layout": layout}
    if op == "scored":
        B = log(1, 32)
        return {"op": op, "B": B, "L": log(1, 17 * 4095 // B), "ragged": rng.random() < 0.5, "layout": layout}
    B = log(1, 4)
    S = log(64, 4096)
    budget = rng.randint(S // 4, S - 1)
    return {"op": op, "B": B, "S": S, "budget": budget, "recent": rng.randint(0, budget // 4), "layers": rng.randint(1, 28),
            "layout": layout}


# ------------------------------------------------------------------------------------------ inputs
def _slots(case):
    """Slots of a layer: the cached ones, the drafted ones and a few that stay free."""
    return case["S"] if "S" in case else case["L"] + case.get("T", 1) + 5


def _lens(case):
    """Cached slots per sequence: the longest has L, the others are spread below it."""
    B, L = case["B"], case["L"]
    return [L if not case["ragged"] or b == 0 else max(1, (L * ((b * 7919) % 97 + 3)) // 100) for b in range(B)]


def _counts(case):
    """Drafted tokens per sequence."""
    B, T = case["B"], case["T"]
    return [T if not case["ragged"] or b == 0 else 1 + (b * 5) % T for b in range(B)]


def _cache(case, g):
    """(k, v, strides): strides are (sequence, layer, slot, head) in elements."""
    B, S, n = case["B"], _slots(case), case.get("layers", 1)
    shape = (B, n * S, NKV, HD) if case["layout"] == "flat" else (B, n, NKV, S, HD)
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    if case["layout"] == "flat":
        return k, v, (n * S * NKV * HD, S * NKV * HD, NKV * HD, HD)
    return k, v, (n * NKV * S * HD, NKV * S * HD, HD, S * HD)


def _rope(rows):
    inv = THETA ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def i64(v):
        return torch.tensor(v, device="cuda", dtype=torch.int64)

    if case["op"] == "gemv":
        N, K, R = case["N"], case["K"], case["R"]
        # weights ~ N(0, 0.02): nibbles spread over the whole range, scales near 0.02 * 2.2 / 8
        q = (randn(N, K // 32, 32) * (8 / 2.2) + 8).round_().clamp_(0, 15).to(torch.uint8)
        d = ((1 + 0.2 * randn(N, K // 32, 1)) * (0.02 * 2.2 / 8)).half()
        s["w"] = torch.cat([d.view(torch.uint8), q[..., :16] | (q[..., 16:] << 4)], -1).reshape(-1)
        s["x"] = randn(R, K).half()
        s["y"] = torch.zeros(R, N, device="cuda", dtype=torch.float16)
        return s
    S = s["S"] = _slots(case)
    s["k"], s["v"], s["strides"] = _cache(case, g)
    B = case["B"]
    if case["op"] in ("tree", "scored"):
        T = case.get("T", 1)
        s["qkv"] = randn(B, T, ROW).half()
        s["q_norm"], s["k_norm"] = ((1 + 0.1 * randn(HD)).half() for _ in range(2))
        lens = _lens(case)
        s["len"] = i64(lens)
        # an earlier eviction: more positions seen than slots held
        s["pos"] = i64([n + (b * 3) % 4 * 11 for b, n in enumerate(lens)])
        s["cos"], s["sin"] = _rope(S + 40 + T)
        s["out"] = torch.zeros(B, T, NQ * HD, device="cuda", dtype=torch.float16)
    if case["op"] == "tree":
        # token i's parent: one of the eight before it, or the last cached token (-1)
        i = torch.arange(T, device="cuda")
        back = (torch.rand(B, T, generator=g, device="cuda") * (i + 1).clamp(max=8)).long()
        s["parents"] = (i - 1 - back).clamp(min=-1).int()
        s["n"] = torch.tensor(_counts(case), device="cuda", dtype=torch.int32)
        s["err"] = torch.zeros(1, device="cuda", dtype=torch.int32)
    elif case["op"] == "commit":
        # the accepted path: a root (the first token, or a later one) and its descendants,
        # numbered level by level, so behind the rows that the path moves to
        T, A = case["T"], case["A"]
        order = torch.rand(B, T - A, generator=g, device="cuda").argsort(-1)[:, :A].sort(-1).values + A
        order[::2, 0] = 0
        s["accepted"] = order.int().contiguous()
        s["n"] = torch.tensor([A - (b * 2) % A for b in range(B)], device="cuda", dtype=torch.int32)
        s["len"] = i64([max(0, S - T - (b * 13) % 64) for b in range(B)])
        s["new_len"] = torch.zeros(B, device="cuda", dtype=torch.int64)
        s["err"] = torch.zeros(1, device="cuda", dtype=torch.int32)
    if case["op"] != "tree":
        n = case.get("layers", 1)
        # weight a slot has drawn over some tens of steps: heavy tailed, largest for the first slots
        w = torch.exp(1.5 * randn(B, n, NKV, S)) * (32.0 / S)
        w[..., :4] += 8
        s["weight"] = w
        # the positions the slots hold: ascending with gaps, where others were evicted
        gap = (torch.rand(B, n, NKV, S, generator=g, device="cuda") < 0.2).int()
        p = torch.arange(S, device="cuda", dtype=torch.int32) + gap.cumsum(-1, dtype=torch.int32)
        s["slot_pos"] = p
        if case["op"] == "commit":
            s["pos"] = s["len"] * 6 // 5
            return s
        s["new_weight"] = torch.zeros_like(w)
        s["err"] = torch.zeros(1, device="cuda", dtype=torch.int32)
        if case["op"] == "evict":
            s["len"] = i64([max(0, S - (b * 37) % (S // 2 + 1)) for b in range(B)])
            held = torch.arange(S, device="cuda") < s["len"][:, None, None, None]
            s["pos"] = torch.where(held, p, -1).amax((1, 2, 3)).long() + 1
            s["new_slot_pos"] = torch.zeros_like(p)
            s["new_len"] = torch.zeros(B, device="cuda", dtype=torch.int64)
    return s


def _head_view(s, x):
    """The cache as [B, layers, 8, S, 128], whatever its layout."""
    n = s.get("layers", 1)
    if s["layout"] == "head":
        return x
    return x.view(s["B"], n, s["S"], NKV, HD).permute(0, 1, 3, 2, 4)


# -------------------------------------------------------------------------------------- plain form
def _norm_rope(x, gamma, cos, sin):
    """RMSNorm over a head, then the rotation of (i, i + 64); each rounded to f16, as the cache holds it.
    In 64 bits: the roundings sit next to borders."""
    x = x.double()
    x = (x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gamma.double()).half().double()
    a, b = x[..., :64], x[..., 64:]
    c, d = cos.double(), sin.double()
    return torch.cat([a * c - b * d, a * d + b * c], -1).half()


def _project(s, depth):
    """The roped queries [B, T, 8, G, 128] and keys [B, T, 8, 128] and the values of the new tokens."""
    B, T = s["qkv"].shape[:2]
    at = (s["pos"][:, None] + depth).clamp(0, s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q, k, v = s["qkv"].view(B, T, NQ + 2 * NKV, HD).split([NQ, NKV, NKV], 2)
    q = _norm_rope(q, s["q_norm"], cos, sin).view(B, T, NKV, G, HD)
    return q, _norm_rope(k, s["k_norm"], cos, sin), v


def _attend(s, q, k_new, v_new, live, mask):
    """Softmax attention of the new tokens over the cached slots and, where `mask` [B, T, T] allows, one another.
    Puts the new rows into the cache. Returns the output and the softmax weights over all slots."""
    B, T = q.shape[:2]
    k, v = (_head_view(s, s[x])[:, 0] for x in "kv")
    slot = torch.arange(s["S"], device="cuda")
    new = s["len"][:, None] + torch.arange(T, device="cuda")
    b, t = torch.where(live)
    k[b, :, new[b, t]] = k_new[b, t]
    v[b, :, new[b, t]] = v_new[b, t]
    sc = torch.matmul(q.float().permute(0, 2, 3, 1, 4).reshape(B, NKV, G * T, HD), k.float().transpose(-1, -2)) * SCALE
    allow = (slot < s["len"][:, None])[:, None].expand(B, T, s["S"]).clone()
    allow.scatter_(2, new[:, None].expand(B, T, T).clamp(max=s["S"] - 1), mask)
    sc = sc.view(B, NKV, G, T, s["S"]).masked_fill(~allow[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = (sc - top.masked_fill(top == float("-inf"), 0)).exp()
    tot = p.sum(-1, keepdim=True)
    p = p / tot.masked_fill(tot == 0, 1)
    vz = torch.where((slot < (s["len"] + live.sum(-1))[:, None])[:, None, :, None], v.float(), 0.0)
    o = torch.matmul(p.view(B, NKV, G * T, s["S"]), vz).view(B, NKV, G, T, HD)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, NQ * HD), p


def _plain_gemv(s):
    blocks = s["w"].view(s["N"], s["K"] // 32, 18)
    d = blocks[..., :2].contiguous().view(torch.float16).float()
    q = torch.cat([blocks[..., 2:] & 15, blocks[..., 2:] >> 4], -1)
    w = (d * (q.float() - 8)).view(s["N"], s["K"])
    s["y"].copy_(torch.matmul(s["x"].float(), w.t()))
    return {"y": s["y"]}


def _plain_tree(s):
    B, T = s["parents"].shape
    i = torch.arange(T, device="cuda")
    live = i < s["n"][:, None]
    step = torch.eye(T, device="cuda", dtype=torch.float64) + (s["parents"][:, :, None] == i)
    mask = (torch.linalg.matrix_power(step, T) > 0) & live[:, :, None] & live[:, None]
    q, k, v = _project(s, mask.sum(-1) - 1)
    o, _ = _attend(s, q, k, v, live, mask)
    s["out"].copy_(torch.where(live[..., None], o, s["out"].float()))
    return {"out": s["out"], "k": s["k"], "v": s["v"]}


def _plain_commit(s):
    i = torch.arange(s["A"], device="cuda")
    b, t = torch.where(i < s["n"][:, None])
    src, dst = s["len"][b] + s["accepted"][b, t], s["len"][b] + t
    k, v = _head_view(s, s["k"]), _head_view(s, s["v"])
    k[b, :, :, dst] = k[b, :, :, src]
    v[b, :, :, dst] = v[b, :, :, src]
    s["new_len"].copy_(s["len"] + s["n"])
    s["weight"][b, :, :, dst] = 0.0
    s["slot_pos"][b, :, :, dst] = (s["pos"][b] + t).int()[:, None, None]
    return {"k": s["k"], "v": s["v"], "weight": s["weight"], "slot_pos": s["slot_pos"], "len": s["new_len"]}


def _plain_scored(s):
    B = s["B"]
    one = torch.ones(B, 1, 1, dtype=torch.bool, device="cuda")
    q, k, v = _project(s, 0)
    o, p = _attend(s, q, k, v, one[:, 0], one)
    s["out"].copy_(o)
    slot = torch.arange(s["S"], device="cuda")
    at = s["len"][:, None, None, None]
    w = torch.where(slot < at, s["weight"], 0.0) + p.sum((2, 3))[:, None]
    s["new_weight"].copy_(torch.where(slot <= at, w, s["new_weight"]))
    s["slot_pos"].copy_(torch.where(slot == at, s["pos"].int()[:, None, None, None], s["slot_pos"]))
    return {"out": s["out"], "k": s["k"], "v": s["v"], "weight": s["new_weight"], "slot_pos": s["slot_pos"]}


def _plain_evict(s):
    S, M = s["S"], s["budget"]
    slot = torch.arange(S, device="cuda")
    at = s["len"][:, None, None, None]
    # newest first, then by weight; a stable sort leaves ties to the lower slot
    rank = torch.where(s["slot_pos"] >= (s["pos"] - s["recent"])[:, None, None, None], float("inf"), s["weight"])
    rank = rank.masked_fill(slot >= at, float("-inf"))
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, order[..., :M], True)
    keep = torch.where(at > M, keep, slot < at)
    b, l, h, src = torch.where(keep & (slot >= M))
    _, _, _, dst = torch.where(~keep & (slot < M) & (at > M))
    k, v = _head_view(s, s["k"]), _head_view(s, s["v"])
    k[b, l, h, dst] = k[b, l, h, src]
    v[b, l, h, dst] = v[b, l, h, src]
    s["new_len"].copy_(s["len"].clamp(max=M))
    for x in ("weight", "slot_pos"):
        y = s[x].clone()
        y[b, l, h, dst] = y[b, l, h, src]
        s["new_" + x].copy_(torch.where(slot < at.clamp(max=M), y, s["new_" + x]))
    return {"k": s["k"], "v": s["v"], "weight": s["new_weight"], "slot_pos": s["new_slot_pos"], "len": s["new_len"]}


# ------------------------------------------------------------------------------------ library calls
def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-iree_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import q3b200

    return q3b200


def _kv(q3, s):
    a, b, c, d = s["strides"]
    return q3.KVCache(s["k"].data_ptr(), s["v"].data_ptr(), a, b, c, d, s["S"], s.get("layers", 1), NQ, NKV)


def _own(s):
    q3 = _library()
    st = torch.cuda.current_stream().cuda_stream
    if s["op"] == "gemv":
        q3.call("q3_gemv_q4", s["w"].data_ptr(), s["x"].data_ptr(), s["y"].data_ptr(), s["N"], s["K"], s["R"], st)
        return {"y": s["y"]}
    kv = _kv(q3, s)
    if s["op"] == "tree":
        q3.call("q3_tree_attention", s["qkv"].data_ptr(), s["q_norm"].data_ptr(), s["k_norm"].data_ptr(),
                s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], kv, 0, s["B"], s["T"],
                s["parents"].data_ptr(), s["n"].data_ptr(), s["len"].data_ptr(), s["pos"].data_ptr(),
                s["out"].data_ptr(), s["err"].data_ptr(), st)
        return {"out": s["out"], "k": s["k"], "v": s["v"]}
    if s["op"] == "commit":
        q3.call("q3_tree_commit", kv, 0, s["layers"], s["B"], s["A"], s["accepted"].data_ptr(), s["n"].data_ptr(),
                s["len"].data_ptr(), s["new_len"].data_ptr(), s["pos"].data_ptr(), s["weight"].data_ptr(),
                s["slot_pos"].data_ptr(), s["err"].data_ptr(), st)
        return {"k": s["k"], "v": s["v"], "weight": s["weight"], "slot_pos": s["slot_pos"], "len": s["new_len"]}
    if s["op"] == "scored":
        q3.call("q3_decode_attention_scored", s["qkv"].data_ptr(), s["q_norm"].data_ptr(), s["k_norm"].data_ptr(),
                s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], kv, 0, s["B"], s["len"].data_ptr(),
                s["pos"].data_ptr(), s["weight"].data_ptr(), s["new_weight"].data_ptr(), s["slot_pos"].data_ptr(),
                s["out"].data_ptr(), s["err"].data_ptr(), st)
        return {"out": s["out"], "k": s["k"], "v": s["v"], "weight": s["new_weight"], "slot_pos": s["slot_pos"]}
    q3.call("q3_cache_evict", kv, 0, s["layers"], s["B"], s["budget"], s["recent"], s["len"].data_ptr(),
            s["pos"].data_ptr(), s["weight"].data_ptr(), s["slot_pos"].data_ptr(), s["new_len"].data_ptr(),
            s["new_weight"].data_ptr(), s["new_slot_pos"].data_ptr(), s["err"].data_ptr(), st)
    return {"k": s["k"], "v": s["v"], "weight": s["new_weight"], "slot_pos": s["new_slot_pos"], "len": s["new_len"]}


_PLAIN = {"gemv": _plain_gemv, "tree": _plain_tree, "commit": _plain_commit, "scored": _plain_scored, "evict": _plain_evict}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


# -------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once, each output written once. K and V of a slot: 2 * 256 bytes a head."""
    op, row = case["op"], 2 * 2 * HD
    if op == "gemv":
        N, K, R = case["N"], case["K"], case["R"]
        return {"bytes": N * K // 32 * 18 + 2 * R * (K + N), "flops": 2 * N * K * R}
    if op in ("tree", "scored"):
        lens, one = _lens(case), op == "scored"
        counts = [1] * case["B"] if one else _counts(case)
        keys = sum(lens) * NKV
        new = sum(counts)
        b = keys * row + new * (2 * ROW + NKV * row + 2 * NQ * HD + 512)
        if one:  # weight in and out, and the new slot's position
            b += 8 * keys + 8 * NKV * case["B"]
        return {"bytes": b, "flops": sum(4 * HD * NQ * n * (c + (n + 1) / 2) for c, n in zip(lens, counts))}
    if op == "commit":
        A = case["A"]
        heads = case["layers"] * NKV
        kept = sum(A - (b * 2) % A for b in range(case["B"]))
        stay = (case["B"] + 1) // 2  # paths that begin with the first token leave it where it is
        return {"bytes": heads * (2 * (kept - stay) * row + 8 * kept), "flops": 0}
    # evict: the weights and positions in and out, and the rows of the kept slots behind the
    # budget, read and written (their number by chance: the newest, and their share of the rest)
    S, M, b = case["S"], case["budget"], 0.0
    for i in range(case["B"]):
        n = max(0, S - (i * 37) % (S // 2 + 1))
        held = min(n, M)
        b += 8 * (n + held)
        if n > M:
            newest = min(case["recent"] / 1.2, n - M)
            b += 2 * row * (newest + (n - M - newest) * (M - newest) / max(1, n - newest))
    return {"bytes": b * case["layers"] * NKV, "flops": 0}


# ------------------------------------------------------------------------------ definition in 64 bits
def _exact_head(x, gamma, angle_cos, angle_sin):
    """One head's vectors [..., 128]: (rounded as the cache holds it, before the last rounding)."""
    x = x.to(torch.float64)
    rms = torch.sqrt(torch.sum(x * x, -1, keepdim=True) / HD + EPS)
    y = (gamma.to(torch.float64) * (x / rms)).to(torch.float16).to(torch.float64)
    half = torch.roll(y, 64, -1)
    sign = torch.ones(HD, device="cuda", dtype=torch.float64)
    sign[:64] = -1
    c, s = (torch.cat([z, z], -1).to(torch.float64) for z in (angle_cos, angle_sin))
    z = y * c + sign * half * s
    return z.to(torch.float16).to(torch.float64), z


def _exact_attention(s, parents, n_new):
    """Per sequence and token, over the slots it sees: output, updated caches, and slot weights."""
    out = s["out"].to(torch.float64)
    k, v = s["k"].to(torch.float64), s["v"].to(torch.float64)
    kh, vh = _head_view(s, k), _head_view(s, v)
    lens, pos = s["len"].tolist(), s["pos"].tolist()
    seen = torch.zeros(s["B"], NKV, s["S"], device="cuda", dtype=torch.float64)
    for b, (m, p0, n) in enumerate(zip(lens, pos, n_new)):
        paths = []
        for t in range(n):
            up = parents[b][t]
            paths.append([t] if up < 0 else paths[up] + [t])
        at = torch.tensor([p0 + len(p) - 1 for p in paths], device="cuda")
        allowed = torch.zeros(n, m + n, dtype=torch.bool, device="cuda")
        allowed[:, :m] = True
        for t, p in enumerate(paths):
            allowed[t, torch.tensor(p, device="cuda") + m] = True
        c, d = s["cos"][at][:, None], s["sin"][at][:, None]
        x = s["qkv"][b, :n].view(n, NQ + 2 * NKV, HD)
        q, _ = _exact_head(x[:, :NQ], s["q_norm"], c, d)
        kn, kz = _exact_head(x[:, NQ:NQ + NKV], s["k_norm"], c, d)
        vn = x[:, NQ + NKV:].to(torch.float64)
        for h in range(NKV):
            keys = torch.cat([kh[b, 0, h, :m], kn[:, h]])
            vals = torch.cat([vh[b, 0, h, :m], vn[:, h]])
            for j in range(G):
                e = torch.softmax((q[:, h * G + j] @ keys.T / HD ** 0.5).masked_fill(~allowed, -torch.inf), -1)
                out[b, :n, (h * G + j) * HD:(h * G + j + 1) * HD] = e @ vals
                seen[b, h, :m + n] += e.sum(0)
        kh[b, 0, :, m:m + n] = kz.transpose(0, 1)
        vh[b, 0, :, m:m + n] = vn.transpose(0, 1)
    return out, k, v, seen


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "gemv":
        w = s["w"].view(case["N"], -1, 18)
        d = w[:, :, :2].reshape(-1).view(torch.float16).view(case["N"], -1, 1).to(torch.float64)
        lo, hi = torch.remainder(w[:, :, 2:], 16), torch.div(w[:, :, 2:], 16, rounding_mode="floor")
        w = torch.stack([lo, hi], 2).flatten(2).to(torch.float64).sub_(8).mul_(d).flatten(1)
        return {"y": s["x"].to(torch.float64) @ w.T}
    if op == "tree":
        out, k, v, _ = _exact_attention(s, s["parents"].tolist(), s["n"].tolist())
        return {"out": out, "k": k, "v": v}
    if op == "scored":
        out, k, v, seen = _exact_attention(s, [[-1]] * case["B"], [1] * case["B"])
        w, sp = s["new_weight"].to(torch.float64), s["slot_pos"].clone()
        for b, m in enumerate(s["len"].tolist()):
            w[b, 0, :, :m] = s["weight"][b, 0, :, :m].to(torch.float64) + seen[b, :, :m]
            w[b, 0, :, m] = seen[b, :, m]
            sp[b, 0, :, m] = int(s["pos"][b])
        return {"out": out, "k": k, "v": v, "weight": w, "slot_pos": sp}
    k, v = _head_view(s, s["k"]), _head_view(s, s["v"])
    lens = s["len"].tolist()
    if op == "commit":
        for b, m in enumerate(lens):
            for i, a in enumerate(s["accepted"][b].tolist()[:int(s["n"][b])]):
                for x in (k, v):
                    x[b, :, :, m + i] = x[b, :, :, m + a].clone()
                s["weight"][b, ..., m + i] = 0
                s["slot_pos"][b, ..., m + i] = int(s["pos"][b]) + i
        return {"k": s["k"], "v": s["v"], "weight": s["weight"], "slot_pos": s["slot_pos"], "len": s["len"] + s["n"]}
    M, w, sp = case["budget"], s["new_weight"], s["new_slot_pos"]
    for b, m in enumerate(lens):
        for l in range(case["layers"]):
            for h in range(NKV):
                a, p = s["weight"][b, l, h, :m].to(torch.float64), s["slot_pos"][b, l, h, :m].long()
                at = torch.arange(m, device="cuda")
                if m > M:
                    new = p >= int(s["pos"][b]) - case["recent"]
                    by = torch.where(new, torch.inf, a).cpu().numpy()
                    kept = torch.from_numpy((-by).argsort(kind="stable")[:M].copy()).cuda()
                    stays = torch.isin(at, kept)
                    at = at[:M].clone()
                    at[~stays[:M]] = torch.nonzero(stays[M:])[:, 0] + M
                    k[b, l, h, :M] = k[b, l, h][at]
                    v[b, l, h, :M] = v[b, l, h][at]
                w[b, l, h, :len(at)] = a[at].float()
                sp[b, l, h, :len(at)] = p[at].int()
    return {"k": s["k"], "v": s["v"], "weight": w, "slot_pos": sp, "len": s["len"].clamp(max=M)}
