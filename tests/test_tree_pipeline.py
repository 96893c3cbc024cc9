"""Model check of k_tree_tc's protocol (csrc/q3_tree.cuh) on the CPU.

A copying warp streams the K and V halves of the tiles into two rings, an MMA
warp issues S(j) = Q K(j)^T into one of two S buffers and then O += P V(j - 1),
and softmax warps turn S(j) into the weights P(j) in place, rescaling O when a
maximum has grown.  The model keeps the rules the kernel relies on: a parity
wait succeeds when the phase of that parity is complete, which includes the
phase before the pending one; copies land in any order; MMAs and commits
complete in the order of their issue, at any later time.  No random schedule may
read a slot that does not hold its tile, rescale O before the products of all
earlier tiles are in it, or reach the end (where the operands' memory becomes
the partial outputs) with a copy or an MMA under way.

The barrier o_done completes a phase for every tile's P V, so a wait for one is
only sound where the phase before it is known to be complete: the MMA warp
waits for the products of tile j - 2 before it issues those of j - 1, after the
last S too.  Without that the last wait can take the phase of tile n - 3 for the
one of n - 1; the model finds such a schedule.
"""
import pathlib
import random
import re

import pytest

from test_battn_pipeline import Barrier, Violation

HDR = pathlib.Path(__file__).resolve().parents[1] / "qwen3-iree_b200" / "csrc" / "q3_tree.cuh"


def _mma_loop():
    src = HDR.read_text()
    src = src[src.index("k_tree_tc("):]
    return src[src.index("for (int j = 0; j <= c.tiles; ++j) {"):]


def _waits_after_the_last_s():
    """Whether the kernel waits for tile j - 2 in every round of its loop, or only where there is an S(j)."""
    loop = _mma_loop()
    wait = re.search(r"if \(j >= 2\) ok &= mbar_wait_own\(&sm\.o_done, j & 1", loop).start()
    return wait < loop.index("if (j < c.tiles) {")


def _rings():
    src = HDR.read_text()
    kd, small, large = re.search(r"kSlots = (\d), vSlots = ROWS == 64 \? (\d) : (\d);", src).groups()
    return [(int(kd), int(small)), (int(kd), int(large))]


def run_cta(tiles, fresh, kd, vd, warps, rng, every_round):
    k_full, k_empty = ([Barrier() for _ in range(kd)] for _ in range(2))
    v_full, v_empty = ([Barrier() for _ in range(vd)] for _ in range(2))
    s_full, p_full, o_done = [Barrier(), Barrier()], [Barrier(warps), Barrier(warps)], Barrier()
    k_at, v_at = [None] * kd, [None] * vd
    s_at = [None, None]             # ("S", tile), then the warps' ("P", tile)
    p_parts = [set(), set()]
    inflight, pipe = [], []         # copies; MMAs and commits in order
    summed = [0]                    # tiles whose P V is in O

    def copier():
        def copy_k(j):
            if j >= fresh:
                inflight.append((k_at, j % kd, j, k_full[j % kd]))

        def copy_v(j):
            if j >= fresh:
                inflight.append((v_at, j % vd, j, v_full[j % vd]))

        for j in range(min(kd, tiles)):
            copy_k(j)
            if j < vd:
                copy_v(j)
        if fresh:
            k_at[0] = v_at[0] = 0
        kj = kd
        for j in range(tiles):
            if j >= vd:
                if kj < tiles:
                    while not k_empty[kj % kd].done((kj // kd - 1) & 1):
                        yield
                    copy_k(kj)
                    kj += 1
                while not v_empty[j % vd].done((j // vd - 1) & 1):
                    yield
                copy_v(j)
            if j < fresh:
                k_full[0].arrive()
                v_full[0].arrive()
            yield
        kj = min(kj, tiles)
        for i in range(max(kj - kd, 0), kj):
            while not k_full[i % kd].done((i // kd) & 1):
                yield
        for i in range(max(tiles - vd, 0), tiles):
            while not v_full[i % vd].done((i // vd) & 1):
                yield

    def mma():
        for j in range(tiles + 1):
            if j < tiles:
                while not k_full[j % kd].done((j // kd) & 1):
                    yield
            if j >= 2 and (every_round or j < tiles):
                while not o_done.done(j & 1):
                    yield
            if j < tiles:
                pipe.append(("S", j))
                pipe.append(s_full[j & 1])
                pipe.append(k_empty[j % kd])
            if j > 0:
                i = j - 1
                while not v_full[i % vd].done((i // vd) & 1):
                    yield
                while not p_full[i & 1].done((i >> 1) & 1):
                    yield
                pipe.append(("PV", i))
                pipe.append(o_done)
                pipe.append(v_empty[i % vd])
            yield
        while tiles and not o_done.done((tiles - 1) & 1):
            yield

    def softmax(w):
        for j in range(tiles):
            while not s_full[j & 1].done((j >> 1) & 1):
                yield
            if s_at[j & 1] != ("S", j):
                raise Violation(f"warp {w} took {s_at[j & 1]} for S({j})")
            yield
            if j > 0 and rng.random() < 0.3:
                while not o_done.done((j - 1) & 1):
                    yield
                if summed[0] != j or any(x[0] == "PV" for x in pipe if isinstance(x, tuple)):
                    raise Violation(f"warp {w} rescaled O with {summed[0]} of {j} tiles in it")
                yield
            p_parts[j & 1].add(w)
            if len(p_parts[j & 1]) == warps:
                s_at[j & 1], p_parts[j & 1] = ("P", j), set()
            p_full[j & 1].arrive()
            yield

    def step_pipe():
        x = pipe.pop(0)
        if isinstance(x, Barrier):
            x.arrive()
        elif x[0] == "S":
            if k_at[x[1] % kd] != x[1]:
                raise Violation(f"S({x[1]}) from K of tile {k_at[x[1] % kd]}")
            s_at[x[1] & 1] = x
        else:
            i = x[1]
            if v_at[i % vd] != i or s_at[i & 1] != ("P", i):
                raise Violation(f"P V({i}) from V of tile {v_at[i % vd]}, weights {s_at[i & 1]}")
            summed[0] += 1

    actors = [copier(), mma(), *(softmax(w) for w in range(warps))]
    live = list(range(len(actors)))
    # some schedules starve the copies, the tensor pipe or neither
    p_land, p_pipe = rng.choice([0.02, 0.3]), rng.choice([0.02, 0.3])
    idle = 0
    while live:
        r = rng.random()
        if inflight and (r < p_land or idle > 200):
            at, s, tile, bar = inflight.pop(rng.randrange(len(inflight)))
            at[s] = tile
            bar.arrive()
            idle = 0
            continue
        if pipe and (r > 1 - p_pipe or idle > 200):
            step_pipe()
            idle = 0
            continue
        a = rng.choice(live)
        idle += 1
        if idle > 5000:
            raise Violation("nothing moves")
        try:
            next(actors[a])
        except StopIteration:
            live.remove(a)
    if inflight or any(isinstance(x, tuple) for x in pipe) or summed[0] != tiles:
        raise Violation(f"the end with {summed[0]} of {tiles} tiles in O")


@pytest.mark.parametrize("kd,vd", _rings())
@pytest.mark.parametrize("warps", [1, 4])
def test_tree_pipeline_schedules(kd, vd, warps):
    rng = random.Random(10 * kd + vd + 100 * warps)
    for n in range(400):
        run_cta(1 + n % 9, rng.randint(0, 1), kd, vd, warps, rng, _waits_after_the_last_s())


def test_the_model_finds_the_wait_that_is_left_out():
    rng = random.Random(3)
    failures = 0
    for n in range(400):
        try:
            run_cta(2 + n % 8, 0, 3, 2, 4, rng, every_round=False)
        except Violation:
            failures += 1
    assert failures > 0
