"""Model check of k_gemv_q4_stream's protocol (csrc/q3_q4.cuh) on the CPU.

A group of two warps takes tiles in turn through a ring of two stages.  The
first warp issues the copies; both wait for a tile's copy (full), each sums its
half of K, the second leaves its sums in a place per stage and arrives (done),
and the first waits for that, adds, refills the stage and stores the tile.  The
rules are those of tests/test_tree_pipeline.py, and waits may give up: a copy
that never lands, as on a device in trouble, must leave NaN in the rows that
have no sum, never a sum of what happened to lie in the stage.
"""
import pathlib
import random
import re

import pytest

from test_battn_pipeline import Barrier, Violation

HDR = pathlib.Path(__file__).resolve().parents[1] / "qwen3-iree_b200" / "csrc" / "q3_q4.cuh"
STAGES = 2


def _stops():
    """Whether the kernel leaves its loop when a wait gives up, for both of its waits."""
    src = HDR.read_text()
    src = src[src.index("k_gemv_q4_stream("):]
    gives_up = r"mbar_wait_own\(&%s\[grp\]\[st\], ph, nullptr, kErrTimeoutFull\);\s*if \(!__all_sync\(0xffffffffu, ok\)\) break;"
    return all(re.search(gives_up % b, src) for b in ("full", "done"))


def run_group(tiles, lost, rng, stops):
    full, done = ([Barrier() for _ in range(STAGES)] for _ in range(2))
    stage, sums = [None] * STAGES, [None] * STAGES
    reading = [set(), set()]
    inflight, y = [], {}
    stuck = [False]                 # nothing else can move: waits give up

    def issue(j):
        s = j % STAGES
        if reading[s] or any(c[0] == s for c in inflight):
            raise Violation(f"stage {s} refilled with tile {j} while in use")
        if j == lost:
            stage[s] = None
        else:
            inflight.append((s, j))

    def wait(bar, parity):
        while not bar.done(parity):
            if stuck[0]:
                return
            yield

    def first():
        for j in range(min(STAGES, tiles)):
            issue(j)
        j = 0
        while j < tiles:
            s, ph = j % STAGES, (j // STAGES) & 1
            yield from wait(full[s], ph)
            if not full[s].done(ph) and stops:
                break
            reading[s].add(0)
            mine = stage[s]
            yield
            reading[s].discard(0)
            yield from wait(done[s], ph)
            if not done[s].done(ph) and stops:
                break
            y[j] = (mine, sums[s])
            if full[s].done(ph) and done[s].done(ph) and j + STAGES < tiles:
                issue(j + STAGES)
            j += 1
            yield
        for i in range(j, min(j + STAGES, tiles) if stops else 0):
            yield from wait(full[i % STAGES], (i // STAGES) & 1)
        for i in range(j, tiles):
            y[i] = "nan"

    def second():
        for j in range(tiles):
            s, ph = j % STAGES, (j // STAGES) & 1
            yield from wait(full[s], ph)
            if not full[s].done(ph) and stops:
                return
            reading[s].add(1)
            got = stage[s]
            yield
            reading[s].discard(1)
            sums[s] = got
            if done[s].pending:
                done[s].arrive()
            yield

    live, idle = [first(), second()], 0
    while live:
        if inflight and rng.random() < 0.2:
            s, j = inflight.pop(rng.randrange(len(inflight)))
            stage[s] = j
            full[s].arrive()
            idle = 0
            continue
        idle += 1
        stuck[0] = idle > 200 and not inflight
        a = rng.choice(live)
        try:
            next(a)
        except StopIteration:
            live.remove(a)
    if inflight:
        raise Violation("a copy in flight at the end")
    for j in range(tiles):
        want = (j, j) if lost is None or j < lost else "nan"
        if y[j] != want:
            raise Violation(f"tile {j} stored as {y[j]}, not {want}")


def test_schedules():
    rng = random.Random(1)
    for n in range(600):
        run_group(1 + n % 9, None, rng, _stops())


def test_a_copy_that_never_lands():
    rng = random.Random(2)
    for n in range(200):
        tiles = 1 + n % 7
        run_group(tiles, rng.randrange(tiles), rng, _stops())


def test_the_model_finds_a_wait_that_is_not_heeded():
    with pytest.raises(Violation):
        run_group(5, 2, random.Random(3), stops=False)
