"""Exhaustive check of how a CTA (or a pair of them) of the 4-bit products
leaves when a bounded wait gives up: no load and no MMA may be in flight when
shared memory and tensor memory are given back, and nothing may be stuck.

The model follows megacu_b200/csrc/kernels/fp4_gemm_kernel.cuh:
  * producers (one per CTA) wait `empty[stage]`, then load; a single CTA's first
    ring of loads, and any producer's, passes that wait at once;
  * a load counts on the leader's `full[stage]`: the leader's arrival announces
    one unit of bytes per CTA, each CTA's load takes one off when it lands, and
    the phase completes when the arrival is there and no unit is left;
  * the MMA warp waits `acc_free` of the tile before (from the second tile on),
    then `full[stage]` per k-block, and commits: to `empty` of both CTAs per
    k-block, to `acc_full` of both per tile (also of a tile it gives up in);
    commits arrive in order;
  * an epilogue per CTA waits `acc_full` and arrives on the leader's `acc_free`;
  * every one of these waits may give up whenever it does not pass, and its
    thread then goes to its end;
  * at their ends the MMA warp waits for its last commit; a single CTA's
    producer waits for the last load of every stage; the producer of a pair's
    leader waits for the MMA warp's end and, if that gave up, for the
    follower's producer's, and runs the drain over both counts;
  * the CTAs of a pair leave together.
The drains' operations come from the kernel's own header (stage_ring.h).

Planted: no wait at the producer's end unless its own wait gave up, none for
the MMAs when the free accumulator's wait gave up, a pair's drain over the
leader's loads alone. Each must be found.
"""
from __future__ import annotations

import ctypes
import functools
import os
import re
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WAIT, ANNOUNCE, COMPLETE = 0, 1, 2


@functools.lru_cache(None)
def _library():
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no C++ compiler")
    with tempfile.TemporaryDirectory() as tmp:
        so = os.path.join(tmp, "ring.so")
        subprocess.run([gxx, "-std=c++20", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                        "-I" + os.path.join(ROOT, "megacu_b200", "csrc"),
                        os.path.join(ROOT, "tests", "cpp", "stage_ring_ops.cc"), "-o", so],
                       check=True)
        return ctypes.CDLL(so)


@functools.lru_cache(None)
def drain_ops(pair, leader, follower, stages):
    out = (ctypes.c_uint32 * 192)()
    n = _library().ring_drain_ops(int(pair), leader, follower, stages, out, 64)
    assert n <= 64
    return tuple((out[3 * i], out[3 * i + 1], out[3 * i + 2]) for i in range(n))


class Violation(Exception):
    pass


def passes(count, parity):
    return (count & 1) != parity


def _set(t, i, v):
    return t[:i] + (v,) + t[i + 1:]


# A `full` barrier: (completed phases, arrivals missing, units announced and not landed).
def _settle(bar):
    phase, missing, units = bar
    return (phase + 1, 1, 0) if missing == 0 and units == 0 else bar


RUN, GAVE_UP, ENDED = 0, 1, 2


def explore(stages, tiles, kbs, ctas, mistake=None, limit=3_000_000):
    total = tiles * kbs
    # state: per producer (loads issued, RUN / GAVE_UP / ENDED, drain position),
    # MMA (k-blocks consumed, tiles committed, status), per epilogue (tiles, status),
    # full barriers, empty phases per CTA, acc_full phases per CTA, acc_free (phases, arrivals),
    # loads in flight, commits in flight (FIFO; a stage, or -1 for a tile), drain position of a pair
    start = (((0, RUN, 0),) * ctas, (0, 0, RUN), ((0, RUN),) * ctas, ((0, 1, 0),) * stages,
             ((0,) * stages,) * ctas, (0,) * ctas, (0, 0), frozenset(), (), 0)
    seen, todo = {start}, [start]
    ends = 0
    while todo:
        st = todo.pop()
        prod, mma, epi, full, empty, acc_full, acc_free, loads, commits, at = st
        nxt = []

        def to(prod=prod, mma=mma, epi=epi, full=full, empty=empty, acc_full=acc_full,
               acc_free=acc_free, loads=loads, commits=commits, at=at):
            nxt.append((prod, mma, epi, full, empty, acc_full, acc_free, loads, commits, at))

        # Loads land in any order.
        for r, i in loads:
            s = i % stages
            phase, missing, units = full[s]
            to(loads=loads - {(r, i)}, full=_set(full, s, _settle((phase, missing, units - 1))))
        # Commits arrive in order.
        if commits:
            c = commits[0]
            if c < 0:
                to(commits=commits[1:], acc_full=tuple(n + 1 for n in acc_full))
            else:
                to(commits=commits[1:], empty=tuple(_set(e, c, e[c] + 1) for e in empty))
        # Producers.
        for r, (issued, status, pos) in enumerate(prod):
            if status == RUN and issued == total:
                to(prod=_set(prod, r, (issued, ENDED, 0)))
            elif status == RUN:
                s = issued % stages
                if passes(empty[r][s], issued // stages & 1 ^ 1):
                    f = full
                    if r == 0:
                        phase, missing, units = full[s]
                        if missing != 1:
                            raise Violation("a stage announced twice")
                        f = _set(full, s, _settle((phase, 0, units + ctas)))
                    if any(i % stages == s and q == r for q, i in loads):
                        raise Violation("a stage loaded twice")
                    to(prod=_set(prod, r, (issued + 1, RUN, 0)), loads=loads | {(r, issued)},
                       full=f)
                else:
                    to(prod=_set(prod, r, (issued, GAVE_UP, 0)))
            elif ctas == 1 and not (mistake == "drain_if_gave_up" and status == ENDED):
                ops = drain_ops(False, issued, 0, stages)
                if pos < len(ops) and passes(full[ops[pos][1]][0], ops[pos][2]):
                    to(prod=_set(prod, r, (issued, status, pos + 1)))
        # MMA warp.
        used, committed, status = mma
        if status == RUN and used == total and committed == tiles:
            to(mma=(used, committed, ENDED))
        elif status == RUN:
            tile, kb = divmod(used, kbs)
            if tile > committed:  # the tile's last k-block is consumed
                to(mma=(used, committed + 1, RUN), commits=commits + (-1,))
            elif kb == 0 and tile > 0 and not passes(acc_free[0], (tile - 1) & 1):
                to(mma=(used, committed, GAVE_UP))
            else:
                s = used % stages
                if passes(full[s][0], used // stages & 1):
                    if any(i % stages == s for _, i in loads):
                        raise Violation("a stage read before its load has landed")
                    to(mma=(used + 1, committed, RUN), commits=commits + (s,))
                else:
                    to(mma=(used, committed + 1, GAVE_UP), commits=commits + (-1,))
        # Epilogues.
        for r, (done, status) in enumerate(epi):
            if status != RUN:
                continue
            if done == tiles:
                to(epi=_set(epi, r, (done, ENDED)))
            elif passes(acc_full[r], done & 1):
                phase, arrived = acc_free
                arrived += 1
                to(epi=_set(epi, r, (done + 1, RUN)),
                   acc_free=(phase + 1, 0) if arrived == ctas else (phase, arrived))
            else:
                to(epi=_set(epi, r, (done, GAVE_UP)))
        # The CTAs' end.
        at_end = mma[2] != RUN and all(e[1] != RUN for e in epi) and all(q[1] != RUN for q in prod)
        last = (mma[1] - 1) & 1
        committed_done = mma[1] == 0 or passes(acc_full[0], last)
        # given up at the free accumulator: no commit of its own stands for it
        if mistake == "no_mma_wait" and mma[2] == GAVE_UP and mma[0] % kbs == 0 and \
                mma[1] == mma[0] // kbs:
            committed_done = True
        leaving = at_end and committed_done
        if ctas == 1:
            issued, status, pos = prod[0]
            drained = pos == len(drain_ops(False, issued, 0, stages)) or (
                mistake == "drain_if_gave_up" and status == ENDED)
            leaving = leaving and drained
        elif mma[2] == GAVE_UP:
            # Once both producers and the MMA warp have ended, whatever the epilogues do.
            leaving = False
            if committed_done and all(q[1] != RUN for q in prod):
                follower = prod[0][0] if mistake == "leaders_loads_only" else prod[1][0]
                ops = drain_ops(True, prod[0][0], follower, stages)
                if at < len(ops):
                    kind, s, parity = ops[at]
                    phase, missing, units = full[s]
                    if kind == ANNOUNCE:
                        if missing != 1:
                            raise Violation("announced twice")
                        to(at=at + 1, full=_set(full, s, _settle((phase, 0, units + 1))))
                    elif kind == COMPLETE:
                        to(at=at + 1, full=_set(full, s, _settle((phase, missing, units - 1))))
                    elif passes(phase, parity):
                        to(at=at + 1)
                else:
                    leaving = at_end
        if leaving:
            if loads:
                raise Violation(f"left with loads in flight: {sorted(loads)}")
            if commits:
                raise Violation(f"left with MMAs in flight: {commits}")
            ends += 1
            continue
        if not nxt:
            raise Violation(f"stuck: {st}")
        for s2 in nxt:
            if s2 not in seen:
                seen.add(s2)
                if len(seen) > limit:
                    raise RuntimeError("state space larger than the limit")
                todo.append(s2)
    assert ends > 0
    return len(seen)


SINGLE = [(n, t, k) for n in (1, 2, 3) for t in (1, 2, 3) for k in (1, 2, 3)]
PAIR = [(1, 1, 2), (1, 2, 1), (1, 3, 2), (2, 1, 1), (2, 1, 4), (2, 2, 2), (2, 3, 1), (3, 1, 3),
        (3, 2, 2), (3, 1, 5), (2, 3, 3), (3, 3, 2), (4, 1, 6)]


@pytest.mark.parametrize("stages,tiles,kbs", SINGLE)
def test_a_cta_leaves_nothing_in_flight(stages, tiles, kbs):
    assert explore(stages, tiles, kbs, 1) > 1


@pytest.mark.parametrize("stages,tiles,kbs", PAIR)
def test_a_pair_leaves_nothing_in_flight(stages, tiles, kbs):
    assert explore(stages, tiles, kbs, 2) > 1


@pytest.mark.parametrize("mistake,ctas,case", [
    ("drain_if_gave_up", 1, (2, 1, 2)), ("drain_if_gave_up", 1, (3, 2, 1)),
    ("no_mma_wait", 1, (2, 2, 1)), ("no_mma_wait", 1, (3, 3, 2)),
    ("leaders_loads_only", 2, (2, 1, 4)), ("leaders_loads_only", 2, (1, 2, 1))])
def test_planted_mistakes_are_found(mistake, ctas, case):
    with pytest.raises(Violation):
        explore(*case, ctas, mistake=mistake)


@pytest.mark.parametrize("stages", [1, 4, 7, 15])
def test_drain_waits_for_the_last_load_of_every_stage(stages):
    for issued in range(4 * stages + 2):
        want = {}
        for i in range(issued):
            want[i % stages] = i // stages & 1
        ops = drain_ops(False, issued, 0, stages)
        assert {s: parity for _, s, parity in ops} == want and len(ops) == len(want)


def test_whole_warps_give_up():
    """A wait that may give up decides once for all lanes of its warp: lanes
    that disagree would meet different warp-wide instructions."""
    path = os.path.join(ROOT, "megacu_b200", "csrc", "kernels", "fp4_gemm_kernel.cuh")
    body = open(path).read().split("fp4_gemm_kernel(__grid_constant__", 1)[1]
    calls = re.findall(r"(\w+)\([^;{]*abort_word, p\.timeout_ns\)", body)
    assert len(calls) == 4 and set(calls) == {"warp_wait"}
