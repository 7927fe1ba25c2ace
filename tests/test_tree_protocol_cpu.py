"""Interleaving check of the barriers of the tree attention kernel with 128-row tiles (csrc/tree_attn_tile_sm100.cu).

Every role of the kernel is a program of steps; a step waits for phases of barriers, then arrives on others.  A barrier's wait knows the
parity of a phase only, as on the GPU: it passes when the phase in progress has the other parity.  Every interleaving of a part's roles is
walked (the tensor core, which runs products in order some time after their issue, is a role of its own); reported are

* an *overrun* - a wait that passed on another phase than its own,
* a *stale* read - query scales of another unit, an output that the next unit has begun to overwrite, and
* a *deadlock*.
"""
from __future__ import annotations

from typing import Optional

import pytest

KST, VST, SLOTS = 2, 2, 8


class Part:
    """The roles' programs for a part whose segments have the given numbers of tiles.  ``idle_groups_wait``: a softmax group waits for a unit's
    queries at the unit's start, even if it has no tile of it.  ``by_hand``: the softmax groups read every value tile themselves (values
    that are not finite)."""

    def __init__(self, segments: list[int], fp8: bool, idle_groups_wait: bool = False, by_hand: bool = False) -> None:
        self.fp8, rst = fp8, 3 if fp8 else 2
        seg_of = [s for s, n in enumerate(segments) for _ in range(n)]
        begin = [sum(segments[:s]) for s in range(len(segments) + 1)]
        tiles = len(seg_of)
        roles: dict[str, list[tuple]] = {n: [] for n in ("k", "v", "mma", "meta", "val", "g0", "g1")}

        def step(role, waits=(), arrives=(), read=None, write=None, issue=None):
            roles[role].append((tuple(waits), tuple(arrives), read, write, issue))

        for j in range(tiles):
            step("k", [(("k_empty", j % KST), j // KST - 1)], [("k_full", j % KST)])
            if fp8:
                step("v", [(("r_empty", j % rst), j // rst - 1)], [("r_full", j % rst)])
            else:
                step("v", [(("pv_done", j % VST), j // VST - 1)], [("r_full", j % rst)])
            step("meta", [(("r_full", j % rst), j // rst)], [("f_ready", j % SLOTS)] + ([("r_empty", j % rst)] if fp8 else []))
        # values and queries
        loaded = 0
        for j in range(tiles):
            s, at = seg_of[j], j - begin[seg_of[j]]
            ahead = at == 1 and loaded == s + 1 and begin[s + 1] < tiles
            if loaded <= s or ahead:
                want = s if loaded <= s else s + 1
                step("val", [(("pv_done", (j - 2) % VST), (j - 2) // VST)] if j >= 2 else [], [("q_ready", want & 1)], write=(want & 1, want))
                loaded = want + 1
            waits = [(("f_ready", j % SLOTS), j // SLOTS)] + ([(("pv_done", j % VST), (j - 2) // VST)] if fp8 and j >= 2 else [])
            step("val", waits, [("v_ready", j % VST)] + ([("r_empty", j % rst)] if fp8 else []))

        # products: issued here, run by the role "tensor" in order
        def scores(j):
            s = seg_of[j]
            waits = [(("q_ready", s & 1), s >> 1)] if j == begin[s] else []
            step("mma", waits + [(("k_full", j % KST), j // KST)], issue=("s", j, s))

        for j in range(min(2, tiles)):
            scores(j)
        for j in range(tiles):
            step("mma", [(("v_ready", j % VST), j // VST), (("p_ready", j & 1), j >> 1)], issue=("o", j, seg_of[j]))
            if j + 2 < tiles:
                scores(j + 2)
        # softmax groups
        turn = 0
        for s in range(len(segments)):
            for g in (0, 1):
                mine = [j for j in range(begin[s], begin[s + 1]) if j & 1 == g]
                if fp8 and (mine or idle_groups_wait):
                    step(f"g{g}", [(("q_ready", s & 1), s >> 1)], read=("q", s))
                for j in mine:
                    step(f"g{g}", [(("s_full", g), j >> 1), (("f_ready", j % SLOTS), j // SLOTS)])
                    step(f"g{g}", [(("v_ready", j % VST), j // VST)] if by_hand else [], [("p_ready", g)])
                step(f"g{g}", arrives=[("xch", 0)])
                last = begin[s + 1] - 1
                step(f"g{g}", [(("xch", 0), turn), (("pv_done", last % VST), last // VST)], read=("o", s))
                step(f"g{g}", arrives=[("xch", 0)])
                step(f"g{g}", [(("xch", 0), turn + 1)])
            turn += 2
        self.names = list(roles) + ["tensor"]
        self.programs = [roles[n] for n in roles]
        self.count = {"xch": 2, "r_empty": 2}          # arrivals per phase (others: one)

    def explore(self) -> Optional[str]:
        start = ((0,) * len(self.programs), (), (), (), 0)         # counters, arrivals per barrier, products issued, query buffers, units begun
        seen, stack = {start}, [start]
        while stack:
            pcs, bars, queue, held, begun = stack.pop()
            arrived, bufs = dict(bars), dict(held)

            def done(b):                                            # phases completed
                return arrived.get(b, 0) // self.count.get(b[0], 1)

            moves = []
            for r, prog in enumerate(self.programs):
                if pcs[r] == len(prog):
                    continue
                waits, arrives, read, write, issue = prog[pcs[r]]
                if any((done(b) & 1) == (phase & 1) for b, phase in waits):
                    continue
                where = f"{self.names[r]}, step {pcs[r]}"
                for b, phase in waits:
                    if done(b) != phase + 1:
                        return f"overrun at {where}: {b} is in phase {done(b)}, waited for the end of {phase}"
                if read is not None:
                    what, s = read
                    if what == "q" and bufs.get(s & 1) != s:
                        return f"stale at {where}: scales of unit {bufs.get(s & 1)}, not {s}"
                    if what == "o" and begun > s:
                        return f"stale at {where}: the output of unit {s} is being overwritten"
                now, kept = dict(arrived), dict(bufs)
                for b in arrives:
                    now[b] = now.get(b, 0) + 1
                if write is not None:
                    kept[write[0]] = write[1]
                moves.append((pcs[:r] + (pcs[r] + 1,) + pcs[r + 1:], tuple(sorted(now.items())), queue + ((issue,) if issue else ()),
                              tuple(sorted(kept.items())), begun))
            if queue:
                kind, j, s = queue[0]
                now = dict(arrived)
                if kind == "s":
                    if bufs.get(s & 1) != s:
                        return f"stale: scores of tile {j} from the queries of unit {bufs.get(s & 1)}, not {s}"
                    hit = [("s_full", j & 1), ("k_empty", j % KST)]
                else:
                    hit = [("pv_done", j % VST)]
                for b in hit:
                    now[b] = now.get(b, 0) + 1
                moves.append((pcs, tuple(sorted(now.items())), queue[1:], held, max(begun, s) if kind == "o" else begun))
            if not moves and any(pc < len(p) for pc, p in zip(pcs, self.programs)):
                return f"deadlock at {dict(zip(self.names, pcs))}"
            for m in moves:
                if m not in seen:
                    seen.add(m)
                    stack.append(m)
        return None


SEGMENTS = [[1], [2], [1, 1, 1], [2, 1, 1], [1, 2, 1], [1, 1, 2], [3, 1]]


@pytest.mark.parametrize("by_hand", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("segments", SEGMENTS, ids=str)
def test_no_role_overruns_another(segments, fp8, by_hand):
    assert Part(segments, fp8, by_hand=by_hand).explore() is None


def test_a_group_without_a_tile_must_not_wait_for_the_queries():
    """A unit of one tile is finished by one group; the queries two units on may then be in the buffer, and its barrier a phase further,
    before the other group has looked."""
    found = [Part(s, True, idle_groups_wait=True).explore() for s in SEGMENTS]
    assert any(f and ("overrun" in f or "stale" in f or "deadlock" in f) for f in found)
