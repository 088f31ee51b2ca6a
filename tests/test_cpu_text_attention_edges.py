"""The language models' attention at its edges, as far as a CPU shows it."""
import re
from pathlib import Path

import pytest

import mojodiffusion_b200

CSRC = Path(mojodiffusion_b200.__file__).parent / "csrc"


def _some_order_ends_in_a_deadlock(places, tiles=7):
    """All orders of the three parties that pass the staged queries of the dk / dv kernel with one score buffer: the warp that stages, another warp of its
    group, and the issuer of the products. A barrier is the number of phases that it has behind it; waiting for phase n, a warp sees only whether the
    phase that now runs has another parity than n, as mbarrier.try_wait.parity tells."""
    stager, other, issuer = [], [], [("end", "scores", 0)]
    for i in range(tiles):
        wait = [("wait", f"staged{i % places}", i // places), ("wait", "scores", i), ("arrive", "probabilities", i)]
        stager += [("end", f"staged{i % places}", i // places)] + wait
        other += wait
        issuer += [("wait", "probabilities", i)] + ([("end", "scores", i + 1)] if i + 1 < tiles else [])
    programs = (stager, other, issuer)
    start = ((0, 0, 0), (("probabilities", 0), ("scores", 0), *((f"staged{p}", 0) for p in range(places))), 0)
    todo, known = [start], {start}
    while todo:
        at, barriers, arrived = todo.pop()
        moved = False
        for w, program in enumerate(programs):
            if at[w] == len(program):
                continue
            do, name, n = program[at[w]]
            phases, here = dict(barriers), arrived
            if do == "wait" and phases[name] % 2 == n % 2:
                continue
            if do == "end":
                phases[name] += 1
            elif do == "arrive":
                here = (here + 1) % 2
                phases[name] += here == 0
            moved = True
            after = (tuple(p + (v == w) for v, p in enumerate(at)), tuple(sorted(phases.items())), here)
            if after not in known:
                known.add(after)
                todo.append(after)
        if not moved and any(at[w] < len(program) for w, program in enumerate(programs)):
            return True
    return False


def test_the_model_of_the_staged_queries():
    assert _some_order_ends_in_a_deadlock(1) and not _some_order_ends_in_a_deadlock(2)


def test_staged_queries_cannot_lose_a_warp():
    """Heads of 64 have one score buffer: the barriers per warpgroup that the kernel declares leave no order in which its warps wait for ever."""
    text = (CSRC / "text_attention_bwd.cu").read_text()
    declared = re.search(r"\blv_full\[2\](?:\[(\w+)\])?", text).group(1)
    given = re.search(r"constexpr int PLACES = 3 - BUFS;", text) if declared == "PLACES" else None
    assert not _some_order_ends_in_a_deadlock(2 if given else 1)
