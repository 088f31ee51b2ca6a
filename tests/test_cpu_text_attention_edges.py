"""The language models' attention at its edges, as far as a CPU shows it."""
import re
import subprocess
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


@pytest.mark.parametrize("stages", [2, 3])
def test_a_prompt_that_gives_up_waits_for_all_its_copies(stages, tmp_path):
    """The forward kernel's loop behind a wait that ran out, compiled for the host with barriers that write down who waits for them: the last copy of Q and
    the last one into every place of K and V, whatever the number of copies so far (K and V of a key tile in turn, one Q per item)."""
    text = (CSRC / "text_attention_fwd.cu").read_text()
    loop = re.search(r"\n( +)for \(int j = max\(loads.*?\n\1}\n", text, re.S)
    assert loop, "the loop over the copies on the way"
    source, program = tmp_path / "landing.cpp", tmp_path / "landing"
    source.write_text("""
#include <algorithm>
#include <cstdint>
#include <cstdio>
using std::max;
constexpr int STAGES = %d;
uint64_t q_full, k_full[STAGES], v_full[STAGES];
uint64_t globaltimer_ns() { return 0; }
bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  if (bar == &q_full) printf(" q,0,%%u", parity);
  else if (bar >= k_full && bar < k_full + STAGES) printf(" k,%%d,%%u", (int)(bar - k_full), parity);
  else printf(" v,%%d,%%u", (int)(bar - v_full), parity);
  return true;
}
int main() {
  for (int loads = 0; loads <= 6 * STAGES + 1; ++loads)
    for (int n_items = 0; n_items <= 4; ++n_items) {
      printf("%%d %%d", loads, n_items);
%s
      printf("\\n");
    }
}
""" % (stages, loop.group(0)))
    subprocess.run(["g++", "-std=c++17", "-o", str(program), str(source)], check=True)
    lines = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == (6 * stages + 2) * 5
    for line in lines:
        loads, items, *waits = line.split()
        want = {("q", 0): (int(items) - 1) % 2} if int(items) else {}
        for j in range(int(loads)):
            want["kv"[j % 2], j // 2 % stages] = j // 2 // stages % 2
        got = {(kind, int(place)): int(parity) for kind, place, parity in (w.split(",") for w in waits)}
        assert len(waits) == len(got) and got == want, line
