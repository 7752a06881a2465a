"""CPU: the turns that two softmax warps take at the special-function pipe end whatever either of them gives up on.  The order of the
barrier operations comes from the kernel's own header, compiled for the host; a walk over every interleaving of the two warps finds
the states in which one of them would wait for ever."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "attention_turns.cuh"
struct Log { void sync() { putchar('s'); } void arrive() { putchar('a'); } };
// every way through the turns: argv = the number of turns; a line per warp and point at which it gives up (-1: it does not),
// before taking turn j (work = 0) or behind passing it on (work = 1), as in the loop over the tiles
int main(int, char** argv) {
    const int turns = atoi(argv[1]), tiles = atoi(argv[2]);
    for (int second = 0; second < 2; ++second)
        for (int stop = -1; stop < tiles; ++stop)
            for (int after = 0; after < (stop < 0 ? 1 : 2); ++after) {
                printf("%d ", second);
                sq::AttnTurns<Log> t = {Log(), turns, second};
                bool ok = true;
                t.open();
                int j = 0;
                for (; j < tiles; ++j) {
                    if (j == stop && !after) { ok = false; break; }
                    t.take(j);
                    t.pass(j);
                    if (j == stop) { ++j; ok = false; break; }
                }
                if (!ok) t.leave(j);
                putchar('\n');
            }
}
"""


def _stuck(ops0, ops1):
    """True if some interleaving leaves a warp waiting for ever.  A barrier completes with the second of two arrivals, whether they
    wait or not, and starts again; warp w waits at barrier w and arrives at barrier 1 - w."""
    seqs = (ops0, ops1)
    seen, todo = set(), [(0, 0, 0, 0, False, False)]             # positions, arrivals at either barrier, waiting
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        moved = False
        for w in (0, 1):
            at, count, wait = list(state[:2]), list(state[2:4]), list(state[4:])
            if wait[w] or at[w] == len(seqs[w]):
                continue
            moved = True
            op = seqs[w][at[w]]
            at[w] += 1
            bar = w if op == "s" else 1 - w
            count[bar] += 1
            wait[w] = op == "s"
            if count[bar] == 2:
                count[bar] = 0
                wait[bar] = False                                # only warp `bar` ever waits there
            todo.append((*at, *count, *wait))
        if not moved and any(state[4:]):
            return True
    return False


def test_the_walk_finds_lost_turns():
    assert not _stuck("sasa", "asas")
    assert _stuck("sasasa", "aasas")                             # two arrivals in a row: the first two complete a phase by themselves
    assert _stuck("sa", "")


@pytest.mark.parametrize("turns", range(0, 7))
def test_every_wait_ends_wherever_a_warp_gives_up(tmp_path, turns):
    src, exe = tmp_path / "turns.cpp", tmp_path / "turns"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "segquant_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    ways = [[], []]
    for tiles in {turns, turns + 2}:                             # a sub-tile may have more tiles than turns
        for line in subprocess.run([str(exe), str(turns), str(tiles)], check=True, capture_output=True, text=True).stdout.splitlines():
            who, _, ops = line.partition(" ")
            ways[int(who)].append(ops)
    for a in set(ways[0]):
        for b in set(ways[1]):
            assert not _stuck(a, b), (a, b)
