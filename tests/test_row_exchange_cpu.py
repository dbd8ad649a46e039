"""The threads of a row in the paged prompts' kernel tell each other their maxima over slots in shared memory, which every tile uses again: whatever the
order in which the row's warps go on, each has to read what the others wrote for the same tile.  The steps are taken from the source, in their order."""
import re
from pathlib import Path

import pytest

TEXT = (Path(__file__).resolve().parent.parent / "runnburn_b200" / "csrc" / "paged_prefill.cuh").read_text()


def steps(text):
    """The barriers, writes and reads of the slots, in their order; the reads behind one barrier are one step."""
    found = []
    for m in re.finditer(r"(?<![\w.])meet\(\);|\*say = |heard\(", re.sub(r"//[^\n]*", "", text)):
        step = {"m": "meet", "*": "write", "h": "read"}[m.group(0)[0]]
        if step != "read" or found[-1:] != ["read"]:
            found.append(step)
    return found


def between(first, last):
    at = TEXT.index(first)
    return TEXT[at:TEXT.index(last, at)]


TILE = steps(between("uint32_t s[KEYS];", "l_run = fmaf(l_run, corr"))
END = steps(between("// ---- the row's end ----", "auto output = "))
GIVEN_UP = steps(between("if (!ok) {   // a row's warps meet in every tile", "uint32_t s[KEYS];"))


def stale_read(warps, tiles):
    """Walks through every order in which the warps can take their steps; a read of another tile's value, or None."""
    program = [(step, t) for t in range(tiles) for step in TILE] + [(step, tiles) for step in END]
    seen, left = set(), [((0,) * warps, (None,) * warps)]
    while left:
        at, slots = left.pop()
        if (at, slots) in seen:
            continue
        seen.add((at, slots))
        waiting = [w for w in range(warps) if at[w] < len(program) and program[at[w]][0] == "meet"]
        if len(waiting) == warps:
            left.append((tuple(a + 1 for a in at), slots))
            continue
        for w in range(warps):
            if at[w] == len(program) or w in waiting:
                continue
            step, t = program[at[w]]
            now = slots
            if step == "write":
                now = slots[:w] + (t,) + slots[w + 1:]
            elif any(x != t for x in slots):
                return f"warp {w} reads {slots} in tile {t}"
            left.append((at[:w] + (at[w] + 1,) + at[w + 1:], now))
        if not any(a < len(program) for a in at):
            continue
    return None


@pytest.mark.parametrize("warps", [2, 4])
def test_a_row_s_warps_read_the_same_tile_s_maxima(warps):
    assert TILE.count("write") == 1 and TILE.count("read") == 1 and END.count("write") == 1 and END.count("read") == 1
    assert stale_read(warps, 3) is None


def test_warps_that_have_given_up_meet_as_often():
    """A barrier counts whole warps: one that skips a tile's work meets the others at each of its barriers."""
    assert GIVEN_UP == ["meet"] * TILE.count("meet")
