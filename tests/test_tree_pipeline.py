"""How far the softmax warps of the tree attention kernel can run apart (no GPU).

A model of the kernel's barriers.  Tiles are numbered through all segments of
a CTA; tile i's scores S(i) and its product PV(i) run in issue order
(S(0), S(1), then PV(i), S(i + 2) for every i), PV(i) once all four warps have
arrived for tile i.  Every warp waits for S(i), cleans V (which has to be
loaded: with a ring of n slots after PV(i - n)), notes a segment that holds a
non-finite draft and arrives.  At a segment's end a warp with rows of its own
waits for the last PV and then reads the note; one without goes on.

One warp is stopped just before it reads its note and all else runs as far as
it can: no note of a later segment may have taken the entry's place.
"""

from __future__ import annotations

import itertools
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "vllm_mps_b200", "csrc", "paged_tree.cu")
WARPS = 4


def _entries():
    masks = {int(x) for x in re.findall(r"odd_seg\[seg & (\d+)\]", open(SOURCE).read())}
    assert len(masks) == 1  # written and read the same way
    return masks.pop() + 1


def _run(lengths, active, stages, stopped, at_segment):
    """The furthest segment in which any warp has cleaned V when ``stopped`` waits before
    reading segment ``at_segment``'s note and nothing else can move."""
    seg_of = [s for s, n in enumerate(lengths) for _ in range(n)]
    tiles = len(seg_of)
    last = [seg_of[i + 1:i + 2] != [seg_of[i]] for i in range(tiles)]
    qk, pv = min(2, tiles), 0  # how many have completed
    arrived = [0] * WARPS      # tiles each warp has arrived for
    reads = [0] * WARPS        # tiles whose segment end it has passed
    cleaned = -1
    moved = True
    while moved:
        moved = False
        if pv < tiles and all(a > pv for a in arrived):
            pv += 1
            qk = min(tiles, qk + 1)
            moved = True
        for w in range(WARPS):
            i = arrived[w]
            if reads[w] < i:  # between arriving for tile i - 1 and what follows
                seg = seg_of[i - 1]
                if last[i - 1] and active[w][seg]:
                    if pv < i or (w == stopped and seg == at_segment):
                        continue
                reads[w] = i
                moved = True
            elif i < tiles and qk > i and pv >= i - stages + 1:
                cleaned = max(cleaned, seg_of[i])
                arrived[w] = i + 1
                moved = True
    return cleaned, arrived[stopped]


@pytest.mark.parametrize("stages", [2, 4])
def test_a_note_is_read_before_its_entry_is_taken_again(stages):
    entries = _entries()
    furthest = 0
    for lengths in itertools.product((1, 2), repeat=5):
        for idle in itertools.product((False, True), repeat=5):
            # Warp 3 always has rows, warp 0 has none where ``idle`` says so.
            active = [[not x for x in idle], [True] * 5, [True] * 5, [True] * 5]
            for seg in range(5):
                ahead, at = _run(lengths, active, stages, 3, seg)
                assert at >= sum(lengths[:seg + 1])  # it did get there
                furthest = max(furthest, ahead - seg)
                for later in range(seg + 1, ahead + 1):
                    assert (later - seg) % entries, (lengths, idle, seg, later)
    assert furthest == 2
