"""The order of copies, waits, barriers and reads of the long-chunk kernel (csrc/paged_attn_chunk.hip), followed tile by tile for
both groups of its wavefronts, with the numbers of its waits as they stand in the source.

A tile is copied by all eight wavefronts, a share each, so that a wavefront may read one only if every wavefront has waited for its own
share before a barrier that both have passed; and a copy may go to the place of an earlier tile only if every wavefront has
done its reads of that before such a barrier."""
import os
import re

import pytest

import mercury_artifact_amd as M

STAGES = 4


def _waits():
    with open(os.path.join(os.path.dirname(M.__file__), "csrc", "paged_attn_chunk.hip")) as f:
        counts = [int(n) for n in re.findall(r's_waitcnt vmcnt\((\d+)\)', f.read())]
    assert len(counts) == 5 and counts[0] == counts[4] == 0      # Q; first tile, loop's first phase, loop; copies past the last tile
    return counts[1:4]


class Wavefront:
    """What one wavefront does in the order of its program; `at` counts the barriers it has passed."""

    def __init__(self):
        self.at = 0
        self.flying = []                   # copies in flight, an entry for each instruction, the oldest first
        self.copied, self.waited, self.reads = {}, {}, {}

    def copy(self, tile):
        self.copied[tile] = self.at
        self.flying += [tile, tile]        # 8 rows are two instructions

    def wait(self, count):
        done, self.flying = self.flying[:max(len(self.flying) - count, 0)], self.flying[max(len(self.flying) - count, 0):]
        for tile in done:
            if tile not in self.flying:
                self.waited.setdefault(tile, self.at)

    def read(self, tile, done_after=0):
        self.reads.setdefault(tile, []).append((self.at, self.at + done_after))

    def barrier(self):
        self.at += 1


def _run(ntiles, group_b, copies_in_matrix_phase, waits):
    first, second, loop = waits
    w = Wavefront()
    for t in range(4):
        w.copy(("K", t))
        if t < 3:
            w.copy(("V", t))
    w.wait(first)
    w.barrier()
    w.read(("K", 0))
    w.wait(second)
    w.barrier()
    if ntiles > 1:
        w.read(("K", 1), int(group_b))      # the first operands: there before the products that take them
    if group_b:
        w.barrier()
    for t in range(ntiles - 1):
        if copies_in_matrix_phase:
            w.copy(("K", t + 4)), w.copy(("V", t + 3))
        w.read(("K", t + 1)), w.read(("V", t))
        w.barrier()
        if not copies_in_matrix_phase:
            w.copy(("K", t + 4)), w.copy(("V", t + 3))
        if t + 2 < ntiles:
            w.read(("K", t + 2), 1)
        w.wait(loop)
        w.barrier()
    w.read(("V", ntiles - 1))
    if not group_b:
        w.barrier()
    return w


def _faults(ntiles, copies_in_matrix_phase, waits):
    wavefronts = [_run(ntiles, b, copies_in_matrix_phase, waits) for b in (False, True)]
    assert wavefronts[0].at == wavefronts[1].at          # as many barriers
    found = []
    for reader in wavefronts:
        for tile, reads in reader.reads.items():
            for begin, end in reads:
                for writer in wavefronts:
                    if not writer.waited.get(tile, 10 ** 9) < begin:
                        found.append(("read before it is there", tile))
                    later = writer.copied.get((tile[0], tile[1] + STAGES))
                    if later is not None and not end < later:
                        found.append(("overwritten while it is read", tile))
    return found


@pytest.mark.parametrize("copies_in_matrix_phase", [False, True])
def test_every_tile_is_there_before_it_is_read_and_until_then(copies_in_matrix_phase):
    for ntiles in range(1, 12):
        assert _faults(ntiles, copies_in_matrix_phase, _waits()) == [], ntiles


def test_the_model_sees_a_wait_that_is_too_short():
    """Each wait by one tile's copies: planted here, in the model alone."""
    waits = [12, 4, 4]
    for i in range(3):
        short = list(waits)
        short[i] += 2
        assert any(_faults(n, m, short) for n in range(1, 12) for m in (False, True)), i
