"""Who sees which key, in the attention over the paged cache with rows in the lanes: four warps write bits into a table, meet at a barrier and read each
other's. Nothing else holds a warp back from the next tile that is masked, so what it writes there must not be what the others still read. Replayed
with the table's place as it stands in the source, since the mistake rarely shows."""
import os
import re

import pytest

from conftest import ROOT

SOURCE = open(os.path.join(ROOT, "sglang_b200", "csrc", "tree_attention.cu")).read()
ROWS_IN_LANES = SOURCE[SOURCE.index("// A thread per row"):SOURCE.index("// (the barrier also says that this segment's tables have been read)")]


def place_of():
    m = re.search(r"words = seen_words \+ (\(.*?\)|\w+) \* NT \* 4;", ROWS_IN_LANES)
    assert m, "no table of words"
    return lambda tile, group: eval(m.group(1), {}, {"own": tile & 1, "group": group})


@pytest.mark.parametrize("first", [0, 1])
def test_no_warp_writes_what_another_may_still_read(first):
    place = place_of()
    writes, barrier, reads = (ROWS_IN_LANES.index(t) for t in ("words[(i0 + i) * 4 + (warp & 3)] = word;", "ptx::any_of(bar, 128, false);", "= words[(token"))
    assert writes < barrier < reads
    tiles = range(first, first + 8)
    for group in (0, 1):
        for t in tiles:
            for later in tiles:
                # A warp that writes at `later` has passed the barrier of the tile before it, which the others reach with the tile before that read
                if later > t and not later - 1 >= t + 1:
                    assert place(later, group) != place(t, group), (group, t, later)


def test_the_tables_of_both_groups_lie_apart_and_fit():
    place = place_of()
    places = {place(t, g) for t in range(4) for g in range(2)}
    assert len(places) == len({(t & 1, g) for t in range(4) for g in range(2)}) == 4 and max(places) == 3
    m = re.search(r"kTables = NT \* 4 \* \(kRowsInLanes \? 4 \+ 2 \+ 2 \+ (\d+) :", SOURCE)
    assert m and int(m.group(1)) >= 4 * len(places)
