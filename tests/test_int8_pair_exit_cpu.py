"""The CTA pairs of the int8 product: every signal that one CTA sends to the other's barriers is waited for before the kernel ends. The
exit barrier of the cluster is relaxed and orders nothing, so a signal that nobody waits for could reach shared memory that its owner
has left. Replayed with the conditions that stand in the source, since a late signal rarely shows."""
import os
import re

import pytest

from conftest import ROOT

SOURCE = open(os.path.join(ROOT, "sglang_b200", "csrc", "int8_gemm_pair.cuh")).read()


def guard_of_the_arrival():
    m = re.search(r"if \(lane == 0(?: && (?P<guard>[^;]*))?\) ptx::mbar_arrive_cluster\(leader_tempty \+ 8 \* b\);", SOURCE)
    assert m, "no arrival on the leader's tempty barriers"
    return m.group("guard") or "True"


@pytest.mark.parametrize("npairs", [1, 2, 5, 74])
def test_every_arrival_on_tempty_is_waited_for(npairs):
    guard = guard_of_the_arrival()
    for tiles in list(range(npairs, 6 * npairs + 3)) + [11 * npairs + 1]:
        for pair in (0, npairs // 2, npairs - 1):
            mine = list(range(pair, tiles, npairs))
            arrived, waited = [0, 0], [0, 0]
            for i, t in enumerate(mine):
                # the issuer's wait before the products of its i-th tile: on the phase that the tile two before it completes
                if i >= 2:
                    waited[i % 2] += 1
                if eval(guard.replace("&&", "and"), {}, {"t": t, "npairs": npairs, "tiles": tiles}):
                    arrived[i % 2] += 1
            assert arrived == waited, (npairs, tiles, pair)


def test_the_other_signals_between_the_ctas_are_waited_for():
    """The producers wait for every stage's last release; full, tfull and the sums' bytes are waited for by whoever uses the data."""
    producer = SOURCE[SOURCE.index("if (warp == Cfg::kProducerWarp) {\n    if (ptx::elect_one())"):SOURCE.index("} else if (warp == Cfg::kMmaWarp)")]
    assert re.search(r"for \(int i = 0; i < S && ok; \+\+i\) \{\s*ok = ptx::mbar_wait\(empty_bar\(s\), phase", producer)
    assert "ptx::mbar_wait(full_bar(s)" in SOURCE and "ptx::mbar_wait(tfull_bar(b)" in SOURCE and "ptx::mbar_wait_cluster(sum_bar" in SOURCE
