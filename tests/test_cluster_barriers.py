"""The cluster barriers are of the aligned kind: a warp has to come to them as one.  So between the block's or warp's
last synchronisation and the barrier no conditional block may have ended, wherever the barrier stands."""
import re

import pytest

from conftest import PKG

SOURCES = sorted((PKG / "csrc").glob("*.cu"))


def places(source):
    """Of each call of cluster_arrive: its line, and whether a block ends between the synchronisation in front and it."""
    lines = [re.sub(r"//.*", "", line).strip() for line in source.splitlines()]
    for at, line in enumerate(lines):
        if "cluster_arrive();" not in line:
            continue
        ended = False
        for before in reversed(lines[:at]):
            if "__syncwarp();" in before or "__syncthreads();" in before:
                break
            ended = ended or before.startswith("}")
        yield at + 1, ended


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_warps_come_to_cluster_barriers_as_one(path):
    assert [line for line, ended in places(path.read_text()) if ended] == []


def test_the_check_sees_a_block_that_ends_in_front_of_a_barrier():
    good = "__syncwarp();\nif (split > 1) {\n  cluster_arrive();  // }\n}\n"
    bad = "__syncthreads();\nif (tid == 0) {\n  x = 1;\n}\ncluster_arrive();\n"
    assert list(places(good)) == [(3, False)] and list(places(bad)) == [(5, True)]
