"""CPU: what the header says of the serving entry points against what the library does, where no device is needed."""
import re
from pathlib import Path

from arke_b200 import _lib, ops

HEADER = (Path(__file__).resolve().parent.parent / "include" / "arke_b200.h").read_text()


def test_the_default_of_paged_prefix_kb_is_the_documented_one():
    """The workspace has room for a prefix of its own from the option's size on: asked for around the documented default,
    the unset option and that value have to agree, and sizes on both sides of it have to differ."""
    told = int(re.search(r'"paged_prefix_kb".*?0 = default, (\d+)\)', HEADER, re.S).group(1))
    B, Hq, Hkv, D = 9, 32, 8, 128
    per = (B - 1) * Hkv * D * 4                         # bytes of re-read keys and values that a position of the prefix saves
    edge = told * 1024 // per
    near = [edge - 1, edge, edge + 1, edge // 2, edge * 2]

    def sizes():
        return [_lib.LIB.arke_b200_paged_gqa_workspace(B, B, Hq, Hkv, D, n) for n in near]

    unset = sizes()
    with ops.options(paged_prefix_kb=told):
        assert sizes() == unset
    assert unset[0] == unset[1] == unset[3] < unset[2] == unset[4]
    with ops.options(paged_prefix_kb=told * 2):
        assert sizes() != unset
