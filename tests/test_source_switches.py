"""The planner that the products on the matrix cores share weighs every tile, however it is compiled."""
import os
import re

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "approxtrain_amd", "csrc", "amsim_tiles.h")


def test_no_switch_forces_a_tile():
    with open(HEADER) as f:
        source = f.read()
    names = re.findall(r"^\s*#\s*(?:ifdef|ifndef|if|elif)\s+(.*?)\s*(?://.*)?$", source, re.M)
    assert names == ["AMSIM_TILES_H_", "__HIP_DEVICE_COMPILE__"]
    planner = source[source.index("Plan make_plan("):]
    loop = re.search(r"for \(int i = 0; i < 4; \+\+i\) \{\s*\n(.*?)\n", planner).group(1)
    assert loop.strip() == "Plan p{i, {}};"
