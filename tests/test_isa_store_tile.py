"""The outputs of the 4-bit products' tiles go from lane to lane of a wave through LDS: in the gfx950 assembly a wave barrier stands between every write
there and the reads behind it, and between reads and the writes that overwrite what they read."""
import re
from pathlib import Path

import pytest

from tests.test_isa_lds_waits import HIPCC
from tests.test_isa_mx4 import _assembly


def unordered(lines):
    """Reads behind writes, and writes behind reads, with no barrier between; and how many barriers there are."""
    last, bad, barriers = None, [], 0
    for line in lines:
        if "wave barrier" in line:
            last, barriers = None, barriers + 1
        op = re.match(r"\s+(ds_read|ds_write)", line)
        if op and last not in (None, op.group(1)):
            bad.append(line.strip())
        if op:
            last = op.group(1)
    return bad, barriers


def test_the_scan():
    assert unordered(["  ds_write_b128 v1, v2", "  ds_read_b128 v3, v1"]) == (["ds_read_b128 v3, v1"], 0)
    assert unordered(["  ds_write_b128 v1, v2", " ; wave barrier", "  ds_read_b128 v3, v1", "  ds_write_b128 v1, v3"]) == (["ds_write_b128 v1, v3"], 1)
    assert unordered([" ; wave barrier", "  ds_write_b128 v1, v2", " ; wave barrier", "  ds_read_b128 v3, v1", " ; wave barrier", "  ds_write_b128 v1, v3"]) == ([], 3)


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not found")
def test_stores(tmp_path):
    _, bodies = _assembly("mx4_api.hip", tmp_path)
    seen = 0
    for k, body in bodies.items():
        if "mx4_tile_kernel" in k or "mx4_wide_kernel" in k:
            bad, barriers = unordered(body[body.rindex("s_barrier"):].split("\n"))
            assert not bad and barriers >= 2, (k, bad[:3], barriers)
            seen += 1
    assert seen == 6
