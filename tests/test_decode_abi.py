"""`ek_launch_list` (include/enceladus_hip.h): what it refuses before any launch (CPU)."""

import struct

import pytest

from enceladus_amd.compiler.errors import HipError
from enceladus_amd.runtime import hip


@pytest.mark.parametrize("packed", [
    b"", b"\0" * 15, struct.pack("<QII", 0, 1, 0), struct.pack("<QII", 0, 0, 8),
    struct.pack("<QII", 0, 1, 8) + b"\0" * 24, struct.pack("<QII", 0, 0xFFFFFFFF, 0),
    struct.pack("<QII", 0, 0, 0) + b"\0"])
def test_sizes_that_do_not_add_up(packed):
    with pytest.raises(HipError, match="ek_launch_list: (no head|the sizes)"):
        hip.call("ek_launch_list", packed, len(packed))


def test_an_empty_list():
    packed = struct.pack("<QII", 0, 0, 4) + b"\0" * 4
    hip.call("ek_launch_list", packed, len(packed))
