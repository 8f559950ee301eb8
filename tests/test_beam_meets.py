"""Arrays of a move that may not share memory, checked without a GPU."""
import ctypes

import pytest

from test_beam_checks import checks, reorder, state  # noqa: F401

# two groups of four beams: parents 0x2000..0x2020, with rows 6 apart 0x2000..0x2028
BAD = [dict(status=0x2000), dict(status=0x201c), dict(status=0x1ffc), dict(status=0x2024, parent_stride=6),
       dict(status=0x5000, lengths=0x5000), dict(status=0x5000, lengths=0x5004), dict(status=0x5004, lengths=0x5000)]
GOOD = [dict(status=0x2020), dict(status=0x1ff8), dict(status=0x2028, parent_stride=6),
        dict(status=0x5000, lengths=0x5008), dict(status=0x5008, lengths=0x5000), dict(status=0x5000, lengths=0x2000)]


@pytest.mark.parametrize("r", BAD)
def test_status_over_what_the_move_reads(checks, r):  # noqa: F811
    msg = checks.check_reorder(ctypes.byref(reorder([state()], **r)))
    assert msg and b"status overlaps" in msg, msg


@pytest.mark.parametrize("r", GOOD)
def test_status_beside_it(checks, r):  # noqa: F811
    assert checks.check_reorder(ctypes.byref(reorder([state(data=0x100000)], **r))) is None
