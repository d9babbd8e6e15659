"""What the page calls refuse before any launch."""
import struct

import pytest
import torch

from llmdivedeep_b200 import _lib, build, ops


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_tables_whose_pages_outgrow_the_sums_are_refused(lib):
    """New tokens for 200 rows of 2^24 pages may ask for more pages than the 32-bit sums of the plan hold."""
    ws = lib.dsa_pages_workspace_bytes(8, 200)
    args = [16, 1 << 24, 1 << 24, 200, 16, 16, 8, 16, 16, 200, 1 << 30, 16, 16, ws, None, None]
    assert lib.dsa_extend_pages(*args) == -1 and b"table entries" in lib.dsa_last_error_string()
    args[9] = 0
    assert lib.dsa_extend_pages(*args) == 0                        # nothing asked for


def test_caches_that_can_be_read_in_two_ways():
    """A pool of two pages: FP8 keys [128, 128] are rows of one layer, what could be layers too is refused, and t[None] says which."""
    entry = lambda t: struct.unpack("=Qqii", ops._page_caches([t], 2)[0])[2:]
    keys = torch.zeros(128, 128, dtype=torch.uint8).view(ops.FP8)
    assert entry(keys) == (1, 128) and entry(keys[None]) == (1, 128)
    assert entry(torch.zeros(128, 416, dtype=torch.uint8)) == (1, 416) and entry(torch.zeros(3, 128)) == (3, 4)
    wide = torch.zeros(128, 128)
    for t in (wide, keys.view(torch.uint8), torch.zeros(128, 128, 4, dtype=torch.uint8)):
        with pytest.raises(ops.DsaError, match="one layer"):
            ops._page_caches([t], 2)
    assert entry(wide[None]) == (1, 512)
    with pytest.raises(ops.DsaError, match="must be"):
        ops._page_caches([torch.zeros(64, 4)], 2)
