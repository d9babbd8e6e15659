"""What the page calls refuse before any launch, and the room that a decode step asks for."""
import struct

import pytest
import torch

from llmdivedeep_b200 import _lib, build, layer, ops


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


@pytest.mark.parametrize("heads", [8, 16, 64, 128])
def test_a_decode_workspace_over_fp8_records_is_no_larger_for_the_4_bit_ones(lib, heads):
    """Its parts are what FP8 records need; the first step over 4-bit records makes room for theirs, once."""
    ws = layer.DecodeWorkspace(64, heads, 4096, 2048, "cpu")
    need = [lib.dsa_sparse_mla_decode_records_workspace_bytes(w, 64, heads, 2048) for w in (656, 416)]
    assert need[0] == lib.dsa_sparse_mla_decode_workspace_bytes(64, heads, 2048)
    assert ws.mla_ws.numel() == need[0]
    assert ws.parts(656) is ws.mla_ws
    four = ws.parts(416)
    assert four.numel() >= need[1] and ws.parts(416) is four
