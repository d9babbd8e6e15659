"""What the page calls refuse before any launch."""
import pytest

from llmdivedeep_b200 import _lib, build


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
