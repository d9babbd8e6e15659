"""How the 4-bit attention of few heads divides a call, on the host: every block of every list once, no CTA with more pieces than its table."""
import numpy as np
import pytest

from llmdivedeep_b200 import _lib, build

PIECES = 1024                                          # of a CTA's table


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def most_pieces(lib, T, K, sms, parts):
    seen = np.zeros((T, max(1, -(-K // 64))), np.uint8)
    n = lib.dsa_test_few_heads_plan(T, K, sms, parts, seen.ctypes.data)
    assert n >= 0 and (seen == 1).all(), (T, K, sms, parts, n)
    return n


@pytest.mark.parametrize("parts", [0, 1])
@pytest.mark.parametrize("sms", [148, 7, 1])
def test_every_block_once(lib, sms, parts):
    rng = np.random.default_rng(sms + parts)
    sizes = [(int(np.exp(rng.uniform(0, np.log(20 * sms)))), int(rng.choice([1, 64, 65, 300, 2048]))) for _ in range(120)]
    for T, K in [(1, 0), (sms, 2048), (sms + 1, 2048), (2 * sms - 1, 1), *sizes]:
        assert 1 <= most_pieces(lib, T, K, sms, parts) <= T // sms + 4


@pytest.mark.parametrize("parts", [0, 1])
def test_calls_of_any_length_fit_the_table(lib, parts):
    """One sequence of 160001 query rows would be 1082 pieces of a CTA in one launch; the cuts are where they fall, inside a sequence too."""
    for T in (512 * 148 - 1, 512 * 148, 512 * 148 + 1, 160001, 300000):
        for K in (1, 200):
            assert most_pieces(lib, T, K, 148, parts) <= PIECES
    assert most_pieces(lib, 5000, 100, 3, parts) <= PIECES


def test_refusals(lib):
    assert lib.dsa_test_few_heads_plan(0, 64, 148, 1, None) == 0
    for args in ((-1, 64, 148, 1, 16), (4, -1, 148, 1, 16), (4, 2049, 148, 1, 16), (4, 64, 0, 1, 16), (4, 64, 148, 1, None)):
        assert lib.dsa_test_few_heads_plan(*args) < 0
