"""Page calls on states that are not what they should be."""
import pytest
import torch

from llmdivedeep_b200 import ops
from tests.test_gpu_pages import Both, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", [-1, 12, 1 << 30])
def test_a_last_page_that_is_none_is_refused(entry):
    """A partly filled last page whose table entry is no page: neither a fork, which would copy it, nor new tokens, which would go into it,
    change anything; a row that gets no tokens and is not forked may have it."""
    s = Both(5, 3, 12)
    s.extend([0, 1], [100, 70], 100)
    s.table[0, 1] = entry
    s.o.table[0, 1] = entry
    before = [t.clone() for t in (s.table, s.ctx, s.refs, *s.caches)]

    def refused():
        with pytest.raises(ops.DsaError, match="out of range"):
            ops.check_status("cuda")
        for got, want in zip((s.table, s.ctx, s.refs, *s.caches), before):
            assert torch.equal(got, want)

    ops.fork_pages(s.table, s.ctx, s.refs, ints([1, 0]), ints([3, 4]), s.caches)
    refused()
    assert bool((ops.extend_pages(s.table, s.ctx, s.refs, ints([1, 0]), ints([3, 4]), 9) == -1).all())
    refused()
    s.extend([0, 1], [0, 5], 9)                                    # none of them in that page
    s.fork([1], [2])


def test_a_key_cache_of_two_pages():
    """[128, 128] in the keys' type: 128 rows of one layer, since a token of one byte is no cache."""
    pages = 2
    keys = torch.randint(0, 256, (128, 128), dtype=torch.uint8, device="cuda")
    lat = torch.randint(0, 256, (128, 416), dtype=torch.uint8, device="cuda")
    want = [t.clone() for t in (keys, lat)]
    for t in want:
        t[64:] = t[:64]
    ops.copy_pages([keys.view(ops.FP8), lat], ints([0]), ints([1]), num_pages=pages)
    ops.check_status("cuda")
    assert torch.equal(keys, want[0]) and torch.equal(lat, want[1])
    table, ctx, refs = ints([[1, -1], [-1, -1]]), ints([9, 0]), ints([0, 1])
    keys[64:] += 1
    ops.fork_pages(table, ctx, refs, ints([0]), ints([1]), [keys.view(ops.FP8), lat])
    ops.check_status("cuda")
    assert torch.equal(keys[:9], keys[64:73]) and ctx.tolist() == [9, 9] and table.tolist() == [[1, -1], [0, -1]]
    ops.free_pages(table, ctx, refs, ints([1]))
    table, refs = ops.compact_pages(table, refs, [keys.view(ops.FP8), lat])
    ops.check_status("cuda")
    assert torch.equal(keys[:64], keys[64:]) and table.tolist() == [[0, -1], [-1, -1]] and refs.tolist() == [1, 0]
