"""Page calls in graphs and on other streams, those with a second kernel under the first one's end among them, against the oracle."""
import numpy as np
import pytest
import torch

from llmdivedeep_b200 import ops
from tests.test_gpu_pages import Both, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("side", [False, True])
def test_a_scheduler_step_in_a_graph(side):
    """Extending (more slots than the planning cluster writes itself), forking, freeing and compacting in place, captured once and
    replayed with other lengths, and the same calls on a stream of their own: every table, slot and byte after every step."""
    B, P, most = 7, 40, 8300
    s = Both(B, P, 150)
    s.extend([0, 1, 2, 3], [64, 1, 200, 63], 200)
    grow, n_new, gone, parents, children = ints([0, 1, 2, 3]), ints([0, 0, 0, 0]), ints([4, 0]), ints([1, 1, 2]), ints([4, 5, 0])
    last = ints([5, 4])

    def step():
        slots = ops.extend_pages(s.table, s.ctx, s.refs, grow, n_new, most)
        ops.free_pages(s.table, s.ctx, s.refs, gone)
        ops.fork_pages(s.table, s.ctx, s.refs, parents, children, s.caches)
        ops.compact_pages(s.table, s.refs, s.caches, out=(s.table, s.refs))
        ops.free_pages(s.table, s.ctx, s.refs, last)
        return slots

    def expect(n):
        slots = s.o.extend([0, 1, 2, 3], n, most)
        s.o.free([4, 0])
        s.o.fork([1, 1, 2], [4, 5, 0])
        s.o.compact()
        s.o.free([5, 4])
        return slots

    lengths = [[1, 2, 3, 4], [64, 0, 65, 500], [300, 129, 1, 0], [7, 64, 64, 63], [0, 0, 0, 0], [130, 1, 100, 200]]
    if side:
        stream = torch.cuda.Stream()
        for n in lengths:
            n_new.copy_(ints(n))
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                slots = step()
            torch.cuda.current_stream().wait_stream(stream)
            np.testing.assert_array_equal(slots.cpu().numpy(), expect(n))
            s.same()
        return
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots = step()
    for n in lengths:
        n_new.copy_(ints(n))
        graph.replay()
        np.testing.assert_array_equal(slots.cpu().numpy(), expect(n))
        s.same()
