"""Page tables on the GPU against the one-step-at-a-time rules of the oracle: whole numbers, equal everywhere."""
import numpy as np
import pytest
import torch

from llmdivedeep_b200 import ops
from oracle import latent4_oracle as L

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def ints(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32).cuda()


def caches_for(pages, layers, seed, widths=(128, 4, 416)):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, 256, (layers, pages * 64, w), dtype=np.uint8) for w in widths]


class Both:
    """A pool on the GPU and the oracle's, taken through the same steps."""

    def __init__(self, B, P, pages, layers=2, seed=0, widths=(128, 4, 416)):
        host = caches_for(pages, layers, seed, widths)
        self.o = L.Pool(np.full((B, P), -1, np.int32), np.zeros(B, np.int32), np.zeros(pages, np.int32), host)
        self.table, self.ctx, self.refs = ints(self.o.table), ints(self.o.ctx), ints(self.o.refs)
        self.caches = [torch.from_numpy(c).cuda() for c in host]

    def same(self, status=0):
        word = ops.status_word(torch.device("cuda", 0))
        assert int(word) == self.o.status == status, (int(word), self.o.status, status)
        word.zero_()
        self.o.status = 0
        for got, want in ((self.table, self.o.table), (self.ctx, self.o.ctx), (self.refs, self.o.refs)):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
        for got, want in zip(self.caches, self.o.caches):
            np.testing.assert_array_equal(got.cpu().numpy(), want)

    def extend(self, rows, n_new, max_new, status=0):
        slots = ops.extend_pages(self.table, self.ctx, self.refs, ints(rows), ints(n_new), max_new)
        np.testing.assert_array_equal(slots.cpu().numpy(), self.o.extend(np.asarray(rows), np.asarray(n_new), max_new))
        self.same(status)
        return slots

    def fork(self, parents, children, status=0):
        ops.fork_pages(self.table, self.ctx, self.refs, ints(parents), ints(children), self.caches)
        self.o.fork(np.asarray(parents), np.asarray(children))
        self.same(status)

    def free(self, rows, status=0):
        ops.free_pages(self.table, self.ctx, self.refs, ints(rows))
        self.o.free(rows)
        self.same(status)

    def compact(self, in_place=False):
        out = (self.table, self.refs) if in_place else None
        old = self.table.clone(), self.refs.clone()
        new = ops.compact_pages(self.table, self.refs, self.caches, out=out)
        if not in_place:
            assert torch.equal(old[0], self.table) and torch.equal(old[1], self.refs)
            self.table, self.refs = new
        self.o.compact()
        self.same()


@pytest.mark.parametrize("pages", [40, 64])
def test_random_traffic(pages):
    rng = np.random.default_rng(pages)
    B, P = 9, 6
    s = Both(B, P, pages)
    for step in range(120):
        r = rng.permutation(B)
        kind = rng.integers(4)
        k = int(rng.integers(1, 4))
        if kind == 0:
            n_new = rng.choice([0, 1, 3, 63, 64, 65, 130, 200], k)
            room = P * 64 - s.o.ctx[r[:k]]
            want = np.minimum(n_new, room)
            lacks = sum(-(-(c + n) // 64) - -(-c // 64) for c, n in zip(s.o.ctx[r[:k]], want)) > (s.o.refs == 0).sum()
            s.extend(r[:k], want, int(rng.integers(want.max(), 210)), status=3 if lacks else 0)
        elif kind == 1:
            empty = [x for x in r if s.o.ctx[x] == 0][:k]
            parents = rng.choice([x for x in r if x not in empty] or [r[0]], len(empty))
            if len(empty) and not set(parents) & set(empty):
                lacks = sum(s.o.ctx[p] % 64 != 0 for p in parents) > (s.o.refs == 0).sum()
                s.fork(parents, empty, status=3 if lacks else 0)
        elif kind == 2:
            s.free(list(r[:k]))
        else:
            s.compact(in_place=bool(rng.integers(2)))


def test_lengths_at_the_edges_of_pages():
    s = Both(8, 4, 40)
    s.extend([0, 1, 2, 3, 4, 5, 6], [0, 1, 63, 64, 65, 255, 256], 256)
    s.extend([0, 1, 2, 3, 4, 5], [1, 63, 1, 64, 0, 1], 64)
    s.fork([6], [7])                                               # full to the last page: nothing is copied
    s.free([7, 7])                                                 # twice: once
    s.fork([0], [7])
    s.extend([], [], 5)
    s.free([])
    s.fork([], [])


def test_calls_with_a_bad_argument_change_nothing():
    s = Both(5, 3, 12)
    s.extend([0, 1], [100, 64], 100)
    for rows, n_new in (([2, 2], [1, 1]), ([5], [1]), ([-1], [1]), ([2], [11]), ([2], [-1]), ([0, 3], [1, 11])):
        s.extend(rows, n_new, 10, status=2)
    s.extend([0], [93], 100, status=2)                             # past the table's end
    s.extend([2, 3, 4], [192, 192, 192], 192)
    s.free([2, 3, 4])
    s.extend([2, 3], [190, 128], 192)
    s.extend([4], [192], 192)
    s.extend([0, 3], [40, 1], 40, status=3)                        # eleven of twelve pages are held, two wanted
    s.free([4])
    for parents, children in (([0], [1]), ([0, 1], [4, 4]), ([0], [0]), ([4], [4]), ([7], [4]), ([0], [9]), ([-1], [4])):
        s.fork(parents, children, status=2)
    s.free([9, 0], status=2)                                       # the one that exists is freed
    s.free([0])


def test_forks_share_pages_and_survive_their_parent():
    s = Both(6, 5, 30, layers=3)
    s.extend([2], [200], 200)
    s.fork([2, 2, 2, 2], [0, 1, 3, 5])
    assert int(s.refs.max()) == 5
    s.extend([0, 1], [1, 60], 64)
    s.free([2])
    s.fork([0, 1], [2, 4])
    s.compact()
    s.free([0, 1, 2, 3, 4, 5])
    assert int(s.refs.sum()) == 0 and bool((s.table == -1).all())
    s.compact()


@pytest.mark.parametrize("pages", [1, 5, 4095, 4096, 4097, 20011, 70000])
def test_pools_of_every_size(pages):
    """One CTA, a cluster, stretches that end inside a group of four; most pages held, the free ones anywhere."""
    rng = np.random.default_rng(pages)
    s = Both(40, 70, pages, layers=1, widths=(4,))
    used = rng.random(pages) < 0.7
    used[rng.integers(0, pages)] = False
    s.o.refs[:] = used
    s.refs.copy_(ints(s.o.refs))
    s.o.table[39, :min(70, used.sum())] = np.nonzero(used)[0][-70:]       # a row that holds the highest of them
    s.o.ctx[39] = 64 * min(70, used.sum())
    s.table.copy_(ints(s.o.table)), s.ctx.copy_(ints(s.o.ctx))
    n = min(int((~used).sum()), 1200)
    each = min(60, n)
    rows = list(range(min(30, n // each)))
    s.extend(rows, [64 * each - (r % 5) for r in rows], 64 * each)
    left = int((s.o.refs == 0).sum())
    if left < 36:
        s.extend(list(range(30, 39)), [64 * 4] * 9, 64 * 4, status=3)
    s.compact()


@pytest.mark.parametrize("layers,widths", [(1, (4,)), (3, (656,)), (2, (128, 4, 416)), (1, (16, 20, 4, 1152)), (5, (300, 4))])
def test_copy_pages(layers, widths):
    pages = 30
    rng = np.random.default_rng(layers)
    host = caches_for(pages, layers, 1, widths)
    ids = rng.permutation(pages)
    src, dst = ids[:14].copy(), ids[14:28].copy()
    src[3], dst[5] = -1, -7                                        # left out
    for tokens in (None, rng.integers(-2, 70, 14)):
        o = L.Pool(np.zeros((1, 1)), np.zeros(1), np.zeros(pages), host)
        o.copy(src, dst, tokens)
        dev = [torch.from_numpy(c).cuda() for c in host]
        ops.copy_pages(dev, ints(src), ints(dst), None if tokens is None else ints(tokens), num_pages=pages)
        ops.check_status("cuda")
        for got, want in zip(dev, o.caches):
            np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_copy_pages_of_many_and_of_strided_caches():
    """More caches than one launch takes, each a tensor of its own; layers with a gap between them; typed caches."""
    pages, rng = 6, np.random.default_rng(3)
    many = [torch.from_numpy(rng.integers(0, 256, (pages * 64, 8), dtype=np.uint8)).cuda() for _ in range(300)]
    wide = torch.from_numpy(rng.integers(0, 256, (4, 2, pages * 64, 32), dtype=np.uint8)).cuda()
    part = wide[:, 1]                                              # four layers, two apart
    typed = torch.randn(pages * 64, 16, device="cuda").to(ops.FP8)
    scale = torch.randn(pages * 64, device="cuda")
    want = [t.clone() for t in (*many, part, typed.view(torch.uint8), scale)]
    other = wide[:, 0].clone()
    for t in want:
        d = 1 if t.dim() == 3 else 0
        t.narrow(d, 0, 64).copy_(t.narrow(d, 4 * 64, 64)), t.narrow(d, 5 * 64, 64).copy_(t.narrow(d, 2 * 64, 64))
    ops.copy_pages([*many, part, typed, scale], ints([4, 2]), ints([0, 5]))
    ops.check_status("cuda")
    for got, w in zip((*many, part, typed.view(torch.uint8), scale), want):
        assert torch.equal(got, w)
    assert torch.equal(wide[:, 0], other)


def test_pages_out_of_range_are_flagged_and_skipped():
    pages = 4
    c = torch.arange(pages * 64 * 8, device="cuda").to(torch.uint8).view(pages * 64, 8)
    before = c.clone()
    ops.copy_pages([c], ints([0, 4, 1]), ints([4, 0, 1 << 30]))
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    assert torch.equal(c, before)
    table, ctx, refs = ints([[9, 1]]), ints([128]), ints([0, 0, 0, 0])
    ops.free_pages(table, ctx, refs, ints([0]))                    # a page that does not exist, one that nobody holds
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    assert bool((refs == 0).all()) and int(ctx) == 0


def test_page_addresses_past_two_gigabytes():
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    pages = 84000
    c = torch.empty(pages * 64, 416, dtype=torch.uint8, device="cuda")
    c[(pages - 1) * 64:] = 5
    c[(pages - 90) * 64:(pages - 89) * 64] = 6
    ops.copy_pages([c], ints([pages - 1, pages - 90]), ints([pages - 2, 0]))
    ops.check_status("cuda")
    assert bool((c[(pages - 2) * 64:] == 5).all() and (c[:64] == 6).all())


def test_streams_and_graphs():
    """Extend, fork and free in a graph that is replayed: a decode loop whose tables never leave the GPU."""
    s = Both(4, 8, 40)
    s.extend([0, 1], [60, 130], 130)
    rows, one = ints([0, 1]), ints([1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.extend_pages(s.table, s.ctx, s.refs, rows, one, 1)
    torch.cuda.current_stream().wait_stream(side)
    s.o.extend([0, 1], [1, 1], 1)
    s.same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots = ops.extend_pages(s.table, s.ctx, s.refs, rows, one, 1)
    for _ in range(10):
        graph.replay()
        np.testing.assert_array_equal(slots.cpu().numpy(), s.o.extend([0, 1], [1, 1], 1))
        s.same()


def test_tensors_of_other_forms_are_refused():
    s = Both(4, 3, 10)
    r, n = ints([0, 1]), ints([1, 1])
    t, c, f = s.table, s.ctx, s.refs
    for args in ((t.long(), c, f, r, n, 1), (t[0], c, f, r, n, 1), (t.t(), c, f, r, n, 1), (t, c[:3], f, r, n, 1), (t, c.long(), f, r, n, 1), (t, c, f[None], r, n, 1),
                 (t, c, f, r[None], n, 1), (t, c, f, r, n[:1], 1), (t, c, f, r.long(), n, 1), (t, c, f, r, n, -1), (t.cpu(), c, f, r, n, 1)):
        with pytest.raises(ops.DsaError):
            ops.extend_pages(*args)
    for caches in ([s.caches[0][0, :64]], [s.caches[0].transpose(1, 2)], [s.caches[0][:, :, ::2]], [torch.zeros(640, 3, dtype=torch.uint8, device="cuda")],
                   [torch.zeros(640, 640, dtype=torch.uint8, device="cuda")], [s.caches[0].cpu()]):
        with pytest.raises(ops.DsaError):
            ops.fork_pages(t, c, f, r, ints([2, 3]), caches)
    with pytest.raises(ops.DsaError):
        ops.copy_pages([torch.zeros(64, 128, 8, dtype=torch.uint8, device="cuda")], r, n)          # 64 layers of two pages, or one of a page
    with pytest.raises(ops.DsaError):
        ops.compact_pages(t, f, s.caches, out=(t[:2], f))
    s.same()
