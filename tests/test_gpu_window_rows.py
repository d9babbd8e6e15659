"""Window attention of sequences with many query rows over records: their records are made bf16 rows first, and the prompts' kernel attends over these -- whole units
where there are enough of them to go round, parts of their keys where there are few."""
import math

import pytest
import torch

from llmdivedeep_b200 import ops
from tests.test_gpu_window import SCALE, Case, check, i32

pytestmark = pytest.mark.gpu

# heads, query tokens a sequence, sequences, tokens of a sequence at most, window, first.  Units of 128 rows and more of them than pairs of SMs: heads that fill a unit, share it, lie
# across two, fewer than four (units of 32 tokens)
WHOLE = [(128, 5, 15, 200, 60, 3), (40, 13, 16, 260, 64, 1), (200, 4, 12, 300, 30, 70), (16, 40, 15, 330, 100, 2), (5, 129, 13, 300, 33, 4), (2, 260, 15, 420, 50, 1), (1, 514, 15, 700, 64, 9)]
# few units, over 1024 keys and more
PARTS = [(128, 5, 2, 1500, 1100, 3), (16, 64, 2, 1300, 1000, 70), (40, 16, 1, 1700, 1 << 30, 1), (3, 214, 2, 1500, 1024, 5), (1, 600, 1, 1900, 1200, 64)]


class Rows(Case):
    """A call of these sizes, of ragged sequences: one is idle, one is drafts alone, one has a single draft."""

    def __init__(self, shape, record, tree, seed=0):
        H, per, B, most, self.window, self.first = shape
        ctx = [max(per, most - 37 * b % (most // 2)) for b in range(B)]
        n_new = [per - b % 3 for b in range(B)]
        if B > 3:
            ctx[1], ctx[2], n_new[1], n_new[2], n_new[3] = 0, per, 0, per, 1
        super().__init__(B, per, H, ctx, record, seed + per + H, n_new, tree)
        self.room = ops._room(torch.cuda.current_device(), "dsa_window_mla_decode_workspace_bytes", record, B, per, H, min(self.window, 0x7fffffff), self.first, self.max_ctx)
        self.clean = self.kv

    def run(self, **changes):
        """The call, which has to have gone by rows: they are in its workspace, the first being the first token of the first sequence."""
        ws = torch.zeros(self.room, dtype=torch.uint8, device="cuda")
        out = torch.full((self.B * self.per, self.q.shape[1], 512), 9.0, dtype=torch.bfloat16, device="cuda")
        args = {**self.args(), **changes}
        ops.window_mla_decode_paged(**args, window=self.window, first=self.first, scale=SCALE, out=out, workspace=ws)
        if bool((args["block_table"][0, 0] >= 0)) and not bool(self.clean[0, 0].isnan().any()):
            assert torch.equal(ws[:1152].view(torch.bfloat16).double(), self.clean[0, 0])
        return out

    def want(self, sees):
        B, per, H = self.B, self.per, self.q.shape[1]
        s = (self.q.double().view(B, per * H, 576) @ self.clean.transpose(1, 2) * SCALE).view(B, per, H, -1)
        s = s.masked_fill(~sees.cuda().view(B, per, 1, -1), -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0)
        return (p.view(B, per * H, -1) @ self.clean[..., :512]).view(B * per, H, 512)

    def seen(self):
        return self.sees(self.window, self.first)

    def dirty(self, at):
        """The records with tokens `at` [(sequence, position)] that are no numbers."""
        rec = self.rec.clone()
        for b, pos in at:
            rec[int(self.table[b, pos // 64]) * 64 + pos % 64] = 255
        return rec


def forms(shapes):
    return [(s, tree) for s in shapes for tree in (False, True) if not tree or s[1] <= 64]


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("shape,tree", forms(WHOLE + PARTS))
def test_against_64_bits(record, shape, tree):
    c = Rows(shape, record, tree)
    want = c.want(c.seen())
    check(c.run(), want)
    # the same over the records themselves, and with room for the rows alone
    for room in (0, (c.room // 256 * 256) if shape in WHOLE else c.room):
        ws = torch.empty(room, dtype=torch.uint8, device="cuda")
        check(ops.window_mla_decode_paged(**c.args(), window=c.window, first=c.first, scale=SCALE, workspace=ws), want)
    ops.check_status("cuda")


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("shape,tree", forms(WHOLE + PARTS))
def test_pages_that_are_none(record, shape, tree):
    """The page of the first draft, one in the window, the last one, all of a sequence's."""
    c = Rows(shape, record, tree)
    table, sees = c.args()["block_table"], c.seen()
    last = c.B - 1
    at = {(0, (c.ctx[0] - c.n_new[0]) // 64), (0, max(0, c.ctx[0] - c.n_new[0] - 2) // 64), (last, (c.ctx[last] - 1) // 64)}
    if c.B > 4:
        at |= {(4, p) for p in range(table.shape[1])}
    for b, page in at:
        table[b, page] = -7 if page % 2 else c.rec.shape[0] // 64
        sees[b * c.per:(b + 1) * c.per, page * 64:page * 64 + 64] = False
    out = c.run(block_table=table)
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    check(out, c.want(sees))
    if c.B > 4:
        assert bool((out.view(c.B, -1)[4] == 0).all())


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("shape,tree", forms(WHOLE + PARTS))
def test_records_that_are_no_numbers(record, shape, tree):
    """A draft's, one that the window's end passes by, a first token's, and one of each beside a page that is none: rows that see them are none, the others right."""
    c = Rows(shape, record, tree)
    sees, last = c.seen(), c.B - 1
    P = c.ctx[0] - c.n_new[0]
    W = min(c.window, P)
    for at in ([(0, P + 1)], [(0, max(0, P - W + 2)), (last, c.ctx[last] - 2)], [(0, 0)], [(0, P), (last, max(0, c.ctx[last] - c.n_new[last]))]):
        bad = torch.zeros_like(sees)
        for b, pos in at:
            bad[b * c.per:(b + 1) * c.per, pos] = True
        for hole in (False, True):
            table, left = c.args()["block_table"], sees.clone()
            if hole:                                       # a page without any of them
                b = last
                page = next(p for p in range(c.max_ctx // 64 - 1, -1, -1) if p * 64 < c.ctx[b] and (b, p) not in {(x, y // 64) for x, y in at})
                table[b, page] = -1
                left[b * c.per:(b + 1) * c.per, page * 64:page * 64 + 64] = False
            touched = (left & bad).any(-1).cuda()
            out = c.run(cache=c.dirty(at), block_table=table) if (0, 0) not in at else \
                ops.window_mla_decode_paged(**{**c.args(), "cache": c.dirty(at), "block_table": table}, window=c.window, first=c.first, scale=SCALE)
            if hole and bool(left.ne(sees).any()):
                ops.status_word("cuda").zero_()
            ops.check_status("cuda")
            assert bool(out[touched].isnan().all())
            check(out[~touched], c.want(left)[~touched])


@pytest.mark.parametrize("record", [656, 416])
def test_more_rows_to_be_done_again_than_a_list_holds(record):
    """A first draft that is no number and that only itself sees, in every sequence, eighteen units to a pair: nearly every unit has rows to be done again."""
    B, per, H = 222, 6, 128
    c = Case(B, per, H, [70 + b % 50 for b in range(B)], record, 5, [per - (b % 5 == 4) for b in range(B)])
    c.tree = torch.tensor([[0, 0, 2, 2, 8, 26]] * B)
    c.window, c.first = 60, 3
    at = [(b, c.ctx[b] - c.n_new[b]) for b in range(B)]
    sees, bad = c.sees(60, 3), torch.zeros(B * per, c.max_ctx, dtype=torch.bool)
    for b, pos in at:
        bad[b * per:(b + 1) * per, pos] = True
    touched = (sees & bad).any(-1).cuda()
    assert int(touched.sum()) == B
    c.clean = c.kv
    dirty = Rows.dirty(c, at)
    out = ops.window_mla_decode_paged(**{**c.args(), "cache": dirty}, window=60, first=3, scale=SCALE)
    ops.check_status("cuda")
    assert bool(out[touched].isnan().all())
    check(out[~touched], Rows.want(c, sees)[~touched])
    dead = torch.tensor([i >= c.n_new[b] for b in range(B) for i in range(per)]).cuda()
    assert bool((out[dead] == 0).all())


def test_lengths_that_make_no_sense():
    c = Rows(WHOLE[0], 416, True)
    lens, new = i32(c.ctx), i32(c.n_new)
    lens[5], new[6], new[7], lens[8], new[8] = c.max_ctx + 1, c.per + 1, -1, 2, 3
    out = c.run(ctx_len=lens, n_new=new)
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    sees = c.seen()
    sees[5 * c.per:9 * c.per] = False
    check(out, c.want(sees))


def test_in_a_graph_with_lengths_that_change():
    c = Rows(WHOLE[0], 656, True)
    a, out = c.args(), torch.zeros(c.B * c.per, 128, 512, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    call = lambda: ops.window_mla_decode_paged(**a, window=c.window, first=c.first, scale=SCALE, out=out)
    call()
    with torch.cuda.graph(graph):
        call()
    for shift in (0, 7, 30):
        c.ctx = [max(n, x - shift) for x, n in zip(c.ctx, c.n_new)]
        a["ctx_len"].copy_(i32(c.ctx))
        c.n_new = [n - (n > 1) for n in c.n_new]
        a["n_new"].copy_(i32(c.n_new))
        out.fill_(9)
        graph.replay()
        ops.check_status("cuda")
        check(out, c.want(c.seen()))


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("shape", [WHOLE[0], WHOLE[5], PARTS[0], PARTS[3]])
@pytest.mark.parametrize("idle", ["tokens", "drafts"])
def test_nobody_has_a_draft(record, shape, idle):
    """Sequences without a token, and sequences without a draft: zeros in every row."""
    c = Rows(shape, record, False)
    none = torch.zeros(c.B, dtype=torch.int32, device="cuda")
    out = torch.full((c.B * c.per, c.q.shape[1], 512), 9.0, dtype=torch.bfloat16, device="cuda")
    changes = dict(n_new=none, ctx_len=none) if idle == "tokens" else dict(n_new=none)
    ops.window_mla_decode_paged(**{**c.args(), **changes}, window=c.window, first=c.first, scale=SCALE, out=out)
    ops.check_status("cuda")
    assert bool((out == 0).all())


def test_two_calls_at_once():
    """On streams of their own, each with its own workspace, whole units beside parts: what each gives alone."""
    cases = [Rows(WHOLE[0], 656, True), Rows(PARTS[0], 416, True), Rows(WHOLE[5], 416, False)]
    call = lambda c, a: ops.window_mla_decode_paged(**a, window=c.window, first=c.first, scale=SCALE)
    args = [c.args() for c in cases]
    want = [call(c, a) for c, a in zip(cases, args)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    for _ in range(10):
        for s, c, a, g in zip(streams, cases, args, got):
            with torch.cuda.stream(s):
                g.append(call(c, a))
    torch.cuda.synchronize()
    ops.check_status("cuda")
    assert all(torch.equal(o, w) for g, w in zip(got, want) for o in g)
