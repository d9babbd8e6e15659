"""Window attention whose scores are sums of two large halves, of either half infinite: a pair of SMs computes half of every score each."""
import random

import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import drafts_oracle as D
from tests.test_gpu_window import MOST, REL, SCALE, check, i32, rows

pytestmark = pytest.mark.gpu
# One SM has latent values 0 .. 255 and rope values 0 .. 31, the other the rest.  Rope values come into the scores and not into the output.
LOW, HIGH = 512 + 5, 544 + 9


def split(q, kv, a, lo, hi, seed):
    """Adds a * b to the first half of each score and -a * b to the second, b a whole number of [lo, hi) and another one for each key: exact in bf16 as
    long as hi <= 256, and nothing in the sum."""
    g = torch.Generator().manual_seed(seed)
    b = torch.randint(lo, hi, (kv.shape[0],), generator=g).to(kv.dtype).to(kv.device)
    q[..., LOW], q[..., HIGH] = a, a
    kv[..., LOW], kv[..., HIGH] = b, -b


# A half of size X comes from fp32 sums: each of a half's 18 products of 16 terms is added to a sum of at most X, whose rounding, towards zero at worst, is 2^-23 of it; the two
# halves' and their own sum's make a score off by 37 * 2^-23 X at most, and P by the scale times as much, relatively.  The output takes P and the sum of P: twice.
def bound(x):
    return 2 * 37 * 2.0 ** -23 * x * SCALE


@pytest.mark.parametrize("a,lo,hi", [(32, 1, 128), (512, 1, 128), (512, 130, 256)])
@pytest.mark.parametrize("T,S,H,window,first", [(70, 600, 128, 300, 4), (70, 600, 16, 300, 4), (9, 2100, 8, 2048, 4), (300, 300, 3, 64, 0), (600, 600, 64, 90, 20)])
def test_prompts_halves_that_cancel(T, S, H, window, first, a, lo, hi):
    q, kv = rows(T, H, seed=1), rows(S, seed=2)
    split(q, kv, a, lo, hi, seed=3)
    out = ops.window_mla_prefill(q, kv, None, None, window, first, SCALE)
    ops.check_status("cuda")
    more = bound(a * hi)
    check(out, D.attend(q, kv, D.prompt_sees(T, S, window, first), SCALE), REL + more, MOST + more)


class Records:
    """Sequences over records whose rope values `touch` sets; what no sequence has reads as NaN."""

    def __init__(self, B, per, H, ctx, record, seed, touch, tree=False):
        g = torch.Generator().manual_seed(seed)
        self.B, self.per, self.ctx = B, per, ctx
        self.max_ctx = -(-max(ctx) // 64) * 64
        P = self.max_ctx // 64
        kv = torch.randn((B * P + 2) * 64, 576, generator=g).to(torch.bfloat16).cuda()
        self.q = torch.randn(B * per, H, 576, generator=g).to(torch.bfloat16).cuda()
        self.table = torch.randperm(B * P + 2, generator=g)[:B * P].int().view(B, P)
        self.at = self.table.long()[:, torch.arange(self.max_ctx) // 64] * 64 + torch.arange(self.max_ctx) % 64
        touch(self, kv)
        self.rec = layer.pack_latent_cache(kv) if record == 656 else ops.pack_latent4(kv)
        used = torch.zeros(kv.shape[0], dtype=torch.bool)
        for b in range(B):
            used[self.at[b, :ctx[b]]] = True
        self.rec[~used.cuda()] = 255
        self.values = D.record_values(self.rec)[self.at].cuda()           # [B, max_ctx, 576]
        self.tree = D.random_tree(random.Random(seed), B, per) if tree else None
        self.args = dict(q=self.q, cache=self.rec, block_table=self.table.cuda(), ctx_len=i32(ctx), tokens_per_seq=per, tree=None if self.tree is None else self.tree.cuda())

    def sees(self, window, first):
        return D.draft_sees(self.B, self.per, self.ctx, self.max_ctx, None, self.tree, window, first)


# one token and several; parts; units over records and over rows that were made of them first
SHAPES = [(1, 1, 128, [2000], 512, 4), (2, 4, 16, [900, 700], 300, 64), (5, 1, 8, [200, 1, 2, 64, 129], 33, 1), (80, 1, 128, [130] * 80, 100, 4), (3, 13, 128, [1400, 1290, 1500], 1200, 4),
          (15, 5, 128, [90 + 7 * b for b in range(15)], 60, 3)]


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("a,lo,hi", [(32, 1, 128), (512, 130, 256)])
@pytest.mark.parametrize("B,per,H,ctx,window,first", SHAPES)
def test_records_halves_that_cancel(record, B, per, H, ctx, window, first, a, lo, hi):
    c = Records(B, per, H, ctx, record, B + per, lambda s, kv: split(s.q, kv, a, lo, hi, seed=per), tree=per > 1)
    out = ops.window_mla_decode_paged(**c.args, window=window, first=first, scale=SCALE)
    ops.check_status("cuda")
    more = bound(a * hi)
    check(out, D.attend(c.q, c.values.repeat_interleave(per, 0), c.sees(window, first), SCALE), REL + more, MOST + more)


@pytest.mark.parametrize("T,S,H,window,first", [(70, 600, 128, 300, 4), (70, 600, 16, 300, 4), (9, 2100, 8, 2048, 4)])
@pytest.mark.parametrize("dim", [100, 300, LOW, HIGH])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_prompts_a_key_that_is_infinite(T, S, H, window, first, dim, bad):
    """A row and head that sees it: where its score is inf the softmax is none, and no value of the output is a number; where it is -inf the key weighs nothing, but for 0 x inf in
    its own column."""
    q, kv = rows(T, H, seed=4), rows(S, seed=5)
    sees = D.prompt_sees(T, S, window, first)
    at = S - 5
    dirty, less = kv.clone(), sees.clone()
    dirty[at, dim] = bad
    less[:, at] = False
    out = ops.window_mla_prefill(q, dirty, None, None, window, first, SCALE)
    ops.check_status("cuda")
    infinite(out, q[..., dim] * (1 if bad > 0 else -1), sees[:, at].cuda(), dim, D.attend(q, kv, less, SCALE), D.attend(q, kv, sees, SCALE))


def infinite(out, toward, seen, dim, less, clean):
    assert bool(seen.any()) and bool((toward != 0).all())
    check(out[~seen], clean[~seen])
    up = seen[:, None] & (toward > 0)
    down = seen[:, None] & (toward < 0)
    assert bool(out[up].isnan().all())
    if dim < 512:
        assert not bool(out[..., dim][down].isfinite().any())
        out, less = out.clone(), less.clone()
        out[..., dim], less[..., dim] = 0, 0
    check(out[down], less[down])


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("dim", [LOW, HIGH])
@pytest.mark.parametrize("B,per,H,ctx,window,first", [(1, 1, 128, [2000], 512, 4), (2, 4, 16, [900, 700], 300, 64), (3, 13, 128, [1400, 1290, 1500], 1200, 4), (15, 5, 128, [90] * 15, 60, 3)])
def test_records_a_key_that_is_infinite(record, dim, B, per, H, ctx, window, first):
    pos = ctx[0] - per - 3

    def touch(s, kv):
        kv[s.at[0, pos], dim] = float("inf")

    c = Records(B, per, H, ctx, record, B + per, touch)
    out = ops.window_mla_decode_paged(**c.args, window=window, first=first, scale=SCALE)
    ops.check_status("cuda")
    sees = c.sees(window, first)
    less = sees.clone()
    less[:per, pos] = False
    seen = torch.zeros(B * per, dtype=torch.bool)
    seen[:per] = sees[:per, pos]
    kv = c.values.clone()
    kv[0, pos, dim] = 0                                                    # (rows that see it are compared without it)
    kv = kv.repeat_interleave(per, 0)
    infinite(out, c.q[..., dim], seen.cuda(), dim, D.attend(c.q, kv, less, SCALE), D.attend(c.q, kv, sees, SCALE))
