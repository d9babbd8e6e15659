"""Window attention and drafted tokens by their definitions, position by position, in 64 bits (test infrastructure; nothing here is on a
product path)."""
import numpy as np
import torch

from oracle import latent4_oracle as L

PAGE = 64


def prompt_sees(T, S, window, first, ks=None, ke=None):
    """[T, S] bool: what row t sees."""
    s = torch.arange(S)
    ks = torch.zeros(T, dtype=torch.long) if ks is None else ks.long().clamp_min(0)
    ke = torch.arange(S - T + 1, S + 1) if ke is None else ke.long().clamp_max(S)
    at = s - ks[:, None]                                   # position within the sequence
    p = (ke - ks)[:, None] - 1
    return (at >= 0) & (at <= p) & ((at < first) | (at > p - window))


def draft_paths(ctx, m, i, tree_row, per):
    """Positions of the tokens on draft i's path, itself last, in order; None for a row without a token."""
    if ctx < 0 or m < 0 or m > per or m > ctx or i >= m:
        return None
    P = ctx - m
    mask = -1 if tree_row is None else int(tree_row[i])
    return list(range(P)) + [P + j for j in range(i) if mask >> j & 1] + [P + i]


def draft_sees(B, per, ctx, max_ctx, n_new=None, tree=None, window=None, first=0):
    """[B * per, max_ctx] bool."""
    sees = torch.zeros(B * per, max_ctx, dtype=torch.bool)
    for b in range(B):
        c = int(ctx[b])
        m = int(n_new[b]) if n_new is not None else min(c, per)
        if c > max_ctx:
            continue
        for i in range(per):
            path = draft_paths(c, m, i, None if tree is None else tree[b], per)
            if path is not None:
                if window is not None:
                    path = [s for k, s in enumerate(path) if k < first or k > len(path) - 1 - window]
                sees[b * per + i, path] = True
    return sees


def attend(q, kv, sees, scale):
    """q [T, H, 576], kv [S, 576] (or [T, S, 576]), sees [T, S] -> [T, H, 512] float64.  What is not seen does not come in, whatever it is."""
    out = torch.zeros(*q.shape[:2], 512, dtype=torch.float64, device=q.device)
    for t in range(q.shape[0]):
        at = torch.nonzero(sees[t])[:, 0].to(kv.device)
        if at.numel():
            x = (kv if kv.dim() == 2 else kv[t])[at].double()
            out[t] = torch.softmax(q[t].double() @ x.t() * scale, -1) @ x[:, :512]
    return out


def record_values(rec):
    """Records uint8 [N, 656 or 416] -> the bf16 rows that the attention works on, float64."""
    if rec.shape[1] == 416:
        return torch.from_numpy(L.decode(rec.cpu().numpy()))
    rec = rec.cpu().contiguous()
    lat = rec[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(-1, 4, 128) * rec[:, 512:528].contiguous().view(torch.float32).view(-1, 4, 1)
    return torch.cat((lat.reshape(-1, 512).to(torch.bfloat16).double(), rec[:, 528:].contiguous().view(torch.bfloat16).double()), 1)


def logits(q, w, k, kscale, sees):
    """q [T, H, 128], w [T, H], k [T, S, 128] and kscale [T, S] of each row's sequence -> float64, -inf where not seen."""
    s = torch.relu(torch.einsum("thd,tsd->ths", q.double(), k.double()))
    s = torch.einsum("ths,th->ts", s, w.double()) * kscale.double()
    return s.masked_fill(~sees, -torch.inf)


def random_tree(rng, B, per):
    """int64 [B, per]: every draft descends from one before it, or from none."""
    masks = []
    for _ in range(B):
        row = []
        for i in range(per):
            up = rng.randint(-1, i - 1)
            row.append((row[up] if up >= 0 else 0) | (1 << i))
        masks.append([x - (1 << 64) if x >> 63 else x for x in row])
    return torch.tensor(masks, dtype=torch.int64).view(B, per)


class Pool(L.Pool):
    def accept(self, rows, n_new, path, n_keep):
        B, P = self.table.shape
        pages = lambda n: -(-n // PAGE)  # noqa: E731
        good = []
        for i, (r, m, keep) in enumerate(zip(map(int, rows), map(int, n_new), map(int, n_keep))):
            ok = 0 <= r < B and r not in [int(x) for x in rows[:i]] and 0 <= keep <= m and keep <= path.shape[1]
            c = int(self.ctx[r]) if ok else 0
            ok = ok and m <= c <= P * PAGE
            if ok:
                p = [int(x) for x in path[i, :keep]]
                ok = all(0 <= x < m for x in p) and all(a < b for a, b in zip(p, p[1:]))
                for j in range((c - m) // PAGE, pages(c)):
                    page = int(self.table[r, j])
                    ok = ok and 0 <= page < len(self.refs) and not (keep < m and j < pages(c - m + keep) and self.refs[page] != 1)
            good.append(ok)
            if not ok:
                self._refuse(2)
        for i in range(len(rows)):
            if good[i]:
                r, m, keep = int(rows[i]), int(n_new[i]), int(n_keep[i])
                c = int(self.ctx[r])
                at = lambda s: int(self.table[r, s // PAGE]) * PAGE + s % PAGE  # noqa: E731
                for cache in self.caches:
                    new = [cache[:, at(c - m + int(path[i, k]))].copy() for k in range(keep)]
                    for k in range(keep):
                        cache[:, at(c - m + k)] = new[k]
                now = c - m + keep
                for j in range(pages(now), pages(c)):
                    self.refs[self.table[r, j]] -= 1
                    self.table[r, j] = -1
                self.ctx[r] = now
