"""Plain forms, in 64 bits, of the operators on beams, and the inputs of their tests."""
import math
import random

import torch


class SharedCase:
    """Groups given as (shared tokens, lengths of the group's sequences); everything no row may read is NaN."""

    def __init__(self, groups, heads, kv_heads, dim, dtype, page_size=16, window=0, scatter=True, seed=0, extra_columns=0, scale=None,
                 behind=0):
        rng = random.Random(seed)
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.dtype = heads, kv_heads, dim, dtype
        self.page_size, self.window = page_size, window
        self.scale = 1.3 * dim ** -0.5 if scale is None else scale
        self.prefix = [p for p, _ in groups]
        self.starts = [0]
        for _, lengths in groups:
            self.starts.append(self.starts[-1] + len(lengths))
        self.lens = [n for _, lengths in groups for n in lengths] + [0] * behind
        rows = len(self.lens)
        # pages: whole shared ones belong to the first sequence of a group, the page in which the shared part ends to each
        need, tables = 0, []
        for p, lengths in groups:
            shared = min(p, max(lengths + [0])) // page_size
            for r, n in enumerate(lengths):
                own = max(0, -(-n // page_size) - shared) if r else max(-(-n // page_size), -(-min(p, max(lengths)) // page_size))
                tables.append((r, shared, own))
                need += own
        ids = list(range(need + 3))
        if scatter:
            rng.shuffle(ids)
        width = max([s + o for _, s, o in tables] + [1])
        self.table = torch.full((rows, width), -1, dtype=torch.int32)
        at, first = 0, []
        for row, (r, shared, own) in enumerate(tables):
            mine = ids[at:at + own]
            at += own
            if r == 0:
                first = mine
                self.table[row, :own] = torch.tensor(mine, dtype=torch.int32)
            else:
                all_pages = first[:shared] + mine
                self.table[row, :len(all_pages)] = torch.tensor(all_pages, dtype=torch.int32)
        self.k, self.v = (torch.full((need + 3, kv_heads, page_size, dim), float("nan"), dtype=dtype) for _ in range(2))
        for g, p in enumerate(self.prefix):
            for r in range(self.starts[g], self.starts[g + 1]):
                n, lead = self.lens[r], self.starts[g]
                lo = max(0, n - window) if window else 0
                for j in range(lo, n):
                    row = lead if j < p and self.starts[g + 1] - lead > 1 else r
                    page, o = int(self.table[row, j // page_size]), j % page_size
                    if torch.isnan(self.k[page, 0, o, 0]):
                        self.k[page, :, o] = torch.randn(kv_heads, dim, generator=gen).to(dtype)
                        self.v[page, :, o] = torch.randn(kv_heads, dim, generator=gen).to(dtype)
        if window:  # pages that no row of the group sees are given back
            for g in range(len(groups)):
                of = range(self.starts[g], self.starts[g + 1])
                lowest = min([max(0, self.lens[r] - window) for r in of] + [1 << 30])
                for r in of:
                    self.table[r, :min(width, lowest // page_size)] = -1
        self.q = torch.randn(rows, heads * dim + extra_columns, generator=gen).to(dtype)

    def keys(self, g, r):
        """(sequence whose pages are read, place) of the keys that row r sees."""
        lead, n = self.starts[g], self.lens[r]
        several = self.starts[g + 1] - lead > 1
        return [(lead if several and j < self.prefix[g] else r, j) for j in range(max(0, n - self.window) if self.window else 0, n)]

    def plain(self):
        """(result, bound) in 64 bits: the bound is what the definition's roundings may amount to."""
        H, G, D = self.heads, self.heads // self.kv_heads, self.dim
        out = torch.zeros((len(self.lens), H, D), dtype=torch.float64)
        size = torch.zeros_like(out)  # sum_j w_j |v_j|
        delta = torch.zeros((len(self.lens), H, 1), dtype=torch.float64)  # error of a score
        longest = max(self.lens + [1])
        for g in range(len(self.prefix)):
            for r in range(self.starts[g], self.starts[g + 1]):
                keys = self.keys(g, r)
                if not keys:
                    continue
                row, j = (torch.tensor(x) for x in zip(*keys))
                pages, offs = self.table[row, j // self.page_size].long(), j % self.page_size
                k, v = self.k[pages, :, offs].double(), self.v[pages, :, offs].double()
                q = self.q[r, :H * D].double().view(self.kv_heads, G, D)
                w = torch.softmax(torch.einsum("hgd,lhd->hgl", q, k) * self.scale, -1)
                out[r] = torch.einsum("hgl,lhd->hgd", w, v).reshape(H, D)
                size[r] = torch.einsum("hgl,lhd->hgd", w, v.abs()).reshape(H, D)
                big = torch.einsum("hgd,lhd->hgl", q.abs(), k.abs()).amax(-1) * self.scale
                delta[r] = (big * (D + 8) * 2.0 ** -24).reshape(H, 1)
        # A weight is off by twice the error of a score, and by the roundings of sums of `longest` terms; bfloat16 rounds the
        # weights and the result to 8 bits (half a unit of the last: 2^-8 relative at most).
        relative = 2 * delta + (longest + 64) * 2.0 ** -24
        if self.dtype == torch.bfloat16:
            relative = relative + 2 * 2.0 ** -8
        return out.reshape(-1, H * D), (relative * size + 1e-30).reshape(-1, H * D)

    def tensors(self, device="cuda:0"):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        return (self.q.to(device)[:, :self.heads * self.dim], self.k.to(device), self.v.to(device), self.table.to(device), i32(self.lens),
                i32(self.starts), i32(self.prefix))

    def run(self, device="cuda:0", out=None):
        from dispec_b200 import ops

        return ops.shared_prefix_attention(*self.tensors(device), scale=self.scale, window=self.window, out=out)

    def check(self, **kw):
        want, bound = self.plain()
        rows = self.starts[-1]
        got = self.run(**kw).double().cpu()
        assert got.shape == want.shape and torch.isfinite(got[:rows]).all()
        worst = ((got - want).abs() / bound)[:rows].max() if rows else torch.tensor(0.0)
        assert worst <= 1.0, float(worst)


def select_keys(logits, scores):
    """Every candidate's key in 64 bits [R, V], -inf where there is none."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(1, keepdim=True)
    away = torch.where(x == top, 0.0, x - top)
    log_sum = torch.log(torch.exp(away).sum(1, keepdim=True)).float().double()
    key = scores.double()[:, None] + away - log_sum
    return torch.where((x == -math.inf) | ~torch.isfinite(scores)[:, None], -math.inf, key)


def plain_select(logits, scores, starts, count):
    """(parent, token, key): the largest keys, ties to the lowest row and token."""
    keys = select_keys(logits, scores)
    V = keys.shape[1]
    parent, token, best = [], [], []
    for a, b in zip(starts, starts[1:]):
        flat = keys[a:b].flatten()
        order = torch.sort(flat, descending=True, stable=True).indices[:count]
        order = order[flat[order] > -math.inf]
        pad = [-1] * (count - len(order))
        parent.append((a + order // V).tolist() + pad)
        token.append((order % V).tolist() + pad)
        best.append(flat[order].tolist() + [-math.inf] * len(pad))
    return torch.tensor(parent), torch.tensor(token), torch.tensor(best, dtype=torch.float64)


def select_tolerance(vocab, largest):
    """How far a key may be off.  A term exp(d) of a row's sum: d is rounded (2^-24), multiplied by a rounded log2 e (2^-24 and
    2^-25): |d| 2.5 2^-24 of the term, and 2^-22 from the exponential; weighted by the terms, |d| is at most log V on average;
    31 additions in 32 bits (2^-24 each), the rest in 64.  The logarithm of the sum is rounded (2^-24 of at most log V), and so is a
    score that is returned."""
    log_v = math.log(max(2, vocab))
    return (4 + 2.5 * log_v + 31 + log_v + largest) * 2.0 ** -24
