"""Plain forms, in 64 bits, of the operators on drafted trees, and the inputs of their tests."""
import random

import torch

from dispec_b200.ops.tree import ancestors


def random_tree(n, rng, chain=False):
    return [i - 1 if chain or i == 0 else rng.randint(max(0, i // 2 - 3), i - 1) for i in range(n)]


def paged(lens, page_size, rng, scatter, spare=3):
    """A page table for requests of these lengths (int64 [S, width], -1 behind each) and the number of pages."""
    need = [-(-n // page_size) for n in lens]
    ids = list(range(sum(need) + spare))
    if scatter:
        rng.shuffle(ids)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    return table, sum(need) + spare


class AttentionCase:
    """Trees given as (stored tokens, parents); everything no row may read is NaN."""

    def __init__(self, trees, heads, kv_heads, dim, dtype, page_size=16, window=0, scatter=True, seed=0, extra_columns=0,
                 scale=None):
        rng = random.Random(seed)
        gen = torch.Generator().manual_seed(seed)
        self.trees, self.heads, self.kv_heads, self.dim, self.dtype = trees, heads, kv_heads, dim, dtype
        self.page_size, self.window = page_size, window
        self.scale = 1.3 * dim ** -0.5 if scale is None else scale
        self.counts = [len(p) for _, p in trees]
        self.ctx = [c for c, _ in trees]
        self.starts = [0]
        for n in self.counts:
            self.starts.append(self.starts[-1] + n)
        rows = self.starts[-1]
        lens = [c + n for c, n in zip(self.ctx, self.counts)]
        self.table, pages = paged(lens, page_size, rng, scatter)
        shape = (pages, kv_heads, page_size, dim)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
        for s, n in enumerate(lens):
            for j in range(n):
                p, o = int(self.table[s, j // page_size]), j % page_size
                self.k[p, :, o] = torch.randn(kv_heads, dim, generator=gen).to(dtype)
                self.v[p, :, o] = torch.randn(kv_heads, dim, generator=gen).to(dtype)
        if window:  # pages behind the root's window are given back
            for s, c in enumerate(self.ctx):
                for j in range(max(0, c - window + 1) // page_size):
                    p = int(self.table[s, j])
                    self.k[p] = self.v[p] = float("nan")
                    self.table[s, j] = -1
        self.q = torch.randn(rows, heads * dim + extra_columns, generator=gen).to(dtype)
        words = max(1, -(-max(self.counts + [1]) // 64))
        self.visible = torch.zeros((rows, words), dtype=torch.int64)
        self.depth = torch.zeros((rows,), dtype=torch.int32)
        for s, (_, parents) in enumerate(trees):
            if parents:
                bits, depth = ancestors(parents)
                for i, (b, d) in enumerate(zip(bits, depth)):
                    self.visible[self.starts[s] + i, :len(b)] = torch.tensor(b)
                    self.depth[self.starts[s] + i] = d

    def sees(self, s, i, k):
        return bool((int(self.visible[self.starts[s] + i, k // 64]) >> (k % 64)) & 1)

    def plain(self):
        """(result, bound) in 64 bits: the bound is what the definition's roundings may amount to."""
        H, G, D, W = self.heads, self.heads // self.kv_heads, self.dim, self.window
        out = torch.zeros((self.starts[-1], H, D), dtype=torch.float64)
        size = torch.zeros_like(out)  # sum_j w_j |v_j|
        delta = torch.zeros((self.starts[-1], H, 1), dtype=torch.float64)  # error of a score
        longest = 1
        for s, (ctx, parents) in enumerate(self.trees):
            n = len(parents)
            if n == 0:
                continue
            longest = max(longest, ctx + n)
            depth = [int(self.depth[self.starts[s] + i]) for i in range(n)]
            for i in range(n):
                row = self.starts[s] + i
                keys = [j for j in range(ctx) if not W or j > ctx + depth[i] - W]
                keys += [ctx + k for k in range(n) if self.sees(s, i, k) and (not W or depth[k] > depth[i] - W)]
                if not keys:
                    continue
                j = torch.tensor(keys)
                pages, offs = self.table[s, j // self.page_size].long(), j % self.page_size
                k = self.k[pages, :, offs].double()  # [keys, KVH, D]
                v = self.v[pages, :, offs].double()
                q = self.q[row, :H * D].double().view(self.kv_heads, G, D)
                sc = torch.einsum("hgd,lhd->hgl", q, k) * self.scale
                w = torch.softmax(sc, -1)
                out[row] = torch.einsum("hgl,lhd->hgd", w, v).reshape(H, D)
                size[row] = torch.einsum("hgl,lhd->hgd", w, v.abs()).reshape(H, D)
                big = torch.einsum("hgd,lhd->hgl", q.abs(), k.abs()).amax(-1) * self.scale
                delta[row] = (big * (D + 8) * 2.0 ** -24).reshape(H, 1)
        # A weight is off by twice the error of a score, and by the roundings of sums of `longest` terms; bfloat16 rounds the
        # weights and the result to 8 bits (half a unit of the last: 2^-9 of up to twice the value, 2^-8).
        relative = 2 * delta + (longest + 64) * 2.0 ** -24
        if self.dtype == torch.bfloat16:
            relative = relative + 2 * 2.0 ** -8
        return out.reshape(-1, H * D), (relative * size + 1e-30).reshape(-1, H * D)

    def run(self, device="cuda:0", out=None):
        from dispec_b200 import ops

        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        q = self.q.to(device)[:, :self.heads * self.dim]
        return ops.tree_attention(q, self.k.to(device), self.v.to(device), self.table.to(device), i32(self.ctx),
                                  i32(self.starts), self.visible.to(device), self.depth.to(device),
                                  max_nodes=max(self.counts + [1]), scale=self.scale, window=self.window, out=out)

    def check(self, **kw):
        want, bound = self.plain()
        got = self.run(**kw).double().cpu()
        assert got.shape == want.shape and torch.isfinite(got).all()
        worst = ((got - want).abs() / bound).max() if want.numel() else torch.tensor(0.0)
        assert worst <= 1.0, float(worst)


class VerifyCase:
    """Logits [T, V], trees of drafted tokens, uniform numbers."""

    def __init__(self, trees, tokens, logits, temperature, uniforms, draws, draft=None):
        self.trees, self.tokens, self.logits, self.temperature = trees, tokens, logits, temperature
        self.uniforms, self.draws, self.draft = uniforms, draws, draft
        self.starts = [0]
        for t in trees:
            self.starts.append(self.starts[-1] + len(t))

    def run(self, device="cuda:0", max_nodes=None, logits_dtype=torch.float32):
        from dispec_b200 import ops

        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        f32 = lambda v: torch.as_tensor(v, dtype=torch.float32).to(device)
        got = ops.verify_tree(self.logits.to(device, logits_dtype), i32(self.tokens), i32([p for t in self.trees for p in t]),
                              i32(self.starts), f32(self.temperature), f32(self.uniforms), f32(self.draws),
                              None if self.draft is None else f32(self.draft),
                              max_nodes=max_nodes or max([len(t) for t in self.trees] + [1]))
        return got.count.tolist(), got.path.tolist(), got.token.tolist()

    def follow(self, s, count, path, token, slack=1e-5):
        """Walks tree s in 64 bits along the given decisions; raises where one of them lies more than ``slack`` on the
        wrong side.  ``slack`` covers the 32-bit exponentials (2^-22 of a mass, arguments up to 100 rounded to 2^-18)
        and masses cut to 2^-40 of the largest."""
        first, tree = self.starts[s], self.trees[s]
        if not tree:
            assert (count, token) == (0, -1)
            return
        t = float(self.temperature[s])

        def target(i):
            x = self.logits[first + i].double()
            x = torch.where(torch.isnan(x), float("-inf"), x)
            if t > 0:
                x = x / t
            top = x.max()
            if t <= 0 or top == float("-inf"):
                p = torch.zeros_like(x)
                p[int((x == top).nonzero()[0])] = 1.0
                return p
            e = torch.where(x == top, 1.0, torch.exp(x - top))
            return e / e.sum()

        assert path[0] == 0 and 1 <= count <= len(tree) and all(v == -1 for v in path[count:])
        cur, at, p = 0, 1, target(0)
        for i in range(1, len(tree)):
            if tree[i] != cur:
                continue
            tok, u = self.tokens[first + i], float(self.uniforms[first + i])
            q = None if self.draft is None else self.draft[first + cur].double()
            limit = u * (float(q[tok]) if q is not None else 1.0)
            if at < count and path[at] == i:
                assert limit <= float(p[tok]) + slack, (s, i, limit, float(p[tok]))
                cur, at, p = i, at + 1, target(i)
                continue
            assert limit >= float(p[tok]) - slack, (s, i, limit, float(p[tok]))
            rest = p.clone()
            if q is not None:
                rest = (rest - q).clamp_min(0)
            else:
                rest[tok] = 0
            if float(rest.sum()) > slack:
                p = rest / rest.sum()
                slack = slack / min(1.0, float(rest.sum()))
            elif float(rest.sum()) > 0:
                return  # what is left is within the roundings: any token may follow
        assert at == count
        below = float(p[:token].sum())
        assert below - slack <= float(self.draws[s]) <= below + float(p[token]) + slack, (s, token)
