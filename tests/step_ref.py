"""64-bit references and input makers of the step operators' and the latent cache's tests."""

import math

import torch

from tests.verify_ref import _weigh, pack_bits, random_tree, see_of


# ------------------------------------------------------------------- pages --
class Pages:
    """A host copy of the page state, and what extend and release do to it, page by page."""

    def __init__(self, table, counts, free, free_count):
        self.table, self.counts = [list(r) for r in table], list(counts)
        self.free, self.count = list(free), free_count

    def extend(self, ctx, new, depths=None):
        slots, positions, short, t = [], [], False, 0
        for b, (c, n) in enumerate(zip(ctx, new)):
            want = -(-(c + n) // 64)
            need = max(0, want - self.counts[b])
            if need and (short or need > self.count):
                short = True
            elif need:
                for _ in range(need):
                    self.count -= 1
                    self.table[b][self.counts[b]] = self.free[self.count]
                    self.counts[b] += 1
            for i in range(n):
                p = c + i
                slots.append(self.table[b][p // 64] * 64 + p % 64 if p // 64 < self.counts[b] else -1)
                positions.append(c + (i if depths is None else depths[t]))
                t += 1
        return slots, positions, short

    def release(self, keep):
        give, short = [], False
        for b, k in enumerate(keep):
            m = max(0, self.counts[b] - -(-k // 64))
            if m and (short or self.count + len(give) + m > len(self.free)):
                short = True
                continue
            give += [(b, self.counts[b] - m + j) for j in range(m)]
        for b, j in reversed(give):
            self.free[self.count] = self.table[b][j]
            self.table[b][j] = -1
            self.counts[b] -= 1
            self.count += 1
        return short


# ------------------------------------------------------------------ verify --
def verify(parents, tokens, target, draft, au, su, max_path):
    """One sequence, by the definition: distributions normalised after every rejection (all fp64)."""
    n = len(parents)
    if n == 0:
        return [], -1
    path = [0]
    good = lambda x: torch.where((x > 0) & (x < math.inf), x, 0.0)
    while True:
        whole = good(target[path[-1]].double())
        p, step = target[path[-1]].double(), None
        p = good(p)
        children = [i for i in range(path[-1] + 1, n) if parents[i] == path[-1]] if len(path) < max_path else []
        for i in children:
            x = int(tokens[i])
            if not 0 <= x < len(p):
                continue
            if draft is not None:
                q = draft[path[-1]].double()
                if float(au[i]) * float(q[x]) < float(p[x]):
                    step = i
                    break
                p = good(p - q)
                p = p / p.sum() if float(p.sum()) > 0 else p
            else:
                if float(au[i]) < float(p[x]):
                    step = i
                    break
                rest = 1.0 - float(p[x])
                p = p.clone()
                p[x] = 0.0
                if rest > 0:
                    p = p / rest
        if step is None:
            break
        path.append(step)
    p = p if float(p.sum()) > 0 else whole
    total = float(p.sum())
    if not total > 0:
        return path, -1
    cdf = p.cumsum(0)
    return path, int((cdf <= float(su) * float(cdf[-1])).sum())


# ------------------------------------------------------------------ latent --
def latent_rows(pool, slots):
    """Rows [N, 576] (fp64) at slots; negative slots give zeros."""
    s = slots.clamp_min(0)
    x = pool[s // 64, 0, :, s % 64].flatten(-2).double()
    return torch.where((slots >= 0)[:, None], x, 0.0)


def turn(x, angle, interleaved):
    """x [N, .., 64] turned by angle [N, 32] (fp64)."""
    x = x.double()
    c, s = torch.cos(angle), torch.sin(angle)
    while c.dim() < x.dim():
        c, s = c.unsqueeze(1), s.unsqueeze(1)
    out = x.clone()
    a, b = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


class LatentCase:
    """One call's inputs: ragged contexts and drafts over a permuted pool, everything else in it NaN."""

    def __init__(self, ctx, nodes, heads, dtype=torch.bfloat16, chain=False, dead=0.0, seed=0, qscale=1.0, poison=True,
                 device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        gc = torch.Generator().manual_seed(seed + 1)
        need = [-(-(c + t) // 64) for c, t in zip(ctx, nodes)]
        nb = sum(need) + 3
        order = torch.randperm(nb, generator=gc)
        self.block_table = torch.full((len(ctx), max(max(need), 1)), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.block_table[b, :n] = order[at:at + n].int()
            at += n
        self.ctx, self.nodes, self.heads = ctx, nodes, heads
        self.pool = torch.randn((nb, 1, 9, 64, 64), generator=g, device=device).to(dtype)
        self.block_table = self.block_table.to(device)
        if poison:
            owned = torch.zeros(nb * 64, dtype=torch.bool, device=device)
            for b, (c, t) in enumerate(zip(ctx, nodes)):
                owned[self.slots(b, 0, c + t)] = True
            self.pool.permute(0, 3, 1, 2, 4)[~owned.view(nb, 64)] = float("nan")
        self.context_lens = torch.tensor(ctx, dtype=torch.int32, device=device)
        self.indptr = [0]
        for t in nodes:
            self.indptr.append(self.indptr[-1] + t)
        self.q_indptr = torch.tensor(self.indptr, dtype=torch.int32, device=device)
        n = self.indptr[-1]
        self.q_latent = (torch.randn((n, heads, 512), generator=g, device=device) * qscale).to(dtype)
        self.q_rope = (torch.randn((n, heads, 64), generator=g, device=device) * qscale).to(dtype)
        self.max_nodes = max(max(nodes), 1)
        if chain:
            self.see = [torch.ones(t, t, dtype=torch.bool).tril() for t in nodes]
            self.mask = None
        else:
            self.see = [see_of(random_tree(t, gc, dead)) for t in nodes]
            self.mask = torch.cat([pack_bits(s, -(-self.max_nodes // 64)) for s in self.see]).to(device)

    def slots(self, b, start, stop):
        p = torch.arange(start, stop, device=self.block_table.device)
        return self.block_table[b].long()[p // 64] * 64 + p % 64

    def args(self):
        return self.q_latent, self.q_rope, self.pool, self.block_table, self.context_lens, self.q_indptr

    def kwargs(self):
        return dict(tree_mask=self.mask, max_nodes=self.max_nodes)

    def reference(self, scale=None):
        """(out, lse, spread) in 64 bits; spread = sum of weight * |latent|, what the error bound goes by."""
        scale = 192**-0.5 if scale is None else scale
        outs, lses, spreads = [], [], []
        for b, (c, t) in enumerate(zip(self.ctx, self.nodes)):
            if t == 0:
                continue
            rows = latent_rows(self.pool, self.slots(b, 0, c + t))
            part = slice(self.indptr[b], self.indptr[b + 1])
            q = torch.cat([self.q_latent[part], self.q_rope[part]], -1).double()
            s = torch.einsum("thd,pd->htp", q, rows) * scale
            see = torch.cat([torch.ones(t, c, dtype=torch.bool), self.see[b]], 1).to(s.device)
            s = s.masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, -1)
            w = torch.where(see & (lse[..., None] > -math.inf), torch.exp(s - lse[..., None]), 0.0)
            v = rows[:, None, :512].expand(-1, self.heads, -1)
            outs.append(_weigh(w, v))
            spreads.append(_weigh(w, v.abs()))
            lses.append(lse.transpose(0, 1))
        return torch.cat(outs), torch.cat(lses), torch.cat(spreads)
