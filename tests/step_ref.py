"""64-bit references and input makers of the step operators' and the latent cache's tests."""

import math

import torch


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
