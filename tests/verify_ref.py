"""64-bit references and input makers of the speculative-verification tests."""

import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def unit_roundoff(dtype):
    return torch.finfo(dtype).eps / 2


def rotate64(x, angle, scale, interleaved):
    """x [T, H, D] turned by angle [T, rotary_dim / 2] (fp64), element by element."""
    x, out = x.double(), x.double().clone()
    half = angle.shape[1]
    c, s = torch.cos(angle)[:, None] * scale, torch.sin(angle)[:, None] * scale
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    out[..., ia] = x[..., ia] * c - x[..., ib] * s
    out[..., ib] = x[..., ib] * c + x[..., ia] * s
    return out


def rows_of(pool, scales, slots):
    """Rows [N, Hkv, D] (fp64) at slots; negative slots give zeros."""
    live = slots >= 0
    s = slots.clamp_min(0)
    x = pool[s // 64, :, :, s % 64].flatten(-2).double()
    if scales is not None:
        x = x * scales[s // 64, :, s % 64].double()[..., None]
    return torch.where(live[:, None, None], x, 0.0)


def make_cache(nb, hkv, dim, cache, gen, device="cuda"):
    """(pool, scales) holding about N(0, 1); scales None for 16-bit pools."""
    if cache in QMAX:
        if cache == torch.int8:
            pool = torch.randint(-127, 128, (nb, hkv, 1, 64, 128), generator=gen, device=device, dtype=torch.int8)
        else:
            pool = (torch.randn((nb, hkv, 1, 64, 128), generator=gen, device=device) * 120).clamp(-448, 448)
            pool = pool.to(torch.float8_e4m3fn)
        step = 0.02 if cache == torch.int8 else 0.008
        return pool, (torch.rand((nb, hkv, 64), generator=gen, device=device) + 0.2) * step
    return torch.randn((nb, hkv, dim // 64, 64, 64), generator=gen, device=device).to(cache), None


def random_tree(n, gen, dead=0.0):
    """parents [n] (local, -1 a root, -2 pruned) of a random tree."""
    parents = []
    for i in range(n):
        u, v = torch.rand(2, generator=gen).tolist()
        parents.append(int(u / 0.85 * i) if i and u < 0.85 else -1)
        if v < dead:
            parents[-1] = -2
    # a pruned node has no children: they hang from its nearest kept predecessor or become roots
    return [(-1 if p >= 0 and parents[p] == -2 else p) for p in parents]


def see_of(parents):
    n = len(parents)
    see = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        if parents[i] == -2:
            continue
        j = i
        while j != -1:
            see[i, j] = True
            j = parents[j]
    return see


def pack_bits(see, words):
    n = see.shape[0]
    bits = torch.zeros(n, words * 64, dtype=torch.int64)
    bits[:, :n] = see.long()
    return (bits.view(n, words, 64) << torch.arange(64)).sum(-1)


class TreeCase:
    """One call's inputs: ragged contexts and drafts over a permuted pool, everything else in it NaN."""

    def __init__(self, ctx, nodes, hq, hkv, dim=128, dtype=torch.float16, cache=None, chain=False, dead=0.0, seed=0,
                 qscale=1.0, poison=True, device="cuda"):
        cache = cache or dtype
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
        self.ctx, self.nodes, self.hq, self.hkv, self.dim = ctx, nodes, hq, hkv, dim
        self.k_pool, self.k_scales = make_cache(nb, hkv, dim, cache, g, device)
        self.v_pool, self.v_scales = make_cache(nb, hkv, dim, cache, g, device)
        self.block_table = self.block_table.to(device)
        if poison:
            self.poison_unowned()
        self.context_lens = torch.tensor(ctx, dtype=torch.int32, device=device)
        self.indptr = [0]
        for t in nodes:
            self.indptr.append(self.indptr[-1] + t)
        self.q_indptr = torch.tensor(self.indptr, dtype=torch.int32, device=device)
        self.q = (torch.randn((self.indptr[-1], hq, dim), generator=g, device=device) * qscale).to(dtype)
        self.max_nodes = max(max(nodes), 1)
        if chain:
            self.parents = None
            self.see = [torch.ones(t, t, dtype=torch.bool).tril() for t in nodes]
            self.mask = None
        else:
            self.parents = [random_tree(t, gc, dead) for t in nodes]
            self.see = [see_of(p) for p in self.parents]
            words = -(-self.max_nodes // 64)
            self.mask = torch.cat([pack_bits(s, words) for s in self.see]).to(device)

    def slots(self, b, start, stop):
        p = torch.arange(start, stop, device=self.block_table.device)
        return self.block_table[b].long()[p // 64] * 64 + p % 64

    def poison_unowned(self):
        owned = torch.zeros(self.k_pool.shape[0] * 64, dtype=torch.bool, device=self.k_pool.device)
        for b, (c, t) in enumerate(zip(self.ctx, self.nodes)):
            owned[self.slots(b, 0, c + t)] = True
        free = ~owned.view(-1, 64)
        for pool, scales in ((self.k_pool, self.k_scales), (self.v_pool, self.v_scales)):
            raw = pool.view(torch.int8) if pool.element_size() == 1 else pool
            sel = free[:, None, None, :, None].expand(pool.shape)
            raw[sel] = 0x7F if pool.element_size() == 1 else float("nan")
            if scales is not None:
                scales[free[:, None, :].expand(scales.shape)] = float("nan")

    def kwargs(self):
        return dict(tree_mask=self.mask, max_nodes=self.max_nodes, k_scales=self.k_scales, v_scales=self.v_scales)

    def args(self):
        return self.q, self.k_pool, self.v_pool, self.block_table, self.context_lens, self.q_indptr

    def reference(self, scale=None):
        """(out, lse, spread) in 64 bits; spread = sum of weight * |v|, what the error bound goes by."""
        scale = 1.0 / math.sqrt(self.dim) if scale is None else scale
        g, outs, lses, spreads = self.hq // self.hkv, [], [], []
        for b, (c, t) in enumerate(zip(self.ctx, self.nodes)):
            if t == 0:
                continue
            sl = self.slots(b, 0, c + t)
            k = rows_of(self.k_pool, self.k_scales, sl).repeat_interleave(g, 1)
            v = rows_of(self.v_pool, self.v_scales, sl).repeat_interleave(g, 1)
            q = self.q[self.indptr[b]:self.indptr[b + 1]].double()
            s = torch.einsum("thd,phd->htp", q, k) * scale
            see = torch.cat([torch.ones(t, c, dtype=torch.bool), self.see[b]], 1).to(s.device)
            s = s.masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, -1)
            w = torch.where(see & (lse[..., None] > -math.inf), torch.exp(s - lse[..., None]), 0.0)
            # a masked place contributes nothing, whatever it holds
            outs.append(_weigh(w, v))
            spreads.append(_weigh(w, v.abs()))
            lses.append(lse.transpose(0, 1))
        return torch.cat(outs), torch.cat(lses), torch.cat(spreads)


def _weigh(w, v):
    if bool(torch.isfinite(v).all()):
        return torch.einsum("htp,phd->thd", w, v)
    bad = ~torch.isfinite(v)
    out = torch.einsum("htp,phd->thd", w, torch.where(bad, 0.0, v))
    for p in bad.flatten(1).any(1).nonzero()[:, 0].tolist():
        seen = (w[:, :, p] > 0).transpose(0, 1)[..., None]
        out = out + torch.where(seen & bad[p][None], v[p][None], 0.0)
    return out


def attention_bound(out, spread, n_keys, dtype):
    """How far a result of `dtype` may be off: u|o| for its own rounding, u times the weighted |v|
    each for the weights and for values rounded to the compute type (u the unit roundoff), weights
    below the smallest normal fp16 number, and fp32 sums and exponentials at 2^-17."""
    u = unit_roundoff(dtype)
    tiny = n_keys * 2.0 ** -24 if dtype == torch.float16 else 0.0
    return u * out.abs() + (2 * u + 2.0 ** -17) * spread + tiny * 4 + 2.0 ** -24
