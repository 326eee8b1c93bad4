"""Drafted decoding over a cache of latent vectors: the operators, their plain forms and measured cases.

The operators (layouts as in include/b200kv.h, tokens in 64-token pages of 128-byte sticks):

* ``pages``   a step's block tables, slots and positions made on the GPU from the requests' lengths: pages
              taken from a stack of free ones, and those past the lengths that are kept given back.
* ``store``   a token's latent vector (normalised) and shared rotary key written to their slots, the heads'
              rotary queries turned beside them; the rows are read back.
* ``latent``  attention of each sequence's new tokens (drafted trees, chains, single ones) over cached latent
              vectors, which are key and value of every head (the absorbed form).
* ``prompt``  attention of prompts with keys and values expanded from latent vectors: a head's own key part and
              value, one rotary key part for all heads; ragged lengths, causal at the end or not.
* ``verify``  drafted tokens accepted or rejected against the target's probabilities, from given random
              numbers, and the token that comes next.
"""

import math
import random

import torch

own = False

PAGE, RANK, ROPE, NOPE = 64, 512, 64, 128
STICKS = (RANK + ROPE) // 64
SCALE = 1.0 / math.sqrt(NOPE + ROPE)
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # A decode step of 64 sequences with drafts of up to 8 nodes: latency counts.
        dict(name="pages_step", op="pages", batch=64, ctx_lo=16, ctx_hi=8192, nodes_lo=1, nodes_hi=8, tree=True),
        # 256 prompts arrive at once.
        dict(name="pages_prompts", op="pages", batch=256, ctx_lo=0, ctx_hi=0, nodes_lo=1, nodes_hi=1024, tree=False),
        # One step's tokens of 32 sequences, all heads on one GPU.
        dict(name="store_step", op="store", dtype="bf16", tokens=32, heads=128, interleaved=True, norm=True,
             max_pos=8192, pad=0.0),
        # A long prompt of odd length, an eighth of the heads, a few padding rows.
        dict(name="store_prompt", op="store", dtype="fp16", tokens=16381, heads=16, interleaved=False, norm=True,
             max_pos=32768, pad=0.02),
        # One sequence, one token, an eighth of the heads, 1000 cached tokens: the smallest attention.
        dict(name="latent_single", op="latent", dtype="bf16", batch=1, heads=16, ctx_lo=1000, ctx_hi=1000, nodes_lo=1,
             nodes_hi=1, chain=True, dead=0.0),
        # A batch on a tensor-parallel shard: an eighth of the heads, ragged contexts, one token each.
        dict(name="latent_shard", op="latent", dtype="fp16", batch=64, heads=16, ctx_lo=512, ctx_hi=8192, nodes_lo=1,
             nodes_hi=1, chain=True, dead=0.0),
        # A batch with all heads on one GPU, one token each.
        dict(name="latent_batch", op="latent", dtype="bf16", batch=32, heads=128, ctx_lo=1024, ctx_hi=8192, nodes_lo=1,
             nodes_hi=1, chain=True, dead=0.0),
        # Drafted trees with all heads on one GPU, long contexts, some nodes pruned.
        dict(name="latent_drafts", op="latent", dtype="bf16", batch=8, heads=128, ctx_lo=4096, ctx_hi=16384, nodes_lo=1,
             nodes_hi=8, chain=False, dead=0.05),
        # Four prompts of ragged lengths, an eighth of the heads.
        dict(name="prompt_batch", op="prompt", dtype="fp16", batch=4, heads=16, past_lo=0, past_hi=0, new_lo=1,
             new_hi=4096, causal=True),
        # Chunks of two long prompts over their expanded past, all heads.
        dict(name="prompt_chunk", op="prompt", dtype="bf16", batch=2, heads=128, past_lo=4001, past_hi=8000, new_lo=777,
             new_hi=1024, causal=True),
        # Drafted trees of 16 sequences, a small vocabulary.
        dict(name="verify_trees", op="verify", dtype="fp32", batch=16, vocab=32000, nodes_lo=2, nodes_hi=32, chain=False,
             draft=True),
        # Chains of four drafted tokens for a large batch, a large vocabulary.
        dict(name="verify_chains", op="verify", dtype="fp32", batch=128, vocab=131072, nodes_lo=5, nodes_hi=5, chain=True,
             draft=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "store", "verify", "prompt", "prompt", "latent", "latent", "latent", "latent"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "pages":
        tree = rng.random() < 0.5
        hi = _log(rng, 1, 64 if tree else 1024)
        ctx = rng.choice([0, _log(rng, 1, 32768)])
        return dict(op=op, batch=_log(rng, 1, 256), ctx_lo=rng.choice([0, ctx // 2, ctx]), ctx_hi=ctx,
                    nodes_lo=rng.randint(0, hi), nodes_hi=hi, tree=tree)
    if op == "store":
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, 16381), heads=rng.choice([0, 1, 5, 16, 20, 32, 128]),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.7, max_pos=_log(rng, 64, 32768),
                    pad=rng.choice([0.0, 0.1]))
    if op == "verify":
        chain = rng.random() < 0.4
        hi = _log(rng, 1, 12 if chain else 64)
        case = dict(op=op, dtype=rng.choice(["fp32", "fp32", "fp16", "bf16"]), batch=_log(rng, 1, 128),
                    vocab=_log(rng, 3, 131072), nodes_lo=rng.randint(1, hi), nodes_hi=hi, chain=chain,
                    draft=rng.random() < 0.6)
        # no more rows of probabilities than the large batch has
        case["batch"] = max(1, min(case["batch"], int(640 * 131072 / case["vocab"] / hi)))
        return case
    if op == "prompt":
        heads = rng.choice([1, 2, 5, 8, 16, 20, 64, 128])
        new, past = _log(rng, 1, 4096), rng.choice([0, _log(rng, 1, 16384)])
        case = dict(op=op, dtype=dtype, batch=_log(rng, 1, 16), heads=heads, past_lo=rng.choice([0, past // 2, past]),
                    past_hi=past, new_lo=rng.randint(0, new), new_hi=new, causal=rng.random() < 0.8)
    else:
        chain = rng.random() < 0.4
        hi, ctx = _log(rng, 1, 64 if chain else 24), _log(rng, 1, 131072)
        case = dict(op=op, dtype=dtype, batch=_log(rng, 1, 96), heads=rng.choice([1, 3, 8, 16, 20, 32, 48, 64, 128]),
                    ctx_lo=rng.choice([0, ctx // 2, ctx]), ctx_hi=ctx, nodes_lo=rng.randint(1, hi), nodes_hi=hi,
                    chain=chain, dead=0.0 if chain else rng.choice([0.0, 0.2]))
    while _over(case):
        if case["batch"] > 1:
            case["batch"] = case["batch"] * 3 // 4
        else:
            for name in ("new", "past") if op == "prompt" else ("ctx",):
                case[name + "_hi"] = max(case[name + "_hi"] * 3 // 4, 1 if name == "new" else 0)
                case[name + "_lo"] = min(case[name + "_lo"], case[name + "_hi"])
    return case


def _over(case):
    """No more cached bytes and no more products than the largest listed cases have."""
    w = work(dict(case, ctx_lo=case["ctx_hi"], nodes_lo=case["nodes_hi"]) if case["op"] == "latent" else
             dict(case, past_lo=case["past_hi"], new_lo=case["new_hi"]))
    bytes_most, flops_most = (3.2e8, 2.9e11) if case["op"] == "latent" else (9.5e8, 9.5e11)
    return w["bytes"] > bytes_most or w["flops"] > flops_most


# ------------------------------------------------------------------ inputs --
def _gen(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _lens(c, lo, hi):
    """One length for each sequence, [lo, hi], the longest among them; the case alone decides them."""
    rng = random.Random(repr((sorted(c.items()), lo, hi)))
    return [hi] + [rng.randint(lo, hi) for _ in range(c["batch"] - 1)]


def _indptr(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _block_table(need, g, device):
    """Pages of each sequence drawn without order from a pool with an eighth to spare; -1 past them."""
    nb = sum(need) + sum(need) // 8 + 1
    order = torch.randperm(nb, generator=g).to(torch.int32)
    bt = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32)
    pos = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[pos:pos + n]
        pos += n
    return nb, bt.to(device), order[pos:].to(device)


def _parents(n, chain, g):
    """Parents of a drafted tree listed parents first; node 0 is the root."""
    if chain:
        return [i - 1 for i in range(n)]
    u = torch.rand((max(n, 1),), generator=g).tolist()
    # near the front more often: drafts branch at their first levels
    return [-1 if i == 0 else int(u[i] ** 1.5 * i) for i in range(n)]


def _see(parents, dead, g):
    """bool [n, n]: which nodes each node sees (itself and its ancestors; a pruned one and its descendants none)."""
    n = len(parents)
    see, u = torch.zeros((n, n), dtype=torch.bool), torch.rand((max(n, 1),), generator=g).tolist()
    gone = [False] * n
    for i, p in enumerate(parents):
        gone[i] = (u[i] < dead) or (p >= 0 and gone[p])
        if gone[i]:
            continue
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


def _pack(see, words):
    """Packs bool [n, n] into int64 [n, words], bit j % 64 of word j / 64."""
    n = see.shape[0]
    bits = torch.zeros((n, words * 64), dtype=torch.int64)
    bits[:, :n] = see.to(torch.int64)
    return (bits.view(n, words, 64) << torch.arange(64, dtype=torch.int64)).sum(-1)


def _angles64(c, device):
    i = torch.arange(ROPE // 2, dtype=torch.float64, device=device)
    pos = torch.arange(c["max_pos"], dtype=torch.float64, device=device)
    return pos[:, None] * 10000.0 ** (-2.0 * i / ROPE)


def _inputs(case, seed):
    device = torch.device("cuda")
    c = case
    g, gc = _gen(seed, device), _gen(seed, "cpu")
    s = dict(case=c)

    def normal(*shape, dtype=None, std=1.0):
        return torch.empty(shape, dtype=DTYPES[c["dtype"]] if dtype is None else dtype, device=device).normal_(
            0.0, std, generator=g)

    if c["op"] == "pages":
        ctx, new = _lens(c, c["ctx_lo"], c["ctx_hi"]), _lens(c, c["nodes_lo"], c["nodes_hi"])
        owned = [-(-n // PAGE) for n in ctx]
        nb, table, free = _block_table(owned, gc, "cpu")
        extra = sum(-(-(n + t) // PAGE) for n, t in zip(ctx, new)) - sum(owned) + 5
        # enough for all, in no order
        free = torch.cat([torch.arange(nb, nb + extra, dtype=torch.int32), free])
        free = free[torch.randperm(len(free), generator=gc)]
        wide = torch.full((c["batch"], max(-(-(n + t) // PAGE) for n, t in zip(ctx, new)) + 2), -1, dtype=torch.int32)
        wide[:, :min(table.shape[1], wide.shape[1])] = table[:, :wide.shape[1]]
        s.update(table=wide.to(device), counts=_int32(owned, device), free=free.to(device),
                 free_count=_int32([len(free)], device), ctx=_int32(ctx, device), indptr=_int32(_indptr(new), device),
                 total=sum(new), mask=None)
        if c["tree"]:
            words = max(1, -(-c["nodes_hi"] // 64))
            masks = [_pack(_see(_parents(n, False, gc), 0.1, gc), words) for n in new]
            s["mask"] = torch.cat(masks).to(device)
    elif c["op"] == "store":
        t = c["tokens"]
        # views of the projections' outputs, as a model has them
        a = normal(t, RANK + ROPE)
        s["latent"], s["k_rope"] = a[:, :RANK], a[:, RANK:]
        s["q_rope"] = normal(t, c["heads"], NOPE + ROPE)[..., NOPE:] if c["heads"] else None
        s["weight"] = 1.0 + normal(RANK, std=0.1) if c["norm"] else None
        s["positions"] = torch.randint(0, c["max_pos"], (t,), dtype=torch.int32, generator=g, device=device)
        nb = t // PAGE + 2
        # the last slot stays free (the plain form writes the padding rows there)
        s["slots"] = torch.randperm(nb * PAGE - 1, generator=g, device=device)[:t].contiguous()
        s["slots"][torch.rand((t,), generator=g, device=device) < c["pad"]] = -1
        s["pool"] = normal(nb, 1, STICKS, PAGE, 64)
        ang = _angles64(c, device)
        s["rope"] = torch.stack([torch.cos(ang), torch.sin(ang)], -1).float()
    elif c["op"] == "latent":
        ctx, new = _lens(c, c["ctx_lo"], c["ctx_hi"]), _lens(c, c["nodes_lo"], c["nodes_hi"])
        nb, s["table"], _ = _block_table([-(-(n + t) // PAGE) for n, t in zip(ctx, new)], gc, device)
        s.update(ctx=ctx, new=new, lens=_int32(ctx, device), indptr=_int32(_indptr(new), device), most=max(new))
        see = [_see(_parents(n, c["chain"], gc), c["dead"], gc) for n in new]
        s["see"] = [m.to(device) for m in see]
        s["mask"] = None if c["chain"] else torch.cat([_pack(m, -(-max(new) // 64)) for m in see]).to(device)
        s["q_latent"], s["q_rope"] = normal(sum(new), c["heads"], RANK), normal(sum(new), c["heads"], ROPE)
        s["pool"] = normal(nb, 1, STICKS, PAGE, 64)
    elif c["op"] == "prompt":
        past, new = _lens(c, c["past_lo"], c["past_hi"]), _lens(c, c["new_lo"], c["new_hi"])
        n, m = sum(new), sum(past) + sum(new)
        s.update(past=past, new=new, q_indptr=_int32(_indptr(new), device),
                 kv_indptr=_int32(_indptr([p + t for p, t in zip(past, new)]), device))
        s["q"] = normal(n, c["heads"], NOPE + ROPE)
        kv = normal(m, c["heads"], 2 * NOPE)
        s["k_nope"], s["v"] = kv[..., :NOPE], kv[..., NOPE:]
        s["k_rope"] = normal(m, RANK + ROPE)[:, RANK:]
    else:
        new = _lens(c, c["nodes_lo"], c["nodes_hi"])
        n, v = sum(new), c["vocab"]
        first = _indptr(new)
        parents = [_parents(t, c["chain"], gc) for t in new]
        s.update(new=new, most=max(new), parents=_int32([p for ps in parents for p in ps], device),
                 indptr=_int32(first, device))
        z = normal(n, v, dtype=torch.float32, std=2.0)
        s["target"] = torch.softmax(z, -1).to(DTYPES[c["dtype"]])
        # the drafter is near the target, not equal to it
        z += normal(n, v, dtype=torch.float32, std=0.7)
        guess = torch.softmax(z, -1)
        del z
        s["draft"] = guess.to(DTYPES[c["dtype"]]) if c["draft"] else None
        row = torch.tensor([first[b] + max(p, 0) for b, ps in enumerate(parents) for p in ps], device=device)
        u = torch.rand((n,), generator=g, device=device, dtype=torch.float64)
        tokens = []
        for i in range(0, n, 64):  # drawn from the drafter's row at the parent
            cdf = guess[row[i:i + 64]].double().cumsum(-1)
            tokens.append((cdf <= (u[i:i + 64] * cdf[:, -1])[:, None]).sum(-1))
        s["tokens"] = torch.cat(tokens).clamp_max(v - 1)
        s["accept_u"] = torch.rand((n,), generator=g, device=device)
        s["sample_u"] = torch.rand((c["batch"],), generator=g, device=device)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------- plain forms --
def _turn(x, cos, sin, interleaved):
    """Pairs of the last axis turned: half layout, or side by side."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x[..., :ROPE // 2], x[..., ROPE // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _rows(pool, slots):
    """Rows [N, 576] of the pool at slots."""
    return pool[slots // PAGE, 0, :, slots % PAGE].flatten(-2)


def _plain_pages(s):
    """Pages taken in the order of the sequences from the top of the stack, then given back."""
    table, counts, free, dev = s["table"], s["counts"], s["free"], s["table"].device
    indptr, ctx = s["indptr"].long(), s["ctx"].long()
    n = torch.arange(s["total"], device=dev)
    new = indptr[1:] - indptr[:-1]
    seq = torch.repeat_interleave(torch.arange(len(new), device=dev), new, output_size=s["total"])
    local = n - indptr[seq]
    pos = ctx[seq] + local
    depth = local
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(64, device=dev)) & 1
        depth = (bits.sum((1, 2)) - 1).clamp_min(0)
    want = (ctx + new + PAGE - 1) // PAGE
    need = (want - counts).clamp_min(0)
    before = need.cumsum(0) - need
    column = torch.arange(table.shape[1], device=dev)
    fresh = (column >= counts[:, None]) & (column < want[:, None])
    rank = (before[:, None] + column - counts[:, None]).clamp(0)
    top = s["free_count"][0].long()
    full = torch.where(fresh, free[(top - 1 - rank).clamp_min(0)], table)
    slots = full[seq, pos // PAGE].long() * PAGE + pos % PAGE
    positions = (ctx[seq] + depth).to(torch.int32)
    # the step ends with nothing kept past the committed tokens: what was taken goes back where it was
    return slots, positions, full


def _plain_store(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    turn = s["rope"][s["positions"].long()]
    x = s["latent"].float()
    if s["weight"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    k = _turn(s["k_rope"].float(), turn[..., 0], turn[..., 1], c["interleaved"])
    live = s["slots"] >= 0
    slots = torch.where(live, s["slots"], s["pool"].shape[0] * PAGE - 1)
    s["pool"][slots // PAGE, 0, :, slots % PAGE] = torch.cat([x, k], -1).to(dt).view(-1, STICKS, 64)
    back = torch.where(live[:, None], _rows(s["pool"], slots), 0.0)
    out = [back[:, :RANK], back[:, RANK:]]
    if s["q_rope"] is not None:
        out.append(_turn(s["q_rope"].float(), turn[:, None, :, 0], turn[:, None, :, 1], c["interleaved"]).to(dt))
    return out


def _softmax(p):
    """Weights of the last axis, in place; a row of -inf gets zeros."""
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _run_latent(s, wide):
    c, pos, outs = s["case"], 0, []
    for b, (ctx, t) in enumerate(zip(s["ctx"], s["new"])):
        pages = s["table"][b, :-(-(ctx + t) // PAGE)].long()
        rows = s["pool"][pages, 0].permute(0, 2, 1, 3).reshape(-1, RANK + ROPE)[:ctx + t].to(wide)
        q = torch.cat([s["q_latent"][pos:pos + t], s["q_rope"][pos:pos + t]], -1).to(wide)
        p = torch.matmul(q.flatten(0, 1), rows.T).mul_(SCALE).view(t, c["heads"], ctx + t)
        p[..., ctx:].masked_fill_(~s["see"][b][:, None], -math.inf)
        outs.append(torch.matmul(_softmax(p).flatten(0, 1), rows[:, :RANK]).view(t, c["heads"], RANK))
        pos += t
    out = torch.cat(outs)
    return out.to(DTYPES[c["dtype"]]) if wide == torch.float32 else out


def _run_prompt(s, wide):
    c, at, kv, outs = s["case"], 0, 0, []
    for past, t in zip(s["past"], s["new"]):
        m = past + t
        q = s["q"][at:at + t].to(wide).transpose(0, 1)
        k = torch.cat([s["k_nope"][kv:kv + m], s["k_rope"][kv:kv + m, None].expand(m, c["heads"], ROPE)], -1)
        k, v = k.to(wide).permute(1, 2, 0), s["v"][kv:kv + m].to(wide).transpose(0, 1)
        out = torch.empty((t, c["heads"], NOPE), dtype=wide, device=q.device)
        hidden = torch.arange(m, device=q.device) > past + torch.arange(t, device=q.device)[:, None]
        for h in range(0, c["heads"], 8) if m and t else ():
            p = torch.matmul(q[h:h + 8], k[h:h + 8]).mul_(SCALE)
            if c["causal"]:
                p.masked_fill_(hidden, -math.inf)
            out[:, h:h + 8] = torch.matmul(_softmax(p), v[h:h + 8]).transpose(0, 1)
        outs.append(out)
        at, kv = at + t, kv + m
    out = torch.cat(outs)
    return out.to(DTYPES[c["dtype"]]) if wide == torch.float32 else out


def _plain_verify(s):
    """All sequences side by side, node after node: a node is tried when its parent is the last one accepted.

    64 bits throughout: whether a token is taken hangs on a comparison.
    """
    c, dev = s["case"], s["tokens"].device
    batch, most = c["batch"], s["most"]
    first, count = s["indptr"][:-1].long(), (s["indptr"][1:] - s["indptr"][:-1]).long()
    lane = torch.arange(batch, device=dev)
    cur = torch.zeros(batch, dtype=torch.int64, device=dev)
    path = torch.full((batch, most), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    taken = torch.ones(batch, dtype=torch.int64, device=dev)
    w = s["target"][first].double()  # what the next token is drawn from, times `mass`
    q = s["draft"][first].double() if c["draft"] else None
    mass = torch.ones(batch, dtype=torch.float64, device=dev)
    for i in range(1, most):
        at = first + torch.clamp(torch.full_like(count, i), max=count - 1)
        tried = (i < count) & (s["parents"][at].long() == cur)
        x = s["tokens"][at]
        wx = w[lane, x]
        limit = s["accept_u"][at].double() * mass.clamp_min(0.0) * (q[lane, x] if c["draft"] else 1.0)
        yes, no = tried & (wx > limit), tried & ~(wx > limit)
        # rejected: what is left of the distribution without what the drafter proposes
        if c["draft"]:
            left = (w - mass[:, None] * q).clamp_min(0.0)
            w = torch.where(no[:, None], left, w)
            mass = torch.where(no, left.sum(-1), mass)
        else:
            mass = torch.where(no, mass - wx, mass)
            w[lane, x] = torch.where(no, 0.0, wx)
        # accepted: on to the node's own distributions
        w = torch.where(yes[:, None], s["target"][at].double(), w)
        if c["draft"]:
            q = torch.where(yes[:, None], s["draft"][at].double(), q)
        mass = torch.where(yes, 1.0, mass)
        cur = torch.where(yes, i, cur)
        path[lane, taken.clamp_max(most - 1)] = torch.where(yes, i, path[lane, taken.clamp_max(most - 1)]).to(torch.int32)
        taken = taken + yes
    p = s["target"][first + cur].double()
    w = torch.where((w.sum(-1) > 0)[:, None], w, p)
    cdf = w.cumsum(-1)
    token = (cdf <= (s["sample_u"].double() * cdf[:, -1])[:, None]).sum(-1)
    return path, taken.to(torch.int32), token


# --------------------------------------------------------------------- run --
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    op = s["case"]["op"]
    if op == "pages":
        return _plain_pages(s) + (s["table"], s["counts"], s["free"], s["free_count"])
    if op == "store":
        return _plain_store(s)
    if op == "latent":
        return _run_latent(s, torch.float32)
    if op == "prompt":
        return _run_prompt(s, torch.float32)
    return _plain_verify(s)


def _run_own(s):
    import torch_spyre_b200 as tsb

    c = s["case"]
    if c["op"] == "pages":
        state = s["table"], s["counts"], s["free"], s["free_count"]
        slots, positions = tsb.extend_pages(*state, s["ctx"], s["indptr"], s["total"], tree_mask=s["mask"])
        full = s["table"].clone()
        tsb.release_pages(*state, s["ctx"])
        return (slots, positions, full) + state
    if c["op"] == "store":
        turned = tsb.latent_store(s["latent"], s["k_rope"], s["pool"], s["slots"], q_rope=s["q_rope"],
                                  norm_weight=s["weight"], eps=EPS, table=s["rope"], positions=s["positions"],
                                  interleaved=c["interleaved"])
        return list(tsb.latent_load(s["pool"], s["slots"])) + ([] if turned is None else [turned])
    if c["op"] == "latent":
        return tsb.latent_attention(s["q_latent"], s["q_rope"], s["pool"], s["table"], s["lens"], s["indptr"],
                                    tree_mask=s["mask"], scale=SCALE, max_nodes=s["most"])
    if c["op"] == "prompt":
        return tsb.latent_prompt_attention(s["q"], s["k_nope"], s["k_rope"], s["v"], s["q_indptr"], s["kv_indptr"],
                                           scale=SCALE, causal=c["causal"])
    return tsb.tree_verify(s["parents"], s["tokens"], s["indptr"], s["target"], s["accept_u"], s["sample_u"],
                           draft_probs=s["draft"], max_path=s["most"])


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    c = case
    if c["op"] == "pages":
        return None
    s = _inputs(c, seed)
    if c["op"] == "latent":
        return _run_latent(s, torch.float64)
    if c["op"] == "prompt":
        return _run_prompt(s, torch.float64)
    if c["op"] == "store":
        z = torch.polar(torch.ones((), dtype=torch.float64, device=s["slots"].device), _angles64(c, s["slots"].device))
        z = z[s["positions"].long()]

        def turned(x, z):
            """Each pair as a complex number, multiplied by the turn."""
            x = x.double()
            if c["interleaved"]:
                return torch.view_as_real(torch.complex(x[..., 0::2], x[..., 1::2]) * z).flatten(-2)
            y = torch.complex(x[..., :ROPE // 2], x[..., ROPE // 2:]) * z
            return torch.cat([y.real, y.imag], -1)

        x = s["latent"].double()
        if c["norm"]:
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].double()
        live = (s["slots"] >= 0)[:, None]
        out = [torch.where(live, x, 0.0), torch.where(live, turned(s["k_rope"], z), 0.0)]
        return out + ([turned(s["q_rope"], z[:, None])] if c["heads"] else [])
    # verify: one sequence after the other, one child after the other, distributions normalised as they come
    parents, tokens, au, su = (s[k].tolist() for k in ("parents", "tokens", "accept_u", "sample_u"))
    paths, lens, nexts, first = [], [], [], 0
    for b, n in enumerate(s["new"]):
        path = [0]
        while True:
            p = s["target"][first + path[-1]].double()
            whole, step = p, None
            for i in range(path[-1] + 1, n):
                if parents[first + i] != path[-1]:
                    continue
                x = tokens[first + i]
                if c["draft"]:
                    q = s["draft"][first + path[-1]].double()
                    if au[first + i] * float(q[x]) < float(p[x]):
                        step = i
                        break
                    p = (p - q).clamp_min(0.0)
                    total = float(p.sum())
                    p = p / total if total > 0 else p
                else:
                    if au[first + i] < float(p[x]):
                        step = i
                        break
                    rest = 1.0 - float(p[x])
                    p = p.clone()
                    p[x] = 0.0
                    p = p / rest if rest > 0 else p
            if step is None:
                break
            path.append(step)
        p = p if float(p.sum()) > 0 else whole
        cdf = p.cumsum(-1)
        nexts.append(int((cdf <= su[b] * float(cdf[-1])).sum()))
        lens.append(len(path))
        paths.append(path + [-1] * (s["most"] - len(path)))
        first += n
    dev = s["tokens"].device
    return _int32(paths, dev), _int32(lens, dev), torch.tensor(nexts, device=dev)


# -------------------------------------------------------------------- work --
def work(case):
    c = case
    if c["op"] == "pages":
        n = c["batch"] * (c["nodes_lo"] + c["nodes_hi"]) / 2.0
        pages = n / PAGE + c["batch"] * 0.5
        # lengths in; slots, positions and table entries out, the entries taken back
        return {"bytes": int(c["batch"] * 24 + n * (12 + (8 if c["tree"] else 0)) + pages * 24), "flops": 0}
    if c["op"] == "store":
        t, e = c["tokens"], ESIZE[c["dtype"]]
        row = (RANK + ROPE) * e
        # rows and the heads' rotary parts in and out, the rows read back and out; the turn, slots
        return {"bytes": t * (4 * row + 2 * c["heads"] * ROPE * e + ROPE * 4 + 12 + 8),
                "flops": t * (4 * RANK + 3 * ROPE * (c["heads"] + 1))}
    if c["op"] == "latent":
        ctx, n = (c["ctx_lo"] + c["ctx_hi"]) / 2.0, (c["nodes_lo"] + c["nodes_hi"]) / 2.0
        seen = ctx + (n / 2.0 if c["chain"] else min(n, 4.0))
        return {"bytes": int(c["batch"] * ((ctx + n) * ((RANK + ROPE) * 2 + 4.0 / PAGE)
                                           + n * c["heads"] * (2 * RANK + ROPE) * 2)),
                "flops": int(c["batch"] * n * c["heads"] * seen * 2 * (2 * RANK + ROPE))}
    if c["op"] == "prompt":
        past, n = (c["past_lo"] + c["past_hi"]) / 2.0, (c["new_lo"] + c["new_hi"]) / 2.0
        seen = past + (n / 2.0 if c["causal"] else n)
        return {"bytes": int(c["batch"] * ((past + n) * (c["heads"] * 2 * NOPE + ROPE) * 2
                                           + n * c["heads"] * (2 * NOPE + ROPE) * 2)),
                "flops": int(c["batch"] * n * c["heads"] * seen * 2 * (2 * NOPE + ROPE))}
    # a row of probabilities a sequence (the drafter's too), the numbers of its nodes
    n = (c["nodes_lo"] + c["nodes_hi"]) / 2.0
    row = c["vocab"] * ESIZE[c["dtype"]] * (2 if c["draft"] else 1)
    return {"bytes": int(c["batch"] * (row + n * 28 + 24)), "flops": int(c["batch"] * c["vocab"] * 4)}
