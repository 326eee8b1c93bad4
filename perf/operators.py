"""Speculative verification over a paged cache: the operators, their plain forms and measured cases.

The operators (layouts as in include/b200kv.h, tokens in 64-token pages of 128-byte sticks):

* ``rotary``   rotary positions of rows [T, H, D], half or interleaved pairs, part of the head,
               table scaled for long contexts; forward and gradient.
* ``store``    K/V rows rotated, quantised (one fp32 scale per token and head) and written to
               their slots, q rotated beside them; the rows are read back.
* ``load``     rows of an 8-bit cache gathered by slot and dequantised.
* ``tree``     attention of each sequence's drafted tokens over its committed tokens and those
               of its own draft that the tree mask shows (no mask: a chain, each sees its past).
* ``commit``   the accepted path's rows moved to the end of the committed tokens.
"""

import math
import random

import torch

own = False

PAGE = 64
QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32,
          "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ESIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "int8": 1, "e4m3": 1}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One decode step of 16 sequences: q and k heads of a fused projection, latency counts.
        dict(name="rotary_decode", op="rotary", dtype="fp16", tokens=16, heads=40, beside=8, dim=128, rotary_dim=128,
             interleaved=False, scaling="none", max_pos=8192, backward=False),
        # A training step's 8k tokens: half the head rotated, pairs side by side, yarn table, gradient.
        dict(name="rotary_train", op="rotary", dtype="bf16", tokens=8192, heads=40, beside=0, dim=128, rotary_dim=64,
             interleaved=True, scaling="yarn", max_pos=32768, backward=True),
        # 16 sequences' drafts of 8 nodes written to an int8 cache.
        dict(name="store_draft", op="store", dtype="fp16", cache="int8", tokens=128, q_heads=32, kv_heads=8,
             dim=128, rotary_dim=128, interleaved=False, scaling="none", max_pos=8192, pad=0.0),
        # A prompt of odd length written to an e4m3 cache, partial rotation, a few padding rows.
        dict(name="store_prompt", op="store", dtype="bf16", cache="e4m3", tokens=16381, q_heads=32, kv_heads=8,
             dim=128, rotary_dim=96, interleaved=True, scaling="linear", max_pos=32768, pad=0.02),
        # A short prefix read back in the compute type.
        dict(name="load_prefix", op="load", cache="int8", dtype="fp16", tokens=777, kv_heads=8, dim=128),
        # The bulk read of 128k tokens.
        dict(name="load_bulk", op="load", cache="e4m3", dtype="bf16", tokens=131072, kv_heads=8, dim=128),
        # 16 sequences accept up to 8 drafted tokens each.
        dict(name="commit_draft", op="commit", cache="int8", batch=16, kv_heads=8, dim=128, nodes=64, path=8,
             ctx_lo=512, ctx_hi=4096),
        # A serving batch of 128 with long drafts (short contexts: the move does not depend on them).
        dict(name="commit_batch", op="commit", cache="fp16", batch=128, kv_heads=8, dim=128, nodes=128, path=64,
             ctx_lo=128, ctx_hi=512),
        # One sequence, 32/32 heads, a draft of 8 nodes over 1k tokens: the smallest attention.
        dict(name="tree_single", op="tree", dtype="fp16", cache="fp16", batch=1, q_heads=32, kv_heads=32, dim=128,
             ctx_lo=1024, ctx_hi=1024, nodes_lo=8, nodes_hi=8, chain=False, dead=0.0),
        # 16 sequences, 32/8 heads, ragged contexts and drafts, some nodes pruned.
        dict(name="tree_ragged", op="tree", dtype="bf16", cache="bf16", batch=16, q_heads=32, kv_heads=8, dim=128,
             ctx_lo=512, ctx_hi=8192, nodes_lo=1, nodes_hi=64, chain=False, dead=0.05),
        # Long contexts in an int8 cache, drafts of 16 nodes.
        dict(name="tree_long", op="tree", dtype="fp16", cache="int8", batch=4, q_heads=32, kv_heads=8, dim=128,
             ctx_lo=32768, ctx_hi=131072, nodes_lo=16, nodes_hi=16, chain=False, dead=0.0),
        # Chunks of a long prompt (a chain) over their committed past, 64/8 heads.
        dict(name="tree_chunk", op="tree", dtype="fp16", cache="fp16", batch=2, q_heads=64, kv_heads=8, dim=128,
             ctx_lo=8001, ctx_hi=8192, nodes_lo=1024, nodes_hi=1024, chain=True, dead=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "store", "load", "commit", "tree", "tree", "tree"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        interleaved = rng.random() < 0.5
        rd = dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)
        return dict(op=op, dtype=rng.choice(["fp16", "bf16", "fp32"]), tokens=_log(rng, 1, 8192),
                    heads=rng.randint(1, 40), beside=rng.choice([0, 0, 1, 8]), dim=dim, rotary_dim=rd, interleaved=interleaved,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), max_pos=_log(rng, 64, 32768),
                    backward=rng.random() < 0.5)
    if op == "store":
        cache = rng.choice(["same", "int8", "e4m3"])
        dim = rng.choice([64, 128]) if cache == "same" else 128
        kv = rng.choice([1, 2, 4, 8])
        return dict(op=op, dtype=dtype, cache=dtype if cache == "same" else cache, tokens=_log(rng, 1, 16381),
                    q_heads=kv * rng.randint(1, 4), kv_heads=kv, dim=dim, rotary_dim=16 * rng.randint(1, dim // 16),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    max_pos=_log(rng, 64, 32768), pad=rng.choice([0.0, 0.1]))
    if op == "load":
        return dict(op=op, cache=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    tokens=_log(rng, 1, 65536), kv_heads=rng.randint(1, 8), dim=128)
    if op == "commit":
        cache = rng.choice(["fp16", "bf16", "int8", "e4m3"])
        nodes = _log(rng, 1, 128)
        return dict(op=op, cache=cache, batch=_log(rng, 1, 128), kv_heads=rng.randint(1, 8), dim=128, nodes=nodes,
                    path=rng.randint(0, nodes), ctx_lo=0, ctx_hi=_log(rng, 1, 512))
    cache = rng.choice(["same", "int8", "e4m3"])
    dim = rng.choice([64, 128]) if cache == "same" else 128
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    chain = rng.random() < 0.3
    hi, ctx_hi = _log(rng, 1, 1024 if chain else 128), _log(rng, 1, 131072)
    case = dict(op=op, dtype=dtype, cache=dtype if cache == "same" else cache, batch=_log(rng, 1, 64),
                q_heads=kv * group, kv_heads=kv, dim=dim, ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]), ctx_hi=ctx_hi,
                nodes_lo=rng.randint(1, hi), nodes_hi=hi, chain=chain, dead=0.0 if chain else rng.choice([0.0, 0.2]))
    # no more cached bytes than the longest listed batch and no more products than the chunked prompt
    while _over(dict(case, ctx_lo=ctx_hi, nodes_lo=case["nodes_hi"])):
        if case["batch"] > 1:
            case["batch"] -= 1
        else:
            case["nodes_hi"] //= 2
            case["nodes_lo"] = min(case["nodes_lo"], case["nodes_hi"])
    return case


def _over(case):
    w = work(case)
    return w["bytes"] > 6.9e8 or w["flops"] > 5.7e11


# ------------------------------------------------------------------ inputs --
def _gen(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


SCALING = {"none": dict(factor=1.0, original=0), "linear": dict(factor=4.0, original=0),
           "ntk": dict(factor=4.0, original=0), "yarn": dict(factor=4.0, original=4096)}
BASE = 10000.0


def _angles64(c, device):
    """fp64 angles [max_pos, rotary_dim / 2] and the factor on cos and sin."""
    rd, s = c["rotary_dim"], SCALING[c["scaling"]]
    base, m = BASE, 1.0
    if c["scaling"] == "ntk":
        base = base * s["factor"] ** (rd / (rd - 2.0)) if rd > 2 else base
    i = torch.arange(rd // 2, dtype=torch.float64, device=device)
    inv = base ** (-2.0 * i / rd)
    if c["scaling"] == "linear":
        inv = inv / s["factor"]
    if c["scaling"] == "yarn":
        def dim_of(turns):
            return rd * math.log(s["original"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        lo, hi = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), rd // 2 - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / s["factor"] * ramp
        m = 0.1 * math.log(s["factor"]) + 1.0
    pos = torch.arange(c["max_pos"], dtype=torch.float64, device=device)
    return pos[:, None] * inv, m


def _table64(c, device):
    ang, m = _angles64(c, device)
    return torch.stack([torch.cos(ang) * m, torch.sin(ang) * m], -1)


def _table(c, device):
    if own:
        import torch_spyre_b200 as tsb

        s = SCALING[c["scaling"]]
        return tsb.rotary_table(c["max_pos"], c["rotary_dim"], base=BASE, scaling=c["scaling"], factor=s["factor"],
                                original_max_pos=s["original"] or None, device=device)
    return _table64(c, device).float()


def _rand_cache(nb, c, g, device):
    """A pool of the case's cache type holding rows of N(0, 1) values (scales for 8-bit types)."""
    kind, hkv, d = c["cache"], c["kv_heads"], c["dim"]
    if kind in QMAX:
        shape = (nb, hkv, d // 128, PAGE, 128)
        if kind == "int8":
            pool = torch.empty(shape, dtype=torch.int8, device=device)
            pool.random_(-127, 128, generator=g)
        else:
            pool = torch.empty(shape, dtype=torch.float16, device=device).normal_(0.0, 120.0, generator=g)
            pool = pool.clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
        scales = torch.rand((nb, hkv, PAGE), generator=g, device=device) * 0.02 + 0.01
        if kind == "e4m3":
            scales = scales * (127.0 / 448.0)
        return pool, scales
    shape = (nb, hkv, d // 64, PAGE, 64)
    return torch.empty(shape, dtype=DTYPES[kind], device=device).normal_(0.0, 1.0, generator=g), None


def _lens(c, lo, hi):
    """One length for each sequence, [lo, hi], the longest among them; the case alone decides them."""
    rng = random.Random(repr((sorted(c.items()), lo, hi)))
    return [hi] + [rng.randint(lo, hi) for _ in range(c["batch"] - 1)]


def _block_table(need, g, device):
    """Pages of each sequence drawn without order from a pool with an eighth to spare."""
    nb = sum(need) + sum(need) // 8 + 1
    order = torch.randperm(nb, generator=g)
    bt = torch.zeros((len(need), max(need)), dtype=torch.int32)
    pos = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[pos:pos + n].to(torch.int32)
        pos += n
    return nb, bt.to(device)


def _draft(n, chain, dead, g):
    """bool [n, n]: which draft nodes each node sees (itself and its ancestors; a pruned node none)."""
    if chain:
        return torch.ones((n, n), dtype=torch.bool).tril_()
    see = torch.zeros((n, n), dtype=torch.bool)
    u = torch.rand((2, n), generator=g)
    for i in range(n):
        if i and float(u[0, i]) < 0.9:
            see[i] = see[int(float(u[0, i]) / 0.9 * i)]
        see[i, i] = True
    see[u[1] < dead] = False
    return see


def _pack(see, words):
    """Packs bool [n, n] into int64 [n, words], bit j % 64 of word j / 64."""
    n = see.shape[0]
    bits = torch.zeros((n, words * 64), dtype=torch.int64)
    bits[:, :n] = see.to(torch.int64)
    return (bits.view(n, words, 64) << torch.arange(64, dtype=torch.int64)).sum(-1)


def _inputs(case, seed):
    device = torch.device("cuda")
    c = case
    g, gc = _gen(seed, device), _gen(seed, "cpu")
    s = dict(case=c)
    if c["op"] == "rotary":
        dt = DTYPES[c["dtype"]]
        shape = (c["tokens"], c["heads"], c["dim"])
        fused = torch.empty((c["tokens"], c["heads"] + c["beside"], c["dim"]), dtype=dt, device=device)
        s["x"] = fused.normal_(0.0, 1.0, generator=g)[:, :c["heads"]]
        s["positions"] = torch.randint(0, c["max_pos"], (c["tokens"],), dtype=torch.int32, generator=g, device=device)
        if c["backward"]:
            s["grad"] = torch.empty(shape, dtype=dt, device=device).normal_(0.0, 1.0, generator=g)
    elif c["op"] == "store":
        dt, t = DTYPES[c["dtype"]], c["tokens"]
        for name, h in (("q", "q_heads"), ("k", "kv_heads"), ("v", "kv_heads")):
            s[name] = torch.empty((t, c[h], c["dim"]), dtype=dt, device=device).normal_(0.0, 1.0, generator=g)
        s["positions"] = torch.randint(0, c["max_pos"], (t,), dtype=torch.int32, generator=g, device=device)
        nb = t // PAGE + 2
        # the last slot stays free (the plain form writes the padding rows there)
        s["slots"] = torch.randperm(nb * PAGE - 1, generator=g, device=device)[:t].contiguous()
        s["slots"][torch.rand((t,), generator=g, device=device) < c["pad"]] = -1
        s["k_pool"], s["k_scales"] = _rand_cache(nb, c, g, device)
        s["v_pool"], s["v_scales"] = _rand_cache(nb, c, g, device)
    elif c["op"] == "load":
        t = c["tokens"]
        nb, bt = _block_table([-(-t // PAGE)], gc, device)
        tok = torch.arange(t, device=device)
        s["slots"] = bt[0].long()[tok // PAGE] * PAGE + tok % PAGE
        s["pool"], s["scales"] = _rand_cache(nb, c, g, device)
    elif c["op"] == "commit":
        ctx = _lens(c, c["ctx_lo"], c["ctx_hi"])
        nb, s["block_table"] = _block_table([-(-(n + c["nodes"]) // PAGE) for n in ctx], gc, device)
        s["ctx"] = ctx
        s["context_lens"] = torch.tensor(ctx, dtype=torch.int32, device=device)
        plen = _lens(c, 0, c["path"])
        path = torch.zeros((c["batch"], max(c["path"], 1)), dtype=torch.int32)
        for b, n in enumerate(plen):
            # a run from the root that is in place already, then nodes past the places to be filled:
            # a second pass over the same state moves the same rows again
            lead = max(int(torch.randint(0, n + 1, (1,), generator=gc)), 2 * n - c["nodes"])
            far = n + torch.randperm(c["nodes"] - n, generator=gc)[:n - lead].sort().values
            path[b, :n] = torch.cat([torch.arange(lead), far]).to(torch.int32)
        s["plen"] = plen
        s["path"], s["path_lens"] = path.to(device), torch.tensor(plen, dtype=torch.int32, device=device)
        s["k_pool"], s["k_scales"] = _rand_cache(nb, c, g, device)
        s["v_pool"], s["v_scales"] = _rand_cache(nb, c, g, device)
    else:
        ctx, nodes = _lens(c, c["ctx_lo"], c["ctx_hi"]), _lens(c, c["nodes_lo"], c["nodes_hi"])
        nb, s["block_table"] = _block_table([-(-(n + t) // PAGE) for n, t in zip(ctx, nodes)], gc, device)
        s["ctx"], s["nodes"] = ctx, nodes
        s["context_lens"] = torch.tensor(ctx, dtype=torch.int32, device=device)
        indptr = [0]
        for t in nodes:
            indptr.append(indptr[-1] + t)
        s["q_indptr"] = torch.tensor(indptr, dtype=torch.int32, device=device)
        see = [_draft(t, c["chain"], c["dead"], gc) for t in nodes]
        words = -(-max(nodes) // 64)
        s["see"] = [m.to(device) for m in see]
        s["tree_mask"] = None if c["chain"] else torch.cat([_pack(m, words) for m in see]).to(device)
        s["max_nodes"] = max(nodes)
        s["q"] = torch.empty((indptr[-1], c["q_heads"], c["dim"]), dtype=DTYPES[c["dtype"]],
                             device=device).normal_(0.0, 1.0, generator=g)
        s["k_pool"], s["k_scales"] = _rand_cache(nb, c, g, device)
        s["v_pool"], s["v_scales"] = _rand_cache(nb, c, g, device)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if "rotary_dim" in case:
        s["table"] = _table(case, s["positions"].device)
    if case.get("backward") and own:
        s["x"].requires_grad_(True)
    return s


# ------------------------------------------------------------- plain forms --
def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 or 64 bits, cos / sin [T, rotary_dim / 2]."""
    half = cos.shape[-1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([rot, rest], -1)


def _quantise(x, kind):
    """(values in steps, scale) of rows x [T, H, D] in an 8-bit cache: one scale per row, amax / qmax."""
    qmax = QMAX[kind]
    scale = x.abs().amax(-1, keepdim=True) / qmax
    q = (x * torch.where(scale > 0, 1.0 / scale, 0.0)).clamp(-qmax, qmax)
    if kind == "int8":
        q = torch.round(q)
    elif x.dtype == torch.float32:
        q = q.to(torch.float8_e4m3fn).to(x.dtype)
    else:  # to the nearest e4m3 number, ties to even: steps of 2^-3 of the power of two below, 2^-9 at least
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3.0)
        q = torch.round(q / step) * step
    return q, scale


def _rows(pool, slots):
    """Rows [N, Hkv, D] of the pool at slots."""
    return pool[slots // PAGE, :, :, slots % PAGE].flatten(-2)


def _run_store(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    cs = s["table"][s["positions"].long()]
    live = s["slots"] >= 0
    slots = torch.where(live, s["slots"], s["k_pool"].shape[0] * PAGE - 1)
    out = [_rotate(s["q"].float(), cs[..., 0], cs[..., 1], c["interleaved"]).to(dt)]
    rotated = _rotate(s["k"].float(), cs[..., 0], cs[..., 1], c["interleaved"])
    for x, pool, scales in ((rotated, s["k_pool"], s["k_scales"]), (s["v"].float(), s["v_pool"], s["v_scales"])):
        if scales is not None:
            x, scale = _quantise(x, c["cache"])
            scales[slots // PAGE, :, slots % PAGE] = scale[..., 0]
        raw = pool if pool.element_size() == 2 else pool.view(torch.int8)
        x = x.to(pool.dtype).view(raw.dtype).view(*x.shape[:2], pool.shape[2], pool.shape[4])
        raw[slots // PAGE, :, :, slots % PAGE] = x
        x = _rows(pool, slots).float()
        if scales is not None:
            x = x * _rows(scales[:, :, None, :, None], slots)
        out.append(torch.where(live[:, None, None], x, 0.0).to(dt))
    return out


def _run_tree(s, wide):
    c = s["case"]
    group, d = c["q_heads"] // c["kv_heads"], c["dim"]
    scale, pos, outs = 1.0 / math.sqrt(d), 0, []
    for b, (ctx, t) in enumerate(zip(s["ctx"], s["nodes"])):
        pages = s["block_table"][b, :-(-(ctx + t) // PAGE)].long()

        def rows(pool, scales):
            x = pool[pages].permute(1, 0, 3, 2, 4).flatten(-2).flatten(1, 2)[:, :ctx + t].to(wide)
            if scales is not None:
                x = x * scales[pages].permute(1, 0, 2).flatten(1)[:, :ctx + t, None].to(wide)
            return x

        q = s["q"][pos:pos + t].to(wide).view(t, c["kv_heads"], group, d).permute(1, 2, 0, 3).flatten(1, 2)
        p = torch.matmul(q, rows(s["k_pool"], s["k_scales"]).transpose(1, 2)).mul_(scale).view(-1, group, t, ctx + t)
        p[..., ctx:].masked_fill_(~s["see"][b], -math.inf)
        top = p.amax(-1, keepdim=True)
        p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.flatten(1, 2), rows(s["v_pool"], s["v_scales"])).view(-1, group, t, d)
        o = torch.where(total > 0, o / total, 0.0)
        outs.append(o.permute(2, 0, 1, 3).reshape(t, c["q_heads"], d))
        pos += t
    out = torch.cat(outs)
    return out.to(DTYPES[c["dtype"]]) if wide == torch.float32 else out


def _commit_slots(s):
    """(source, destination) slots of every accepted node, all sequences one after the other."""
    dev = s["path"].device
    seq, step, at = [], [], []
    for b, (ctx, n) in enumerate(zip(s["ctx"], s["plen"])):
        seq += [b] * n
        step += list(range(n))
        at += [ctx] * n
    seq, step, at = (torch.tensor(v, dtype=torch.int64, device=dev) for v in (seq, step, at))
    src, dst = at + s["path"][seq, step].long(), at + step
    return [s["block_table"][seq, t // PAGE].long() * PAGE + t % PAGE for t in (src, dst)]


def _run_commit(s):
    if "moves" not in s:
        s["moves"] = _commit_slots(s)  # kept with the plain form's plan: the host knows the lengths
    src, dst = s["moves"]
    for pool, scales in ((s["k_pool"], s["k_scales"]), (s["v_pool"], s["v_scales"])):
        raw = pool.view(torch.int16) if pool.element_size() == 2 else pool.view(torch.int8)
        raw[dst // PAGE, :, :, dst % PAGE] = raw[src // PAGE, :, :, src % PAGE]
        if scales is not None:
            scales[dst // PAGE, :, dst % PAGE] = scales[src // PAGE, :, src % PAGE]
    return s["context_lens"] + s["path_lens"]


def _commit_out(s, lens):
    """The updated state: the pools as they are, in 8 bits as whole bytes beside their scales."""
    def raw(pool):
        return pool.view(torch.uint8) if pool.element_size() == 1 else pool
    out = [raw(s["k_pool"]), raw(s["v_pool"]), lens]
    return out + [x for x in (s["k_scales"], s["v_scales"]) if x is not None]


# --------------------------------------------------------------------- run --
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        cs = s["table"][s["positions"].long()]
        y = _rotate(s["x"].float(), cs[..., 0], cs[..., 1], c["interleaved"]).to(s["x"].dtype)
        if not c["backward"]:
            return y
        # y is linear in x: the gradient is the transposed map, the turn by the opposite angle
        return y, _rotate(s["grad"].float(), cs[..., 0], -cs[..., 1], c["interleaved"]).to(s["x"].dtype)
    if c["op"] == "store":
        return _run_store(s)
    if c["op"] == "load":
        x = _rows(s["pool"], s["slots"]).float() * _rows(s["scales"][:, :, None, :, None], s["slots"])
        return x.to(DTYPES[c["dtype"]])
    if c["op"] == "commit":
        return _commit_out(s, _run_commit(s))
    return _run_tree(s, torch.float32)


def _run_own(s):
    import torch_spyre_b200 as tsb

    c = s["case"]
    if c["op"] == "rotary":
        y = tsb.rotary(s["x"], s["table"], s["positions"], interleaved=c["interleaved"])
        if not c["backward"]:
            return y
        return y.detach(), torch.autograd.grad(y, s["x"], s["grad"])[0]
    if c["op"] == "store":
        q = tsb.kv_store(s["k"], s["v"], s["k_pool"], s["v_pool"], s["slots"], k_scales=s["k_scales"],
                         v_scales=s["v_scales"], q=s["q"], table=s["table"], positions=s["positions"],
                         interleaved=c["interleaved"])
        dt = DTYPES[c["dtype"]]
        return [q, tsb.kv_load(s["k_pool"], s["slots"], scales=s["k_scales"], dtype=dt),
                tsb.kv_load(s["v_pool"], s["slots"], scales=s["v_scales"], dtype=dt)]
    if c["op"] == "load":
        return tsb.kv_load(s["pool"], s["slots"], scales=s["scales"], dtype=DTYPES[c["dtype"]])
    if c["op"] == "commit":
        lens = tsb.tree_commit(s["k_pool"], s["v_pool"], s["block_table"], s["context_lens"], s["path"],
                               s["path_lens"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return _commit_out(s, lens)
    return tsb.tree_attention(s["q"], s["k_pool"], s["v_pool"], s["block_table"], s["context_lens"], s["q_indptr"],
                              tree_mask=s["tree_mask"], max_nodes=s["max_nodes"], k_scales=s["k_scales"],
                              v_scales=s["v_scales"])


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    c = case
    if c["op"] == "commit":
        return None
    s = _inputs(c, seed)
    if c["op"] == "tree":
        return _run_tree(s, torch.float64)
    if c["op"] == "load":
        return _rows(s["pool"], s["slots"]).double() * _rows(s["scales"][:, :, None, :, None], s["slots"]).double()
    ang, m = _angles64(c, s["positions"].device)
    turn = torch.polar(torch.full_like(ang, m), ang)[s["positions"].long()][:, None, :]
    half = c["rotary_dim"] // 2

    def rotated(x, turn):
        """Each pair as a complex number, multiplied by the turn."""
        x = x.double()
        if c["interleaved"]:
            z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn
            head = torch.view_as_real(z).reshape(*x.shape[:-1], 2 * half)
        else:
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
            head = torch.cat([z.real, z.imag], -1)
        return torch.cat([head, x[..., 2 * half:]], -1)

    if c["op"] == "rotary":
        y = rotated(s["x"], turn)
        return (y, rotated(s["grad"], turn.conj())) if c["backward"] else y
    out = [rotated(s["q"], turn)]
    for x in (rotated(s["k"], turn), s["v"].double()):
        if c["cache"] in QMAX:
            x, scale = _quantise(x, c["cache"])
            x = x * scale
        out.append(torch.where((s["slots"] >= 0)[:, None, None], x, 0.0))
    return out


# -------------------------------------------------------------------- work --
def work(case):
    c = case
    if c["op"] == "rotary":
        n, times = c["tokens"] * c["heads"], 2 if c["backward"] else 1
        return {"bytes": times * (2 * n * c["dim"] * ESIZE[c["dtype"]] + c["tokens"] * (4 + 4 * c["rotary_dim"])),
                "flops": times * 3 * n * c["rotary_dim"]}
    if c["op"] == "store":
        t, d, e = c["tokens"], c["dim"], ESIZE[c["dtype"]]
        row = d * ESIZE[c["cache"]] + (4 if c["cache"] in QMAX else 0)
        # read q, k, v and the turn; write q and the cache; read the cache back and write it out
        return {"bytes": t * (2 * c["q_heads"] * d * e + 2 * c["kv_heads"] * (2 * d * e + 2 * row)
                              + 4 * c["rotary_dim"] + 28),
                "flops": t * (3 * c["rotary_dim"] * (c["q_heads"] + c["kv_heads"]) + 8 * d * c["kv_heads"])}
    if c["op"] == "load":
        n = c["tokens"] * c["kv_heads"]
        return {"bytes": n * (c["dim"] * (ESIZE[c["cache"]] + ESIZE[c["dtype"]]) + 4) + 8 * c["tokens"],
                "flops": n * c["dim"]}
    if c["op"] == "commit":
        n = c["batch"] * c["path"] / 2.0 * c["kv_heads"]
        row = c["dim"] * ESIZE[c["cache"]] + (4 if c["cache"] in QMAX else 0)
        return {"bytes": int(4 * n * row + c["batch"] * (2 * c["path"] + 12)), "flops": 0}
    ctx, nodes = (c["ctx_lo"] + c["ctx_hi"]) / 2.0, (c["nodes_lo"] + c["nodes_hi"]) / 2.0
    row = c["dim"] * ESIZE[c["cache"]] + (4 if c["cache"] in QMAX else 0)
    seen = ctx + (nodes / 2.0 if c["chain"] else min(nodes, 4.0))
    return {"bytes": int(c["batch"] * ((ctx + nodes) * (2 * c["kv_heads"] * row + 4.0 / PAGE)
                                       + 2 * nodes * c["q_heads"] * c["dim"] * ESIZE[c["dtype"]])),
            "flops": int(c["batch"] * nodes * c["q_heads"] * seen * 4 * c["dim"])}
