"""Sampled decoding with drafted trees over a paged latent cache, without the host.

    python examples/serve_latent.py [--dtype float16|bfloat16] [--steps 24] [--no-graph]

A small random decoder with latent attention writes its prompts in chunks, in the
expanded form, then takes steps in the absorbed one.  A step's lengths, pages,
slots and accepted tokens stay on the GPU, so it is captured into a graph once:

    slots, positions = extend_pages(table, counts, free, free_count, lens, ...)   room for the drafts
    per layer:
      q_rope = latent_store(latent, k_rope, pool, slots, q_rope, norm, ...)       rows normalised, turned, written
      x = latent_attention(q_latent, q_rope, pool, table, lens, ..., mask)        nodes over the cache and the tree
    path, path_lens, token = tree_verify(parents, tokens, ..., p, draft_probs=q)  what stays, what comes next
    lens = latent_commit(pool, table, lens, path, path_lens)                      per layer, the accepted path
    release_pages(table, counts, free, free_count, lens)                          pages of the rejected drafts

The drafter is a table of what follows a token.  In the end every text is run once
more without a cache (a plain attention in fp32), and the probabilities that its
tokens were taken with must be the plain run's up to rounding.
"""

from __future__ import annotations

import argparse
import random
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import torch_spyre_b200 as tsb  # noqa: E402

LAYERS, HEADS, HIDDEN, VOCAB, MAX_LEN, PAGE = 2, 8, 512, 600, 640, 64
RANK, ROPE, NOPE = 512, 64, 128
PARENTS, DEPTH = [-1, 0, 0, 1, 1, 2, 3, 6], 5  # a drafted tree, nodes of its longest path


class Decoder:
    """Random weights; one latent attention and one linear layer per block."""

    def __init__(self, dtype: torch.dtype, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape, fan):
            return (torch.randn(shape, generator=g, device="cuda") * fan**-0.5).to(dtype)

        self.embed = weight(VOCAB, HIDDEN, fan=1)
        self.down = [weight(HIDDEN, RANK + ROPE, fan=HIDDEN) for _ in range(LAYERS)]
        self.norm = [1 + weight(RANK, fan=100) for _ in range(LAYERS)]
        self.query = [weight(HIDDEN, HEADS * (NOPE + ROPE), fan=HIDDEN) for _ in range(LAYERS)]
        self.key = [weight(HEADS, NOPE, RANK, fan=RANK) for _ in range(LAYERS)]
        self.value = [weight(HEADS, RANK, NOPE, fan=RANK) for _ in range(LAYERS)]
        self.out = [weight(HEADS * NOPE, HIDDEN, fan=HEADS * NOPE) for _ in range(LAYERS)]
        self.mlp = [weight(HIDDEN, HIDDEN, fan=HIDDEN) for _ in range(LAYERS)]
        self.head = weight(HIDDEN, VOCAB, fan=HIDDEN)
        self.drafter = self.probs(self.embed)  # [VOCAB, VOCAB]: after a token, the decoder without its layers

    def probs(self, h):
        return torch.softmax((F.rms_norm(h, (HIDDEN,)) @ self.head).float(), -1)

    def run(self, tokens, attend):
        """Distributions after tokens [N]; attend(layer, latent, k_rope, q) is the attention of the rows,
        q [N, HEADS, 192], its result [N, HEADS, 128]."""
        h = self.embed[tokens]
        for layer in range(LAYERS):
            x = F.rms_norm(h, (HIDDEN,))
            latent, k_rope = (x @ self.down[layer]).split((RANK, ROPE), 1)
            q = (x @ self.query[layer]).view(-1, HEADS, NOPE + ROPE)
            h = h + attend(layer, latent, k_rope, q).reshape(-1, HEADS * NOPE) @ self.out[layer]
            h = h + F.silu(F.rms_norm(h, (HIDDEN,)) @ self.mlp[layer])
        return self.probs(h)


class Cache:
    """Latent rows of every layer in pages that all sequences share."""

    def __init__(self, model: Decoder, batch: int, blocks: int, dtype: torch.dtype):
        self.model, self.blocks = model, blocks
        self.pools = [tsb.empty_latent_pool(blocks, dtype, "cuda") for _ in range(LAYERS)]
        self.table = torch.full((batch, MAX_LEN // PAGE), -1, dtype=torch.int32, device="cuda")
        self.counts, self.lens = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(2))
        self.free = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.free_count = torch.tensor([blocks], dtype=torch.int32, device="cuda")
        self.flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.turn = tsb.rotary_table(MAX_LEN, ROPE, device="cuda")

    def extend(self, indptr, total, mask=None):
        return tsb.extend_pages(self.table, self.counts, self.free, self.free_count, self.lens, indptr, total, mask,
                                error_flag=self.flag)

    def release(self, lens):
        tsb.release_pages(self.table, self.counts, self.free, self.free_count, lens, error_flag=self.flag)

    def store(self, layer, latent, k_rope, q, slots, positions):
        return tsb.latent_store(latent, k_rope, self.pools[layer], slots, q[..., NOPE:], self.model.norm[layer],
                                table=self.turn, positions=positions, error_flag=self.flag)

    def prompts(self, chunks, before):
        """Distributions after the tokens of `chunks`, which follow before[b] tokens of sequence b."""
        def offsets(counts):
            return F.pad(torch.tensor(counts, device="cuda").cumsum(0), (1, 0)).to(torch.int32)

        after = [n + len(c) for n, c in zip(before, chunks)]
        indptr, kv_indptr = offsets([len(c) for c in chunks]), offsets(after)
        slots, positions = self.extend(indptr, sum(map(len, chunks)))
        seq = torch.repeat_interleave(torch.arange(len(after), device="cuda"), torch.tensor(after, device="cuda"))
        pos = torch.arange(len(seq), device="cuda") - kv_indptr.long()[seq]
        seen = self.table[seq, pos // PAGE].long() * PAGE + pos % PAGE  # of all tokens, old and new

        def attend(layer, latent, k_rope, q):
            q_rope = self.store(layer, latent, k_rope, q, slots, positions)
            c, r = tsb.latent_load(self.pools[layer], seen, error_flag=self.flag)
            k, v = (torch.einsum(how, c, w[layer]) for how, w in
                    (("nr,hdr->nhd", self.model.key), ("nr,hrd->nhd", self.model.value)))
            return tsb.latent_prompt_attention(torch.cat((q[..., :NOPE], q_rope), 2), k, r, v, indptr, kv_indptr,
                                               error_flag=self.flag)

        probs = self.model.run(torch.tensor([t for c in chunks for t in c], device="cuda"), attend)
        self.lens += torch.tensor([len(c) for c in chunks], dtype=torch.int32, device="cuda")
        return probs

    def nodes(self, tokens, indptr, mask):
        """Distributions after the nodes of drafted trees."""
        slots, positions = self.extend(indptr, len(tokens), mask)

        def attend(layer, latent, k_rope, q):
            q_rope = self.store(layer, latent, k_rope, q, slots, positions)
            q_latent = torch.einsum("nhd,hdr->nhr", q[..., :NOPE], self.model.key[layer])
            x = tsb.latent_attention(q_latent, q_rope, self.pools[layer], self.table, self.lens, indptr, mask,
                                     max_nodes=len(PARENTS), error_flag=self.flag)
            return torch.einsum("nhr,hrd->nhd", x, self.model.value[layer])

        return self.model.run(tokens, attend)

    def commit(self, path, path_lens):
        for pool in self.pools:
            lens = tsb.latent_commit(pool, self.table, self.lens, path, path_lens, error_flag=self.flag)
        self.lens.copy_(lens)
        self.release(self.lens)


class Server:
    """Steps of a batch.  What a step needs lies in tensors of its own, so that a graph can repeat it."""

    def __init__(self, model, cache, batch, steps, seed):
        n, g = len(PARENTS), torch.Generator(device="cuda").manual_seed(seed)
        self.model, self.cache, self.batch = model, cache, batch
        self.parents = torch.tensor(PARENTS * batch, dtype=torch.int32, device="cuda")
        self.indptr = torch.arange(0, batch * n + 1, n, dtype=torch.int32, device="cuda")
        self.mask = tsb.tree_mask(self.parents, self.indptr, n)
        self.last = torch.zeros(batch, dtype=torch.int64, device="cuda")
        # random numbers of all steps: drafts, acceptance, the next token
        self.random = torch.rand((steps, 2 * n + 1, batch), generator=g, device="cuda")
        self.at = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.taken = torch.full((steps, batch, DEPTH), -1, dtype=torch.int64, device="cuda")
        self.taken_probs = torch.zeros((steps, batch, DEPTH), device="cuda")

    def first(self, probs, u):
        """The token after each prompt: a tree that is its root."""
        nodes = torch.arange(self.batch + 1, dtype=torch.int32, device="cuda")
        roots = torch.full((self.batch,), -1, dtype=torch.int32, device="cuda")
        _, _, token = tsb.tree_verify(roots, self.last, nodes, probs, u, u, max_path=1, error_flag=self.cache.flag)
        self.last.copy_(token)

    def step(self):
        n = len(PARENTS)
        u = self.random[self.at][0]
        tokens = [self.last]
        for i in range(1, n):  # a child is drawn from what the drafter gives its parent
            p = self.model.drafter[tokens[PARENTS[i]]]
            tokens.append(torch.searchsorted(p.cumsum(1), u[i][:, None])[:, 0].clamp(max=VOCAB - 1))
        tokens = torch.stack(tokens, 1)
        flat = tokens.view(-1)
        p = self.cache.nodes(flat, self.indptr, self.mask)
        path, path_lens, token = tsb.tree_verify(
            self.parents, flat, self.indptr, p, u[n:2 * n].t().reshape(-1), u[2 * n], draft_probs=self.model.drafter[flat],
            max_path=DEPTH, error_flag=self.cache.flag)
        self.cache.commit(path, path_lens)
        # what was taken: the path's tokens behind the root, then the next one
        after = torch.cat((path[:, 1:], path[:, :1]), 1).long()
        taken = tokens.gather(1, after.clamp(min=0))
        last = path_lens.long()[:, None] - 1
        taken.scatter_(1, last, token[:, None])
        places = torch.arange(DEPTH, device="cuda")
        probs = p.view(self.batch, n, VOCAB)[torch.arange(self.batch, device="cuda")[:, None], path.long().clamp(min=0), taken]
        self.taken.index_copy_(0, self.at, torch.where(places <= last, taken, -1)[None])
        self.taken_probs.index_copy_(0, self.at, probs[None])
        self.last.copy_(token)
        self.at += 1


def generate(model, prompts, dtype, steps, graph, seed=3):
    """(texts, the probability that each new token but the first was taken with, cache, tokens a step)."""
    batch = len(prompts)
    cache = Cache(model, batch, batch * MAX_LEN // PAGE, dtype)
    server = Server(model, cache, batch, steps + 2, seed)
    ends = torch.zeros((batch, VOCAB), device="cuda")
    for at in range(0, max(map(len, prompts)), 100):  # the prompts, 100 tokens at a time
        chunks = [p[at:at + 100] for p in prompts]
        probs = cache.prompts(chunks, [min(at, len(p)) for p in prompts])
        end = 0
        for b, c in enumerate(chunks):
            end += len(c)
            if c and len(prompts[b]) <= at + 100:
                ends[b] = probs[end - 1]
    server.first(ends, server.random[-1, 0])
    first = server.last.tolist()
    server.step()  # (what a graph records has run once: workspaces are there)
    replay = server.step
    if graph:
        recorded = torch.cuda.CUDAGraph()
        with torch.cuda.graph(recorded):
            server.step()
        replay = recorded.replay
    for _ in range(steps - 1):
        replay()
    texts, probs = [p + [f] for p, f in zip(prompts, first)], [[] for _ in prompts]
    for tokens, ps in zip(server.taken[:steps].tolist(), server.taken_probs[:steps].tolist()):
        for b in range(batch):
            texts[b] += [t for t in tokens[b] if t >= 0]
            probs[b] += [p for t, p in zip(tokens[b], ps[b]) if t >= 0]
    assert int(cache.flag) == 0, f"device error flag {int(cache.flag):#x}"
    assert cache.lens.tolist() == [len(t) - 1 for t in texts]
    return texts, probs, cache, sum(map(len, probs)) / (steps * batch)


def plain_probs(model, cache, text):
    """Distributions after the tokens of a text, without a cache."""
    positions = torch.arange(len(text), dtype=torch.int32, device="cuda")
    seen = torch.ones((len(text), len(text)), dtype=torch.bool, device="cuda").tril()

    def attend(layer, latent, k_rope, q):
        c = F.rms_norm(latent.float(), (RANK,), model.norm[layer].float(), 1e-6)
        q_rope = tsb.rotary(q[..., NOPE:], cache.turn, positions).float()
        k_rope = tsb.rotary(k_rope[:, None], cache.turn, positions)[:, 0].float()
        k = torch.einsum("nr,hdr->nhd", c, model.key[layer].float())
        v = torch.einsum("nr,hrd->nhd", c, model.value[layer].float())
        scores = torch.einsum("ihd,jhd->hij", q[..., :NOPE].float(), k) + torch.einsum("ihd,jd->hij", q_rope, k_rope)
        weights = torch.softmax((scores * (NOPE + ROPE)**-0.5).masked_fill(~seen, float("-inf")), -1)
        return torch.einsum("hij,jhd->ihd", weights, v).to(q.dtype)

    return model.run(torch.tensor(text, device="cuda"), attend)


def main(dtype: str = "float16", steps: int = 24, graph: bool = True):
    dtype, rng = getattr(torch, dtype), random.Random(2)
    model = Decoder(dtype)
    prompts = [[rng.randrange(VOCAB) for _ in range(n)] for n in (1, 64, 130, 301)]
    texts, probs, cache, per_step = generate(model, prompts, dtype, steps, graph)
    worst = 0.0
    for text, prompt, p in zip(texts, prompts, probs):
        new = len(prompt) + 1  # the first that a step took
        plain = plain_probs(model, cache, text[:-1])[new - 1:].gather(1, torch.tensor(text[new:], device="cuda")[:, None])
        worst = max(worst, float((plain[:, 0].log() - torch.tensor(p, device="cuda").log()).abs().max()))
    used = cache.blocks - int(cache.free_count)
    cache.release(torch.zeros_like(cache.lens))  # the requests have ended
    print(f"{str(dtype)[6:]}: {per_step:.2f} tokens a step, {used} of {cache.blocks} pages in use at the end; the plain "
          f"run's log-probabilities of the tokens taken are within {worst:.4f}")
    return texts, per_step, worst, used, cache


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--dtype", default="float16", choices=("float16", "bfloat16"))
    parser.add_argument("--steps", type=int, default=24)
    parser.add_argument("--no-graph", action="store_true")
    args = parser.parse_args()
    main(args.dtype, args.steps, not args.no_graph)
