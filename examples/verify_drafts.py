"""Speculative decoding with drafted token trees over a paged 8-bit cache.

    python examples/verify_drafts.py [--cache int8|float8_e4m3fn|float16] [--new-tokens 48]

A small random decoder writes its prompts in chunks (a chunk is a chain: no
mask), then verifies one drafted tree per sequence and step:

    table = rotary_table(...)                                  once
    mask = tree_mask(parents, q_indptr, ...)                   once a step
    per layer:
      q = kv_store(k, v, pools, slots, q=q, table, positions)  rows turned, quantised, written
      x = tree_attention(q, pools, ..., mask)                  nodes over the cache and the tree
    lens = tree_commit(pools, ..., path, path_lens)            per layer, the accepted path

The drafter here is a stand-in that knows some of the right tokens.  In the end
the whole text is run once more without a cache (rotary and a plain attention in
fp32 over the rows that kv_load reads back), and every token taken must be the
most likely one up to rounding.
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

LAYERS, HQ, HKV, DIM, HIDDEN, VOCAB, MAX_LEN, PAGE = 2, 8, 2, 128, 512, 600, 512, 64


class Decoder:
    """Random weights; one attention and one linear layer per block."""

    def __init__(self, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn((rows, cols), generator=g, device="cuda") * rows**-0.5).half()

        self.embed = torch.randn((VOCAB, HIDDEN), generator=g, device="cuda").half()
        self.qkv = [weight(HIDDEN, (HQ + 2 * HKV) * DIM) for _ in range(LAYERS)]
        self.out = [weight(HQ * DIM, HIDDEN) for _ in range(LAYERS)]
        self.mlp = [weight(HIDDEN, HIDDEN) for _ in range(LAYERS)]
        self.head = weight(HIDDEN, VOCAB)

    def run(self, tokens, attend):
        """Logits of tokens [N]; attend(layer, q, k, v) is the attention of the rows [N, heads, DIM]."""
        h = self.embed[tokens]
        for layer in range(LAYERS):
            qkv = (F.rms_norm(h, (HIDDEN,)) @ self.qkv[layer]).view(len(tokens), HQ + 2 * HKV, DIM)
            q, k, v = qkv.split((HQ, HKV, HKV), 1)
            h = h + attend(layer, q, k, v).view(len(tokens), HQ * DIM) @ self.out[layer]
            h = h + F.silu(F.rms_norm(h, (HIDDEN,)) @ self.mlp[layer])
        return (F.rms_norm(h, (HIDDEN,)) @ self.head).float()


class Cache:
    """Paged K/V of every layer, one block table for all of them."""

    def __init__(self, batch: int, dtype: torch.dtype):
        blocks = batch * MAX_LEN // PAGE
        self.layers = [[tsb.empty_row_pool(blocks, HKV, DIM, dtype, device="cuda") for _ in range(2)]
                       for _ in range(LAYERS)]
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(1))
        self.table = order.view(batch, -1).to(torch.int32).cuda()
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def slots(self, seq, pos):
        return self.table[seq, pos // PAGE].long() * PAGE + pos % PAGE

    def attend(self, counts, depths, turn, mask=None):
        """The attention of rows appended to the sequences (counts[b] rows of sequence b, row i
        at position lens[b] + depths[i]), for Decoder.run."""
        counts = torch.tensor(counts, device="cuda")
        indptr = F.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
        total = len(depths)
        seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=total)
        start = self.lens.long()[seq]
        slots = self.slots(seq, start + torch.arange(total, device="cuda") - indptr.long()[seq])
        positions = (start + torch.tensor(depths, device="cuda")).to(torch.int32)

        def layer_attention(layer, q, k, v):
            (kp, ks), (vp, vs) = self.layers[layer]
            q = tsb.kv_store(k, v, kp, vp, slots, ks, vs, q=q, table=turn, positions=positions, error_flag=self.flag)
            return tsb.tree_attention(q, kp, vp, self.table, self.lens, indptr, mask, k_scales=ks, v_scales=vs,
                                      error_flag=self.flag)

        return layer_attention

    def commit(self, path, path_lens):
        for (kp, ks), (vp, vs) in self.layers:
            lens = tsb.tree_commit(kp, vp, self.table, self.lens, path, path_lens, ks, vs, error_flag=self.flag)
        self.lens = lens


def draft(rng, right):
    """(tokens, parents) of a tree under node 0: the right tokens as far as they go, each level with a
    sibling or two, and sometimes a wrong turn."""
    tokens, parents, at = [0], [-1], 0
    for token in right:
        level = [token if rng.random() < 0.8 else rng.randrange(VOCAB)] + \
                [rng.randrange(VOCAB) for _ in range(rng.randrange(3))]
        place = rng.randrange(len(level))  # the likely one is not always the first
        level[0], level[place] = level[place], level[0]
        tokens += level
        parents += [at] * len(level)
        at = len(tokens) - len(level) + place
    return tokens, parents


def generate(model, prompts, turn, new_tokens, dtype, hints=None, seed=0):
    """Texts (prompt and new tokens) and the tokens taken per step; without hints one token a step."""
    rng, cache = random.Random(seed), Cache(len(prompts), dtype)
    texts, steps = [list(p) for p in prompts], 0
    for at in range(0, max(map(len, prompts)), 100):  # the prompts, 100 tokens at a time
        chunks = [p[at:at + 100] for p in prompts]
        counts = [len(c) for c in chunks]
        depths = [i for n in counts for i in range(n)]
        tokens = torch.tensor([t for c in chunks for t in c], device="cuda")
        logits = model.run(tokens, cache.attend(counts, depths, turn))
        cache.lens = cache.lens + torch.tensor(counts, dtype=torch.int32, device="cuda")
        end = 0
        for b, n in enumerate(counts):
            end += n
            if n and len(prompts[b]) <= at + 100:
                texts[b].append(int(logits[end - 1].argmax()))
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < new_tokens:
        # a text's last token is not in the cache yet: it is the tree's root
        trees = [draft(rng, hints[b][len(t):len(t) + 4] if hints else []) for b, t in enumerate(texts)]
        counts = [len(p) for _, p in trees]
        depths = []
        for (tokens, parents), text in zip(trees, texts):
            tokens[0] = text[-1]
            first = len(depths)
            for p in parents:
                depths.append(0 if p < 0 else depths[first + p] + 1)
        parents = torch.tensor([p for _, ps in trees for p in ps], dtype=torch.int32, device="cuda")
        indptr = F.pad(torch.tensor(counts, device="cuda").cumsum(0), (1, 0)).to(torch.int32)
        mask = tsb.tree_mask(parents, indptr, max(counts), error_flag=cache.flag)
        tokens = torch.tensor([t for ts, _ in trees for t in ts], device="cuda")
        best = model.run(tokens, cache.attend(counts, depths, turn, mask)).argmax(1).tolist()
        paths, first = [], 0
        for (tokens, parents), text in zip(trees, texts):
            path, node = [0], 0
            while True:  # down the tree as long as a child is what the model says
                text.append(best[first + node])
                node = next((i for i, p in enumerate(parents) if p == node and tokens[i] == text[-1]), None)
                if node is None:
                    break
                path.append(node)
            paths.append(path)
            first += len(parents)
        width = max(map(len, paths))
        path = torch.tensor([p + [0] * (width - len(p)) for p in paths], dtype=torch.int32, device="cuda")
        cache.commit(path, torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda"))
        steps += 1
    assert int(cache.flag) == 0, f"device error flag {int(cache.flag):#x}"
    made = sum(len(t) - len(p) - 1 for t, p in zip(texts, prompts))
    return texts, made / (steps * len(prompts)), cache


def shortfall(model, text, prompt_len, turn, cache, b):
    """How far (in logits) the tokens of a text are from the most likely ones, by a plain run of it; and the
    largest difference between its K rows and the cache's, over a row's largest element."""
    n = len(text) - 1  # the last token has no successor
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    seen = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
    slots = cache.slots(torch.full_like(positions, b).long(), positions.long())
    worst_row = 0.0

    def attend(layer, q, k, v):
        nonlocal worst_row
        (kp, ks), (vp, vs) = cache.layers[layer]
        q, k = (tsb.rotary(x, turn, positions).float() for x in (q, k))
        kc, vc = tsb.kv_load(kp, slots, ks, torch.float32), tsb.kv_load(vp, slots, vs, torch.float32)
        worst_row = max(worst_row, float(((k - kc).abs().amax(-1) / k.abs().amax(-1)).max()))
        kc, vc = (x.repeat_interleave(HQ // HKV, 1) for x in (kc, vc))
        scores = torch.einsum("ihd,jhd->hij", q, kc) * DIM**-0.5
        weights = torch.softmax(scores.masked_fill(~seen, float("-inf")), -1)
        return torch.einsum("hij,jhd->ihd", weights, vc).to(v.dtype).contiguous()

    logits = model.run(torch.tensor(text[:-1], device="cuda"), attend)[prompt_len - 1:]
    taken = torch.tensor(text[prompt_len:], device="cuda")
    return float((logits.amax(1) - logits.gather(1, taken[:, None])[:, 0]).max()), worst_row


def main(cache: str = "int8", new_tokens: int = 48):
    dtype = getattr(torch, cache)
    model, rng = Decoder(), random.Random(2)
    prompts = [[rng.randrange(VOCAB) for _ in range(n)] for n in (1, 64, 130, 301)]
    turn = tsb.rotary_table(MAX_LEN, DIM, device="cuda")
    plain, _, _ = generate(model, prompts, turn, new_tokens, dtype)  # one token a step, to have hints
    texts, taken, pages = generate(model, prompts, turn, new_tokens, dtype, hints=plain)
    short, row = zip(*(shortfall(model, t, len(p), turn, pages, b) for b, (t, p) in enumerate(zip(texts, prompts))))
    print(f"{cache} cache: {taken:.2f} tokens a step; the plain run's best logit is at most {max(short):.4f} above a "
          f"taken token's, its K rows within {max(row):.4f} of the cache's")
    return taken, max(short), max(row)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--cache", default="int8", choices=("int8", "float8_e4m3fn", "float16"))
    parser.add_argument("--new-tokens", type=int, default=48)
    args = parser.parse_args()
    main(args.cache, args.new_tokens)
