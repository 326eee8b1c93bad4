"""Caches and rows whose offsets pass 32 bits: the same call over tensors that hold only
what it reads has to give the same.

Where the line of work is cut differently (another number of tokens before), partial sums
meet in another order: then weights and outputs are rounded to 16 bits on either side, so
a result may differ by 2 roundings of a weight and 2 of the output, 4 half steps of the
largest value.
"""

import pytest
import torch

import torch_spyre_b200 as tsb

pytestmark = pytest.mark.gpu


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


@pytest.mark.parametrize("heads", [16, 128])
def test_a_pool_of_more_than_two_to_the_31_elements(heads):
    blocks, ctx, nodes = 60000, [200, 70], [3, 2]
    assert blocks * 9 * 64 * 64 > 2**31
    g = torch.Generator(device="cuda").manual_seed(heads)
    near, far = tsb.empty_latent_pool(7, device="cuda"), tsb.empty_latent_pool(blocks, device="cuda")
    small = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 0]], dtype=torch.int32, device="cuda")
    large = torch.where(small % 2 == 0, blocks - 1 - small, blocks // 2 + small).to(torch.int32)
    lens, indptr = ints(*ctx), ints(0, 3, 5)
    mask = tsb.tree_mask(ints(-1, 0, 0, -1, 0), indptr, 3)
    q = torch.randn((5, heads, 576), generator=g, device="cuda").bfloat16()
    outs = []
    rows = torch.randn((sum(ctx) + 5, 576), generator=g, device="cuda").bfloat16()
    for pool, table in ((near, small), (far, large)):
        seq = torch.repeat_interleave(torch.arange(2, device="cuda"), ints(*(c + n for c, n in zip(ctx, nodes))).long())
        pos = torch.cat([torch.arange(c + n, device="cuda") for c, n in zip(ctx, nodes)])
        slots = table[seq, pos // 64].long() * 64 + pos % 64
        tsb.latent_store(rows[:, :512], rows[:, 512:], pool, slots)
        assert all(torch.equal(x, y) for x, y in zip(tsb.latent_load(pool, slots), rows.split((512, 64), 1)))
        out = tsb.latent_attention(q[..., :512], q[..., 512:], pool, table, lens, indptr, mask)
        new = tsb.latent_commit(pool, table, lens, ints(0, 2, 0, 1).view(2, 2), ints(2, 2))
        outs.append((out, new, *tsb.latent_load(pool, slots)))
    assert all(torch.equal(x, y) for x, y in zip(*outs))


def test_expanded_keys_of_more_than_two_to_the_31_elements():
    heads, total, last = 128, 140000, 300
    assert total * heads * 128 > 2**31
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.empty((total, heads, 128), dtype=torch.float16, device="cuda").normal_(generator=g) for _ in range(2))
    r = torch.randn((total, 64), generator=g, device="cuda").half()
    q = torch.randn((41, heads, 192), generator=g, device="cuda").half()
    out = tsb.latent_prompt_attention(q, k, r, v, ints(0, 1, 41), ints(0, total - last, total))
    want = tsb.latent_prompt_attention(q[1:], k[-last:], r[-last:], v[-last:], ints(0, 40), ints(0, last))
    largest = float(v[-last:].abs().max())
    assert float((out[1:].float() - want.float()).abs().max()) <= 4 * 2.0**-11 * largest


def test_rows_of_probabilities_past_two_to_the_31_elements():
    nodes, vocab = 17000, 131072
    assert nodes * vocab > 2**31
    g = torch.Generator(device="cuda").manual_seed(2)
    batch = 17
    probs = torch.zeros((nodes, vocab), dtype=torch.float16, device="cuda")
    indptr = torch.arange(0, nodes + 1, nodes // batch, dtype=torch.int32, device="cuda")
    parents = (torch.arange(nodes, device="cuda", dtype=torch.int32) % (nodes // batch)) - 1  # chains of 1000
    tokens = torch.randint(0, vocab, (nodes,), generator=g, device="cuda")
    after = torch.roll(tokens, -1)
    probs[torch.arange(nodes, device="cuda"), after] = 0.75  # every drafted token likely, and the one after the last
    u = torch.rand(nodes, generator=g, device="cuda")
    u[::4] *= 0.1
    s = torch.rand(batch, generator=g, device="cuda")
    path, path_lens, nxt = tsb.tree_verify(parents, tokens, indptr, probs, u, s, max_path=nodes // batch)
    rejected = (u >= 0.75).view(batch, -1)
    rejected[:, 0] = False
    for b in range(batch):
        hits = rejected[b].nonzero()
        n = int(hits[0]) if len(hits) else nodes // batch
        assert int(path_lens[b]) == n
        # (after a rejection nothing is left but what the row gave the rejected token: the row again)
        assert int(nxt[b]) == int(after[int(indptr[b]) + n - 1])
