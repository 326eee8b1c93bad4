"""The width of verification's paths: a sequence has 1024 nodes at most, so no path is longer."""

import pytest
import torch

import torch_spyre_b200 as tsb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,nodes", [(3, 5), (100, 11), (2, 1024), (300, 64)])
def test_the_default_width_does_not_grow_past_the_longest_path(batch, nodes):
    n, vocab = batch * nodes, 16
    parents = (torch.arange(n, device="cuda", dtype=torch.int32) % nodes) - 1
    tokens = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    probs = torch.zeros((n, vocab), device="cuda")
    probs[torch.arange(n, device="cuda"), torch.roll(tokens, -1)] = 1.0  # every drafted token is certain
    indptr = torch.arange(0, n + 1, nodes, dtype=torch.int32, device="cuda")
    u, s = torch.full((n,), 0.5, device="cuda"), torch.full((batch,), 0.5, device="cuda")
    path, path_lens, _ = tsb.tree_verify(parents, tokens, indptr, probs, u, s)
    assert path.shape == (batch, min(n, 1024))
    assert path_lens.tolist() == [nodes] * batch
    assert torch.equal(path[:, :nodes], torch.arange(nodes, dtype=torch.int32, device="cuda").expand(batch, -1))
    assert bool((path[:, nodes:] == -1).all())
