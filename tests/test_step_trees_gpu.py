"""Positions of drafted trees whose tokens are more than the threads of a CTA, and more than one CTA places."""

import random

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_step_gpu import State, indptr, int32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("words", [1, 2])
@pytest.mark.parametrize("nodes,batch", [(60, 3), (64, 25), (62, 100)])
def test_positions_of_many_trees_are_depths(words, nodes, batch):
    """Masked tokens past the first of a thread, and those of a launch of their own (over 4096)."""
    rng = random.Random(nodes + words)
    parents, depths, new, ctx = [], [], [], []
    for b in range(batch):
        n = rng.choice([nodes, rng.randint(nodes - 9, nodes)])
        kept = []  # nodes that may have children
        tree = []
        for i in range(n):
            u = rng.random()
            if i > 0 and u < 0.1:
                tree.append((-2, 0))  # pruned: it sees nothing, its position is the root's
                continue
            p = rng.choice(kept) if kept and u < 0.95 else -1
            tree.append((p, tree[p][1] + 1 if p >= 0 else 0))
            kept.append(i)
        parents += [p for p, _ in tree]
        depths += [d for _, d in tree]
        new.append(n)
        ctx.append(rng.choice([0, 63, 64, 500, rng.randint(0, 900)]))
    ptr = indptr(new)
    mask = tsb.tree_mask(int32(parents), ptr, 64 * words)
    assert mask.shape == (sum(new), words)
    s = State(ctx, 20, 2 * batch)
    slots, positions = tsb.extend_pages(*s.args(), int32(ctx), ptr, sum(new), mask, error_flag=s.flag)
    want, want_at, short = s.host.extend(ctx, new, depths)
    assert not short
    assert torch.equal(slots.cpu(), torch.tensor(want)) and torch.equal(positions.cpu().long(), torch.tensor(want_at))
    s.check()
    assert int(s.flag) == 0
