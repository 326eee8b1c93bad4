"""Absorbed attention over batches whose sequences are not alike."""

import pytest

from tests.step_ref import LatentCase
from tests.test_latent_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [8, 16, 64])
def test_one_large_tree_among_single_tokens(heads):
    # few rows on the average (64 / heads nodes a sequence at most): the tree's many blocks are of the kernel for up to 64 rows
    tree = max(640 // heads, 40)
    assert 50 + tree <= 101 * (64 // heads)
    check(LatentCase([100, 0] * 50 + [700], [1, 0] * 50 + [tree], heads, seed=heads, dead=0.1))
