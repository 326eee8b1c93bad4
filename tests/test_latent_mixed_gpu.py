"""Absorbed attention over batches whose sequences are not alike."""

import pytest

from tests.step_ref import LatentCase
from tests.test_latent_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [8, 16, 64])
def test_one_large_tree_among_single_tokens(heads):
    # few rows on the average: the tree's many blocks are of the kernel for up to 64 rows
    check(LatentCase([100, 0] * 50 + [700], [1] * 100 + [max(40 * 16 // heads, 12)], heads, seed=heads, dead=0.1))
