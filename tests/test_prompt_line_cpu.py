"""Which numbers of rows, tokens and heads prompt attention takes (no GPU: a call that passes those checks is
refused for its workspace)."""

import pytest

from tests.test_latent_step_cpu import prompt
from torch_spyre_b200 import _lib


@pytest.mark.parametrize("batch,tokens,heads", [(96, 4096, 128), (1024, 400, 128), (4, 131072, 64), (1024, 3300, 1),
                                                (200, 10000, 16)])
def test_batches_that_fit_are_taken(batch, tokens, heads):
    n = batch * tokens
    assert prompt(B=batch, N=n, M=n, H=heads) == 3 and "workspace" in _lib.last_error()


@pytest.mark.parametrize("over", [dict(N=1 << 22, M=1 << 26, H=256), dict(N=(1 << 31) - 1, M=(1 << 30) - 1, H=1),
                                  dict(N=1 << 15, M=(1 << 30) - 1, H=65535)])
def test_more_steps_than_can_be_counted_are_refused(over):
    assert prompt(**over) == 2 and "2^31" in _lib.last_error()
