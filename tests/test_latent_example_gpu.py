"""The example that runs a step's plan, latent attention and verification together.

Tolerance of the log-probabilities.  Logits have unit variance by construction.  A
hidden state takes about ten roundings on its way (of elements a few units in
size, u = 2^-11 for fp16, 2^-8 for bf16), the cached rows and the absorbed products
a few more; each reaches a logit as a sum of 512 random signs over sqrt(512), so
a logit is off by some 20 u of its own size, with four times that for the largest of
some hundred: 80 u, and a log-probability by twice that at most.
"""

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.parametrize("dtype,u", [("float16", 2.0**-11), ("bfloat16", 2.0**-8)])
def test_steps_take_tokens_with_the_plain_runs_probabilities(dtype, u):
    import serve_latent

    texts, per_step, worst, used, cache = serve_latent.main(dtype, steps=16, graph=True)
    assert 1 <= per_step <= serve_latent.DEPTH
    assert worst <= 160 * u
    # in use at the end: the pages of what is cached; then all are back, each once
    assert used == sum((len(t) - 1 + 63) // 64 for t in texts)
    assert int(cache.free_count) == cache.blocks
    assert sorted(cache.free.tolist()) == list(range(cache.blocks))
    assert (cache.table == -1).all() and (cache.counts == 0).all()


def test_a_recorded_step_takes_the_same_tokens():
    import serve_latent

    graph = serve_latent.main("float16", steps=10, graph=True)
    plain = serve_latent.main("float16", steps=10, graph=False)
    assert graph[0] == plain[0]
