"""Outputs of disjoint sets of tokens joined by their log-sum-exps, in the type that they come in."""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_latent_prompt_gpu import Case

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,result", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("parts", [1, 2, 5])
def test_against_the_formula(dtype, result, parts):
    g = torch.Generator(device="cuda").manual_seed(parts)
    o = [torch.randn((7, 3, 100), generator=g, device="cuda").to(dtype) for _ in range(parts)]
    lses = [torch.randn((7, 3), generator=g, device="cuda") * 3 for _ in range(parts)]
    lses[0][2] = -float("inf")
    for x in lses:
        x[4, 1] = -float("inf")  # nothing anywhere
    out, lse = tsb.merge_attention_states(o, lses)
    assert out.dtype == result and out.shape == (7, 3, 100) and lse.dtype == F32
    w = torch.stack(lses).double()
    want_lse = torch.logsumexp(w, 0)
    w = torch.where(torch.isfinite(want_lse), torch.exp(w - want_lse), 0.0)
    want = (w[..., None] * torch.stack(o).double()).sum(0)
    spread = (w[..., None] * torch.stack(o).double().abs()).sum(0)
    # the result's rounding, and fp32 weights and sums of a few terms (2^-20)
    bound = torch.finfo(result).eps / 2 * want.abs() + 2.0**-20 * spread + 2.0**-25
    assert bool(((out.double() - want).abs() <= bound).all())
    assert not out[4, 1].any() and float(lse[4, 1]) == -float("inf")
    live = torch.isfinite(want_lse)
    assert bool(((lse - want_lse).abs()[live] <= 2.0**-20 * (1 + want_lse.abs()[live])).all())


def test_large_bf16_values_stay_finite():
    # past the largest number of fp16
    o = [torch.full((2, 8), v, dtype=BF16, device="cuda") for v in (1e6, 3e6)]
    out, _ = tsb.merge_attention_states(o, [torch.zeros(2, device="cuda")] * 2)
    assert out.dtype == BF16 and bool((out.float() - 2e6).abs().max() <= 2e6 * 2.0**-8)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_chunk_and_past_are_joined(dtype):
    """A chunk's own tokens (causal) and its past (not causal), merged, are the whole."""
    case = Case([150], [700], 4, dtype, seed=22)
    whole, whole_lse = tsb.latent_prompt_attention(*case.args(), return_lse=True)
    outs, lses = [], []
    for part, causal in ((slice(0, 550), False), (slice(550, 700), True)):
        m = torch.tensor([0, part.stop - part.start], dtype=torch.int32, device="cuda")
        o, x = tsb.latent_prompt_attention(case.q, case.k_nope[part], case.k_rope[part], case.v[part], case.q_indptr, m,
                                           causal=causal, return_lse=True)
        outs.append(o)
        lses.append(x)
    merged, lse = tsb.merge_attention_states(outs, lses)
    assert merged.dtype == dtype
    # two roundings of the parts and one of the result, on both sides
    size = float(case.v.float().abs().max())
    assert float((merged.float() - whole.float()).abs().max()) <= 4 * torch.finfo(dtype).eps / 2 * size
    assert float((lse - whole_lse).abs().max()) <= 1e-3


def test_types_are_checked():
    lse = torch.zeros(2, device="cuda")
    for o in (torch.zeros((2, 8), device="cuda", dtype=torch.float64), torch.zeros((2, 8), device="cuda", dtype=torch.int32)):
        with pytest.raises(ValueError, match="fp16, bf16 or fp32"):
            tsb.merge_attention_states([o], [lse])
