"""Prompt attention of many prompts: every row meets its own sequence's tokens only, so how much there is to
do does not follow from the numbers of rows and tokens of the batch."""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_latent_prompt_gpu import Case
from tests.verify_ref import attention_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
def test_a_batch_of_many_prompts(causal):
    # rows / 256 * tokens / 80 * 4 of the whole batch are more than 2^31; its blocks have some 10^7 steps
    g = torch.Generator().manual_seed(3)
    new = torch.randint(3000, 3700, (1024,), generator=g).tolist()
    past = torch.randint(0, 70, (1024,), generator=g).tolist()
    new[0], new[1023], new[500] = 1, 129, 0
    lens = [n + p for n, p in zip(new, past)]
    assert sum(new) // 256 * (sum(lens) // 80) * 4 > 2**31
    case = Case(new, lens, 1, torch.bfloat16, causal, seed=31)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.latent_prompt_attention(*case.args(), causal=causal, return_lse=True, error_flag=flag)
    assert int(flag) == 0
    for b in (0, 1, 2, 499, 501, 700, 1022, 1023):  # one sequence at a time against 64 bits
        a, c = int(case.q_indptr[b]), int(case.kv_indptr[b])
        one = Case([new[b]], [lens[b]], 1, torch.bfloat16, causal)
        one.q = case.q[a:a + new[b]]
        one.k_nope, one.v, one.k_rope = (x[c:c + lens[b]] for x in (case.k_nope, case.v, case.k_rope))
        ref, ref_lse, spread = one.reference()
        bound = attention_bound(ref, spread, lens[b], out.dtype)
        assert bool(((out[a:a + new[b]].double() - ref).abs() <= bound).all())
        assert bool(((lse[a:a + new[b]].double() - ref_lse).abs() <= 2e-4 * (1 + ref_lse.abs())).all())
