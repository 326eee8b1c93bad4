"""A step's plan with lengths that cannot be: such a sequence adds no tokens, so it gets no slot."""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_step_gpu import State, int32

pytestmark = pytest.mark.gpu


def test_committed_rows_of_a_wrong_length_are_left_as_they_are():
    s = State([64, 64], 4, 4)
    pool = tsb.empty_latent_pool(6, device="cuda")
    tsb.latent_store(torch.ones((384, 512), device="cuda").bfloat16(), torch.ones((384, 64), device="cuda").bfloat16(), pool,
                     torch.arange(384, device="cuda"))
    before = pool.clone()
    slots, _ = tsb.extend_pages(*s.args(), int32([-7, 64]), int32([0, 5, 6]), 6, error_flag=s.flag)
    rows = torch.zeros((6, 576), device="cuda").bfloat16()
    tsb.latent_store(rows[:, :512], rows[:, 512:], pool, slots)
    changed = (pool != before).permute(0, 3, 1, 2, 4).flatten(2).any(2).view(-1).nonzero()[:, 0].tolist()
    assert changed == [int(slots[5])] and slots[:5].tolist() == [-1] * 5
