"""A step's plan with lengths that cannot be: such a sequence adds no tokens, so it takes no page and gets no slot."""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_step_gpu import State, indptr, int32
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu

WIDTH = 100  # pages of a row of the table


@pytest.mark.parametrize("wrong", [-1, -(2**31), WIDTH * 64 + 1, 2**31 - 1])
# tokens placed by the CTA that moves the pages, one or several to a thread, and by a launch of their own
@pytest.mark.parametrize("tokens", [2, 700, 2500])
def test_a_wrong_length_takes_no_page_and_no_slot(wrong, tokens):
    ctx, new = [130, 70, 64, 10], [tokens, 3, tokens, 1]
    s = State(ctx, WIDTH, 90)
    slots, positions = tsb.extend_pages(*s.args(), int32([130, wrong, 64, 10]), indptr(new), sum(new), error_flag=s.flag)
    # the others get what they would get without it
    want, want_at, short = s.host.extend(ctx, [new[0], 0, new[2], new[3]])
    assert not short
    at = new[0]
    want[at:at] = [-1] * new[1]
    assert torch.equal(slots.cpu(), torch.tensor(want))
    got_at = positions.tolist()
    assert torch.equal(torch.tensor(got_at[:at] + got_at[at + new[1]:]), torch.tensor(want_at))
    s.check()
    assert int(s.flag) == _lib.DEVERR_BAD_LEN


def test_a_wrong_length_does_not_empty_the_stack():
    # enough pages for those that are right, far fewer than the table has room for
    ctx, new = [64, 64, 64], [1, 1, 1]
    s = State(ctx, WIDTH, 2)
    slots, _ = tsb.extend_pages(*s.args(), int32([10**6, 64, 64]), indptr(new), 3, error_flag=s.flag)
    want, _, short = s.host.extend(ctx, [0, 1, 1])
    assert not short and slots.tolist() == [-1] + want
    s.check()
    assert int(s.flag) == _lib.DEVERR_BAD_LEN


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


def test_offsets_that_descend_take_no_pages():
    # the second sequence has a length that its table row could hold and pages that do not reach it
    s = State([64, 64], 8, 6)
    tsb.extend_pages(*s.args(), int32([64, 300]), int32([0, 2, 1]), 2, error_flag=s.flag)
    s.host.extend([64], [2])
    s.check()
    assert int(s.flag) == _lib.DEVERR_BAD_LEN
