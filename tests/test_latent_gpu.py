"""Latent attention, absorbed form, against a 64-bit reference.

The bound (verify_ref.attention_bound): a result's own rounding, the weights' rounding to the pool's type and
fp32 sums and exponentials.  Scores are fp32 sums of 576 exact products: off by at most a few 2^-24 of
sum |q||c| * scale, some 3e-5 here; log-sum-exps are allowed 2e-4 of their size, as those of tree attention.
"""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.step_ref import LatentCase
from tests.verify_ref import attention_bound, pack_bits
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def check(case, **kw):
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.latent_attention(*case.args(), **case.kwargs(), return_lse=True, error_flag=flag, **kw)
    assert int(flag.item()) == 0
    ref, ref_lse, spread = case.reference(kw.get("scale"))
    n_keys = max(c + t for c, t in zip(case.ctx, case.nodes))
    bound = attention_bound(ref, spread, n_keys, out.dtype)
    err = (out.double() - ref).abs()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert bool(((err <= bound) | torch.isnan(ref) | (out.double() == ref)).all()), \
        f"off by {float((err / bound).nan_to_num().max()):.3g} of the bound"
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((out[empty] == 0).all())
    assert bool(((lse.double() - ref_lse).abs() <= 2e-4 * (1 + ref_lse.abs()))[~empty].all())
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [16, 128, 1])
def test_one_token(dtype, heads):
    check(LatentCase([5], [1], heads, dtype, chain=True, seed=1))
    check(LatentCase([0, 1, 63, 64, 65, 127, 128, 1000], [1] * 8, heads, dtype, chain=True, seed=heads))


@pytest.mark.parametrize("heads", [1, 2, 3, 5, 8, 16, 20, 31, 32, 33, 48, 63, 64, 65, 80, 128, 130, 192, 512])
def test_heads(heads):
    check(LatentCase([200, 0, 77], [9, 3, 1], heads, seed=heads))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [4, 16, 40, 128])
def test_trees_ragged(dtype, heads):
    check(LatentCase([0, 1, 63, 64, 65, 127, 128, 129, 500, 1000], [1, 7, 2, 64, 65, 33, 1, 100, 17, 5], heads, dtype,
                     dead=0.1, seed=heads))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [8, 64, 128])
def test_chains(dtype, heads):
    check(LatentCase([0, 5, 300, 64], [130, 1, 70, 64], heads, dtype, chain=True, seed=3))


@pytest.mark.parametrize("heads", [1, 16, 64, 128])
def test_long_context_is_split(heads):
    check(LatentCase([70001], [1], heads, F16, chain=True, seed=5))
    check(LatentCase([33000, 7], [6, 3], heads, BF16, seed=6))


def test_many_sequences():
    g = torch.Generator().manual_seed(2)
    ctx = torch.randint(0, 400, (300,), generator=g).tolist()
    nodes = torch.randint(0, 6, (300,), generator=g).tolist()  # sequences without a draft among them
    check(LatentCase(ctx, nodes, 16, seed=7))
    check(LatentCase([3] * 1024, [1] * 1024, 2, seed=8))


def test_rows_without_anything_to_see():
    case = LatentCase([0, 0, 130], [4, 70, 9], 16, seed=12)
    for s in case.see:
        s[::2] = False
    case.mask = torch.cat([pack_bits(s, 2) for s in case.see]).cuda()
    check(case)


def test_mask_is_taken_as_it_is():
    # any bits: nodes that see later ones, or not themselves; bits past the draft are ignored
    case = LatentCase([10, 0], [70, 20], 8, seed=13)
    g = torch.Generator().manual_seed(0)
    case.see = [torch.rand(s.shape, generator=g) < 0.3 for s in case.see]
    mask = torch.cat([pack_bits(s, 2) for s in case.see])
    mask[70:, 0] |= -(1 << 20)
    mask[:, 1] |= -(1 << 6)
    case.mask = mask.cuda()
    check(case)


def test_large_scores_and_rising_maxima():
    check(LatentCase([900, 64], [33, 3], 16, qscale=12.0, seed=14))
    for heads in (16, 128):
        case = LatentCase([1500], [3], heads, seed=15, poison=False)
        # keys that grow along the context: every page raises some row's maximum
        ramp = torch.linspace(0.05, 3.0, 1503, device="cuda")
        sl = case.slots(0, 0, 1503)
        q = torch.cat([case.q_latent[0, 0], case.q_rope[0, 0]]).view(1, 9, 64).float()
        case.pool[sl // 64, 0, :, sl % 64] = (q * ramp[:, None, None]).to(BF16)
        check(case)


@pytest.mark.parametrize("scale", [0.3, -0.05, 0.0])
def test_scales(scale):
    check(LatentCase([100, 30], [12, 40], 16, F16, seed=16), scale=scale)


def test_strides():
    case = LatentCase([100, 30], [12, 40], 16, seed=16)
    fused = torch.randn(52, 20, 640, device="cuda", dtype=BF16)
    fused[:, 2:18, 64:576] = case.q_latent
    fused[:, 2:18, 576:] = case.q_rope
    case.q_latent, case.q_rope = fused[:, 2:18, 64:576], fused[:, 2:18, 576:]
    first = check(case)
    across = torch.empty(16, 52, 512, device="cuda", dtype=BF16)  # head-major, as a batched product leaves it
    across.copy_(case.q_latent.transpose(0, 1))
    case.q_latent = across.transpose(0, 1)
    assert torch.equal(check(case), first)
    table = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    table[:, :case.block_table.shape[1]] = case.block_table
    case.block_table = table[:, :case.block_table.shape[1]]
    assert torch.equal(check(case), first)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads", [8, 128])
def test_non_finite_rows_of_unseen_nodes(value, heads):
    """A node's NaN or inf reaches the rows that see it and no other."""
    case = LatentCase([70, 0, 128], [12, 5, 1], heads, seed=17)
    sl = case.slots(0, 70 + 3, 70 + 4)[0]
    case.pool[sl // 64, 0, 2, sl % 64, 5] = value
    out = tsb.latent_attention(*case.args(), **case.kwargs())
    ref, _, spread = case.reference()
    sees = case.see[0][:, 3]
    assert bool(sees.any()) and not bool(sees.all())
    keep = torch.cat([~sees, torch.ones(6, dtype=torch.bool)]).cuda()
    assert bool(torch.isfinite(out[keep]).all())
    bound = attention_bound(ref, spread, 200, BF16)
    assert bool(((out.double() - ref).abs() <= bound)[keep].all())
    # whoever sees it has the score's NaN or inf - inf in it
    if math.isnan(value):
        assert bool(torch.isnan(out[:12][sees.cuda()]).all())


def test_inputs_outside_their_range_are_flagged():
    case = LatentCase([100, 30], [12, 40], 8, seed=19)

    def flag_of(**over):
        names = ["q_latent", "q_rope", "pool", "block_table", "context_lens", "q_indptr"]
        args = dict(zip(names, case.args()), **case.kwargs())
        args.update(over)
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = tsb.latent_attention(**args, error_flag=flag)
        return int(flag.item()), out

    assert flag_of()[0] == 0
    table = case.block_table.clone()
    table[0, 1] = case.pool.shape[0]
    assert flag_of(block_table=table)[0] & _lib.DEVERR_BAD_BLOCK
    table[0, 1] = -1
    assert flag_of(block_table=table)[0] & _lib.DEVERR_BAD_BLOCK
    int32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    assert flag_of(context_lens=int32(100, 128))[0] & _lib.DEVERR_BAD_LEN
    assert flag_of(context_lens=int32(-1, 30))[0] & _lib.DEVERR_BAD_LEN
    got, out = flag_of(max_nodes=39)
    assert got & _lib.DEVERR_BAD_LEN and not out[51].any()
    got, out = flag_of(q_indptr=int32(0, 12, 51))
    assert got & _lib.DEVERR_BAD_LEN and not out[51].any()
    assert flag_of(q_indptr=int32(0, 53, 52))[0] & _lib.DEVERR_BAD_LEN


def test_offsets_that_descend_give_zeros():
    case = LatentCase([100, 30, 5], [12, 40, 3], 8, seed=19)
    case.q_indptr = torch.tensor([0, 40, 30, 55], dtype=torch.int32, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.latent_attention(*case.args(), **case.kwargs(), return_lse=True, error_flag=flag)
    assert int(flag) & _lib.DEVERR_BAD_LEN and not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("heads", [16, 128])
def test_repeat_graph_and_streams(heads):
    case = LatentCase([3000, 700, 64], [4, 1, 3], heads, seed=20)
    first = tsb.latent_attention(*case.args(), **case.kwargs())
    for _ in range(10):
        assert torch.equal(tsb.latent_attention(*case.args(), **case.kwargs()), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tsb.latent_attention(*case.args(), **case.kwargs())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    by_op = torch.ops.b200kv.latent_attention(*case.args(), case.mask, 192**-0.5, case.max_nodes, None)[0]
    assert torch.equal(by_op, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tsb.latent_attention(*case.args(), **case.kwargs())
    captured.zero_()
    graph.replay()
    assert torch.equal(captured, first)
    case.context_lens.copy_(torch.tensor([2000, 100, 0], dtype=torch.int32))  # the plan is made on the device
    graph.replay()
    assert torch.equal(captured, tsb.latent_attention(*case.args(), **case.kwargs()))


def test_absorbed_agrees_with_heads_of_their_own():
    """Against plain attention over keys and values multiplied out, all in 64 bits but the absorbed query's rounding."""
    g = torch.Generator(device="cuda").manual_seed(0)
    heads, ctx = 4, 300
    case = LatentCase([ctx], [1], heads, F16, chain=True, seed=21)
    wk, wv = (torch.randn((heads, 512, 128), generator=g, device="cuda", dtype=torch.float64) / 512**0.5 for _ in range(2))
    q = torch.randn((1, heads, 128), generator=g, device="cuda", dtype=torch.float64)
    case.q_latent = torch.einsum("nhd,hcd->nhc", q, wk).half()
    out = tsb.latent_attention(*case.args(), **case.kwargs())
    from tests.step_ref import latent_rows

    rows = latent_rows(case.pool, case.slots(0, 0, ctx + 1))
    k, v = torch.einsum("pc,hcd->hpd", rows[:, :512], wk), torch.einsum("pc,hcd->hpd", rows[:, :512], wv)
    s = (torch.einsum("hd,hpd->hp", q[0], k) + case.q_rope[0].double() @ rows[:, 512:].T) * 192**-0.5
    want = torch.einsum("hp,hpd->hd", torch.softmax(s, -1), v)
    got = torch.einsum("hc,hcd->hd", out[0].double(), wv)
    # fp16 roundings of q, weights and output, as random signs over 512 elements of unit size
    assert float((got - want).abs().max()) < 2.0**-8
