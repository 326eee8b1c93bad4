"""Tree attention over long contexts, where one lost or misjoined tile is a large error.

Every 128-token tile of a context has one loud key, whose score is the same for all of them, and a V row that
is zero but for one element; all loud keys together hold nearly all of the weight.  A tile that is skipped,
taken twice or joined with a wrong weight so changes an element by a quarter of itself, some hundred times
the bound, and the log-sum-exp by one part in the number of tiles.

The bound (u: unit roundoff of the output's type, u_p: of the weights'; w: the softmax weights):
  u |o|                              the output's own rounding
  (u_p + 2 c) sum w |v|              the weights' rounding; scores that are off by c, which is
                                     (D + 2) 2^-24 of the largest sum |q k| scale, fp32 sums of exact products
  2^-25 sum_p |step_p| max w s       fp16 weights: half a subnormal step, relative to the largest weight times V
                                     scale s (1 in a 16-bit cache, where the steps are V itself)
  2^-18 sum w |v| + 2^-25            exponentials, sums over tiles and pieces, subnormal outputs
"""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.verify_ref import QMAX, TreeCase, rows_of, unit_roundoff

pytestmark = pytest.mark.gpu

F16, BF16, I8, F8 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def make_loud(case, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    sign = torch.where(torch.rand(case.dim, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    size = 0.8 + 0.45 * torch.rand((*case.q.shape[:2], 1), generator=g, device="cuda")
    case.q = (size * sign).to(case.q.dtype)  # a row's loud score: 0.8 to 1.25 of sqrt(dim)
    eight = case.k_pool.dtype in QMAX
    qmax = QMAX.get(case.k_pool.dtype, 1.0)
    for b, c in enumerate(case.ctx):
        if c == 0:
            continue
        if eight:
            sl = case.slots(b, 0, c)
            case.k_scales[sl // 64, :, sl % 64] *= 0.05
        else:
            sl = case.slots(b, 0, c)
            case.k_pool[sl // 64, :, :, sl % 64] *= 0.05
        tiles = torch.arange(-(-c // 128), device="cuda")
        at = tiles * 128 + torch.tensor([0, 127, 63, 64], device="cuda")[tiles % 4]
        at = torch.minimum(at, torch.tensor(c - 1, device="cuda"))
        table = case.block_table[b].long()
        slots = table[at // 64] * 64 + at % 64
        for pool, scales, rows, size in (
                (case.k_pool, case.k_scales, sign.expand(len(at), -1), 1.0),
                (case.v_pool, case.v_scales,
                 torch.nn.functional.one_hot(tiles % case.dim, case.dim).float(), 100.0)):
            steps = (rows * (qmax if eight else size)).to(pool.dtype)
            raw = pool.view(torch.uint8) if eight else pool
            steps = (steps.view(torch.uint8) if eight else steps).view(len(at), 1, pool.shape[2], pool.shape[4])
            raw[slots // 64, :, :, slots % 64] = steps.expand(-1, case.hkv, -1, -1)
            if scales is not None:
                scales[slots // 64, :, slots % 64] = size / qmax
    return case


def check(case):
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.tree_attention(*case.args(), **case.kwargs(), return_lse=True, error_flag=flag)
    assert int(flag.item()) == 0
    dtype, scale, g = case.q.dtype, case.dim**-0.5, case.hq // case.hkv
    eight = case.k_pool.dtype in QMAX
    u, u_p = unit_roundoff(dtype), unit_roundoff(F16 if eight else dtype)
    for b, (c, t) in enumerate(zip(case.ctx, case.nodes)):
        if t == 0:
            continue
        rows = slice(case.indptr[b], case.indptr[b + 1])
        sl = case.slots(b, 0, c + t)
        k, v = rows_of(case.k_pool, case.k_scales, sl), rows_of(case.v_pool, case.v_scales, sl)
        see = torch.cat([torch.ones(t, c, dtype=torch.bool), case.see[b]], 1).cuda()
        for h in range(case.hkv):  # a KV head at a time
            q = case.q[rows, h * g:(h + 1) * g].double()
            s = (torch.einsum("tgd,pd->tgp", q, k[:, h]) * scale).masked_fill(~see[:, None], -math.inf)
            ref_lse = torch.logsumexp(s, -1)
            w = torch.exp(s - ref_lse[..., None])
            ref, spread = w @ v[:, h], w @ v[:, h].abs()
            most = float((q.abs() @ k[:, h].abs().T * scale).max())
            off = (case.dim + 2) * 2.0**-24 * most
            sc = case.v_scales[sl // 64, h, sl % 64].double() if eight else torch.ones_like(w[0, 0])
            live = sc > 0
            steps = torch.where(live[:, None], v[:, h].abs() / sc.clamp_min(1e-300)[:, None], 0.0).sum(0)
            tiny = 2.0**-25 * steps * (w * sc).amax(-1, keepdim=True) if u_p == 2.0**-11 else 0.0
            bound = u * ref.abs() + (u_p + 2 * off + 2.0**-18) * spread + tiny + 2.0**-25
            err = (out[rows, h * g:(h + 1) * g].double() - ref).abs()
            assert bool((err <= bound).all()), f"sequence {b}, head {h}: {float((err / bound).max()):.3g} of the bound"
            lse_err = (lse[rows, h * g:(h + 1) * g].double() - ref_lse).abs()
            assert bool((lse_err <= off + 2.0**-17 + 2.0**-22 * ref_lse.abs()).all()), float(lse_err.max())
    return out


CASES = [([70001], [16], 8, 1, False), ([33000, 7], [200, 3], 8, 2, False), ([12345, 20001, 128], [1, 1, 1], 16, 4, False),
         ([9000], [70], 12, 4, False), ([5000, 2500], [300, 129], 8, 2, True)]


@pytest.mark.parametrize("dtype,cache,dim", [(F16, F16, 128), (BF16, BF16, 128), (F16, F16, 64), (F16, I8, 128),
                                             (BF16, I8, 128), (F16, F8, 128)])
@pytest.mark.parametrize("ctx,nodes,hq,hkv,chain", CASES)
def test_no_tile_is_lost(dtype, cache, dim, ctx, nodes, hq, hkv, chain):
    check(make_loud(TreeCase(ctx, nodes, hq, hkv, dim, dtype, cache, chain=chain, seed=31)))


@pytest.mark.parametrize("cache", [F16, I8, F8])
@pytest.mark.parametrize("ctx,nodes,hq,hkv,chain", CASES)
def test_random_rows_over_long_contexts(cache, ctx, nodes, hq, hkv, chain):
    check(TreeCase(ctx, nodes, hq, hkv, cache=cache, chain=chain, seed=32))


def test_the_bound_sees_a_lost_tile():
    """On the reference alone: what is left of a tile is far outside the bound."""
    case = make_loud(TreeCase([70001], [16], 8, 1, seed=31))
    sl = case.slots(0, 0, 70017)
    k, v = rows_of(case.k_pool, None, sl)[:, 0], rows_of(case.v_pool, None, sl)[:, 0]
    s = (case.q[0, 0].double() @ k.T) * 128**-0.5
    s[70001:] = -math.inf
    s[70001] = case.q[0, 0].double() @ k[70001] * 128**-0.5
    want = torch.softmax(s, 0) @ v
    for tile in (0, 1, 273, 546):
        cut = s.clone()
        cut[tile * 128:(tile + 1) * 128] = -math.inf
        err = (torch.softmax(cut, 0) @ v - want).abs()
        spread = torch.softmax(s, 0) @ v.abs()
        bound = 2.0**-11 * want.abs() + (2.0**-11 + 2.0**-11) * spread + 2.0**-20
        assert float((err / bound).max()) > 50
