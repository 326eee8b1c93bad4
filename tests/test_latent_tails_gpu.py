"""Attention to one loud token before a long flat tail: every token of the tail has a weight far below the
loud one's, and all of them together have one that counts.

The loud token scores 23.5 (in powers of 2) above the others, so a quiet one has 2^-23.5 of its weight, 1.41
times the smallest number of fp16.  With all quiet values alike, roundings of their weights add up instead of averaging
out.  A result may be off by its own rounding (u |o|), its weights' (u of the weighted values, each), exponentials
(2^-17 of the same), what is cut off quiet weights at 2^-25, in units in which the loud one has 2^7 at least (n 2^-32 of
the largest value), and by the fp32 sums: products are added to a sum one after the other, and of each what lies below
the sum's last place, 2^-23 of it, may be dropped, n 2^-23 of the weighted values in all.  (That is 2^-8 of a result that the
loud token has most of: at 2^-23.5 a quiet one is hardly more than a last place.  In the first half of the elements, where the loud
one is zero, it is 2^-8 of the tail.)
"""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.verify_ref import unit_roundoff

pytestmark = pytest.mark.gpu

LOUD, TOKENS = 23.5, 32768
SCALE = LOUD * math.log(2.0) / 64.0  # a query of 1 and a key of 64 in one element


def values(width, dtype, g):
    """(loud, quiet) values; the first half of the loud one is zeros, where the tail is all there is."""
    loud, quiet = (torch.randn(width, generator=g, device="cuda").to(dtype) for _ in range(2))
    loud[:width // 2] = 0
    return loud, quiet


def check(out, lse, loud, quiet, seen, dtype):
    """out [.., width], lse [..], seen [..]: tokens that a row sees, the loud one among them."""
    scale = float(torch.tensor(SCALE, dtype=torch.float32))
    tail = (seen.double() - 1) * math.exp(-64.0 * scale)
    v0, v1 = loud.double(), quiet.double()
    want = (v0 + tail[..., None] * v1) / (1 + tail[..., None])
    spread = (v0.abs() + tail[..., None] * v1.abs()) / (1 + tail[..., None])
    u = unit_roundoff(dtype)
    cut = TOKENS * 2.0**-32 * float(v1.abs().max()) if dtype == torch.float16 else 0.0
    bound = u * want.abs() + (u + 2.0**-17 + TOKENS * 2.0**-23) * spread + cut + 2.0**-24
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), f"off by {float((err / bound).max()):.3g} of the bound"
    want_lse = 64.0 * scale + torch.log1p(tail)
    assert bool(((lse.double() - want_lse).abs() <= 2e-4 * (1 + want_lse.abs())).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [16, 128])
def test_absorbed(heads, dtype):
    # as many sequences as shares, so that a share has the loud token and the whole tail
    batch, g = 148, torch.Generator(device="cuda").manual_seed(heads)
    loud, quiet = values(512, dtype, g)
    rows = torch.zeros((TOKENS, 576), dtype=dtype, device="cuda")
    rows[:, :512] = quiet
    rows[0, :512] = loud
    rows[0, 512] = 64
    pool = tsb.empty_latent_pool(TOKENS // 64, dtype, "cuda")
    tsb.latent_store(rows[:, :512], rows[:, 512:], pool, torch.arange(TOKENS, device="cuda"))
    q = torch.zeros((batch, heads, 576), dtype=dtype, device="cuda")
    q[..., 512] = 1
    table = torch.arange(TOKENS // 64, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lens = torch.full((batch,), TOKENS - 1, dtype=torch.int32, device="cuda")
    lens[1] = TOKENS // 2  # (and one that is shorter)
    indptr = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    out, lse = tsb.latent_attention(q[..., :512], q[..., 512:], pool, table, lens, indptr, scale=SCALE, return_lse=True)
    check(out, lse, loud, quiet, (lens + 1)[:, None].expand(batch, heads), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [200, 100])
def test_expanded(rows, dtype):
    heads, g = 148, torch.Generator(device="cuda").manual_seed(rows)
    loud, quiet = values(128, dtype, g)
    k = torch.zeros((TOKENS, heads, 128), dtype=dtype, device="cuda")
    k[0, :, 5] = 64
    v = quiet.expand(TOKENS, heads, 128).contiguous()
    v[0] = loud
    q = torch.zeros((rows, heads, 192), dtype=dtype, device="cuda")
    q[..., 5] = 1
    ptr = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (rows, TOKENS)]
    r = torch.zeros((TOKENS, 64), dtype=dtype, device="cuda")
    out, lse = tsb.latent_prompt_attention(q, k, r, v, *ptr, scale=SCALE, return_lse=True)
    seen = TOKENS - rows + 1 + torch.arange(rows, device="cuda")
    check(out, lse, loud, quiet, seen[:, None].expand(rows, heads), dtype)
