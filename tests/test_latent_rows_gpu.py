"""Rows of a latent cache written, read back and moved, against 64-bit references.

Tolerances.  The rotary key and queries: table entries are fp32 (2^-24), each product and the sum rounded in
fp32, so an element is off by at most 4 * 2^-24 of the pair's length, then half a step of the type.  The
norm: a sum of 512 squares in fp32 (each of the at most 16 + 5 additions of a lane's chain, the product and
the square root off by 2^-24, together under 32 * 2^-24 of the factor), two products: 40 * 2^-24, then half a step.
"""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.step_ref import latent_rows, turn
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu


def angles(positions):
    i = torch.arange(32, dtype=torch.float64, device="cuda")
    return positions.double()[:, None] * 10000.0 ** (-2.0 * i / 64)


def close(got, want, slack, size=None):
    u = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * u
    bound = want.abs() * u + (want.abs() if size is None else size) * slack * (1 + u) + tiny
    worst = ((got.double() - want).abs() - bound).max() if got.numel() else -1.0
    assert worst <= 0, worst


def pair_size(x, interleaved):
    x = x.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :32], x[..., 32:])
    r = torch.sqrt(a * a + b * b)
    return torch.stack([r, r], -1).flatten(-2) if interleaved else torch.cat([r, r], -1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads", [(1, 0), (1, 1), (3, 5), (65, 16), (7, 33), (130, 128), (2, 20)])
@pytest.mark.parametrize("interleaved,norm", [(False, True), (True, True), (True, False)])
def test_store_and_load(dtype, tokens, heads, interleaved, norm):
    g = torch.Generator(device="cuda").manual_seed(tokens + heads)
    nb, max_pos = 5, 700
    pool = torch.full((nb, 1, 9, 64, 64), float("nan"), dtype=dtype, device="cuda")
    fused = torch.randn((tokens, 640), generator=g, device="cuda").to(dtype)
    latent, k_rope = fused[:, 8:520], fused[:, 576:]
    q = torch.randn((tokens, heads, 192), generator=g, device="cuda").to(dtype)[..., 128:] if heads else None
    weight = (1 + 0.2 * torch.randn(512, generator=g, device="cuda")).to(dtype) if norm else None
    slots = torch.randperm(nb * 64, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[1] = -1
    positions = torch.randint(0, max_pos, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    table = tsb.rotary_table(max_pos, 64, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = pool.clone()
    out = tsb.latent_store(latent, k_rope, pool, slots, q_rope=q, norm_weight=weight, eps=1e-5, table=table,
                           positions=positions, interleaved=interleaved, error_flag=flag)
    assert int(flag) == 0
    ang = angles(positions)
    live = slots >= 0
    got = pool[slots[live] // 64, 0, :, slots[live] % 64].flatten(-2)
    want = latent.double()
    if norm:
        want = want / torch.sqrt((want * want).mean(-1, keepdim=True) + 1e-5) * weight.double()
        close(got[:, :512], want[live], 40 * 2.0**-24)
    else:
        assert torch.equal(got[:, :512], latent[live])
    close(got[:, 512:], turn(k_rope, ang, interleaved)[live], 4 * 2.0**-24, pair_size(k_rope, interleaved)[live])
    if heads:
        assert out.shape == (tokens, heads, 64) and out.is_contiguous()
        close(out, turn(q, ang, interleaved), 4 * 2.0**-24, pair_size(q, interleaved))
    else:
        assert out is None
    # what has no token is untouched
    rest = torch.ones(nb * 64, dtype=torch.bool, device="cuda")
    rest[slots[live]] = False
    rest = rest.view(nb, 64)
    assert torch.equal(pool.view(torch.int16).permute(0, 3, 1, 2, 4)[rest], before.view(torch.int16).permute(0, 3, 1, 2, 4)[rest])
    for out_dtype in (None, torch.float32):
        a, b = tsb.latent_load(pool, slots, dtype=out_dtype)
        assert torch.equal(torch.cat([a, b], -1).double(), latent_rows(pool, slots))


def test_rows_as_they_are_without_a_table():
    pool = tsb.empty_latent_pool(2, torch.float16, "cuda")
    x = torch.randn((4, 576), device="cuda").half()
    assert tsb.latent_store(x[:, :512], x[:, 512:], pool, torch.tensor([3, 127, 0, 64], device="cuda")) is None
    a, b = tsb.latent_load(pool, torch.tensor([3, 127, 0, 64, -1], device="cuda"))
    assert torch.equal(torch.cat([a, b], -1), torch.cat([x, torch.zeros_like(x[:1])]))


def test_a_single_token_of_any_stride_and_expanded_rows():
    pool = tsb.empty_latent_pool(1, torch.bfloat16, "cuda")
    x = torch.randn((1, 581), device="cuda").bfloat16()
    base = torch.randn((2, 584), device="cuda").bfloat16()
    row = base.as_strided((1, 512), (3, 1))
    tsb.latent_store(row, base[1:, :64], pool, torch.tensor([5], device="cuda"))
    assert torch.equal(tsb.latent_load(pool, torch.tensor([5], device="cuda"))[0], row)
    one = torch.randn((1, 512), device="cuda").bfloat16().expand(3, 512)
    tsb.latent_store(one, base[:1, :64].expand(3, 64), pool, torch.tensor([1, 2, 3], device="cuda"))
    assert torch.equal(tsb.latent_load(pool, torch.tensor([1, 2, 3], device="cuda"))[0], one)
    del x


def test_bad_slots_and_positions_are_flagged():
    pool = torch.zeros((1, 1, 9, 64, 64), dtype=torch.float16, device="cuda")
    x, flag = torch.randn((2, 576), device="cuda").half(), torch.zeros(1, dtype=torch.int32, device="cuda")
    tsb.latent_store(x[:, :512], x[:, 512:], pool, torch.tensor([64, -3], device="cuda"), error_flag=flag)
    assert int(flag) == _lib.DEVERR_BAD_SLOT and not pool.any()
    flag.zero_()
    table = tsb.rotary_table(4, 64, device="cuda")
    pos = torch.tensor([9, -1], dtype=torch.int32, device="cuda")
    tsb.latent_store(x[:, :512], x[:, 512:], pool, torch.tensor([0, 1], device="cuda"), table=table, positions=pos,
                     error_flag=flag)
    assert int(flag) == _lib.DEVERR_BAD_LEN
    other = torch.zeros_like(pool)
    tsb.latent_store(x[:, :512], x[:, 512:], other, torch.tensor([0, 1], device="cuda"), table=table,
                     positions=pos.clamp(0, 3))
    assert torch.equal(pool, other)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,path", [(1, 1), (3, 7), (5, 64), (2, 130)])
def test_commit_moves_the_path(dtype, batch, path):
    g = torch.Generator().manual_seed(path)
    nodes, ctx = 2 * path, [int(x) for x in torch.randint(0, 200, (batch,), generator=g)]
    pages = -(-(max(ctx) + nodes) // 64)
    pool = torch.randn((batch * pages + 2, 1, 9, 64, 64), device="cuda").to(dtype)
    table = torch.randperm(batch * pages, generator=g).to(torch.int32).view(batch, pages).cuda()
    lens = [path] + [int(x) for x in torch.randint(0, path + 1, (batch - 1,), generator=g)]
    rows = torch.full((batch, path), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        rows[b, :n] = torch.randperm(nodes, generator=g)[:n].sort().values.int()
    want = pool.clone()
    slot = lambda b, t: int(table[b, t // 64]) * 64 + t % 64
    for b, n in enumerate(lens):
        for i in range(n):
            src, dst = slot(b, ctx[b] + int(rows[b, i])), slot(b, ctx[b] + i)
            want[dst // 64, :, :, dst % 64] = pool[src // 64, :, :, src % 64]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    new = tsb.latent_commit(pool, table, torch.tensor(ctx, dtype=torch.int32, device="cuda"), rows.cuda(),
                            torch.tensor(lens, dtype=torch.int32, device="cuda"), error_flag=flag)
    assert int(flag) == 0 and new.tolist() == [c + n for c, n in zip(ctx, lens)]
    assert torch.equal(pool, want)
