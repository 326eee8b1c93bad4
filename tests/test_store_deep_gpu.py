"""kv_store where a lane group takes several rows (many tokens) and over the rotary dims, against the
same rows stored a few tokens at a time and against 64 bits."""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_rotary_rows_gpu import check_store
from tests.verify_ref import rotate64

pytestmark = pytest.mark.gpu

F16, BF16, I8, F8 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("tokens,hq,hkv,dim,dtype,cache", [
    (2500, 32, 8, 128, F16, I8),
    (7001, 6, 3, 128, BF16, F8),
    (9000, 7, 1, 128, BF16, BF16),
    (9000, 9, 5, 64, F16, F16),
    (12001, 4, 2, 128, F16, F8),
])
@pytest.mark.parametrize("rotary_dim,interleaved", [(16, False), (64, False), (128, False), (10, True), (64, True),
                                                    (96, False), (126, True), (128, True)])
def test_store_many_rows(tokens, hq, hkv, dim, dtype, cache, rotary_dim, interleaved):
    if rotary_dim > dim:
        rotary_dim = dim
    g = torch.Generator(device="cuda").manual_seed(tokens + rotary_dim)

    def rows(heads):  # strided: heads of a wider projection
        return torch.randn((tokens, heads + 2, dim), generator=g, device="cuda").to(dtype)[:, 1:heads + 1]

    q, k, v = rows(hq), rows(hkv), rows(hkv)
    table = tsb.rotary_table(500, rotary_dim, device="cuda")
    pos = torch.randint(0, 500, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    nb = tokens // 64 + 2
    slots = torch.randperm(nb * 64, generator=g, device="cuda")[:tokens].contiguous()
    slots[5::11] = -1

    def pools():
        made = [tsb.empty_row_pool(nb, hkv, dim, cache, device="cuda") for _ in range(2)]
        for pool, scales in made:
            pool.view(torch.uint8).fill_(0x55)
            if scales is not None:
                scales.fill_(7.0)
        return made

    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    (kp, ks), (vp, vs) = pools()
    out = tsb.kv_store(k, v, kp, vp, slots, ks, vs, q=q, table=table, positions=pos, interleaved=interleaved,
                       error_flag=flag)
    (kp2, ks2), (vp2, vs2) = pools()
    parts = [tsb.kv_store(k[i:i + 300], v[i:i + 300], kp2, vp2, slots[i:i + 300].contiguous(), ks2, vs2,
                          q=q[i:i + 300], table=table, positions=pos[i:i + 300].contiguous(), interleaved=interleaved,
                          error_flag=flag) for i in range(0, tokens, 300)]
    assert int(flag.item()) == 0
    assert torch.equal(out, torch.cat(parts))
    assert torch.equal(out, tsb.rotary(q, table, pos, interleaved=interleaved))
    for a, b in ((kp, kp2), (vp, vp2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in ((ks, ks2), (vs, vs2)):
        assert a is None or torch.equal(a, b)
    inv = 10000.0 ** (-2.0 * torch.arange(rotary_dim // 2, dtype=torch.float64, device="cuda") / rotary_dim)
    k64 = rotate64(k, pos.double()[:, None] * inv, 1.0, interleaved)
    check_store(k64, 16 * 2.0 ** -24 * k64.abs().amax(-1, keepdim=True), kp, ks, slots, cache, dtype)
    check_store(v.double(), 0.0, vp, vs, slots, cache, dtype)
