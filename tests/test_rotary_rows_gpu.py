"""GPU parity of rotary positions and of K/V rows stored and loaded, against 64-bit references."""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.verify_ref import QMAX, rotate64, rows_of, unit_roundoff
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu

F16, BF16, F32, I8, F8 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def turn_bound(ref, x, half, interleaved, dtype, scale=1.0):
    """Own rounding, three fp32 roundings of |a| + |b| and the table's two: 5 * 2^-24 (|a| + |b|)."""
    mag = torch.zeros_like(ref)
    a = x.double().abs()
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    mag[..., ia] = mag[..., ib] = (a[..., ia] + a[..., ib]) * scale
    tiny = 2.0 ** -25 if dtype == F16 else 0.0  # half the spacing of fp16's subnormal numbers
    return unit_roundoff(dtype) * ref.abs() + 5 * 2.0 ** -24 * mag * (1 + unit_roundoff(dtype)) + tiny


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rd", [(128, 128), (128, 64), (64, 16), (80, 80), (96, 20), (6, 4), (256, 250), (2, 2),
                                    (130, 8)])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (7, 5), (33, 40)])
def test_rotary(dtype, interleaved, dim, rd, tokens, heads):
    g = gen(dim + rd)
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 500, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    table = tsb.rotary_table(500, rd, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = tsb.rotary(x, table, pos, interleaved=interleaved, error_flag=flag)
    inv = 10000.0 ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64, device="cuda") / rd)
    ref = rotate64(x, pos.double()[:, None] * inv, 1.0, interleaved)
    assert int(flag.item()) == 0 and y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    assert bool(((y.double() - ref).abs() <= turn_bound(ref, x, rd // 2, interleaved, dtype)).all())
    assert torch.equal(y[..., rd:], x[..., rd:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_many_tokens(interleaved):
    # enough rows for several heads per thread; odd counts
    g = gen(1)
    for heads, dim, rd in ((41, 128, 96), (3, 64, 64)):
        tokens = 2501 if heads == 41 else 50001
        x = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(BF16)
        pos = torch.randint(0, 4000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        y = tsb.rotary(x, tsb.rotary_table(4000, rd, device="cuda"), pos, interleaved=interleaved)
        inv = 10000.0 ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64, device="cuda") / rd)
        ref = rotate64(x, pos.double()[:, None] * inv, 1.0, interleaved)
        assert bool(((y.double() - ref).abs() <= turn_bound(ref, x, rd // 2, interleaved, BF16)).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides(interleaved):
    g = gen(2)
    table = tsb.rotary_table(64, 64, device="cuda")
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    big = torch.randn(9, 12, 128, generator=g, device="cuda").to(F16)
    want = lambda x: tsb.rotary(x.contiguous(), table, pos, interleaved=interleaved)  # noqa: E731
    for x in (big[:, 3:7], big.transpose(0, 1).contiguous().transpose(0, 1), big[:, ::3], big[:, :, :66], big[:, :, 1:65],
              big[:, :1].expand(9, 5, 128), big.view(-1)[3:3 + 8 * 12 * 128].view(8, 12, 128)):
        n = x.shape[0]
        got = tsb.rotary(x, table, pos[:n].contiguous(), interleaved=interleaved)
        ref = tsb.rotary(x.contiguous().clone(), table, pos[:n].contiguous(), interleaved=interleaved)
        assert torch.equal(got, ref)
    assert torch.equal(want(big)[:, :, 64:], big[:, :, 64:])


def test_rotary_keeps_non_finite_values_apart():
    x = torch.ones(1, 1, 128, device="cuda", dtype=F32)
    x[0, 0, 70], x[0, 0, 127] = math.inf, math.nan
    table = tsb.rotary_table(8, 66, device="cuda")
    for inter in (False, True):
        y = tsb.rotary(x, table, torch.tensor([3], dtype=torch.int32, device="cuda"), interleaved=inter)
        assert bool(torch.isfinite(y[0, 0, :66]).all()) and torch.equal(y[0, 0, 66:127], x[0, 0, 66:127])


def test_rotary_flags_positions():
    x = torch.randn(2, 3, 64, device="cuda", dtype=F16)
    table = tsb.rotary_table(16, 64, device="cuda")
    for bad in (-1, 16):
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        y = tsb.rotary(x, table, torch.tensor([4, bad], dtype=torch.int32, device="cuda"), error_flag=flag)
        assert int(flag.item()) == _lib.DEVERR_BAD_LEN
        near = tsb.rotary(x, table, torch.tensor([4, max(0, min(bad, 15))], dtype=torch.int32, device="cuda"))
        assert torch.equal(y, near)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_tables(scaling):
    kw = dict(scaling=scaling, factor=8.0, original_max_pos=2048)
    t = tsb.rotary_table(16384, 64, base=1e5, device="cuda", **kw).double()
    i = torch.arange(32, dtype=torch.float64)
    inv, scale = 1e5 ** (-i / 32), 1.0
    if scaling == "linear":
        inv = inv / 8
    if scaling == "ntk":
        inv = (1e5 * 8 ** (64 / 62)) ** (-i / 32)
        assert math.isclose(float(inv[-1] * 8), float(1e5 ** (-i[-1] / 32)), rel_tol=1e-12)
    if scaling == "yarn":
        scale = 0.1 * math.log(8.0) + 1
        turns = 2048 * inv / (2 * math.pi)
        got = torch.atan2(t[1, :, 1], t[1, :, 0]).cpu()
        assert torch.allclose(got[turns > 40], inv[turns > 40], rtol=1e-6)
        assert torch.allclose(got[turns < 0.8], inv[turns < 0.8] / 8, rtol=1e-6)
        mid = (turns < 30) & (turns > 1.1)
        assert bool(((got < inv * (1 + 1e-6)) & (got > inv / 8))[mid].all())
        inv = got  # the ramp's own values: checked between its ends above
    p = 16383.0 if scaling != "yarn" else 1.0
    assert torch.allclose(t[int(p), :, 0].cpu(), torch.cos(p * inv) * scale, atol=1e-6)
    assert torch.allclose(t[int(p), :, 1].cpu(), torch.sin(p * inv) * scale, atol=1e-6)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rotary_gradient(interleaved, dtype):
    g = gen(5)
    x = torch.randn(5, 3, 24, generator=g, device="cuda").to(dtype).requires_grad_(True)
    pos = torch.randint(0, 50, (5,), generator=g, device="cuda", dtype=torch.int32)
    table = tsb.rotary_table(50, 16, scaling="yarn", factor=2.0, original_max_pos=32, device="cuda")
    w = torch.randn(5, 3, 24, generator=g, device="cuda").to(dtype)
    y = tsb.rotary(x, table, pos, interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, w)
    # the formula: the transposed map of w
    scale = 0.1 * math.log(2.0) + 1
    angle = torch.atan2(table[..., 1].double(), table[..., 0].double())[pos.long()]
    ref = rotate64(w, -angle, scale, interleaved)
    ref[..., 16:] = w[..., 16:].double()
    assert bool(((dx.double() - ref).abs() <= turn_bound(ref, w, 8, interleaved, dtype, scale) + 2e-7).all())
    # differences: y is linear, so <w, y(x + e) - y(x)> = <dx, e> up to the roundings of y
    if dtype == F32:
        e = torch.randn(5, 3, 24, generator=g, device="cuda")
        d = (w.double() * (tsb.rotary(x.detach() + e, table, pos, interleaved=interleaved).double()
                           - y.detach().double())).sum()
        assert abs(float(d - (dx.double() * e.double()).sum())) < 1e-4
    # a broadcast input and an expanded gradient
    one = torch.randn(5, 1, 24, generator=g, device="cuda").to(dtype).requires_grad_(True)
    tsb.rotary(one.expand(5, 3, 24), table, pos, interleaved=interleaved).sum().backward()
    ones = rotate64(torch.ones(5, 3, 24, device="cuda", dtype=dtype), -angle, scale, interleaved)
    ones[..., 16:] = 1.0
    assert torch.allclose(one.grad.double(), ones.sum(1, keepdim=True), atol=20 * unit_roundoff(dtype), rtol=0)


def test_rotary_second_gradient():
    x = torch.randn(2, 2, 8, device="cuda", requires_grad=True)
    table = tsb.rotary_table(4, 8, device="cuda")
    pos = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    (dx,) = torch.autograd.grad((tsb.rotary(x, table, pos) ** 2).sum(), x, create_graph=True)
    # |R x|^2 = |x|^2: the gradient is 2x, its sum's gradient 2
    assert torch.allclose(dx, 2 * x, atol=1e-5)
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    assert torch.allclose(ddx, torch.full_like(ddx, 2.0), atol=1e-5)


# --------------------------------------------------------------- store, load --
def steps(x, cache):
    """(steps, scale) in 64 bits of rows x (fp64)."""
    qmax = QMAX[cache]
    s = x.abs().amax(-1, keepdim=True) / qmax
    return torch.where(s > 0, x / s, 0.0), s


def check_store(x64, slack, pool, scales, slots, cache, dtype):
    """Rows in the cache against fp64 rows: a 16-bit row within its rounding, an 8-bit row within
    half a step of the true value (slack: what x64 may be off, in units of x)."""
    got = rows_of(pool, scales, slots)
    live = (slots >= 0)[:, None, None]
    if scales is None:
        bound = unit_roundoff(dtype) * x64.abs() + slack + (2.0 ** -25 if dtype == F16 else 0.0)
    else:
        q, s = steps(x64, cache)
        if cache == I8:
            half = torch.full_like(q, 0.5)
        else:  # half the spacing of e4m3 numbers at q, 2^-10 at least
            half = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 4.0)
            half = half * (1 + 2.0 ** -20)
        bound = half * s * (1 + 2.0 ** -19) + slack + 2.0 ** -21 * x64.abs()
    assert bool(((got - torch.where(live, x64, 0.0)).abs() <= bound)[live.expand_as(got)].all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cache,dim", [(None, 64), (None, 128), (I8, 128), (F8, 128)])
@pytest.mark.parametrize("turn", ["none", "half", "interleaved"])
@pytest.mark.parametrize("tokens,hq,hkv", [(1, 4, 1), (37, 6, 3), (1500, 32, 8)])
def test_store_and_load(dtype, cache, dim, turn, tokens, hq, hkv):
    cache = cache or dtype
    g = gen(tokens)
    k, v = (torch.randn(tokens, hkv, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(tokens, hq, dim, generator=g, device="cuda").to(dtype)
    nb = tokens // 64 + 2
    (kp, ks), (vp, vs) = (tsb.empty_row_pool(nb, hkv, dim, cache, device="cuda") for _ in range(2))
    for p in (kp, vp):
        p.view(torch.uint8).fill_(0x55)
    slots = torch.randperm(nb * 64, generator=g, device="cuda")[:tokens].contiguous()
    if tokens > 1:
        slots[::7] = -1
    kw = {}
    if turn != "none":
        rd = 48
        pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        kw = dict(q=q, table=tsb.rotary_table(300, rd, device="cuda"), positions=pos,
                  interleaved=turn == "interleaved")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    free = torch.ones(nb * 64, dtype=torch.bool, device="cuda")
    free[slots[slots >= 0]] = False
    out = tsb.kv_store(k, v, kp, vp, slots, k_scales=ks, v_scales=vs, error_flag=flag, **kw)
    assert int(flag.item()) == 0
    k64, slack = k.double(), torch.zeros(1, device="cuda", dtype=torch.float64)
    if turn == "none":
        assert out is None
    else:
        assert torch.equal(out, tsb.rotary(q, kw["table"], pos, interleaved=kw["interleaved"]))
        inv = 10000.0 ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64, device="cuda") / rd)
        k64 = rotate64(k, pos.double()[:, None] * inv, 1.0, kw["interleaved"])
        slack = 8 * 2.0 ** -24 * k64.abs().amax(-1, keepdim=True) * 2
    check_store(k64, slack, kp, ks, slots, cache, dtype)
    check_store(v.double(), 0.0, vp, vs, slots, cache, dtype)
    # nothing else was written
    for p in (kp, vp):
        rows = p.view(torch.uint8).permute(0, 3, 1, 2, 4).reshape(nb * 64, -1)
        assert bool((rows[free] == 0x55).all())
    for to in (F16, BF16, F32):
        got = tsb.kv_load(kp, slots, scales=ks, dtype=to)
        assert torch.equal(got, rows_of(kp, ks, slots).float().to(to))  # one product, exact in fp64, rounded twice
    assert tsb.kv_load(vp, slots, scales=vs).dtype == (cache if cache in (F16, BF16) else F16)


@pytest.mark.parametrize("cache", [I8, F8])
def test_store_special_rows(cache):
    k = torch.randn(8, 1, 128, device="cuda", dtype=BF16)
    k[0] = 0
    k[1, 0, 3] = math.nan
    k[2, 0, 3] = math.inf
    k[3] = 1e-40
    k[4] *= 1e30
    k[5] *= 1e-30
    k[6, 0, 1:] = 0
    (kp, ks), (vp, vs) = (tsb.empty_row_pool(1, 1, 128, cache, device="cuda") for _ in range(2))
    slots = torch.arange(8, device="cuda")
    tsb.kv_store(k, k, kp, vp, slots, k_scales=ks, v_scales=vs)
    y = tsb.kv_load(kp, slots, scales=ks, dtype=F32)
    assert torch.equal(kp.view(torch.uint8)[0, 0, 0, :8], vp.view(torch.uint8)[0, 0, 0, :8])  # the rows written
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2]).all())
    assert bool((y[3] == 0).all())  # a subnormal scale
    for i in (4, 5, 6, 7):
        top = k[i].float().abs().max()
        assert bool(((y[i] - k[i].float()).abs() <= top / (253 if cache == I8 else 27)).all())
    assert float(y[6, 0, 0]) == pytest.approx(float(k[6, 0, 0]), rel=1e-6)


def test_store_strides_flags_and_padding():
    g = gen(9)
    fused = torch.randn(70, 20, 128, generator=g, device="cuda").to(F16)
    (kp, ks), (vp, vs) = (tsb.empty_row_pool(2, 4, device="cuda") for _ in range(2))
    slots = torch.randperm(128, generator=g, device="cuda")[:70].contiguous()
    pos = torch.arange(70, device="cuda", dtype=torch.int32)
    table = tsb.rotary_table(70, 128, device="cuda")
    q, k, v = fused[:, :12], fused[:, 12:16], fused[:, 16:]
    out = tsb.kv_store(k, v, kp, vp, slots, k_scales=ks, v_scales=vs, q=q, table=table, positions=pos)
    (kp2, ks2), (vp2, vs2) = (tsb.empty_row_pool(2, 4, device="cuda") for _ in range(2))
    out2 = tsb.kv_store(k.contiguous(), v.transpose(0, 1).contiguous().transpose(0, 1), kp2, vp2, slots, k_scales=ks2,
                        v_scales=vs2, q=q.contiguous(), table=table, positions=pos)
    assert torch.equal(out, out2)
    for a, b, sa, sb in ((kp, kp2, ks, ks2), (vp, vp2, vs, vs2)):
        assert torch.equal(tsb.kv_load(a, slots, scales=sa), tsb.kv_load(b, slots, scales=sb))
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = slots.clone()
    bad[5] = 128
    tsb.kv_store(k, v, kp, vp, bad, k_scales=ks, v_scales=vs, error_flag=flag)
    assert int(flag.item()) == _lib.DEVERR_BAD_SLOT
    flag.zero_()
    assert bool((tsb.kv_load(kp, bad, scales=ks, error_flag=flag)[5] == 0).all())
    assert int(flag.item()) == _lib.DEVERR_BAD_SLOT
    flag.zero_()
    tsb.kv_store(k, v, kp, vp, slots, k_scales=ks, v_scales=vs, q=q, table=table, positions=pos + 1, error_flag=flag)
    assert int(flag.item()) == _lib.DEVERR_BAD_LEN


def test_nothing_to_do():
    (kp, ks), (vp, vs) = (tsb.empty_row_pool(2, 4, device="cuda") for _ in range(2))
    none = torch.empty(0, 4, 128, device="cuda", dtype=F16)
    slots = torch.empty(0, dtype=torch.int64, device="cuda")
    tsb.kv_store(none, none, kp, vp, slots, k_scales=ks, v_scales=vs)
    assert tsb.kv_load(kp, slots, scales=ks).shape == (0, 4, 128)
    table = tsb.rotary_table(4, 128, device="cuda")
    assert tsb.rotary(none, table, torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 128)
