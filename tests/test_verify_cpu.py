"""Refusals and host-side parts of the speculative-verification operators (no GPU)."""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from torch_spyre_b200 import _lib

F16, BF16, F32, I8, U8 = 0, 1, 2, 3, 99
A = 1 << 20  # an aligned address that is never touched: every call here is refused, or has nothing to do


def rotary(**over):
    a = dict(x=A, dtype=F16, st=512, sh=128, out=A, table=A, max_pos=16, rd=128, pos=A, T=2, H=4, D=128, inter=0,
             tr=0, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_rotary(*a.values())


def store(**over):
    a = dict(q=A, qn=512, qh=128, qo=A, k=A, kn=512, kh=128, v=A, vn=512, vh=128, rdt=F16, kp=A, vp=A, pdt=I8, ks=A,
             vs=A, slots=A, table=A, max_pos=16, rd=128, pos=A, inter=0, N=2, Hq=4, Hkv=2, D=128, NB=4, flag=None,
             stream=None)
    a.update(over)
    return _lib.lib().b200kv_kv_store(*a.values())


def load(**over):
    a = dict(pool=A, pdt=I8, sc=A, slots=A, out=A, odt=F16, N=2, H=2, D=128, NB=4, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_kv_load(*a.values())


def tree(**over):
    a = dict(q=A, qdt=F16, qt=512, qh=128, kp=A, vp=A, pdt=F16, ks=None, vs=None, bt=A, bts=4, ctx=A, ip=A, mask=A,
             words=1, out=A, lse=None, N=8, B=2, Hq=4, Hkv=2, D=128, NB=8, MB=4, mn=8, scale=0.1, ws=None, wsb=0,
             flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_tree_attention(*a.values())


def commit(**over):
    a = dict(kp=A, vp=A, pdt=F16, ks=None, vs=None, bt=A, bts=4, ctx=A, path=A, ps=8, pl=A, nl=A, B=2, Hkv=2, D=128,
             NB=8, MB=4, mp=8, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_tree_commit(*a.values())


@pytest.mark.parametrize("call,over,status,msg", [
    (rotary, dict(dtype=I8), 1, "dtype"),
    (rotary, dict(rd=3), 1, "rotary_dim"),
    (rotary, dict(rd=130), 1, "rotary_dim"),
    (rotary, dict(rd=0), 1, "rotary_dim"),
    (rotary, dict(max_pos=0), 1, "max_pos"),
    (rotary, dict(T=-1), 1, "num_tokens"),
    (rotary, dict(x=None), 1, "null"),
    (rotary, dict(table=A + 4), 1, "aligned"),
    (store, dict(rdt=F32), 1, "row dtype"),
    (store, dict(pdt=U8), 1, "pool dtype"),
    (store, dict(pdt=BF16), 1, "rows' dtype"),
    (store, dict(D=64), 2, "head_dim"),
    (store, dict(pdt=F16, D=256), 2, "head_dim"),
    (store, dict(rd=24), 2, "multiples of 16"),
    (store, dict(table=None), 1, "table"),
    (store, dict(pos=None), 1, "positions"),
    (store, dict(ks=None), 1, "k_scales"),
    (store, dict(k=A + 8), 1, "aligned"),
    (store, dict(kn=516), 1, "multiples of 8"),
    (store, dict(qo=None), 1, "q_out"),
    (store, dict(N=-1), 1, "num_tokens"),
    (load, dict(odt=I8), 1, "out dtype"),
    (load, dict(sc=None), 1, "scales"),
    (load, dict(D=64), 2, "head_dim"),
    (load, dict(slots=None), 1, "null"),
    (load, dict(NB=0), 1, "num_blocks"),
    (tree, dict(qdt=F32), 1, "q dtype"),
    (tree, dict(pdt=BF16), 1, "q's dtype"),
    (tree, dict(pdt=I8), 1, "k_scales"),
    (tree, dict(pdt=I8, ks=A, vs=A, D=64), 2, "head_dim"),
    (tree, dict(D=96), 2, "head_dim"),
    (tree, dict(Hq=5), 1, "multiple"),
    (tree, dict(Hq=258), 2, "group"),
    (tree, dict(B=1025), 2, "batch"),
    (tree, dict(B=0), 1, "without a sequence"),
    (tree, dict(bts=3), 1, "block_table_stride"),
    (tree, dict(mn=65), 1, "mask_words"),
    (tree, dict(mn=0), 1, "max_nodes"),
    (tree, dict(scale=math.inf), 1, "finite"),
    (tree, dict(q=A + 2), 1, "aligned"),
    (tree, dict(qh=0), 1, "positive"),
    (tree, dict(ctx=None), 1, "null"),
    (tree, dict(), 3, "workspace"),
    (commit, dict(pdt=F32), 1, "dtype"),
    (commit, dict(D=96), 2, "head_dim"),
    (commit, dict(pdt=I8), 1, "scales"),
    (commit, dict(ps=7), 1, "path_stride"),
    (commit, dict(path=None), 1, "null"),
    (commit, dict(B=70000), 1, "batch"),
])
def test_refusals(call, over, status, msg):
    assert call(**over) == status
    assert msg in _lib.last_error()


def test_calls_with_nothing_to_do_succeed():
    assert rotary(T=0, x=None) == 0
    assert store(N=0, k=None) == 0
    assert load(N=0, pool=None) == 0
    assert tree(N=0, q=None) == 0
    assert commit(B=0, kp=None) == 0
    assert _lib.lib().b200kv_tree_mask(None, None, 0, 0, 1, None, None, None) == 0
    assert _lib.lib().b200kv_tree_mask(A, A, 0, 3, 1, A, None, None) == 1
    assert _lib.lib().b200kv_tree_mask(A, A, 1, 3, 0, A, None, None) == 1


def test_workspace_bytes():
    size = _lib.lib().b200kv_tree_workspace_bytes
    assert size(8, 2, 32, 8, 128) > 0
    assert size(8, 2, 30, 8, 128) == -1 and size(8, 2, 32, 8, 96) == -1


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        tsb.rotary(x, tsb.rotary_table(4, 64), torch.zeros(1, dtype=torch.int32))


def test_pools_and_tables_are_checked():
    with pytest.raises(ValueError):
        tsb.empty_row_pool(1, 1, 64, torch.int8)
    with pytest.raises(ValueError):
        tsb.empty_row_pool(1, 1, 256, torch.float16)
    with pytest.raises(ValueError):
        tsb.empty_row_pool(1, 1, 128, torch.float32)
    for bad in (dict(rotary_dim=3), dict(max_pos=0), dict(scaling="cubic"), dict(factor=0.5), dict(scaling="yarn")):
        with pytest.raises(ValueError):
            tsb.rotary_table(**{**dict(max_pos=8, rotary_dim=8), **bad})
    assert tsb.rotary_table(5, 6, scaling="ntk", factor=2.0).shape == (5, 3, 2)


def test_table_angles_hold_at_large_positions():
    t = tsb.rotary_table(131072, 8)
    for i in range(4):
        a = 131071 * 10000.0 ** (-i / 4)
        assert abs(float(t[131071, i, 0]) - math.cos(a)) < 1e-7 and abs(float(t[131071, i, 1]) - math.sin(a)) < 1e-7


def test_fake_kernels_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(3, 4, 128, dtype=torch.float16, device="cuda")
        pool = torch.empty(2, 4, 1, 64, 128, dtype=torch.int8, device="cuda")
        slots = torch.empty(3, dtype=torch.int64, device="cuda")
        assert torch.ops.b200kv.kv_load(pool, slots, None, torch.bfloat16, None).dtype == torch.bfloat16
        out, lse = torch.ops.b200kv.tree_attention(x, pool, pool, slots, slots, slots, None, 1.0, 4, None, None, None)
        assert out.shape == x.shape and lse.shape == (3, 4) and lse.dtype == torch.float32
        assert torch.ops.b200kv.tree_mask(slots, slots, 2, None).shape == (3, 2)
