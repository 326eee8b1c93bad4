"""Refusals and host-side parts of latent attention and of a step's plan (no GPU)."""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from torch_spyre_b200 import _lib

F16, BF16, F32, I8 = 0, 1, 2, 3
A = 1 << 20  # an aligned address that is never touched: every call here is refused, or has nothing to do


def extend(**over):
    a = dict(bt=A, bts=4, counts=A, free=A, cap=8, fc=A, ctx=A, ip=A, mask=None, words=0, slots=A, pos=A, N=4, B=2,
             MB=4, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_extend_pages(*a.values())


def release(**over):
    a = dict(bt=A, bts=4, counts=A, free=A, cap=8, fc=A, keep=A, B=2, MB=4, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_release_pages(*a.values())


def verify(**over):
    a = dict(par=A, tok=A, ip=A, p=A, ps=64, q=None, qs=0, dt=F32, u=A, s=A, path=A, pl=A, nt=A, N=4, B=2, V=64, mp=4,
             flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_tree_verify(*a.values())


def store(**over):
    a = dict(c=A, cs=512, k=A, ks=64, q=A, qn=256, qh=64, qo=A, dt=F16, w=A, eps=1e-6, pool=A, slots=A, table=A, mp=16,
             pos=A, inter=0, N=2, H=4, NB=4, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_latent_store(*a.values())


def commit(**over):
    a = dict(pool=A, dt=F16, bt=A, bts=4, ctx=A, path=A, ps=8, pl=A, nl=A, B=2, NB=8, MB=4, mp=8, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_latent_commit(*a.values())


def latent(**over):
    a = dict(ql=A, qlt=2048, qlh=512, qr=A, qrt=256, qrh=64, dt=F16, pool=A, bt=A, bts=4, ctx=A, ip=A, mask=A, words=1,
             out=A, lse=None, N=8, B=2, H=4, NB=8, MB=4, mn=8, scale=0.1, ws=None, wsb=0, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_latent_attention(*a.values())


def prompt(**over):
    a = dict(q=A, qt=768, qh=192, k=A, kt=512, kh=128, r=A, rt=64, v=A, vt=512, vh=128, dt=F16, qi=A, ki=A, out=A,
             lse=None, N=8, M=9, B=2, H=4, scale=0.1, causal=1, ws=None, wsb=0, flag=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_latent_prompt_attention(*a.values())


@pytest.mark.parametrize("call,over,status,msg", [
    (extend, dict(B=-1), 1, "batch"),
    (extend, dict(B=1025), 2, "batch"),
    (extend, dict(B=0), 1, "without a sequence"),
    (extend, dict(MB=0), 1, "max_blocks_per_seq"),
    (extend, dict(MB=1 << 21, bts=1 << 21), 1, "max_blocks_per_seq"),
    (extend, dict(bts=3), 1, "block_table_stride"),
    (extend, dict(cap=-1), 1, "capacity"),
    (extend, dict(cap=1 << 31), 1, "capacity"),
    (extend, dict(N=-1), 1, "num_tokens"),
    (extend, dict(N=1 << 31), 1, "num_tokens"),
    (extend, dict(mask=A), 1, "mask_words"),
    (extend, dict(free=None), 1, "null"),
    (extend, dict(ctx=None), 1, "null"),
    (extend, dict(ip=None), 1, "null"),
    (extend, dict(slots=None), 1, "null"),
    (release, dict(B=1025), 2, "batch"),
    (release, dict(bts=3), 1, "block_table_stride"),
    (release, dict(cap=-1), 1, "capacity"),
    (release, dict(keep=None), 1, "null"),
    (verify, dict(dt=I8), 1, "dtype"),
    (verify, dict(B=65536), 1, "batch"),
    (verify, dict(N=-1), 1, "total_q"),
    (verify, dict(V=0), 1, "vocab"),
    (verify, dict(V=1 << 30), 1, "vocab"),
    (verify, dict(mp=0), 1, "max_path"),
    (verify, dict(path=None), 1, "null"),
    (verify, dict(u=None), 1, "null"),
    (verify, dict(p=A + 2), 1, "aligned"),
    (verify, dict(q=A + 1, dt=F16), 1, "aligned"),
    (store, dict(dt=F32), 1, "dtype"),
    (store, dict(N=-1), 1, "num_tokens"),
    (store, dict(H=65537), 1, "num_q_heads"),
    (store, dict(NB=0), 1, "num_blocks"),
    (store, dict(N=1 << 30, H=64), 1, "num_tokens"),
    (store, dict(mp=0), 1, "max_pos"),
    (store, dict(table=None), 1, "table"),
    (store, dict(pos=None), 1, "positions"),
    (store, dict(eps=-1.0), 1, "eps"),
    (store, dict(qo=None), 1, "null"),
    (store, dict(c=A + 8), 1, "aligned"),
    (store, dict(cs=516), 1, "multiples of 8"),
    (store, dict(qh=68), 1, "multiples of 8"),
    (commit, dict(dt=F32), 1, "dtype"),
    (commit, dict(ps=7), 1, "path_stride"),
    (commit, dict(path=None), 1, "null"),
    (commit, dict(pool=None), 1, "null"),
    (commit, dict(pool=A + 8), 1, "aligned"),
    (commit, dict(bts=3), 1, "block_table_stride"),
    (latent, dict(dt=F32), 1, "dtype"),
    (latent, dict(H=0), 1, "num_heads"),
    (latent, dict(H=513), 2, "heads"),
    (latent, dict(B=1025), 2, "batch"),
    (latent, dict(B=0), 1, "without a sequence"),
    (latent, dict(N=1 << 30), 1, "total_q"),
    (latent, dict(NB=0), 1, "num_blocks"),
    (latent, dict(bts=3), 1, "block_table_stride"),
    (latent, dict(mn=65), 1, "mask_words"),
    (latent, dict(mn=0), 1, "max_nodes"),
    (latent, dict(scale=math.nan), 1, "finite"),
    (latent, dict(N=1 << 28, MB=1 << 20, bts=1 << 20), 2, "2^31"),
    (latent, dict(qr=None), 1, "null"),
    (latent, dict(qlh=516), 1, "multiples of 8"),
    (latent, dict(qrt=-256), 1, "multiples of 8"),
    (latent, dict(pool=A + 8), 1, "aligned"),
    (latent, dict(), 3, "workspace"),
    (latent, dict(ws=A + 128, wsb=1 << 40), 3, "aligned"),
    (prompt, dict(dt=F32), 1, "dtype"),
    (prompt, dict(H=0), 1, "num_heads"),
    (prompt, dict(B=1025), 2, "batch"),
    (prompt, dict(B=0), 1, "without a sequence"),
    (prompt, dict(M=-1), 1, "total_kv"),
    (prompt, dict(M=1 << 30), 1, "total_kv"),
    (prompt, dict(N=1 << 20, M=1 << 24, H=512), 2, "2^31"),
    (prompt, dict(scale=math.inf), 1, "finite"),
    (prompt, dict(k=None), 1, "null"),
    (prompt, dict(v=A + 8), 1, "aligned"),
    (prompt, dict(kt=516), 1, "multiples of 8"),
    (prompt, dict(rt=0), 1, "multiples of 8"),
    (prompt, dict(), 3, "workspace"),
    (prompt, dict(ws=A + 128, wsb=1 << 40), 3, "aligned"),
])
def test_refusals(call, over, status, msg):
    assert call(**over) == status
    assert msg in _lib.last_error()


def test_calls_with_nothing_to_do_succeed():
    assert extend(B=0, N=0, bt=None) == 0
    assert release(B=0, bt=None) == 0
    assert verify(B=0, ip=None) == 0
    assert store(N=0, c=None) == 0
    assert commit(B=0, pool=None) == 0
    assert latent(N=0, ql=None) == 0
    assert prompt(N=0, q=None) == 0


def test_workspace_bytes():
    L = _lib.lib()
    assert L.b200kv_latent_workspace_bytes(8, 2, 16) > 0
    assert L.b200kv_latent_workspace_bytes(8, 2, 0) == -1 and L.b200kv_latent_workspace_bytes(8, 2, 513) == -1
    assert L.b200kv_prompt_workspace_bytes(8, 9, 2, 16) > 0
    assert L.b200kv_prompt_workspace_bytes(8, -1, 2, 16) == -1 and L.b200kv_prompt_workspace_bytes(8, 9, 2, 0) == -1


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    pool = tsb.empty_latent_pool(1)
    rows = torch.zeros((1, 576), dtype=torch.bfloat16)
    table = torch.zeros((1, 1), dtype=torch.int32)
    q = torch.zeros((1, 1, 512), dtype=torch.bfloat16)
    for call in (
            lambda: tsb.extend_pages(table, i[:1], i, i[:1], i[:1], i, 0),
            lambda: tsb.release_pages(table, i[:1], i, i[:1], i[:1]),
            lambda: tsb.tree_verify(i[:1], i[:1].long(), i, torch.zeros(1, 8), torch.zeros(1), torch.zeros(1)),
            lambda: tsb.latent_store(rows[:, :512], rows[:, 512:], pool, i[:1].long()),
            lambda: tsb.latent_load(pool, i[:1].long()),
            lambda: tsb.latent_commit(pool, table, i[:1], table, i[:1]),
            lambda: tsb.latent_attention(q, q[..., :64], pool, table, i[:1], i),
            lambda: tsb.latent_prompt_attention(q[..., :192], q[..., :128], rows[:, :64], q[..., :128], i, i)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_pools_are_checked():
    assert tsb.empty_latent_pool(3, torch.float16).shape == (3, 1, 9, 64, 64)
    with pytest.raises(ValueError):
        tsb.empty_latent_pool(1, torch.float32)
    with pytest.raises(ValueError):
        tsb.latent_load(torch.zeros((1, 1, 8, 64, 64), dtype=torch.float16), torch.zeros(1, dtype=torch.int64))


def test_fake_kernels_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.b200kv
    with FakeTensorMode():
        i = torch.empty(3, dtype=torch.int32, device="cuda")
        table = torch.empty((2, 4), dtype=torch.int32, device="cuda")
        slots, positions = ops.extend_pages(table, i[:2], i, i[:1], i[:2], i, 5, None, None)
        assert (slots.shape, slots.dtype) == ((5,), torch.int64) and (positions.shape, positions.dtype) == ((5,), torch.int32)
        assert ops.release_pages(table, i[:2], i, i[:1], i[:2], None) is None
        probs, u = torch.empty((3, 32), device="cuda"), torch.empty(3, device="cuda")
        path, path_lens, tokens = ops.tree_verify(i, i.long(), i, probs, u, u[:2], None, 7, None)
        assert path.shape == (2, 7) and path_lens.shape == tokens.shape == (2,) and tokens.dtype == torch.int64
        pool = torch.empty((4, 1, 9, 64, 64), dtype=torch.bfloat16, device="cuda")
        rows = torch.empty((3, 576), dtype=torch.bfloat16, device="cuda")
        q = torch.empty((3, 6, 512), dtype=torch.bfloat16, device="cuda")
        turned = ops.latent_store(rows[:, :512], rows[:, 512:], pool, i.long(), q[..., :64], None, 1e-6, u, i, False, None)
        assert turned.shape == (3, 6, 64)
        assert ops.latent_store(rows[:, :512], rows[:, 512:], pool, i.long(), None, None, 1e-6, None, None, False,
                                None).shape == (3, 0, 64)
        assert ops.latent_commit(pool, table, i[:2], table, i[:2], None).shape == (2,)
        out, lse = ops.latent_attention(q, turned, pool, table, i[:2], i, None, 1.0, 3, None)
        assert out.shape == q.shape and lse.shape == (3, 6) and lse.dtype == torch.float32
        out, lse = ops.latent_prompt_attention(q[..., :192], q[..., :128], rows[:, :64], q[..., :128], i, i, 1.0, True, None)
        assert out.shape == (3, 6, 128) and out.dtype == torch.bfloat16 and lse.shape == (3, 6)
