"""The verification operators by their different ways in: the short ways of plain
eager calls, the registered operators, torch.compile, gradients and modes.  All of
them launch the same kernels, so they give the same bits."""

import pytest
import torch

import torch_spyre_b200 as tsb
from torch_spyre_b200 import _eager, kv_rows, rotations, tree

pytestmark = pytest.mark.gpu


class Step:
    """Inputs of one small verify step over an int8 cache."""

    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(11)

        def rows(n, heads):
            return torch.randn((n, heads, 128), generator=g, device="cuda").half()

        (self.kp, self.ks), (self.vp, self.vs) = (tsb.empty_row_pool(4, 2, 128, torch.int8, "cuda") for _ in range(2))
        self.block_table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device="cuda")
        self.lens = torch.tensor([64, 70], dtype=torch.int32, device="cuda")
        self.indptr = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
        self.parents = torch.tensor([-1, 0, 0, -1, 0], dtype=torch.int32, device="cuda")
        self.pos = torch.tensor([64, 65, 65, 70, 71], dtype=torch.int32, device="cuda")
        self.slots = torch.tensor([0, 1, 2, 3 * 64 + 6, 3 * 64 + 7], device="cuda")
        self.path = torch.tensor([[0, 2], [0, 1]], dtype=torch.int32, device="cuda")
        self.path_lens = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
        self.turn = tsb.rotary_table(128, 128, device="cuda")
        self.q, self.k, self.v = rows(5, 8), rows(5, 2), rows(5, 2)
        old = torch.arange(256, device="cuda")
        tsb.kv_store(rows(256, 2), rows(256, 2), self.kp, self.vp, old, self.ks, self.vs)

    def public(self):
        q = tsb.kv_store(self.k, self.v, self.kp, self.vp, self.slots, self.ks, self.vs, q=self.q, table=self.turn,
                         positions=self.pos)
        mask = tsb.tree_mask(self.parents, self.indptr, 3)
        out, lse = tsb.tree_attention(q, self.kp, self.vp, self.block_table, self.lens, self.indptr, mask,
                                      k_scales=self.ks, v_scales=self.vs, return_lse=True)
        lens = tsb.tree_commit(self.kp, self.vp, self.block_table, self.lens, self.path, self.path_lens, self.ks, self.vs)
        back = tsb.kv_load(self.kp, self.slots, self.ks)
        return q, mask, out, lse, lens, back, tsb.rotary(self.k, self.turn, self.pos)

    def by(self, store, mask_op, attention, commit, load, rotary):
        q = store(self.k, self.v, self.kp, self.vp, self.slots, self.ks, self.vs, self.q, self.turn, self.pos, False, None)
        mask = mask_op(self.parents, self.indptr, 1, None)
        out, lse = attention(q, self.kp, self.vp, self.block_table, self.lens, self.indptr, mask, 128**-0.5, 5, self.ks,
                             self.vs, None)
        lens = commit(self.kp, self.vp, self.block_table, self.lens, self.path, self.path_lens, self.ks, self.vs, None)
        back = load(self.kp, self.slots, self.ks, torch.float16, None)
        return q, mask, out, lse, lens, back, rotary(self.k, self.turn, self.pos, False, False, None)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_public_calls_take_the_short_way(monkeypatch):
    step = Step()
    first = step.public()  # makes the workspace of this stream

    def never(*a, **k):
        raise AssertionError("a plain call left the short way")

    for module, name in ((kv_rows, "_kv_store_impl"), (kv_rows, "_kv_load_impl"), (tree, "_tree_mask_impl"),
                         (tree, "_attend"), (tree, "_tree_commit_impl"), (rotations, "_rotary_impl")):
        monkeypatch.setattr(module, name, never)
    assert same(Step().public(), first)
    x = step.k.clone().requires_grad_(True)
    tsb.rotary(x, step.turn, step.pos).sum().backward()


def test_python_and_registered_operators_agree():
    want = Step().public()
    ops = torch.ops.b200kv
    assert same(Step().by(kv_rows._kv_store_impl, tree._tree_mask_impl, tree._tree_attention_impl,
                          tree._tree_commit_impl, kv_rows._kv_load_impl, rotations._rotary_impl), want)
    assert same(Step().by(ops.kv_store, ops.tree_mask, ops.tree_attention, ops.tree_commit, ops.kv_load, ops.rotary), want)


def test_compiled_step_agrees():
    want = Step().public()
    got = torch.compile(lambda s: s.public(), backend="eager", fullgraph=True)(Step())
    assert same(got, want)


def test_inputs_that_require_a_gradient():
    # no operator but rotary has one: the result must not pretend to
    step, want = Step(), Step().public()
    step.q.requires_grad_(True)
    q = tsb.kv_store(step.k, step.v, step.kp, step.vp, step.slots, step.ks, step.vs, q=step.q, table=step.turn,
                     positions=step.pos)
    assert torch.equal(q, want[0])
    with pytest.raises(RuntimeError):
        q.float().sum().backward()
    with torch.no_grad():
        assert not tsb.rotary(step.q, step.turn, step.pos).requires_grad


def test_rotary_gradients_agree():
    step = Step()
    w = torch.randn_like(step.k)
    grads = []
    for rotary in (lambda x: tsb.rotary(x, step.turn, step.pos, interleaved=True),
                   lambda x: rotations._Rotary.apply(x, step.turn, step.pos, True, False, None),
                   lambda x: torch.ops.b200kv.rotary(x, step.turn, step.pos, True, False, None)):
        x = step.k.clone().requires_grad_(True)
        y = rotary(x)
        assert y.requires_grad
        grads.append(torch.autograd.grad(y, x, w)[0])
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


def test_rotary_gradient_sees_a_changed_table():
    step = Step()
    x = step.k.clone().requires_grad_(True)
    y = tsb.rotary(x, step.turn, step.pos)
    step.turn.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_forward_derivatives_are_not_dropped():
    import torch.autograd.forward_ad as fwad

    step = Step()
    with fwad.dual_level():
        x = fwad.make_dual(step.k, torch.randn_like(step.k))
        assert _eager.fast.rotary(x, step.turn, step.pos, False, False, None) is None
        assert not _eager.direct(x)


def test_written_tensors_count_as_changed():
    step = Step()
    before = [t._version for t in (step.kp, step.vp, step.ks, step.vs)]
    step.public()
    assert all(t._version > b for t, b in zip((step.kp, step.vp, step.ks, step.vs), before))
