"""A step's plan, latent attention and verification by their different ways in: the short
ways of plain eager calls, the Python and the registered operators, torch.compile,
traces, streams and host threads.  All of them launch the same kernels, so they give
the same bits."""

import threading

import pytest
import torch

import torch_spyre_b200 as tsb
from torch_spyre_b200 import _eager, latent, pages, tree

pytestmark = pytest.mark.gpu

HEADS, VOCAB = 6, 500


class Step:
    """Inputs of one small step: drafted trees of 3 and 2 nodes over 64 and 70 tokens, then two prompts."""

    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(11)

        def rows(*shape):
            return torch.randn(shape, generator=g, device="cuda").bfloat16()

        def ints(*values, dtype=torch.int32):
            return torch.tensor(values, dtype=dtype, device="cuda")

        self.pool = tsb.empty_latent_pool(5, device="cuda")
        self.block_table = torch.tensor([[2, -1, -1], [1, 3, -1]], dtype=torch.int32, device="cuda")
        self.counts, self.free, self.free_count = ints(1, 2), ints(4, 0, -1, -1, -1), ints(2)
        self.lens, self.indptr, self.parents = ints(64, 70), ints(0, 3, 5), ints(-1, 0, 0, -1, 0)
        self.tokens = ints(1, 2, 3, 4, 5, dtype=torch.int64)
        self.turn = tsb.rotary_table(128, 64, device="cuda")
        self.down, self.q, self.q_latent, self.norm = rows(5, 576), rows(5, HEADS, 192), rows(5, HEADS, 512), rows(512)
        self.p, self.d = (torch.rand((5, VOCAB), generator=g, device="cuda") for _ in range(2))
        self.u, self.s = (torch.rand(n, generator=g, device="cuda") for n in (5, 2))
        self.kv, self.k_rope, self.q_prompt = rows(140, HEADS, 256), rows(140, 64), rows(100, HEADS, 192)
        self.q_indptr, self.kv_indptr = ints(0, 70, 100), ints(0, 70, 140)
        tsb.latent_store(rows(320, 512), rows(320, 64), self.pool, torch.arange(320, device="cuda"))

    def public(self):
        mask = tsb.tree_mask(self.parents, self.indptr, 3)
        slots, positions = tsb.extend_pages(self.block_table, self.counts, self.free, self.free_count, self.lens,
                                            self.indptr, 5, mask)
        turned = tsb.latent_store(self.down[:, :512], self.down[:, 512:], self.pool, slots, self.q[..., 128:], self.norm,
                                  table=self.turn, positions=positions)
        out, lse = tsb.latent_attention(self.q_latent, turned, self.pool, self.block_table, self.lens, self.indptr, mask,
                                        return_lse=True)
        path, path_lens, tokens = tsb.tree_verify(self.parents, self.tokens, self.indptr, self.p, self.u, self.s, self.d)
        lens = tsb.latent_commit(self.pool, self.block_table, self.lens, path, path_lens)
        tsb.release_pages(self.block_table, self.counts, self.free, self.free_count, lens)
        c, r = tsb.latent_load(self.pool, slots)
        x, x_lse = tsb.latent_prompt_attention(self.q_prompt, self.kv[..., :128], self.k_rope, self.kv[..., 128:],
                                               self.q_indptr, self.kv_indptr, return_lse=True)
        return (slots, positions, turned, out, lse, path, path_lens, tokens, lens, c, r, x, x_lse, self.block_table,
                self.counts, self.free, self.free_count)

    def by(self, extend, store, attention, verify, commit, release, prompt):
        mask = tsb.tree_mask(self.parents, self.indptr, 3)
        slots, positions = extend(self.block_table, self.counts, self.free, self.free_count, self.lens, self.indptr, 5,
                                  mask, None)
        turned = store(self.down[:, :512], self.down[:, 512:], self.pool, slots, self.q[..., 128:], self.norm, 1e-6,
                       self.turn, positions, False, None)
        out, lse = attention(self.q_latent, turned, self.pool, self.block_table, self.lens, self.indptr, mask, 192**-0.5,
                             5, None)
        path, path_lens, tokens = verify(self.parents, self.tokens, self.indptr, self.p, self.u, self.s, self.d, 5, None)
        lens = commit(self.pool, self.block_table, self.lens, path, path_lens, None)
        release(self.block_table, self.counts, self.free, self.free_count, lens, None)
        c, r = tsb.latent_load(self.pool, slots)
        x, x_lse = prompt(self.q_prompt, self.kv[..., :128], self.k_rope, self.kv[..., 128:], self.q_indptr,
                          self.kv_indptr, 192**-0.5, True, None)
        return (slots, positions, turned, out, lse, path, path_lens, tokens, lens, c, r, x, x_lse, self.block_table,
                self.counts, self.free, self.free_count)


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_public_calls_take_the_short_way(monkeypatch):
    first = Step().public()  # makes the workspace of this stream

    def never(*a, **k):
        raise AssertionError("a plain call left the short way")

    for module, name in ((pages, "_extend_pages_impl"), (pages, "_release_pages_impl"), (latent, "_latent_store_impl"),
                         (latent, "_latent_commit_impl"), (latent, "_attend"), (latent, "_attend_prompt"),
                         (tree, "_tree_verify_impl")):
        monkeypatch.setattr(module, name, never)
    assert same(Step().public(), first)


def test_python_and_registered_operators_agree():
    want, ops = Step().public(), torch.ops.b200kv
    assert same(Step().by(pages._extend_pages_impl, latent._latent_store_impl, latent._latent_attention_impl,
                          tree._tree_verify_impl, latent._latent_commit_impl, pages._release_pages_impl,
                          latent._latent_prompt_attention_impl), want)
    assert same(Step().by(ops.extend_pages, ops.latent_store, ops.latent_attention, ops.tree_verify, ops.latent_commit,
                          ops.release_pages, ops.latent_prompt_attention), want)


def test_compiled_step_agrees():
    want = Step().public()
    assert same(torch.compile(lambda s: s.public(), backend="eager", fullgraph=True)(Step()), want)


def test_calls_without_the_module_give_the_same_bits(monkeypatch):
    want = Step().public()
    monkeypatch.setattr(_eager, "fast", _eager._Absent())
    assert same(Step().public(), want)


def test_written_tensors_count_as_changed():
    step = Step()
    written = (step.pool, step.block_table, step.counts, step.free, step.free_count)
    before = [t._version for t in written]
    step.public()
    assert all(t._version > b for t, b in zip(written, before))


def test_inputs_that_require_a_gradient():
    # none of these operators has one: a result must not pretend to
    step, want = Step(), Step().public()
    step.q.requires_grad_(True)
    step.q_prompt.requires_grad_(True)
    got = step.public()
    assert same(got, want)
    for result in (got[2], got[11]):
        with pytest.raises(RuntimeError):
            result.float().sum().backward()


def test_traced_calls_are_recorded():
    Step().public()

    def run(step, q, q_prompt):
        step.q, step.q_prompt = q, q_prompt
        return step.public()

    step = Step()
    traced = torch.jit.trace(lambda q, p: run(step, q, p), (step.q, step.q_prompt), check_trace=False)
    kinds = {n.kind() for n in traced.graph.nodes()}
    assert {f"b200kv::{n}" for n in ("extend_pages", "release_pages", "latent_store", "latent_attention", "tree_verify",
                                     "latent_commit", "latent_prompt_attention")} <= kinds


def test_another_stream_and_its_own_workspace():
    want = Step().public()
    step, side = Step(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step.public()
    side.synchronize()
    assert same(got, want)


def test_a_captured_step_replays():
    want, step = Step().public(), Step()
    state = [step.pool, step.block_table, step.counts, step.free, step.free_count]
    saved = [t.clone() for t in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step.public()
    for _ in range(3):
        for t, s in zip(state, saved):
            t.copy_(s)
        graph.replay()
        assert same(got, want)


def test_attentions_in_turn_share_a_workspace():
    """Operators of different sizes one after the other, decode's counters among them, on one workspace."""
    from tests.step_ref import LatentCase

    step, small, large = Step(), LatentCase([300, 7], [2, 3], 16, seed=1), LatentCase([9000, 100], [5, 1], 128, seed=2)
    g = torch.Generator(device="cuda").manual_seed(5)
    kp, vp = (torch.randn((40, 2, 2, 64, 64), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((1, 8, 128), generator=g, device="cuda").half()
    table, lens = torch.arange(40, dtype=torch.int32, device="cuda")[None], torch.tensor([2500], dtype=torch.int32, device="cuda")
    calls = [lambda: tsb.latent_attention(*small.args(), **small.kwargs()),
             lambda: tsb.decode_attention(q, kp, vp, table, lens),
             lambda: tsb.latent_prompt_attention(step.q_prompt, step.kv[..., :128], step.k_rope, step.kv[..., 128:],
                                                 step.q_indptr, step.kv_indptr),
             lambda: tsb.latent_attention(*large.args(), **large.kwargs())]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    for order in ((0, 1, 2, 3), (3, 1, 0, 2), (1, 3, 1, 2), (2, 1, 3, 0)):
        got = [calls[i]() for i in order]
        assert all(torch.equal(x, want[i]) for x, i in zip(got, order))


def test_host_threads_share_a_stream():
    """Calls of several host threads on one stream and workspace: each gives the bits that it gives alone."""
    from tests.step_ref import LatentCase

    step, stream = Step(), torch.cuda.current_stream()
    cases = [LatentCase([5000], [3], 16, seed=1), LatentCase([900, 0, 3000], [4, 1, 2], 128, seed=2)]

    def absorbed(c):  # the registered operator: its entry is called without the interpreter lock
        return torch.ops.b200kv.latent_attention(*c.args(), c.mask, 192**-0.5, c.max_nodes, None)

    def expanded(s):
        return torch.ops.b200kv.latent_prompt_attention(s.q_prompt, s.kv[..., :128], s.k_rope, s.kv[..., 128:], s.q_indptr,
                                                        s.kv_indptr, 192**-0.5, True, None)

    work = [(absorbed, c) for c in cases] + [(expanded, step)] * 2
    want = [call(c) for call, c in work]
    torch.cuda.synchronize()
    results = [None] * len(work)

    def run(i):
        try:
            call, c = work[i]
            with torch.cuda.stream(stream):
                results[i] = [call(c) for _ in range(60)]
                stream.synchronize()
        except Exception as e:  # noqa: BLE001 (shown below)
            results[i] = e

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got, one in zip(results, want):
        if isinstance(got, Exception):
            raise got
        assert all(torch.equal(x, y) for pair in got for x, y in zip(pair, one))


def test_arguments_are_checked_before_anything_is_written():
    step = Step()
    q, k, v, r = step.q_prompt, step.kv[..., :128], step.kv[..., 128:], step.k_rope
    mask = tsb.tree_mask(step.parents, step.indptr, 3)
    plan = (step.block_table, step.counts, step.free, step.free_count, step.lens, step.indptr)
    slots = torch.zeros(5, dtype=torch.int64, device="cuda")
    c, kr = step.down[:, :512], step.down[:, 512:]
    attend = (step.q_latent, step.q[..., 128:], step.pool, step.block_table, step.lens, step.indptr)
    verify = (step.parents, step.tokens, step.indptr, step.p, step.u, step.s)
    bad = [
        lambda: tsb.extend_pages(*plan[:5], step.indptr.long(), 5),
        lambda: tsb.extend_pages(*plan, -1),
        lambda: tsb.extend_pages(*plan, 4, mask),
        lambda: tsb.extend_pages(step.block_table.t(), *plan[1:], 5),
        lambda: tsb.extend_pages(step.block_table, step.counts[:1], *plan[2:], 5),
        lambda: tsb.release_pages(*plan[:4], step.lens[:1]),
        lambda: tsb.release_pages(*plan[:4], step.lens.cpu()),
        lambda: tsb.latent_store(c.float(), kr, step.pool, slots),
        lambda: tsb.latent_store(c[:, :500], kr, step.pool, slots),
        lambda: tsb.latent_store(c, kr, step.pool, slots, step.q[..., 128:]),
        lambda: tsb.latent_store(c, kr, step.pool, slots[:4]),
        lambda: tsb.latent_store(c, kr, step.pool, slots, table=step.turn),
        lambda: tsb.latent_store(c, kr, step.pool, slots, table=tsb.rotary_table(8, 32, device="cuda"),
                                 positions=step.parents),
        lambda: tsb.latent_store(c, kr, step.pool, slots, norm_weight=step.norm[:500]),
        lambda: tsb.latent_load(step.pool, slots.int()),
        lambda: tsb.latent_commit(step.pool, step.block_table, step.lens, step.parents, step.lens),
        lambda: tsb.latent_attention(step.q_latent.half(), *attend[1:]),
        lambda: tsb.latent_attention(step.q_latent[:, :3], *attend[1:]),
        lambda: tsb.latent_attention(*attend, mask[:4]),
        lambda: tsb.latent_attention(*attend, mask, max_nodes=65),
        lambda: tsb.latent_attention(*attend, scale=float("inf")),
        lambda: tsb.tree_verify(*verify[:3], step.p[:4], *verify[4:]),
        lambda: tsb.tree_verify(*verify, draft_probs=step.d.half()),
        lambda: tsb.tree_verify(*verify, max_path=0),
        lambda: tsb.latent_prompt_attention(q[..., :128], k, r, v, step.q_indptr, step.kv_indptr),
        lambda: tsb.latent_prompt_attention(q, k[:139], r, v, step.q_indptr, step.kv_indptr),
        lambda: tsb.latent_prompt_attention(q, k, r, v, step.q_indptr, step.kv_indptr[:2]),
        lambda: tsb.latent_prompt_attention(q.float(), k, r, v, step.q_indptr, step.kv_indptr),
    ]
    state = [t.clone() for t in (step.pool, *plan)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert all(torch.equal(a, b) for a, b in zip(state, (step.pool, *plan)))
