"""Workspaces that are made while a graph is captured: zeros before any replay, no part of the graph."""

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.step_ref import LatentCase
from tests.test_latent_prompt_gpu import Case
from tests.verify_ref import TreeCase
from torch_spyre_b200 import ops
from torch_spyre_b200.workloads import DECODE_CONFIGS, make_decode_inputs

pytestmark = pytest.mark.gpu

WORKSPACE = 1 << 26  # at least what any of these takes


def latent():
    case = LatentCase([3000, 700, 64], [4, 1, 3], 16, seed=20)
    return lambda: tsb.latent_attention(*case.args(), **case.kwargs())


def prompt():
    case = Case([300, 700, 64], [400, 700, 1000], 4, seed=23)
    return lambda: tsb.latent_prompt_attention(*case.args())


def tree():
    case = TreeCase([3000, 700], [4, 1], 8, 2, seed=3)
    return lambda: tsb.tree_attention(*case.args(), **case.kwargs())


def decode():
    inp = make_decode_inputs(DECODE_CONFIGS["gqa_b16"], device="cuda", ctx=[5000, 300])
    return lambda: tsb.decode_attention(inp.q, inp.k_pool, inp.v_pool, inp.block_table, inp.context_lens)


@pytest.fixture
def fresh(monkeypatch):
    """No workspace of any stream, to the Python and the short ways."""
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_outgrown", [])
    monkeypatch.setattr(tsb._eager, "fast", tsb._eager._Absent())


def capture(stream, run):
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    return graph, out


@pytest.mark.parametrize("make", [latent, prompt, tree, decode])
def test_replays_do_not_fill_the_workspace(make, fresh):
    call = make()
    want, stream = call(), torch.cuda.Stream()
    ops._workspaces.clear()
    graph, out = capture(stream, call)
    (ws,) = ops._workspaces.values()
    torch.cuda.synchronize()
    assert not ws.any()  # before the first replay
    ws[-64:] = 7  # (past what a call uses)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert bool((ws[-64:] == 7).all())


@pytest.mark.parametrize("make", [latent, prompt, tree, decode])
def test_memory_of_the_graph_is_not_the_workspaces(make, fresh):
    call = make()
    want, stream, places = call(), torch.cuda.Stream(), []
    ops._workspaces.clear()

    def run():
        temps = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (1 << 20, 1 << 24, WORKSPACE, 1 << 25)]
        places.extend((t.data_ptr(), t.data_ptr() + t.numel()) for t in temps)
        del temps  # their memory is the graph's to give to what follows
        return call()

    graph, out = capture(stream, run)
    (ws,) = ops._workspaces.values()
    first, last = ws.data_ptr(), ws.data_ptr() + ws.numel()
    assert all(last <= a or first >= b for a, b in places)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_the_second_graph_may_be_replayed_first(fresh):
    calls = [decode(), tree(), latent()]
    want, stream = [call() for call in calls], torch.cuda.Stream()
    ops._workspaces.clear()
    graphs = [capture(stream, call) for call in calls]
    for i in (1, 0, 2, 0, 1):
        graph, out = graphs[i]
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[i])
