"""Edges of the verification operators: inputs that are out of range or out of order, extreme scales,
rows that no sequence has, and calls from several host threads."""

import math
import threading

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_verify_paths_gpu import Step, same
from tests.verify_ref import TreeCase, make_cache, unit_roundoff
from torch_spyre_b200 import _eager, _lib
from torch_spyre_b200.rotations import DTYPE_CODES

pytestmark = pytest.mark.gpu

F16, BF16, I8, F8 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def int32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------- rows --
def attend_into(case, out, lse, context_lens=None, q_indptr=None, max_nodes=None):
    """The C entry with outputs that the caller has filled; returns the error flag."""
    ctx = case.context_lens if context_lens is None else context_lens
    indptr = case.q_indptr if q_indptr is None else q_indptr
    N, Hq, D = case.q.shape
    batch = len(ctx)
    size = _lib.lib().b200kv_tree_workspace_bytes(N, batch, Hq, case.hkv, D)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    sc = [None if s is None else s.data_ptr() for s in (case.k_scales, case.v_scales)]
    mask, words = (None, 0) if case.mask is None else (case.mask.data_ptr(), case.mask.shape[1])
    table = case.block_table
    st = _lib.lib().b200kv_tree_attention(
        case.q.data_ptr(), DTYPE_CODES[case.q.dtype], case.q.stride(0), case.q.stride(1), case.k_pool.data_ptr(),
        case.v_pool.data_ptr(), DTYPE_CODES[case.k_pool.dtype], *sc, table.data_ptr(), table.stride(0), ctx.data_ptr(),
        indptr.data_ptr(), mask, words, out.data_ptr(), lse.data_ptr(), N, batch, Hq, case.hkv, D, case.k_pool.shape[0],
        table.shape[1], max_nodes or case.max_nodes, D**-0.5, ws.data_ptr(), size, flag.data_ptr(),
        torch.cuda.current_stream().cuda_stream)
    assert st == 0, _lib.last_error()
    torch.cuda.synchronize()
    return int(flag.item())


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("over,cut", [
    (dict(max_nodes=20), range(32, 52)),
    (dict(context_lens=(100, 128)), range(12, 52)),
    (dict(context_lens=(100, 120)), range(20, 52)),
    (dict(q_indptr=(0, 12, 45)), range(45, 52)),
    (dict(q_indptr=(3, 12, 52)), range(0, 3)),
    (dict(q_indptr=(0, 53, 52)), range(28, 52)),  # 100 committed tokens leave 28 of the two pages
])
def test_rows_that_no_sequence_has_are_zero(cache, over, cut):
    case = TreeCase([100, 30], [12, 40], 8, 2, cache=cache, seed=19, poison=False)
    over = {k: v if isinstance(v, int) else int32(*v) for k, v in over.items()}
    out, lse = torch.full_like(case.q, math.nan), torch.full((52, 8), math.nan, device="cuda")
    assert attend_into(case, out, lse, **over) & _lib.DEVERR_BAD_LEN
    cut = torch.tensor(list(cut), device="cuda")
    assert bool((out[cut] == 0).all()) and bool((lse[cut] == -math.inf).all())
    kept = torch.ones(52, dtype=torch.bool, device="cuda")
    kept[cut] = False
    assert bool(torch.isfinite(lse[kept]).all())


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("indptr", [(0, 40, 12, 52), (52, 0, 0, 52), (0, 60, -3, 52), (0, 52, 0, 52)])
def test_no_row_has_a_sequence_where_the_offsets_descend(cache, indptr):
    case = TreeCase([100, 30, 7], [12, 30, 10], 8, 2, cache=cache, seed=19, poison=False)
    out, lse = torch.full_like(case.q, math.nan), torch.full((52, 8), math.nan, device="cuda")
    assert attend_into(case, out, lse, q_indptr=int32(*indptr), max_nodes=64) & _lib.DEVERR_BAD_LEN
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("cache", [F16, I8])
def test_store_takes_any_stride_of_a_single_row_or_head(cache):
    g = torch.Generator(device="cuda").manual_seed(3)
    fused = torch.randn(1, 6 * 128 + 3, generator=g, device="cuda").half()
    q, k, v = (fused.as_strided((1, n, 128), (771, 128 if n > 1 else 771, 1), at * 128) for at, n in ((0, 4), (4, 1), (5, 1)))
    tight = tuple(torch.empty(x.shape, dtype=F16, device="cuda").copy_(x) for x in (q, k, v))
    table, pos, slots = tsb.rotary_table(8, 128, device="cuda"), int32(5), torch.tensor([70], device="cuda")
    got = []
    for q, k, v in ((q, k, v), tight):
        (kp, ks), (vp, vs) = (tsb.empty_row_pool(2, 1, 128, cache, device="cuda") for _ in range(2))
        out = tsb.kv_store(k, v, kp, vp, slots, ks, vs, q=q, table=table, positions=pos)
        got.append((out, tsb.kv_load(kp, slots, ks), tsb.kv_load(vp, slots, vs)))
    assert same(*got)


# -------------------------------------------------------------------- flags --
@pytest.mark.parametrize("flag", [torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64),
                                  torch.zeros(0, dtype=torch.int32)])
def test_flags_that_a_kernel_cannot_write_are_refused(flag):
    if flag.dtype == torch.int64 or flag.numel() == 0:
        flag = flag.cuda()
    case = TreeCase([10], [2], 2, 1, cache=I8, seed=1)
    rows = torch.randn(2, 1, 128, device="cuda", dtype=F16)
    slots, pos, table = torch.arange(2, device="cuda"), int32(0, 1), tsb.rotary_table(4, 128, device="cuda")
    kv = (case.k_pool, case.v_pool)
    for call in (lambda: tsb.rotary(rows, table, pos, error_flag=flag),
                 lambda: tsb.kv_store(rows, rows, *kv, slots, case.k_scales, case.v_scales, error_flag=flag),
                 lambda: tsb.kv_load(case.k_pool, slots, case.k_scales, error_flag=flag),
                 lambda: tsb.tree_mask(int32(-1, 0), int32(0, 2), 2, error_flag=flag),
                 lambda: tsb.tree_attention(*case.args(), **case.kwargs(), error_flag=flag),
                 lambda: tsb.tree_commit(*kv, case.block_table, case.context_lens, int32(0).view(1, 1), int32(1),
                                         case.k_scales, case.v_scales, error_flag=flag)):
        with pytest.raises(ValueError, match="error_flag"):
            call()


# ------------------------------------------------------------------ scales --
def scaled_case(ctx, nodes, hq, hkv, cache, v_scales, seed=0):
    """An 8-bit cache whose V rows have scales v_scales(number of rows)."""
    case = TreeCase(ctx, nodes, hq, hkv, dtype=BF16, cache=cache, seed=seed)
    for b, (c, t) in enumerate(zip(ctx, nodes)):
        sl = case.slots(b, 0, c + t)
        case.v_scales[sl // 64, :, sl % 64] = v_scales(c + t).float().cuda()[:, None].expand(-1, hkv)
    return case


def uniform(n):
    return (torch.rand(n, generator=torch.Generator().manual_seed(n)) + 0.2) * 0.02


RAMPS = {
    "tiny": lambda n: uniform(n) * 2.0**-115,
    "large": lambda n: uniform(n) * 2.0**100,
    "tiny first": lambda n: uniform(n) * torch.where(torch.arange(n) < 200, 2.0**-116, 1.0),
    "tiny last": lambda n: uniform(n) * torch.where(torch.arange(n) < n - 200, 1.0, 2.0**-80),
    "rising": lambda n: uniform(n) * torch.exp2(-115.0 + 10.0 * (torch.arange(n) // 128).clamp(max=12)),
    "zeros first": lambda n: uniform(n) * torch.where(torch.arange(n) < 200, 0.0, 2.0**-100),
    "zeros between large": lambda n: uniform(n) * torch.where(torch.arange(n) % 2 == 0, 0.0, 2.0**30),
    "all zero": lambda n: torch.zeros(n),
}


@pytest.mark.parametrize("cache", [I8, F8])
@pytest.mark.parametrize("ramp", RAMPS)
@pytest.mark.parametrize("ctx,nodes,hq,hkv", [([300, 5], [3, 1], 4, 2), ([1700, 64], [16, 9], 8, 2),
                                              ([257, 40], [60, 40], 4, 1), ([9000], [11], 8, 1)])
def test_scales_of_v_over_their_whole_range(cache, ramp, ctx, nodes, hq, hkv):
    """The result is right relative to the rows' own size (the bound: rounding of out and of the weights), and the
    lse does not know V at all."""
    case = scaled_case(ctx, nodes, hq, hkv, cache, RAMPS[ramp])
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.tree_attention(*case.args(), **case.kwargs(), return_lse=True, error_flag=flag)
    assert int(flag.item()) == 0
    ref, ref_lse, spread = case.reference()
    u = unit_roundoff(BF16)
    bound = u * ref.abs() + (2 * u + 2.0**-17) * spread + 2.0**-133
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert bool(((lse - ref_lse).abs() <= 2e-4 * (1 + ref_lse.abs())).all())


@pytest.mark.parametrize("cache", [I8, F8])
@pytest.mark.parametrize("nodes,hq", [(3, 4), (12, 8), (60, 4)])
@pytest.mark.parametrize("where", ["committed", "node"])
def test_a_nan_v_row_leaves_the_lse(cache, nodes, hq, where):
    case = TreeCase([1000, 40], [nodes, 2], hq, 2, cache=cache, seed=23)
    at = 700 if where == "committed" else 1000 + nodes // 2
    sl = case.slots(0, at, at + 1)[0]
    case.v_scales[sl // 64, :, sl % 64] = math.nan
    out, lse = tsb.tree_attention(*case.args(), **case.kwargs(), return_lse=True)
    _, ref_lse, _ = case.reference()
    sees = torch.ones(nodes, dtype=torch.bool) if where == "committed" else case.see[0][:, nodes // 2]
    sees = torch.cat([sees, torch.zeros(2, dtype=torch.bool)]).cuda()
    assert bool(torch.isnan(out[sees]).all()) and bool(torch.isfinite(out[~sees]).all())
    assert bool(((lse - ref_lse).abs() <= 2e-4 * (1 + ref_lse.abs())).all())


# ------------------------------------------------------------------- pages --
@pytest.mark.parametrize("cache", [F16, I8, F8])
@pytest.mark.parametrize("bad", [-1, -(1 << 31), 1 << 20])
@pytest.mark.parametrize("ctx,at", [([700, 30], 3), ([9000, 64], 64), ([40, 5], 0)])
def test_a_page_outside_the_pool_reads_as_zeros(cache, bad, ctx, at):
    """The same bits as with a page of zeros in its place, whatever the pool's first page holds."""
    case = TreeCase(ctx, [9, 2], 8, 2, cache=cache, seed=29)
    zeros = int((set(range(case.k_pool.shape[0])) - set(case.block_table.flatten().tolist()) - {0}).pop())
    if (case.block_table == 0).any():  # page 0 moves to a free place, so that no sequence has it
        free = int((set(range(case.k_pool.shape[0])) - set(case.block_table.flatten().tolist()) - {0, zeros}).pop())
        case.block_table[case.block_table == 0] = free
    else:
        free = zeros
    for pool, scales in ((case.k_pool, case.k_scales), (case.v_pool, case.v_scales)):
        raw = pool.view(torch.uint8)
        if free != zeros:
            raw[free] = raw[0]
            if scales is not None:
                scales[free] = scales[0]
        raw[0], raw[zeros] = 0x7F, 0  # NaN in e4m3 and fp16
        if scales is not None:
            scales[0], scales[zeros] = 1.0, 0.0
    table = case.block_table.clone()
    case.block_table[0, at] = zeros
    want = tsb.tree_attention(*case.args(), **case.kwargs(), return_lse=True)
    assert all(bool(torch.isfinite(x).all()) for x in want)
    table[0, at] = bad
    case.block_table = table
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = tsb.tree_attention(*case.args(), **case.kwargs(), return_lse=True, error_flag=flag)
    assert int(flag.item()) == _lib.DEVERR_BAD_BLOCK and all(torch.equal(x, y) for x, y in zip(got, want))


# ------------------------------------------------------------------- masks --
def test_descendants_of_a_pruned_node_see_nothing():
    parents = [-1, -2, 1, 2, 0] + [-1] + list(range(5, 100)) + [70, -2]  # a second sequence of several mask words
    parents = parents[:5] + [p if p < 0 else p - 5 for p in parents[5:]]
    parents[5 + 66] = -2
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    mask = tsb.tree_mask(int32(*parents), int32(0, 5, len(parents)), len(parents) - 5, error_flag=flag).cpu()
    assert int(flag.item()) == 0
    assert mask[:5].tolist() == [[1, 0], [0, 0], [0, 0], [0, 0], [17, 0]]
    for i in range(len(parents) - 5):  # a chain as far as node 65, pruned from 66 on; then a child of node 65
        want = [0, 0]
        if i < 66 or parents[5 + i] == 65:
            for j in list(range(min(i, 65) + 1)) + [i]:
                want[j // 64] |= 1 << (j % 64)
        assert [w & (2**64 - 1) for w in mask[5 + i].tolist()] == want, i


@pytest.mark.parametrize("grad", [False, True])
def test_tables_that_the_entry_refuses(grad):
    x = torch.randn(2, 1, 8, device="cuda", requires_grad=grad)
    odd = torch.zeros(1 + 4 * 8, device="cuda")[1:].view(4, 4, 2)  # 4 bytes past an 8-byte boundary
    for table, what in ((odd, "aligned"), (torch.zeros(0, 4, 2, device="cuda"), "max_pos")):
        with pytest.raises(tsb.B200KVError, match=what):
            tsb.rotary(x, table, int32(0, 1))


# ------------------------------------------------------------------ commit --
@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("ctx", [0, 3, 100])
@pytest.mark.parametrize("path,kept", [
    # (path, the entries that move): a run of negatives that ascends, entries below their own index
    ([0, -5, -4, 9], [0, 3]),
    ([-7, -6, -2, 3, 8], [3, 4]),
    ([5, 1, 2, 3, 7], [0, 3, 4]),
    (list(range(0, 140, 2)) + [0, 1, 2, 500], list(range(70)) + [73]),
    (list(range(1, 65)) + [-1000, -999, -998, 70], list(range(64)) + [67]),
])
def test_commit_skips_entries_that_do_not_ascend(cache, ctx, path, kept):
    g = torch.Generator(device="cuda").manual_seed(1)
    (kp, ks), (vp, vs) = (make_cache(24, 2, 128, cache, g) for _ in range(2))
    # the sequence's row of the table comes first, then one that must not be read
    table = torch.stack([torch.arange(10), torch.arange(10, 20)]).int().cuda()
    before = [None if t is None else t.clone() for t in (kp, vp, ks, vs)]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    paths = torch.tensor([path, [0] * len(path)], dtype=torch.int32, device="cuda")
    new = tsb.tree_commit(kp, vp, table, int32(ctx, 0), paths, int32(len(path), 0), ks, vs, error_flag=flag)
    assert int(flag.item()) == _lib.DEVERR_BAD_SLOT and new.tolist() == [ctx + len(path), 0]
    for now, was, is_pool in zip((kp, vp, ks, vs), before, (True, True, False, False)):
        if now is None:
            continue
        now, was = (t.view(torch.uint8) if is_pool else t for t in (now, was))
        want = was.clone()
        for i in kept:
            src, dst = ctx + path[i], ctx + i
            if is_pool:
                want[dst // 64, :, :, dst % 64] = was[src // 64, :, :, src % 64]
            else:
                want[dst // 64, :, dst % 64] = was[src // 64, :, src % 64]
        assert torch.equal(now, want)


@pytest.mark.parametrize("registered", [False, True])
@pytest.mark.parametrize("view", ["expanded", "wider", "one column", "overlapping"])
def test_commit_takes_paths_of_any_row_stride(view, registered):
    g = torch.Generator(device="cuda").manual_seed(2)
    table = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3)
    rows = int32(*range(2, 40))
    path = {"expanded": lambda: int32(1, 4, 9).expand(3, 3), "wider": lambda: rows[:36].view(3, 12)[:, :5],
            "one column": lambda: int32(7).expand(3, 1), "overlapping": lambda: rows.as_strided((3, 5), (2, 1))}[view]()
    tight = path.contiguous()
    lens, n = int32(3, 60, 100), torch.full((3,), path.shape[1], dtype=torch.int32, device="cuda")
    pools = [make_cache(9, 2, 128, I8, g) for _ in range(2)]
    after = []
    commit = torch.ops.b200kv.tree_commit if registered else lambda *a: tsb.tree_commit(*a[:-1], error_flag=a[-1])
    for p in (path, tight):
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        (kp, ks), (vp, vs) = ((a.clone(), s.clone()) for a, s in pools)
        if view == "overlapping" and p is path:  # refused: rows of one path must not run into the next's
            with pytest.raises(tsb.B200KVError, match="path_stride"):
                commit(kp, vp, table, lens, p, n, ks, vs, flag)
            return
        new = commit(kp, vp, table, lens, p, n, ks, vs, flag)
        assert int(flag.item()) == 0
        after.append((kp, ks, vp, vs, new))
    assert all(torch.equal(x, y) for x, y in zip(*after))


# ----------------------------------------------------------------- threads --
def in_threads(calls):
    """What the calls return (or raise), each by a thread of its own."""
    results = [None] * len(calls)

    def run(i):
        try:
            results[i] = calls[i]()
        except Exception as e:  # noqa: BLE001 (shown by the caller)
            results[i] = e

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in results:
        if isinstance(r, Exception):
            raise r
    return results


@pytest.mark.parametrize("cache", [F16, I8])
def test_first_call_of_a_host_thread(cache):
    """A thread's first use of CUDA can be a call that encodes tensor maps."""
    case = TreeCase([300, 7], [9, 3], 8, 2, cache=cache, seed=1)
    want = tsb.tree_attention(*case.args(), **case.kwargs())
    torch.cuda.synchronize()
    (got,) = in_threads([lambda: tsb.tree_attention(*case.args(), **case.kwargs())])
    assert torch.equal(got, want)
    if cache == F16:
        one = TreeCase([300, 7], [1, 1], 8, 2, seed=1)
        args = (one.q, one.k_pool, one.v_pool, one.block_table.clamp_min(0), one.context_lens + 1)
        want = tsb.decode_attention(*args)
        torch.cuda.synchronize()
        assert torch.equal(in_threads([lambda: tsb.decode_attention(*args)])[0], want)


def test_host_threads_share_a_stream():
    """Calls of several host threads on one stream and workspace, of the widest difference in rows, beside
    decode calls: each gives the bits that it gives alone."""
    cases = [TreeCase([5000], [3], 8, 2, seed=1), TreeCase([900, 0, 3000], [300, 200, 500], 8, 2, seed=2),
             TreeCase([20000, 70], [16, 1], 8, 2, cache=I8, seed=3), TreeCase([64], [1], 8, 2, cache=F8, seed=4)]
    decode = TreeCase([4000] * 20, [1] * 20, 8, 2, seed=5)
    table, lens = decode.block_table.clamp_min(0), decode.context_lens + 1
    stream = torch.cuda.current_stream()

    def tree_call(c):  # the registered operator: its entry is called without the interpreter lock
        return torch.ops.b200kv.tree_attention(*c.args(), c.mask, 128**-0.5, c.max_nodes, c.k_scales, c.v_scales, None)

    def decode_call(c):
        return torch.ops.b200kv.decode_attention(c.q, c.k_pool, c.v_pool, table, lens, 128**-0.5, 0, None)

    work = [(tree_call, c) for c in cases] + [(decode_call, decode)] * 2
    want = [call(c) for call, c in work]
    torch.cuda.synchronize()

    def run(call, c):
        with torch.cuda.stream(stream):
            got = [call(c) for _ in range(60)]
            stream.synchronize()
        return got

    for got, one in zip(in_threads([lambda call=call, c=c: run(call, c) for call, c in work]), want):
        assert all(torch.equal(x, y) for pair in got for x, y in zip(pair, one))


# ------------------------------------------------------------------ traces --
def test_traced_calls_are_recorded():
    first = Step()
    first.public()

    def run(step, q, k, v):
        step.q, step.k, step.v = q, k, v
        return step.public()

    step = Step()
    traced = torch.jit.trace(lambda q, k, v: run(step, q, k, v), (step.q, step.k, step.v), check_trace=False)
    kinds = {n.kind() for n in traced.graph.nodes()}
    assert {f"b200kv::{n}" for n in ("kv_store", "kv_load", "tree_mask", "tree_attention", "tree_commit", "rotary")} <= kinds
    fresh = Step()
    for t, s in ((step.kp, fresh.kp), (step.vp, fresh.vp), (step.ks, fresh.ks), (step.vs, fresh.vs)):
        t.copy_(s)
    assert same(traced(fresh.q, fresh.k, fresh.v), Step().public())


def test_traced_gradient():
    step = Step()
    x = step.k.clone().requires_grad_(True)
    traced = torch.jit.trace(lambda x: tsb.rotary(x, step.turn, step.pos), (x,), check_trace=False)
    w = torch.randn_like(x)
    assert torch.equal(torch.autograd.grad(traced(x), x, w)[0],
                       torch.autograd.grad(tsb.rotary(x, step.turn, step.pos), x, w)[0])


# ------------------------------------------------------------- without _fast --
def test_calls_without_the_module_give_the_same_bits(monkeypatch):
    want = Step().public()
    x = Step().k.clone().requires_grad_(True)
    step, w = Step(), torch.randn_like(x)
    grad = torch.autograd.grad(tsb.rotary(x, step.turn, step.pos), x, w)[0]
    monkeypatch.setattr(_eager, "fast", _eager._Absent())
    assert same(Step().public(), want)
    assert torch.equal(torch.autograd.grad(tsb.rotary(x, step.turn, step.pos), x, w)[0], grad)
