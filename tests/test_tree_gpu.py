"""GPU parity of tree attention, tree masks and the commit against 64-bit references."""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.verify_ref import TreeCase, attention_bound, make_cache, pack_bits, random_tree, rows_of, see_of
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu

F16, BF16, I8, F8 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def check(case, **kw):
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.tree_attention(*case.args(), **case.kwargs(), return_lse=True, error_flag=flag, **kw)
    assert int(flag.item()) == 0
    ref, ref_lse, spread = case.reference(kw.get("scale"))
    n_keys = max(c + t for c, t in zip(case.ctx, case.nodes))
    bound = attention_bound(ref, spread, n_keys, case.q.dtype)
    err = (out.double() - ref).abs()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert bool(((err <= bound) | torch.isnan(ref) | (out.double() == ref)).all()), \
        f"off by {float((err / bound).nan_to_num().max()):.3g} of the bound"
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((out[empty] == 0).all())
    # scores: fp32 sums of D exact products of 16-bit (or 8-bit) values
    assert bool(((lse.double() - ref_lse).abs() <= 2e-4 * (1 + ref_lse.abs()))[~empty].all())
    return out


TYPES = [(F16, F16, 128), (BF16, BF16, 128), (F16, F16, 64), (BF16, BF16, 64), (F16, I8, 128), (BF16, I8, 128),
         (F16, F8, 128), (BF16, F8, 128)]


@pytest.mark.parametrize("dtype,cache,dim", TYPES)
@pytest.mark.parametrize("hq,hkv", [(4, 4), (6, 2), (8, 1), (16, 2)])
def test_trees_ragged(dtype, cache, dim, hq, hkv):
    # contexts around page and tile ends, drafts of one node up to two mask words
    case = TreeCase([0, 1, 63, 64, 65, 127, 128, 129, 500, 1000], [1, 7, 2, 64, 65, 33, 1, 100, 17, 5], hq, hkv, dim,
                    dtype, cache, dead=0.1, seed=hq)
    check(case)


@pytest.mark.parametrize("dtype,cache,dim", TYPES)
def test_chains(dtype, cache, dim):
    case = TreeCase([0, 5, 300, 64], [130, 1, 257, 64], 8, 2, dim, dtype, cache, chain=True, seed=3)
    check(case)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 12, 32, 100, 128])
def test_groups(group):
    case = TreeCase([200, 0, 77], [9, 3, 1], group * 2, 2, seed=group)
    check(case)
    check(TreeCase([200, 0, 77], [9, 3, 1], group * 2, 2, cache=I8, seed=group))


@pytest.mark.parametrize("cache", [F16, I8])
def test_one_token_equals_decode_lengths(cache):
    # the single-token form over contexts from nothing to several tiles per SM
    case = TreeCase([0, 1, 127, 128, 4096, 20000], [1] * 6, 32, 8, cache=cache, seed=11)
    check(case)


@pytest.mark.parametrize("cache", [F16, I8, F8])
def test_long_context_is_split(cache):
    check(TreeCase([70001], [16], 8, 1, cache=cache, seed=5))
    check(TreeCase([33000, 7], [200, 3], 8, 2, cache=cache, seed=6))


def test_many_sequences():
    g = torch.Generator().manual_seed(2)
    ctx = torch.randint(0, 400, (300,), generator=g).tolist()
    nodes = torch.randint(0, 6, (300,), generator=g).tolist()  # sequences without a draft among them
    check(TreeCase(ctx, nodes, 4, 2, seed=7))


def test_chunk_of_a_long_prompt():
    check(TreeCase([2000], [700], 16, 2, chain=True, seed=8))
    check(TreeCase([0], [1025], 8, 8, dtype=BF16, chain=True, seed=9))


def test_rows_without_anything_to_see():
    case = TreeCase([0, 0, 130], [4, 70, 9], 8, 2, seed=12)
    for s in case.see:
        s[::2] = False
    case.mask = torch.cat([pack_bits(s, 2) for s in case.see]).cuda()
    check(case)


def test_mask_is_taken_as_it_is():
    # any bits: nodes that see later ones, or not themselves; bits past the draft are ignored
    case = TreeCase([10, 0], [70, 20], 4, 1, seed=13)
    g = torch.Generator().manual_seed(0)
    case.see = [torch.rand(s.shape, generator=g) < 0.3 for s in case.see]
    mask = torch.cat([pack_bits(s, 2) for s in case.see])
    mask[70:, 0] |= -(1 << 20)
    mask[:, 1] |= -(1 << 6)
    case.mask = mask.cuda()
    check(case)


def test_large_scores_and_rising_maxima():
    # scores of +-100: the running maximum moves far, and most weights vanish
    check(TreeCase([900, 64], [33, 3], 8, 2, qscale=30.0, seed=14))
    case = TreeCase([1500], [8], 8, 1, seed=15, poison=False)
    # keys that grow along the context: every tile raises the maximum
    ramp = torch.linspace(0.1, 8.0, 1508, device="cuda")
    sl = case.slots(0, 0, 1508)
    case.k_pool[sl // 64, :, :, sl % 64] = (case.q[0, 0].view(1, 1, 2, 64).float()
                                            * ramp[:, None, None, None]).half().expand(-1, 1, 2, 64)
    check(case)


def test_explicit_scale_and_strides():
    case = TreeCase([100, 30], [12, 40], 8, 2, seed=16)
    check(case, scale=0.3)
    wide = torch.randn(case.q.shape[0], 20, 128, device="cuda", dtype=F16)
    wide[:, 5:13] = case.q
    case.q = wide[:, 5:13]  # a slice of a fused projection
    check(case)
    across = torch.empty(8, case.q.shape[0], 128, device="cuda", dtype=F16)
    across.copy_(case.q.transpose(0, 1))
    case.q = across.transpose(0, 1)  # head-major
    check(case)
    table = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    table[:, :case.block_table.shape[1]] = case.block_table
    case.block_table = table[:, :case.block_table.shape[1]]
    check(case)


@pytest.mark.parametrize("cache", [F16, I8, F8])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_rows_of_unseen_nodes(cache, value):
    """A node's NaN or inf reaches the rows that see it and no other."""
    case = TreeCase([70, 0, 128], [12, 5, 1], 8, 2, cache=cache, seed=17)
    sl = case.slots(0, 70 + 3, 70 + 4)[0]
    for pool, scales in ((case.k_pool, case.k_scales), (case.v_pool, case.v_scales)):
        if scales is None:
            pool[sl // 64, :, 0, sl % 64, 5] = value
        else:
            scales[sl // 64, :, sl % 64] = value
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = tsb.tree_attention(*case.args(), **case.kwargs(), error_flag=flag)
    ref, _, spread = case.reference()
    sees = torch.cat(case.see[:1])[:, 3]
    assert bool(sees.any()) and not bool(sees.all())
    keep = torch.cat([~sees, torch.ones(6, dtype=torch.bool)]).cuda()
    assert bool(torch.isfinite(out[keep]).all())
    bound = attention_bound(ref, spread, 200, F16)
    assert bool(((out.double() - ref).abs() <= bound)[keep].all())
    # whoever sees it has the key's NaN (inf - inf included) in every element
    if math.isnan(value):
        assert bool(torch.isnan(out[:12][sees]).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_with_finite_keys(value):
    case = TreeCase([70, 3], [12, 130], 8, 2, seed=18)
    for b, node in ((0, 3), (1, 100)):
        sl = case.slots(b, case.ctx[b] + node, case.ctx[b] + node + 1)[0]
        case.v_pool[sl // 64, 1, 1, sl % 64, 9] = value
    check(case)


def test_inputs_outside_their_range_are_flagged():
    case = TreeCase([100, 30], [12, 40], 8, 2, seed=19)

    def flag_of(**over):
        names = ["q", "k_pool", "v_pool", "block_table", "context_lens", "q_indptr"]
        args = dict(zip(names, case.args()), **case.kwargs())
        args.update(over)
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        tsb.tree_attention(**args, error_flag=flag)
        return int(flag.item())

    assert flag_of() == 0
    table = case.block_table.clone()
    table[0, 1] = case.k_pool.shape[0]
    assert flag_of(block_table=table) & _lib.DEVERR_BAD_BLOCK
    table[0, 1] = -1
    assert flag_of(block_table=table) & _lib.DEVERR_BAD_BLOCK
    assert flag_of(context_lens=torch.tensor([100, 128], dtype=torch.int32, device="cuda")) & _lib.DEVERR_BAD_LEN
    assert flag_of(context_lens=torch.tensor([-1, 30], dtype=torch.int32, device="cuda")) & _lib.DEVERR_BAD_LEN
    assert flag_of(max_nodes=39) & _lib.DEVERR_BAD_LEN
    assert flag_of(q_indptr=torch.tensor([0, 12, 51], dtype=torch.int32, device="cuda")) & _lib.DEVERR_BAD_LEN
    assert flag_of(q_indptr=torch.tensor([0, 53, 52], dtype=torch.int32, device="cuda")) & _lib.DEVERR_BAD_LEN


def test_repeat_graph_and_streams():
    case = TreeCase([3000, 700, 64], [40, 1, 16], 16, 2, cache=I8, seed=20)
    first = tsb.tree_attention(*case.args(), **case.kwargs())
    for _ in range(3):
        assert torch.equal(tsb.tree_attention(*case.args(), **case.kwargs()), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tsb.tree_attention(*case.args(), **case.kwargs())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tsb.tree_attention(*case.args(), **case.kwargs())
    captured.zero_()
    graph.replay()
    assert torch.equal(captured, first)
    case.context_lens.copy_(torch.tensor([2000, 100, 0], dtype=torch.int32))  # the plan is made on the device
    graph.replay()
    assert torch.equal(captured, tsb.tree_attention(*case.args(), **case.kwargs()))


@pytest.mark.parametrize("cache", [F16, I8, F8])
def test_long_contexts_give_the_same_bits_every_time(cache):
    # a cache that stays in L2, so that loads come back fast, and blocks of every width
    for nodes in (3, 12, 200):
        case = TreeCase([33000, 700], [nodes, 3], 8, 2, cache=cache, seed=6)
        first = check(case)
        for _ in range(10):
            assert torch.equal(tsb.tree_attention(*case.args(), **case.kwargs()), first)


def test_one_node_agrees_with_decode_attention():
    case = TreeCase([900, 17, 64], [1, 1, 1], 32, 8, seed=21)
    out = tsb.tree_attention(*case.args(), **case.kwargs())
    table = case.block_table.clamp_min(0)
    dec = tsb.decode_attention(case.q, case.k_pool, case.v_pool, table, case.context_lens + 1)
    torch.testing.assert_close(out.float(), dec.float(), atol=2e-3, rtol=1e-2)


# ------------------------------------------------------------------- masks --
@pytest.mark.parametrize("nodes", [[1], [3, 0, 64, 65, 1, 200], [130] * 3])
def test_tree_mask(nodes):
    g = torch.Generator().manual_seed(4)
    trees = [random_tree(n, g, 0.1) for n in nodes]
    indptr = torch.tensor([0] + torch.tensor(nodes).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    mask = tsb.tree_mask(parents, indptr, max(nodes), error_flag=flag)
    words = -(-max(nodes) // 64)
    want = torch.cat([pack_bits(see_of(t), words) for t in trees])
    assert int(flag.item()) == 0 and torch.equal(mask.cpu(), want)


def test_tree_mask_flags_a_parent_after_its_child():
    for parents in ([-1, 1], [-1, 2, 0], [-3]):
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        indptr = torch.tensor([0, len(parents)], dtype=torch.int32, device="cuda")
        tsb.tree_mask(torch.tensor(parents, dtype=torch.int32, device="cuda"), indptr, 8, error_flag=flag)
        assert int(flag.item()) & _lib.DEVERR_BAD_LEN


# ------------------------------------------------------------------ commit --
@pytest.mark.parametrize("cache,dim", [(F16, 128), (BF16, 64), (I8, 128), (F8, 128)])
@pytest.mark.parametrize("max_path", [0, 1, 9, 150, 600])
def test_commit(cache, dim, max_path):
    g, gc = torch.Generator(device="cuda").manual_seed(1), torch.Generator().manual_seed(1)
    ctx = [0, 1, 63, 200, 64]
    room = max_path + 40
    need = [-(-(c + room) // 64) for c in ctx]
    nb = sum(need) + 2
    order, table, at = torch.randperm(nb, generator=gc), torch.full((5, max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    pools = [make_cache(nb, 3, dim, cache, g) for _ in range(2)]
    lens = [max_path, max_path // 2, 0, max_path // 3, max_path]
    path = torch.zeros(5, max_path, dtype=torch.int32)
    for b, n in enumerate(lens):
        # ascending, so that sources and destinations overlap (the last: all in place)
        path[b, :n] = (torch.randperm(room, generator=gc)[:n].sort().values if b < 4 else torch.arange(n)).int()
    want = [(p.clone(), None if s is None else s.clone()) for p, s in pools]
    slot = lambda b, t: (int(table[b, t // 64]), t % 64)  # noqa: E731
    for (p, s), (p0, s0) in zip(want, pools):
        for b, n in enumerate(lens):
            for i in range(n):
                sb, so = slot(b, ctx[b] + int(path[b, i]))
                db, do = slot(b, ctx[b] + i)
                p.view(torch.uint8)[db, :, :, do] = p0.view(torch.uint8)[sb, :, :, so]
                if s is not None:
                    s[db, :, do] = s0[sb, :, so]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    new = tsb.tree_commit(pools[0][0], pools[1][0], table.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"),
                          path.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), k_scales=pools[0][1],
                          v_scales=pools[1][1], error_flag=flag)
    assert int(flag.item()) == 0
    assert new.tolist() == [c + n for c, n in zip(ctx, lens)]
    for (p, s), (p1, s1) in zip(want, pools):
        assert torch.equal(p.view(torch.uint8), p1.view(torch.uint8))
        assert s is None or torch.equal(s, s1)


def test_commit_flags():
    pool, _ = tsb.empty_row_pool(4, 2, dtype=F16, device="cuda")
    pool.zero_()
    ctx = torch.tensor([60], dtype=torch.int32, device="cuda")

    def flag_of(path, n, table=((0, 1),), ctx=ctx):
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        new = tsb.tree_commit(pool, pool.clone(), torch.tensor(table, dtype=torch.int32, device="cuda"), ctx,
                              torch.tensor([path], dtype=torch.int32, device="cuda"),
                              torch.tensor([n], dtype=torch.int32, device="cuda"), error_flag=flag)
        return int(flag.item()), int(new.item())

    assert flag_of([0, 3, 5], 3) == (0, 63)
    assert flag_of([0, 3, 3], 3)[0] & _lib.DEVERR_BAD_SLOT
    assert flag_of([0, -1, 3], 3)[0] & _lib.DEVERR_BAD_SLOT
    assert flag_of([0, 3, 1 << 30], 3)[0] & _lib.DEVERR_BAD_SLOT
    assert flag_of([0, 3, 5], 4) == (_lib.DEVERR_BAD_LEN, 60)
    assert flag_of([0, 3, 5], -1) == (_lib.DEVERR_BAD_LEN, 60)
    assert flag_of([0, 1, 5], 3, table=((0, 9),))[0] & _lib.DEVERR_BAD_BLOCK
    assert flag_of([0, 3, 5], 3, ctx=torch.tensor([129], dtype=torch.int32, device="cuda"))[0] & _lib.DEVERR_BAD_LEN


def test_rows_written_then_committed_are_what_is_read():
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(10, 2, 128, generator=g, device="cuda", dtype=F16) for _ in range(2))
    (kp, ks), (vp, vs) = (tsb.empty_row_pool(3, 2, device="cuda") for _ in range(2))
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    pos = torch.arange(60, 70, device="cuda")
    slots = table[0].long()[pos // 64] * 64 + pos % 64
    tsb.kv_store(k, v, kp, vp, slots, k_scales=ks, v_scales=vs)
    before = tsb.kv_load(kp, slots, scales=ks, dtype=torch.float32)
    path = torch.tensor([[1, 4, 8]], dtype=torch.int32, device="cuda")
    tsb.tree_commit(kp, vp, table, torch.tensor([60], dtype=torch.int32, device="cuda"), path,
                    torch.tensor([3], dtype=torch.int32, device="cuda"), k_scales=ks, v_scales=vs)
    after = tsb.kv_load(kp, slots[:3], scales=ks, dtype=torch.float32)
    assert torch.equal(after, before[[1, 4, 8]])
    assert torch.equal(after.double(), rows_of(kp, ks, slots[:3]).float().double())
