"""Pages, slots and positions of a step, and the verification of drafted tokens, against plain references.

Everything here is whole numbers and has to be equal.  The verification's comparisons are in 64 bits on both
sides and differ by a few 2^-53 of their operands, so a random number would have to fall that close to a border
to tell them apart.
"""

import math
import random

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.step_ref import Pages, verify
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def indptr(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return int32(out)


class State:
    def __init__(self, ctx, width, spare, seed=0, room=0, stride=None):
        rng = random.Random(seed)
        owned = [-(-c // 64) for c in ctx]
        ids = list(range(sum(owned) + spare))
        rng.shuffle(ids)
        rows, at = [], 0
        for n in owned:
            rows.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        self.host = Pages(rows, owned, ids[at:] + [-5] * room, spare)
        stride = stride or width
        self.buffer = torch.full((len(ctx), stride), -9, dtype=torch.int32, device="cuda")
        self.table = self.buffer[:, :width]
        if ctx:
            self.table.copy_(torch.tensor(rows, dtype=torch.int32).view(len(ctx), width))
        self.counts, self.free, self.count = int32(owned), int32(self.host.free), int32([spare])
        self.flag = int32([0])

    def args(self):
        return self.table, self.counts, self.free, self.count

    def check(self):
        assert self.table.tolist() == self.host.table
        assert self.counts.tolist() == self.host.counts
        assert int(self.count) == self.host.count
        assert self.free.tolist()[:self.host.count] == self.host.free[:self.host.count]
        assert (self.buffer[:, self.table.shape[1]:] == -9).all()


@pytest.mark.parametrize("batch,ctx_hi,new_hi", [(1, 0, 1), (1, 200, 1), (3, 65, 130), (33, 700, 9), (64, 5000, 1),
                                                 (257, 300, 40), (1024, 130, 3), (2, 64, 4000), (5, 0, 3000)])
@pytest.mark.parametrize("stride", [None, 101])
def test_pages_follow_the_lengths(batch, ctx_hi, new_hi, stride):
    rng = random.Random(batch + new_hi)
    ctx = [rng.choice([0, 63, 64, 65, ctx_hi, rng.randint(0, ctx_hi)]) if ctx_hi >= 65 else rng.randint(0, ctx_hi)
           for _ in range(batch)]
    new = [rng.choice([0, 1, new_hi, rng.randint(0, new_hi)]) for _ in range(batch)]
    s = State(ctx, 80 if max(c + n for c, n in zip(ctx, new)) <= 5120 else 100, sum(-(-n // 64) + 1 for n in new), batch,
              stride=stride)
    for step in range(3):  # extend, keep a part, extend again
        slots, positions = tsb.extend_pages(*s.args(), int32(ctx), indptr(new), sum(new), error_flag=s.flag)
        want = s.host.extend(ctx, new)
        assert not want[2]
        assert slots.tolist() == want[0] and positions.tolist() == want[1]
        s.check()
        ctx = [c + rng.randint(0, min(n, 7)) for c, n in zip(ctx, new)]
        new = [min(n, 5) for n in new]
        tsb.release_pages(*s.args(), int32(ctx), error_flag=s.flag)
        s.host.release(ctx)
        s.check()
    assert int(s.flag) == 0


def test_an_extend_that_is_released_leaves_the_stack_as_it_was():
    ctx, new = [5, 64, 0, 200], [100, 64, 300, 1]
    s = State(ctx, 8, 20)
    before = [t.clone() for t in s.args()]
    tsb.extend_pages(*s.args(), int32(ctx), indptr(new), sum(new))
    assert not torch.equal(before[0], s.table)
    tsb.release_pages(*s.args(), int32(ctx))
    assert all(torch.equal(x, y) for x, y in zip(before, s.args()))


def test_ended_sequences_give_everything_back():
    s = State([130, 1, 64], 4, 0, room=9)
    owned = [p for r in s.host.table for p in r if p >= 0]
    tsb.release_pages(*s.args(), int32([0, 0, 0]))
    assert s.counts.tolist() == [0, 0, 0] and (s.table == -1).all()
    assert sorted(s.free.tolist()[:int(s.count)]) == sorted(owned)


def test_sequences_that_find_no_page_are_skipped():
    ctx, new = [64, 10, 64, 100, 0], [1, 3, 200, 1, 64]
    s = State(ctx, 8, 3)
    slots, positions = tsb.extend_pages(*s.args(), int32(ctx), indptr(new), sum(new), error_flag=s.flag)
    want = s.host.extend(ctx, new)
    assert want[2] and slots.tolist() == want[0] and positions.tolist() == want[1]
    s.check()
    assert int(s.flag) == _lib.DEVERR_NO_PAGES
    # and a stack that has no room takes none
    full = State([130, 70], 4, 0, room=2)
    tsb.release_pages(*full.args(), int32([64, 0]), error_flag=full.flag)
    assert full.host.release([64, 0])
    full.check()
    assert int(full.flag) == _lib.DEVERR_NO_PAGES


def test_positions_of_a_tree_are_depths():
    parents = int32([-1, 0, 0, 1, 3, -1, 0, -2, 2, 1])
    ptr = int32([0, 5, 10])
    mask = tsb.tree_mask(parents, ptr, 70)
    s = State([100, 3], 4, 6)
    _, positions = tsb.extend_pages(*s.args(), int32([100, 3]), ptr, 10, tree_mask=mask)
    assert positions.tolist() == [100, 101, 101, 102, 103, 3, 4, 3, 3, 5]


def test_bad_lengths_are_clamped_and_flagged():
    s = State([64, 10], 2, 4)
    # the second sequence would pass its row of the table
    slots, positions = tsb.extend_pages(*s.args(), int32([64, 100]), int32([0, 1, 61]), 61, error_flag=s.flag)
    assert int(s.flag) == _lib.DEVERR_BAD_LEN
    assert (slots[1:29] >= 0).all() and (slots[29:] == -1).all()
    assert positions.tolist()[1:] == list(range(100, 160))
    for ctx, ptr, tokens in (([-5, 10], [0, 1, 2], 2), ([1, 10], [0, 2, 1], 2), ([1, 1], [1, 2, 3], 3), ([1, 1], [0, 1, 9], 3)):
        s = State([64, 10], 2, 4)
        slots, _ = tsb.extend_pages(*s.args(), int32(ctx), int32(ptr), tokens, error_flag=s.flag)
        assert int(s.flag) & _lib.DEVERR_BAD_LEN
        assert slots.max() < 6 * 64 and slots.min() >= -1
        if ptr[0] > 0:
            assert int(slots[0]) == -1
    s = State([64, 10], 2, 4)
    tsb.release_pages(*s.args(), int32([-1, 0]), error_flag=s.flag)
    # (the stack of this state has no room either)
    assert s.counts.tolist() == [1, 1] and int(s.flag) == _lib.DEVERR_BAD_LEN | _lib.DEVERR_NO_PAGES
    s = State([64, 10], 2, 4, room=2)
    tsb.release_pages(*s.args(), int32([-1, 0]), error_flag=s.flag)
    assert s.counts.tolist() == [1, 0] and int(s.flag) == _lib.DEVERR_BAD_LEN


def test_nothing_to_plan():
    s = State([64, 10], 2, 4)
    slots, positions = tsb.extend_pages(*s.args(), int32([64, 10]), int32([0, 0, 0]), 0)
    assert slots.shape == (0,) and positions.shape == (0,)
    s.check()
    empty = State([], 2, 4)
    tsb.extend_pages(*empty.args(), int32([]), int32([0]), 0)
    tsb.release_pages(*empty.args(), int32([]))


def test_a_captured_plan_goes_on_with_the_state():
    s = State([60, 0], 8, 12)
    ctx, ptr = int32([60, 0]), int32([0, 3, 5])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        tsb.extend_pages(*State([60, 0], 8, 12).args(), ctx, ptr, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, positions = tsb.extend_pages(*s.args(), ctx, ptr, 5)
        ctx.add_(torch.diff(ptr))
    lens = [60, 0]
    for _ in range(40):
        graph.replay()
        want = s.host.extend(lens, [3, 2])
        assert slots.tolist() == want[0] and positions.tolist() == want[1]
        lens = [lens[0] + 3, lens[1] + 2]
    s.check()


# ------------------------------------------------------------------ verify --
def draft_case(new, vocab, dtype, seed, with_draft=True, wide=None, sharp=2.0, chain=False):
    g = torch.Generator().manual_seed(seed)
    n = sum(new)
    z = torch.randn((n, vocab), generator=g) * sharp
    target = torch.softmax(z, -1)
    draft = torch.softmax(z + 0.7 * torch.randn((n, vocab), generator=g), -1)
    parents, tokens = [], []
    for m in new:
        first = len(parents)
        for i in range(m):
            p = i - 1 if chain else (-1 if i == 0 else int(torch.rand((), generator=g) ** 1.5 * i))
            parents.append(p)
            tokens.append(int(torch.multinomial(draft[first + max(p, 0)], 1, generator=g)))

    def place(x):
        x = x.to(dtype)
        if wide:  # rows of another stride
            big = torch.full((n, vocab + wide), float("nan"), dtype=dtype)
            big[:, :vocab] = x
            return big.cuda()[:, :vocab]
        return x.cuda()

    return dict(parents=int32(parents), tokens=torch.tensor(tokens, device="cuda", dtype=torch.int64), q_indptr=indptr(new),
                target_probs=place(target), accept_u=torch.rand(n, generator=g).cuda(),
                sample_u=torch.rand(len(new), generator=g).cuda(), draft_probs=place(draft) if with_draft else None)


def check_verify(case, new, max_path=None, flag=None):
    path, lens, nxt = tsb.tree_verify(**case, max_path=max_path, error_flag=flag)
    host = {k: None if v is None else v.cpu() for k, v in case.items()}
    width, first = path.shape[1], 0
    for b, n in enumerate(new):
        rows = slice(first, first + n)
        want, token = verify(host["parents"][rows].tolist(), host["tokens"][rows], host["target_probs"][rows],
                             None if host["draft_probs"] is None else host["draft_probs"][rows], host["accept_u"][rows],
                             host["sample_u"][b], width)
        assert int(lens[b]) == len(want), b
        assert path[b].tolist() == want + [-1] * (width - len(want)), b
        assert int(nxt[b]) == token, b
        first += n
    return path, lens, nxt


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("new,vocab", [([1], 1), ([2], 3), ([5, 1, 0, 9], 33), ([33, 64, 7], 1000), ([4] * 40, 4099),
                                       ([17, 3], 32000), ([6] * 3, 70001), ([2] * 300, 257)])
def test_paths_and_tokens(dtype, with_draft, new, vocab):
    check_verify(draft_case(new, vocab, dtype, seed=len(new) + vocab, with_draft=with_draft), new)


@pytest.mark.parametrize("wide", [1, 8, 24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_any_stride(dtype, wide):
    new = [9, 12, 1]
    check_verify(draft_case(new, 997 if wide == 1 else 1000, dtype, seed=wide, wide=wide), new)


def test_many_rejections_at_one_node():
    # 60 children of the root, drawn from a drafter that is far off
    n, vocab = 61, 512
    case = draft_case([n], vocab, torch.float32, 5)
    case["parents"] = int32([-1] + [0] * (n - 1))
    far = torch.softmax(6 * torch.randn(n, vocab, generator=torch.Generator().manual_seed(6)), -1)
    case["draft_probs"] = far.cuda()
    case["tokens"] = torch.multinomial(far[0], n, replacement=True, generator=torch.Generator().manual_seed(7)).cuda()
    check_verify(case, [n])
    check_verify(dict(case, draft_probs=None), [n])


@pytest.mark.parametrize("max_path", [1, 2, 3, 200])
def test_short_paths(max_path):
    new = [8, 1, 20]
    case = draft_case(new, 64, torch.float32, 3, chain=True)
    case["accept_u"].mul_(0.05)  # nearly all accepted
    _, lens, _ = check_verify(case, new, max_path=max_path)
    assert int(lens.max()) == min(max_path, max(int(x) for x in lens))


def test_edges_of_the_random_numbers():
    new = [3] * 64
    for value in (0.0, 1.0 - 2.0**-24):
        case = draft_case(new, 130, torch.float32, 9)
        case["accept_u"].fill_(value)
        case["sample_u"].fill_(value)
        check_verify(case, new)


def test_rows_with_little_left():
    case = draft_case([2, 2, 2, 2, 1], 300, torch.float32, 4)
    t, d = case["target_probs"], case["draft_probs"]
    case["tokens"][:] = 7
    t[0] = 0.0
    t[0, 11] = 1.0  # certain, the draft elsewhere
    d[0] = 0.0
    d[0, 7] = 1.0
    t[2] = d[2] = 0.0
    t[2, 5], d[2, 7], d[2, 5] = 1.0, 0.5, 1.0  # nothing left of p - q: from p again
    t[4] = float("nan")
    t[4, 9] = 0.25  # what is not a number has no weight
    t[6] = 0.0  # no weight at all
    t[8] = float("nan")
    flag = int32([0])
    path, lens, nxt = tsb.tree_verify(**case, error_flag=flag)
    assert lens.tolist() == [1, 1, 1, 1, 1] and nxt.tolist() == [11, 5, 9, -1, -1]
    assert int(flag) == _lib.DEVERR_BAD_TOKEN


def test_tokens_and_parents_that_cannot_be():
    new = [4, 4]
    case = draft_case(new, 50, torch.float32, 8, chain=True)
    case["accept_u"].zero_()
    case["tokens"][1] = 50
    case["tokens"][6] = -1
    flag = int32([0])
    check_verify(case, new, flag=flag)
    assert int(flag) == _lib.DEVERR_BAD_TOKEN
    case = draft_case(new, 50, torch.float32, 8, chain=True)
    case["accept_u"].zero_()
    case["parents"][2], case["parents"][7] = -2, 3
    flag.zero_()
    _, lens, _ = tsb.tree_verify(**case, error_flag=flag)
    assert lens.tolist() == [2, 3] and int(flag) == _lib.DEVERR_BAD_LEN


def test_bad_offsets_take_nothing():
    case = draft_case([3, 3], 20, torch.float32, 1)
    for ptr in ([0, 7, 6], [-1, 3, 6], [0, 5, 3]):
        flag = int32([0])
        path, lens, nxt = tsb.tree_verify(**dict(case, q_indptr=int32(ptr)), error_flag=flag)
        assert int(flag) == _lib.DEVERR_BAD_LEN and 0 in lens.tolist()


def test_a_long_draft():
    new = [1024, 1025]
    case = draft_case(new, 40, torch.float32, 2, chain=True)
    case["accept_u"].zero_()
    flag = int32([0])
    path, lens, _ = tsb.tree_verify(**case, error_flag=flag)
    assert lens.tolist() == [1024, 1024] and int(flag) == _lib.DEVERR_BAD_LEN
    assert path[0, :1024].tolist() == list(range(1024))


@pytest.mark.parametrize("children,with_draft", [(1, True), (3, True), (2, False)])
def test_tokens_have_the_targets_distribution(children, with_draft):
    """40000 sequences of one p and q: the first new token's frequencies are p's, to 5 standard deviations."""
    batch, vocab = 40000, 6
    g = torch.Generator().manual_seed(children)
    p = torch.tensor([0.05, 0.4, 0.1, 0.25, 0.15, 0.05])
    q = torch.tensor([0.3, 0.1, 0.2, 0.1, 0.05, 0.25])
    n = 1 + children
    drawn = torch.multinomial(q.expand(batch, vocab), children, replacement=True, generator=g) if with_draft \
        else torch.tensor([3, 0]).expand(batch, 2)
    tokens = torch.cat([torch.zeros((batch, 1), dtype=torch.int64), drawn], 1)
    path, lens, nxt = tsb.tree_verify(
        int32([-1] + [0] * children).repeat(batch), tokens.flatten().cuda(), int32([n] * (batch + 1)).cumsum(0, dtype=torch.int32) - n,
        p.cuda().expand(batch * n, vocab).contiguous(), torch.rand(batch * n, generator=g).cuda(),
        torch.rand(batch, generator=g).cuda(), q.cuda().expand(batch * n, vocab).contiguous() if with_draft else None)
    taken = tokens.gather(1, path[:, 1:2].clamp_min(0).long().cpu())[:, 0]
    first = torch.where(lens.cpu() > 1, taken, nxt.cpu())
    freq = torch.bincount(first, minlength=vocab).double() / batch
    assert ((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / batch)).all()


def test_the_same_bits_every_time_and_from_a_graph():
    new = [30, 12, 1, 40] * 4
    case = draft_case(new, 20011, torch.float32, 6)
    eager = tsb.tree_verify(**case)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tsb.tree_verify(**case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tsb.tree_verify(**case)
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(eager, out))
    by_op = torch.ops.b200kv.tree_verify(*case.values(), max(1, len(case["parents"])), None)
    assert all(torch.equal(x, y) for x, y in zip(eager, by_op))
